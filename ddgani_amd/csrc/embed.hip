// Table lookup with a scale and its gradient.
//
//     y[i, :]  = scale * E[id_i, :]                       dE[v, :] (+)= scale * sum over {i : id_i = v} of dy[i, :]
//
// Both are bound by HBM traffic: the lookup reads n rows and writes n rows, the gradient reads the n rows of dy and writes
// the V rows of dE (with `accumulate`: reads and writes only the rows that a token names).
//
// The gradient sorts the tokens instead of adding with atomics: (id, position) pairs go through a stable counting sort, so
// every table row finds its positions in ascending order and is summed in registers, in one fixed order (bitwise
// reproducible), and written once.  Frequent ids are long rows: sorted positions are cut into aligned chunks of 64, and a
// chunk that belongs to ONE id is summed beforehand by k_embg_part (4 096-chunks of such sums by a second launch), so the
// longest walk a row can need is 63 + 63 single tokens, 63 + 63 sums of 64 and n / 4 096 sums of 4 096.
#include "types.h"

#define EMB_NT 256
#define EMB_VEC 8                     // elements per thread and row: 16 bytes of a 16-bit type

template <class ID> __device__ __forceinline__ uint32_t emb_key(const ID *ids, int64_t i, int64_t V, int64_t padding_idx) {
    const int64_t v = (int64_t)ids[i];
    return (uint64_t)v < (uint64_t)V && v != padding_idx ? (uint32_t)v : (uint32_t)V;      // V: no row
}

// U rows per thread group: their id loads, then their row loads, are in flight together
template <class TI, class TO, class ID, int U>
__global__ __launch_bounds__(EMB_NT) void k_embed(const ID *__restrict__ ids, int64_t n, const TI *__restrict__ table, int64_t V,
                                                  int D, int64_t ld, float scale, TO *__restrict__ out, int64_t ldo, int lg_tpr) {
    const int tpr = 1 << lg_tpr, rpb = EMB_NT >> lg_tpr;
    const int col = (blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * EMB_VEC;
    const int64_t row0 = (int64_t)blockIdx.x * (rpb * U) + (threadIdx.x >> lg_tpr);
    if (col >= D) return;
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = row0 + (int64_t)u * rpb < n ? (int64_t)ids[row0 + (int64_t)u * rpb] : -1;
    float v[U][EMB_VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool ok = (uint64_t)id[u] < (uint64_t)V;
        load_n<EMB_VEC>(table + (ok ? id[u] : 0) * ld + col, ok ? D - col : 0, v[u]);      // outside the table: zeros
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t r = row0 + (int64_t)u * rpb;
        if (r >= n) return;
#pragma unroll
        for (int i = 0; i < EMB_VEC; ++i) v[u][i] *= scale;
        store_n<EMB_VEC>(out + r * ldo + col, D - col, v[u]);
    }
}

static inline int emb_lg_tpr(int D) {          // lanes per row: the power of two that covers D / 8, at most a workgroup
    int lg = 0;
    while (lg < 8 && (EMB_VEC << lg) < D) ++lg;
    return lg;
}

extern "C" int ddg_embedding(const void *ids, int ids_64, int64_t n, const void *table, int table_type, int64_t V, int D,
                             int64_t ld_table, float scale, void *out, int out_type, int64_t ld_out, void *stream) {
    if (n < 0 || V < 1 || V > 0x7FFFFFFF || D < 1 || ld_table < D || ld_out < D || !ddg_type_ok(table_type) ||
        !ddg_type_ok(out_type) || (ids_64 != 0 && ids_64 != 1))
        return DDG_E_ARG;
    if (n == 0) return DDG_OK;
    if (!ids || !table || !out) return DDG_E_ARG;
    const int lg = emb_lg_tpr(D), rpb = EMB_NT >> lg;
    const int slabs = (D + (EMB_VEC << lg) - 1) / (EMB_VEC << lg);
    // four rows per thread once that still leaves two workgroups per CU; one row below (few rows: latency, not bandwidth)
    const bool wide = ceil_div64(n, 4 * rpb) * slabs >= 512;
    const int64_t gx = ceil_div64(n, wide ? 4 * rpb : rpb);
    if (gx > 0x7FFFFFFF || slabs > 65535) return DDG_E_UNSUPPORTED;
    return ddg_with_type(table_type, [&](auto ti) {
        return ddg_with_type(out_type, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            auto go = [&](auto id) {
                using ID = decltype(id);
                const dim3 grid((unsigned)gx, (unsigned)slabs);
                if (wide)
                    k_embed<TI, TO, ID, 4><<<grid, EMB_NT, 0, (hipStream_t)stream>>>(
                        (const ID *)ids, n, (const TI *)table, V, D, ld_table, scale, (TO *)out, ld_out, lg);
                else
                    k_embed<TI, TO, ID, 1><<<grid, EMB_NT, 0, (hipStream_t)stream>>>(
                        (const ID *)ids, n, (const TI *)table, V, D, ld_table, scale, (TO *)out, ld_out, lg);
                DDG_CHECK_LAUNCH();
                return (int)DDG_OK;
            };
            return ids_64 ? go(int64_t()) : go(int32_t());
        });
    });
}

// ---------------------------------------------------------------------------------------------
// gradient: stable counting sort of (id, position), digits of at most 9 bits, least significant first
// ---------------------------------------------------------------------------------------------
#define SORT_NT 512
#define SORT_WAVES (SORT_NT / 64)
#define SORT_BINS 512
#define SORT_MAX_TILES 128            // a tile's workgroup reads every earlier tile's counts: 128 x 512 words at most
#define SORT_SMALL 4096               // up to this many tokens one workgroup sorts in LDS
#define CHUNK1 64
#define CHUNK2 4096

struct SortPlan {
    int bits, passes, digit;          // id bits, number of passes, bits per pass
    int64_t tile, tiles;              // tokens per tile: a multiple of SORT_NT
};
static inline SortPlan sort_plan(int64_t n, int64_t V) {
    SortPlan p;
    p.bits = 1;
    while (((int64_t)1 << p.bits) < V + 1) ++p.bits;              // keys are 0 ... V
    p.passes = (p.bits + 8) / 9;
    p.digit = (p.bits + p.passes - 1) / p.passes;
    p.tile = ceil_div64(ceil_div64(n, SORT_MAX_TILES), SORT_NT) * SORT_NT;
    if (p.tile < 2048) p.tile = 2048;
    p.tiles = ceil_div64(n, p.tile);
    return p;
}

// where a pass reads its pairs: the caller's ids (first pass; the position is the index) or the previous pass's output
template <class ID> struct SortSrc {
    const ID *ids;
    const uint32_t *key, *pos;
    int64_t V, padding_idx;
    __device__ __forceinline__ uint32_t k(int64_t i) const { return ids ? emb_key(ids, i, V, padding_idx) : key[i]; }
    __device__ __forceinline__ uint32_t p(int64_t i) const { return ids ? (uint32_t)i : pos[i]; }
};

template <class ID>
__global__ __launch_bounds__(SORT_NT) void k_embg_hist(SortSrc<ID> src, int64_t n, int64_t tile, int shift, int bins,
                                                       uint32_t *__restrict__ hist) {
    __shared__ uint32_t c[SORT_BINS];
    const int t = threadIdx.x;
    c[t] = 0;
    __syncthreads();
    const int64_t lo = blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
    for (int64_t i = lo + t; i < hi; i += SORT_NT) atomicAdd(&c[(src.k(i) >> shift) & (bins - 1)], 1u);
    __syncthreads();
    if (t < bins) hist[(int64_t)blockIdx.x * SORT_BINS + t] = c[t];
}

// exclusive prefix sum over the SORT_NT threads of a workgroup
__device__ __forceinline__ uint32_t block_exclusive(uint32_t x, uint32_t *wsum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t s = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(s, d);
        if (lane >= d) s += y;
    }
    if (lane == 63) wsum[w] = s;
    __syncthreads();
    uint32_t before = 0;
    for (int i = 0; i < w; ++i) before += wsum[i];
    __syncthreads();
    return before + s - x;
}

// the lanes of this wave that are live and hold the same digit
__device__ __forceinline__ uint64_t match_digit(uint32_t d, bool live, int digit_bits) {
    uint64_t m = __ballot(live);
    for (int b = 0; b < digit_bits; ++b) {
        const uint64_t s = __ballot((d >> b) & 1);
        m &= (d >> b) & 1 ? s : ~s;
    }
    return m;
}

// One wave places the pairs of [lo, hi) in their order; next[digit] is the wave's next free place.  A volatile pointer: the
// wave's LDS accesses are executed in program order, so the count of one group of 64 is seen by the next.
template <class GetK, class GetP, class Put>
__device__ __forceinline__ void place_segment(int64_t lo, int64_t hi, int shift, int digit_bits, volatile uint32_t *next,
                                              const GetK &getk, const GetP &getp, const Put &put) {
    const int lane = threadIdx.x & 63;
    for (int64_t g = lo; g < hi; g += 64) {
        const bool live = g + lane < hi;
        const uint32_t k = live ? getk(g + lane) : 0, p = live ? getp(g + lane) : 0;
        const uint32_t d = (k >> shift) & ((1u << digit_bits) - 1);
        const uint64_t m = match_digit(d, live, digit_bits);
        const uint32_t rank = __popcll(m & (((uint64_t)1 << lane) - 1));
        if (live) {
            const uint32_t at = next[d];
            put(at + rank, k, p);
            if (rank == 0) next[d] = at + __popcll(m);
        }
    }
}

template <class ID>
__global__ __launch_bounds__(SORT_NT) void k_embg_scatter(SortSrc<ID> src, int64_t n, int64_t tile, int tiles, int shift,
                                                          int digit_bits, const uint32_t *__restrict__ hist,
                                                          uint32_t *__restrict__ okey, uint32_t *__restrict__ opos) {
    __shared__ uint32_t next[SORT_WAVES][SORT_BINS];
    __shared__ uint32_t wsum[SORT_WAVES];
    const int t = threadIdx.x, w = t >> 6, bins = 1 << digit_bits;
    for (int i = 0; i < SORT_WAVES; ++i) next[i][t] = 0;
    __syncthreads();
    const int64_t lo = blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n, seg = tile / SORT_WAVES;
    const int64_t slo = lo + w * seg < hi ? lo + w * seg : hi, shi = slo + seg < hi ? slo + seg : hi;
    for (int64_t i = slo + (t & 63); i < shi; i += 64) atomicAdd(&next[w][(src.k(i) >> shift) & (bins - 1)], 1u);
    uint32_t before = 0, total = 0;
    if (t < bins)
        for (int b = 0; b < tiles; ++b) {
            const uint32_t h = hist[(int64_t)b * SORT_BINS + t];
            total += h;
            if (b < (int)blockIdx.x) before += h;
        }
    __syncthreads();
    uint32_t at = block_exclusive(total, wsum) + before;
    for (int i = 0; i < SORT_WAVES; ++i) {
        const uint32_t c = next[i][t];
        next[i][t] = at;
        at += c;
    }
    __syncthreads();
    place_segment(slo, shi, shift, digit_bits, next[w], [&](int64_t i) { return src.k(i); }, [&](int64_t i) { return src.p(i); },
                  [&](uint32_t d, uint32_t k, uint32_t p) {
                      okey[d] = k;
                      opos[d] = p;
                  });
}

// n <= SORT_SMALL: every pass in LDS, one workgroup, one launch
template <class ID>
__global__ __launch_bounds__(SORT_NT) void k_embg_sort_small(const ID *__restrict__ ids, int n, int64_t V, int64_t padding_idx,
                                                             int passes, int digit_bits, uint32_t *__restrict__ okey,
                                                             uint32_t *__restrict__ opos) {
    __shared__ uint32_t key[2][SORT_SMALL];
    __shared__ uint16_t pos[2][SORT_SMALL];
    __shared__ uint32_t next[SORT_WAVES][SORT_BINS];
    __shared__ uint32_t wsum[SORT_WAVES];
    const int t = threadIdx.x, w = t >> 6, bins = 1 << digit_bits;
    for (int i = t; i < n; i += SORT_NT) {
        key[0][i] = emb_key(ids, i, V, padding_idx);
        pos[0][i] = (uint16_t)i;
    }
    const int seg = ((n + SORT_NT - 1) / SORT_NT) * 64, slo = w * seg < n ? w * seg : n, shi = slo + seg < n ? slo + seg : n;
    for (int pass = 0; pass < passes; ++pass) {
        const int a = pass & 1, shift = pass * digit_bits;
        for (int i = 0; i < SORT_WAVES; ++i) next[i][t] = 0;
        __syncthreads();
        for (int i = slo + (t & 63); i < shi; i += 64) atomicAdd(&next[w][(key[a][i] >> shift) & (bins - 1)], 1u);
        __syncthreads();
        uint32_t total = 0;
        for (int i = 0; i < SORT_WAVES; ++i) total += next[i][t];
        uint32_t at = block_exclusive(total, wsum);
        for (int i = 0; i < SORT_WAVES; ++i) {
            const uint32_t c = next[i][t];
            next[i][t] = at;
            at += c;
        }
        __syncthreads();
        place_segment(slo, shi, shift, digit_bits, next[w], [&](int64_t i) { return key[a][i]; },
                      [&](int64_t i) { return (uint32_t)pos[a][i]; }, [&](uint32_t d, uint32_t k, uint32_t p) {
                          key[1 - a][d] = k;
                          pos[1 - a][d] = (uint16_t)p;
                      });
        __syncthreads();
    }
    for (int i = t; i < n; i += SORT_NT) {
        okey[i] = key[passes & 1][i];
        opos[i] = pos[passes & 1][i];
    }
}

// ---------------------------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------------------------
// acc += rows src[index(j)] (columns from col on) for j in [a, b), four rows in flight
template <class T, class Idx>
__device__ __forceinline__ void add_rows(const T *__restrict__ src, int64_t ld, int col, int D, int64_t a, int64_t b,
                                         const Idx &index, float (&acc)[EMB_VEC]) {
    float v[4][EMB_VEC];
    for (; a + 4 <= b; a += 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u) load_n<EMB_VEC>(src + (int64_t)index(a + u) * ld + col, D - col, v[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < EMB_VEC; ++i) acc[i] += v[u][i];
    }
    for (; a < b; ++a) {
        load_n<EMB_VEC>(src + (int64_t)index(a) * ld + col, D - col, v[0]);
#pragma unroll
        for (int i = 0; i < EMB_VEC; ++i) acc[i] += v[0][i];
    }
}

// LEVEL 1: part[c] = sum of the dy rows of sorted positions [64 c, 64 c + 64) if they all belong to one row of the table;
// LEVEL 2: part[c] = sum of the LEVEL-1 sums of [4 096 c, ...), under the same condition.  Other chunks are never read.
template <class T, int LEVEL>
__global__ __launch_bounds__(EMB_NT) void k_embg_part(const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos,
                                                      int64_t chunks, uint32_t V, const T *__restrict__ src, int64_t ld, int D,
                                                      float *__restrict__ part, int lg_tpr) {
    const int tpr = 1 << lg_tpr;
    const int col = (blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * EMB_VEC;
    const int64_t c = (int64_t)blockIdx.x * (EMB_NT >> lg_tpr) + (threadIdx.x >> lg_tpr);
    const int len = LEVEL == 1 ? CHUNK1 : CHUNK2;
    if (c >= chunks || col >= D) return;
    const uint32_t k = key[c * len];
    if (k >= V || k != key[c * len + len - 1]) return;
    float acc[EMB_VEC] = {};
    if (LEVEL == 1)
        add_rows(src, ld, col, D, c * CHUNK1, (c + 1) * CHUNK1, [&](int64_t j) { return pos[j]; }, acc);
    else
        add_rows(src, ld, col, D, c * (CHUNK2 / CHUNK1), (c + 1) * (CHUNK2 / CHUNK1), [](int64_t j) { return j; }, acc);
    store_n<EMB_VEC>(part + c * D + col, D - col, acc);
}

#define ROWS_MAX 32                   // table rows per workgroup of k_embg_rows

template <class T, class TO>
__global__ __launch_bounds__(EMB_NT) void k_embg_rows(const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos, int64_t n,
                                                      int64_t V, const T *__restrict__ dy, int64_t ld, int D,
                                                      const float *__restrict__ part1, const float *__restrict__ part2, float scale,
                                                      int accumulate, TO *__restrict__ out, int64_t ldo, int lg_tpr, int rows) {
    __shared__ int64_t start[ROWS_MAX + 1];
    const int64_t v0 = (int64_t)blockIdx.x * rows;
    if (threadIdx.x <= rows) {                          // first sorted position whose key is >= v
        const uint64_t v = v0 + threadIdx.x;
        int64_t a = 0, b = n;
        while (a < b) {
            const int64_t mid = (a + b) >> 1;
            if (key[mid] < v) a = mid + 1; else b = mid;
        }
        start[threadIdx.x] = a;
    }
    __syncthreads();
    const int tpr = 1 << lg_tpr;
    const int col = (blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * EMB_VEC;
    if (col >= D) return;
    for (int r = threadIdx.x >> lg_tpr; r < rows && v0 + r < V; r += EMB_NT >> lg_tpr) {
        int64_t a = start[r];
        const int64_t b = start[r + 1];
        if (accumulate && a == b) continue;
        float acc[EMB_VEC] = {};
        while (a < b) {                                 // the longest whole chunk that starts here, else single tokens
            if (a % CHUNK2 == 0 && a + CHUNK2 <= b) {
                const int64_t m = (b - a) / CHUNK2;
                add_rows(part2, D, col, D, a / CHUNK2, a / CHUNK2 + m, [](int64_t j) { return j; }, acc);
                a += m * CHUNK2;
            } else if (a % CHUNK1 == 0 && a + CHUNK1 <= b) {
                int64_t m = (b - a) / CHUNK1;           // up to the next multiple of CHUNK2 (a whole one is taken above)
                const int64_t to2 = (CHUNK2 - a % CHUNK2) / CHUNK1;
                if (m > to2) m = to2;
                add_rows(part1, D, col, D, a / CHUNK1, a / CHUNK1 + m, [](int64_t j) { return j; }, acc);
                a += m * CHUNK1;
            } else {
                const int64_t next1 = (a / CHUNK1 + 1) * CHUNK1, e = next1 < b ? next1 : b;
                add_rows(dy, ld, col, D, a, e, [&](int64_t j) { return pos[j]; }, acc);
                a = e;
            }
        }
        TO *o = out + (v0 + r) * ldo + col;
        float old[EMB_VEC] = {};
        if (accumulate) load_n<EMB_VEC>(o, D - col, old);
#pragma unroll
        for (int i = 0; i < EMB_VEC; ++i) acc[i] = old[i] + scale * acc[i];
        store_n<EMB_VEC>(o, D - col, acc);
    }
}

static inline size_t eal(size_t x) { return (x + 255) & ~(size_t)255; }
struct EmbWs {
    uint32_t *key[2], *pos[2], *hist;
    float *part1, *part2;
    size_t bytes;
};
static inline EmbWs emb_carve(void *base, int64_t n, int D) {
    EmbWs w;
    char *p = (char *)base;
    size_t o = 0;
    auto take = [&](size_t b) {
        char *q = p ? p + o : nullptr;
        o += eal(b);
        return q;
    };
    for (int i = 0; i < 2; ++i) {
        w.key[i] = (uint32_t *)take((size_t)n * 4);
        w.pos[i] = (uint32_t *)take((size_t)n * 4);
    }
    w.hist = (uint32_t *)take((size_t)SORT_MAX_TILES * SORT_BINS * 4);
    w.part1 = (float *)take((size_t)(n / CHUNK1) * D * 4);
    w.part2 = (float *)take((size_t)(n / CHUNK2) * D * 4);
    w.bytes = o;
    return w;
}

extern "C" size_t ddg_embedding_grad_workspace_bytes(int64_t n, int D) {
    if (n < 0 || n > 0x7FFFFFFF || D < 1) return 0;
    return emb_carve(nullptr, n, D).bytes;
}

extern "C" int ddg_embedding_grad(const void *ids, int ids_64, int64_t n, const void *dy, int dy_type, int64_t ld_dy, int64_t V,
                                  int D, float scale, int64_t padding_idx, int accumulate, void *out, int out_type, int64_t ld_out,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    if (n < 0 || V < 1 || D < 1 || ld_dy < D || ld_out < D || !ddg_type_ok(dy_type) || !ddg_type_ok(out_type) ||
        (ids_64 != 0 && ids_64 != 1) || !out)
        return DDG_E_ARG;
    if (n > 0x7FFFFFFF || V > 0x7FFFFFFE) return DDG_E_UNSUPPORTED;
    if (n == 0 && accumulate) return DDG_OK;
    if (n > 0 && (!ids || !dy)) return DDG_E_ARG;
    if (!workspace || workspace_bytes < ddg_embedding_grad_workspace_bytes(n, D)) return DDG_E_WORKSPACE;
    if ((uintptr_t)workspace & 15) return DDG_E_ARG;
    const EmbWs w = emb_carve(workspace, n, D);
    const SortPlan sp = sort_plan(n > 0 ? n : 1, V);
    const hipStream_t s = (hipStream_t)stream;
    int cur = 0;                                        // which of the two pair buffers holds the result
    if (n > 0) {
        auto sort = [&](auto id) {
            using ID = decltype(id);
            if (n <= SORT_SMALL) {
                k_embg_sort_small<ID><<<1, SORT_NT, 0, s>>>((const ID *)ids, (int)n, V, padding_idx, sp.passes, sp.digit, w.key[0],
                                                            w.pos[0]);
                return;
            }
            for (int p = 0; p < sp.passes; ++p) {
                const int from = (p + 1) & 1, to = p & 1;
                const SortSrc<ID> src = {p == 0 ? (const ID *)ids : nullptr, w.key[from], w.pos[from], V, padding_idx};
                k_embg_hist<ID><<<(unsigned)sp.tiles, SORT_NT, 0, s>>>(src, n, sp.tile, p * sp.digit, 1 << sp.digit, w.hist);
                k_embg_scatter<ID><<<(unsigned)sp.tiles, SORT_NT, 0, s>>>(src, n, sp.tile, (int)sp.tiles, p * sp.digit, sp.digit,
                                                                          w.hist, w.key[to], w.pos[to]);
                cur = to;
            }
        };
        if (ids_64) sort(int64_t()); else sort(int32_t());
        DDG_CHECK_LAUNCH();
    }
    const int lg = emb_lg_tpr(D), rpb = EMB_NT >> lg;
    const int slabs = (D + (EMB_VEC << lg) - 1) / (EMB_VEC << lg);
    if (slabs > 65535) return DDG_E_UNSUPPORTED;
    const int rows = rpb > 8 ? (rpb < ROWS_MAX ? rpb : ROWS_MAX) : 8;
    return ddg_with_type(dy_type, [&](auto ti) {
        using TI = decltype(ti);
        const int64_t c1 = n / CHUNK1, c2 = n / CHUNK2;
        if (c1)
            k_embg_part<TI, 1><<<dim3((unsigned)ceil_div64(c1, rpb), slabs), EMB_NT, 0, s>>>(
                w.key[cur], w.pos[cur], c1, (uint32_t)V, (const TI *)dy, ld_dy, D, w.part1, lg);
        if (c2)
            k_embg_part<float, 2><<<dim3((unsigned)ceil_div64(c2, rpb), slabs), EMB_NT, 0, s>>>(
                w.key[cur], w.pos[cur], c2, (uint32_t)V, w.part1, D, D, w.part2, lg);
        return ddg_with_type(out_type, [&](auto to) {
            using TO = decltype(to);
            k_embg_rows<TI, TO><<<dim3((unsigned)ceil_div64(V, rows), slabs), EMB_NT, 0, s>>>(
                w.key[cur], w.pos[cur], n, V, (const TI *)dy, ld_dy, D, w.part1, w.part2, scale, accumulate, (TO *)out, ld_out, lg,
                rows);
            DDG_CHECK_LAUNCH();
            return (int)DDG_OK;
        });
    });
}
