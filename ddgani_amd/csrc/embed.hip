// Table lookup with a scale and its gradient.
//
//     y[i, :]  = scale * E[id_i, :]                       dE[v, :] (+)= scale * sum over {i : id_i = v} of dy[i, :]
//
// Both are bound by HBM traffic: the lookup reads n rows and writes n rows, the gradient reads the n rows of dy and writes
// the V rows of dE (with `accumulate`: reads and writes only the rows that a token names).
//
// The gradient sorts the tokens instead of adding with atomics: (id, position) pairs go through a stable counting sort, so
// every table row finds its positions in ascending order and is summed in registers, in one fixed order (bitwise
// reproducible), and written once.  Frequent ids are long rows: sorted positions are cut into aligned chunks (of 16, 32 or 64), and
// a chunk that belongs to ONE id is summed beforehand by k_embg_part, chunks of 16, 32 or 64 such sums by a second launch.
#include <type_traits>
#include "types.h"

#define EMB_NT 256
#define EMB_MAX_D (1 << 26)           // columns are counted in 32 bits, slabs of them by the grid's second dimension
#define EMB_STREAM (16 << 20)         // elements of a gradient from which it is stored past the caches (2 % less time at 262 million)
#define EMB_VEC 8                     // elements per thread and row: 16 bytes of a 16-bit type

// A lane's eight columns of rows of D: [at, at + 8) is what it loads, always whole and inside the row, so that no load sits
// behind a branch and several stay in flight; `col` on is what it writes (the last lane's piece overlaps its neighbour's, a
// lane behind the row repeats the last piece and writes nothing).  TINY: D < 8, one lane, element by element.
struct Columns {
    int col, at, D;
    __device__ Columns(int c, int d) : col(c), at(c < d - EMB_VEC ? c : d > EMB_VEC ? d - EMB_VEC : 0), D(d) {}
};
template <bool TINY, bool STREAM = false, class T> __device__ __forceinline__ vec8<T> load_row(const T *row, const Columns &c) {
    vec8<T> v;
    if (TINY) {
#pragma unroll
        for (int i = 0; i < EMB_VEC; ++i) v[i] = i < c.D ? row[i] : (T)0.f;
    } else {
        v = load_whole<STREAM>(row + c.at);
    }
    return v;
}
template <bool TINY, bool STREAM = false, class T>
__device__ __forceinline__ void store_row(T *row, const Columns &c, const float (&v)[EMB_VEC]) {
    if (!TINY && c.col == c.at) {
        store_n<EMB_VEC, STREAM>(row + c.at, EMB_VEC, v);
    } else {
#pragma unroll
        for (int i = 0; i < EMB_VEC; ++i)
            if (c.at + i >= c.col && c.at + i < c.D) row[c.at + i] = (T)v[i];
    }
}
template <class T> __device__ __forceinline__ void add_row(float (&acc)[EMB_VEC], const vec8<T> &v) {
#pragma unroll
    for (int i = 0; i < EMB_VEC; ++i) acc[i] += (float)v[i];
}

template <class ID> __device__ __forceinline__ uint32_t emb_key(const ID *ids, int64_t i, int64_t V, int64_t padding_idx) {
    const int64_t v = (int64_t)ids[i];
    return (uint64_t)v < (uint64_t)V && v != padding_idx ? (uint32_t)v : (uint32_t)V;      // V: no row
}

// U rows per thread group: their id loads, then their row loads, are in flight together.  Large results (U > 1) are stored past
// the caches: 65 488 rows of 1 024 fp32 -> bf16 50.6 us with ordinary stores, 42.0 us so.
template <class TI, class TO, class ID, int U, bool TINY>
__global__ __launch_bounds__(EMB_NT) void k_embed(const ID *__restrict__ ids, int64_t n, const TI *__restrict__ table, int64_t V,
                                                  int D, int64_t ld, float scale, TO *__restrict__ out, int64_t ldo, int lg_tpr) {
    const int tpr = 1 << lg_tpr, rpb = EMB_NT >> lg_tpr;
    const Columns c((blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * EMB_VEC, D);
    const int64_t row0 = (int64_t)blockIdx.x * (rpb * U) + (threadIdx.x >> lg_tpr);
    if (c.col >= D) return;
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = row0 + (int64_t)u * rpb < n ? (int64_t)ids[row0 + (int64_t)u * rpb] : -1;
    vec8<TI> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_row<TINY>(table + ((uint64_t)id[u] < (uint64_t)V ? id[u] : 0) * ld, c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t r = row0 + (int64_t)u * rpb;
        if (r >= n) return;
        float f[EMB_VEC];
#pragma unroll
        for (int i = 0; i < EMB_VEC; ++i) f[i] = (uint64_t)id[u] < (uint64_t)V ? (float)v[u][i] * scale : 0.f;
        store_row<TINY, (U > 1)>(out + r * ldo, c, f);
    }
}

static inline int emb_lg_tpr(int D) {          // lanes per row: the power of two that covers D / 8, at most a workgroup
    int lg = 0;
    while (lg < 8 && (EMB_VEC << lg) < D) ++lg;
    return lg;
}

extern "C" int ddg_embedding(const void *ids, int ids_64, int64_t n, const void *table, int table_type, int64_t V, int D,
                             int64_t ld_table, float scale, void *out, int out_type, int64_t ld_out, void *stream) {
    if (n < 0 || V < 1 || V > 0x7FFFFFFF || D < 1 || D > EMB_MAX_D || ld_table < D || ld_out < D || !ddg_type_ok(table_type) ||
        !ddg_type_ok(out_type) || (ids_64 != 0 && ids_64 != 1))
        return DDG_E_ARG;
    if (n == 0) return DDG_OK;
    if (!ids || !table || !out) return DDG_E_ARG;
    const int lg = emb_lg_tpr(D), rpb = EMB_NT >> lg;
    const int slabs = (D + (EMB_VEC << lg) - 1) / (EMB_VEC << lg);
    // four rows per thread once that still leaves two workgroups per CU; one row below (few rows: latency, not bandwidth)
    const bool wide = ceil_div64(n, 4 * rpb) * slabs >= 512;
    const int64_t gx = ceil_div64(n, wide ? 4 * rpb : rpb);
    if (gx > ddg_max_grid(EMB_NT)) return DDG_E_UNSUPPORTED;
    return ddg_with_type(table_type, [&](auto ti) {
        return ddg_with_type(out_type, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            auto go = [&](auto id) {
                using ID = decltype(id);
                auto launch = [&](auto u, auto tiny) {
                    k_embed<TI, TO, ID, decltype(u)::value, decltype(tiny)::value>
                        <<<dim3((unsigned)gx, (unsigned)slabs), EMB_NT, 0, (hipStream_t)stream>>>(
                            (const ID *)ids, n, (const TI *)table, V, D, ld_table, scale, (TO *)out, ld_out, lg);
                };
                const std::integral_constant<int, 4> four;
                const std::integral_constant<int, 1> one;
                if (D < EMB_VEC) wide ? launch(four, std::true_type()) : launch(one, std::true_type());
                else wide ? launch(four, std::false_type()) : launch(one, std::false_type());
                DDG_CHECK_LAUNCH();
                return (int)DDG_OK;
            };
            return ids_64 ? go(int64_t()) : go(int32_t());
        });
    });
}

// ---------------------------------------------------------------------------------------------
// gradient: stable counting sort of (id, position), digits of at most 9 bits, least significant first.  Bound by latency: per pass 5
// us for the counts and 8 (20 000 tokens) to 15 us (262 144) for the scatter, whose workgroups each add up the counts of all
// tiles themselves instead of a third launch for them; up to 4 096 tokens 5 us in all
// ---------------------------------------------------------------------------------------------
#define SORT_NT 512
#define SORT_WAVES (SORT_NT / 64)
#define SORT_BINS 512
#define SORT_MAX_TILES 128            // a tile's workgroup reads every earlier tile's counts: 128 x 512 words at most
#define SORT_SMALL 4096               // up to this many tokens one workgroup sorts in LDS
// Sums beforehand, of chunks of 2^lg1 positions and of 2^lg2: the longest walk that a row can need is 2 (2^lg1 - 1) single tokens, 2
// (2^(lg2 - lg1) - 1) sums of 2^lg1 and n / 2^lg2 sums of 2^lg2
struct Chunks {
    int lg1, lg2;
};
// Small ones where the walk's latency counts, larger ones where the number of the largest does.  Word-like ids: 5 000 tokens of 64
// elements 31 us (with 64 and 4 096: 48), 65 536 of 256 73 (32 and 1 024: 80; 64 and 4 096: 92), of eight ids 61 (71; 112), of
// 200 50 (51; 71), but all of one id 117, 69 and 62: its row's n / 2^lg2 sums are added by one group of lanes; 262 144 of 64 in 5 000 rows 79 (64 and 4 096: 99), 262 144 of 2 048 523 (538).  Fewer than 1 024 tokens: a second launch (3 us)
// is dearer than 64 sums at most.
static constexpr int64_t CHUNKS_SMALL = 65536, CHUNKS_MIDDLE = 1 << 20;
static inline Chunks chunks_of(int64_t n) {
    return n < 1024 ? Chunks{4, 10} : n <= CHUNKS_SMALL ? Chunks{4, 8} : n <= CHUNKS_MIDDLE ? Chunks{5, 10} : Chunks{6, 12};
}

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
// wave's LDS accesses are executed in program order, so the count of one group of 64 is seen by the next.  Four groups are
// loaded at a time, by get(first, k, p), the first four by the caller, the others while the four before them are placed.
template <class Get, class Put>
__device__ __forceinline__ void place_segment(int64_t lo, int64_t hi, int shift, int digit_bits, volatile uint32_t *next,
                                              uint32_t (&k)[4], uint32_t (&p)[4], const Get &get, const Put &put) {
    const int lane = threadIdx.x & 63;
    for (int64_t g0 = lo; g0 < hi; g0 += 256) {
        uint32_t k1[4] = {}, p1[4] = {};
        if (g0 + 256 < hi) get(g0 + 256, k1, p1);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (g0 + u * 64 >= hi) break;
            const bool live = g0 + u * 64 + lane < hi;
            const uint32_t d = (k[u] >> shift) & ((1u << digit_bits) - 1);
            const uint64_t m = match_digit(d, live, digit_bits);
            const uint32_t rank = __popcll(m & (((uint64_t)1 << lane) - 1));
            if (live) {
                const uint32_t at = next[d];
                put(at + rank, k[u], p[u]);
                if (rank == 0) next[d] = at + __popcll(m);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            k[u] = k1[u];
            p[u] = p1[u];
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
    const int64_t lo = blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n, seg = tile / SORT_WAVES;
    const int64_t slo = lo + w * seg < hi ? lo + w * seg : hi, shi = slo + seg < hi ? slo + seg : hi;
    auto get = [&](int64_t first, uint32_t (&k)[4], uint32_t (&p)[4]) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = first + u * 64 + (t & 63);
            k[u] = i < shi ? src.k(i) : 0;
            p[u] = i < shi ? src.p(i) : 0;
        }
    };
    // the segment's first pairs (all of them, up to 262 144 tokens) and the counts of the tiles are on the way together
    uint32_t k[4], p[4], before = 0, total = 0;
    get(slo, k, p);
    if (t < bins)
        for (int b = 0; b < tiles; b += 32) {           // (32 loads in flight: a loop of single ones took 30 us)
            uint32_t h[32];
#pragma unroll
            for (int u = 0; u < 32; ++u) h[u] = b + u < tiles ? hist[(int64_t)(b + u) * SORT_BINS + t] : 0;
#pragma unroll
            for (int u = 0; u < 32; ++u) {
                total += h[u];
                if (b + u < (int)blockIdx.x) before += h[u];
            }
        }
    for (int i = 0; i < SORT_WAVES; ++i) next[i][t] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (slo + u * 64 + (t & 63) < shi) atomicAdd(&next[w][(k[u] >> shift) & (bins - 1)], 1u);
    for (int64_t i0 = slo + 256; i0 < shi; i0 += 256) {
        uint32_t more[4], unused[4];
        get(i0, more, unused);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * 64 + (t & 63) < shi) atomicAdd(&next[w][(more[u] >> shift) & (bins - 1)], 1u);
    }
    uint32_t at = block_exclusive(total, wsum) + before;
    for (int i = 0; i < SORT_WAVES; ++i) {
        const uint32_t c = next[i][t];
        next[i][t] = at;
        at += c;
    }
    __syncthreads();
    place_segment(slo, shi, shift, digit_bits, next[w], k, p, get, [&](uint32_t d, uint32_t key, uint32_t pos) {
        okey[d] = key;
        opos[d] = pos;
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
        auto get = [&](int64_t first, uint32_t (&k)[4], uint32_t (&p)[4]) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = (int)first + u * 64 + (t & 63);
                k[u] = i < shi ? key[a][i] : 0;
                p[u] = i < shi ? pos[a][i] : 0;
            }
        };
        uint32_t k[4], p[4];
        get(slo, k, p);
        place_segment(slo, shi, shift, digit_bits, next[w], k, p, get, [&](uint32_t d, uint32_t to_key, uint32_t to_pos) {
            key[1 - a][d] = to_key;
            pos[1 - a][d] = (uint16_t)to_pos;
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
// acc += rows [a, b) of src
template <bool TINY>
__device__ __forceinline__ void add_rows(const float *__restrict__ src, const Columns &c, uint32_t a, uint32_t b,
                                         float (&acc)[EMB_VEC]) {
#pragma unroll 1
    for (; a < b; a += 2) {                             // (two in flight: more would cost every wave registers)
        const vec8<float> x = load_row<TINY>(src + (int64_t)a * c.D, c);
        const vec8<float> y = load_row<TINY>(src + (int64_t)(a + 1 < b ? a + 1 : a) * c.D, c);
        add_row<float>(acc, x);
        if (a + 1 < b) add_row<float>(acc, y);
    }
}

// LEVEL 1: part[c] = sum of the dy rows of the c-th 2^lg1 sorted positions if they all belong to one row of the table;
// LEVEL 2: part[c] = sum of the LEVEL-1 sums of the c-th 2^lg2 positions, under the same condition.  Other chunks are never read.  Bound by
// HBM (the rows of frequent ids among 262 144 tokens of 2 048 elements: 87 us), LEVEL 2 by latency (7 us).
template <class T, int LEVEL, bool TINY>
__global__ __launch_bounds__(EMB_NT) void k_embg_part(const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos,
                                                      int64_t chunks, Chunks ch, uint32_t V, const T *__restrict__ src, int64_t ld, int D,
                                                      float *__restrict__ part, int lg_tpr) {
    const int tpr = 1 << lg_tpr;
    const Columns cs((blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * EMB_VEC, D);
    const int64_t c = (int64_t)blockIdx.x * (EMB_NT >> lg_tpr) + (threadIdx.x >> lg_tpr);
    const int len = 1 << (LEVEL == 1 ? ch.lg1 : ch.lg2), adds = LEVEL == 1 ? len : 1 << (ch.lg2 - ch.lg1);
    if (c >= chunks || cs.col >= D) return;
    const uint32_t k = key[c * len];
    if (k >= V || k != key[c * len + len - 1]) return;
    float acc[EMB_VEC] = {};
    uint32_t p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) p[u] = LEVEL == 1 ? pos[c * adds + u] : (uint32_t)(c * adds + u);
    for (int j = 0; j < adds; j += 8) {                   // eight rows in flight, and with them the next eight positions
        vec8<T> v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = load_row<TINY, true>(src + (int64_t)p[u] * ld, cs);
        const int next = j + 8 < adds ? j + 8 : j;
#pragma unroll
        for (int u = 0; u < 8; ++u) p[u] = LEVEL == 1 ? pos[c * adds + next + u] : (uint32_t)(c * adds + next + u);
#pragma unroll
        for (int u = 0; u < 8; ++u) add_row<T>(acc, v[u]);
    }
    store_row<TINY>(part + c * D, cs, acc);
}

// How the sorted positions [a, b) of a row divide: single tokens [a, a1) and [b1, b), sums of 2^lg1 [a1, a2) and [b2, b1), sums
// of 2^lg2 [a2, b2)
struct RowParts {
    uint32_t a, a1, a2, b2, b1, b;
};
__device__ __forceinline__ RowParts row_parts(uint32_t a, uint32_t b, const Chunks &ch) {
    RowParts p = {a, b, b, b, b, b};
    const uint32_t up1 = (a + (1u << ch.lg1) - 1) >> ch.lg1 << ch.lg1, dn1 = b >> ch.lg1 << ch.lg1;
    if (up1 >= dn1) return p;                           // no whole chunk
    p.a1 = up1;
    p.b1 = dn1;
    const uint32_t up2 = (a + (1u << ch.lg2) - 1) >> ch.lg2 << ch.lg2, dn2 = b >> ch.lg2 << ch.lg2;
    p.a2 = up2 < dn2 ? up2 : dn1;
    p.b2 = up2 < dn2 ? dn2 : dn1;
    return p;
}

#define ROWS_MAX 32                   // table rows per wave, at most: one lane finds the positions of one row

// Lane l: the first of n sorted keys that is >= v + min(l, rows), for l <= rows <= ROWS_MAX; by the whole wave (v and rows the same
// in every lane).  64 probes at a time for the first and the last of them (two or three rounds of loads where a search by
// halves needs 8 to 18, one after the other), then the few keys in between at once.
__device__ __forceinline__ uint32_t wave_lower_bounds(const uint32_t *__restrict__ key, uint32_t n, uint32_t v, uint32_t rows) {
    const uint32_t lane = threadIdx.x & 63, to[2] = {v, v + rows};
    uint32_t lo[2] = {0, 0}, len[2] = {n, n};           // the place is in [lo, lo + len]
    while (len[0] | len[1]) {
        uint64_t less[2];
        uint32_t step[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            step[i] = (len[i] + 63) / 64;
            const uint32_t at = (lane + 1) * step[i] - 1;
            less[i] = __ballot(at < len[i] && key[lo[i] + at] < to[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!len[i]) continue;
            const uint32_t skip = __popcll(less[i]) * step[i], left = len[i] > skip ? len[i] - skip : 0;
            lo[i] += skip;
            len[i] = left < step[i] - 1 ? left : step[i] - 1;
        }
    }
    const uint32_t count = lo[1] - lo[0];
    uint32_t x = lane < rows ? lane : rows;
    if (count > 128) {                                  // frequent rows
        uint32_t a = lo[0], b = lo[1];
        while (__any(a < b)) {
            const uint32_t mid = a + (b - a) / 2;
            const bool go = a < b, is_less = go && key[mid] < v + x;
            if (go && is_less) a = mid + 1;
            if (go && !is_less) b = mid;
        }
        return a;
    }
    // how many of the keys are below, bit by bit from the top: `same` agree with x so far
    uint32_t before = 0, d[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) d[i] = i * 64 + lane < count ? key[lo[0] + i * 64 + lane] - v : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint64_t same = __ballot(i * 64 + lane < count), below = 0;
#pragma unroll
        for (int bit = 5; bit >= 0; --bit) {
            const uint64_t ones = __ballot((d[i] >> bit) & 1);
            if ((x >> bit) & 1) below |= same & ~ones;
            same &= (x >> bit) & 1 ? ones : ~ones;
        }
        before += __popcll(below);
    }
    return lo[0] + before;
}
static_assert(ROWS_MAX < 64, "six bits");

// A group of 2^lg lanes owns `rows` consecutive rows of the table and as many columns as it has lanes x 8.  The single tokens
// of all its rows form one list, which is walked four at a time with the next four loads in flight, across the rows' borders:
// most rows have few tokens, and a walk row by row would wait out the memory's latency for each of them (609 us, now
// 370 us, for 262 144 tokens of 2 048 elements in 128 000 rows).
template <class T, class TO, bool TINY>
__global__ __launch_bounds__(EMB_NT, sizeof(T) == 2 ? 5 : 4) void k_embg_rows(const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos, int64_t n, Chunks ch,
                                                      int64_t V, const T *__restrict__ dy, int64_t ld, int D,
                                                      const float *__restrict__ part1, const float *__restrict__ part2, float scale,
                                                      int accumulate, TO *__restrict__ out, int64_t ldo, int lg, int rows, int slabs, int stream) {
    const uint32_t rblock = blockIdx.x / slabs, slab = blockIdx.x - rblock * slabs;
    const int lane = threadIdx.x & 63, lanes = 1 << lg, in_group = lane & (lanes - 1), group = lane >> lg;
    const int64_t wave0 = ((int64_t)rblock * (EMB_NT / 64) + (threadIdx.x >> 6)) * ((64 >> lg) * rows);
    if (wave0 >= V) return;
    // lane l: where row wave0 + l begins, up to the one behind the wave's last
    uint32_t begin;
    if (rows > 1) {                                     // enough waves to hide a search by halves, which is less work (2 % of 500 us)
        uint32_t lo = 0, hi = (uint32_t)n;
        const uint64_t v = wave0 + lane;
        while (__any(lo < hi)) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const bool go = lo < hi, less = go && key[mid] < v;
            if (go && less) lo = mid + 1;
            if (go && !less) hi = mid;
        }
        begin = lo;
    } else {                                            // (65 536 tokens of 256 elements in 32 000 rows 63 -> 58 us)
        const int here = V - wave0 < (64 >> lg) * rows ? (int)(V - wave0) : (64 >> lg) * rows;
        begin = wave_lower_bounds(key, (uint32_t)n, (uint32_t)__builtin_amdgcn_readfirstlane((int)wave0), here);
    }
    const Columns c((slab * lanes + in_group) * EMB_VEC, D);
    const int64_t v0 = wave0 + group * rows;
    // lane r of the group: row r's positions and single tokens, and how many the rows up to it have.  From here on groups go
    // their own ways and exchange data within themselves only
    const int own = group * rows + (in_group < rows ? in_group : rows - 1);
    const int first = __shfl((int)begin, own), behind = __shfl((int)begin, own + 1);
    const RowParts rp = row_parts(first, behind, ch);
    const int singles = in_group < rows && v0 + in_group < V ? (int)(rp.a1 - rp.a + rp.b - rp.b1) : 0;
    int upto = singles;                                 // inclusive prefix over the group's rows
    for (int d = 1; d < lanes; d <<= 1) {
        const int y = __shfl_up(upto, d, lanes);
        if (in_group >= d) upto += y;
    }
    const int total = __shfl(upto, lanes - 1, lanes);

    float acc[EMB_VEC] = {};
    int row = 0;                                        // row of the group whose sum acc is
    auto finish = [&]() {                               // writes row `row`, begins the next
        const int64_t v = v0 + row;
        const uint32_t a = __shfl(first, row, lanes), b = __shfl(behind, row, lanes);
        if (v < V && c.col < D && !(accumulate && a == b)) {
            const RowParts p = row_parts(a, b, ch);
            if (p.a1 < p.b1) {
                add_rows<TINY>(part1, c, p.a1 >> ch.lg1, p.a2 >> ch.lg1, acc);
                add_rows<TINY>(part2, c, p.a2 >> ch.lg2, p.b2 >> ch.lg2, acc);
                add_rows<TINY>(part1, c, p.b2 >> ch.lg1, p.b1 >> ch.lg1, acc);
            }
            TO *o = out + v * ldo;
            vec8<TO> old = {};
            if (accumulate) old = load_row<TINY>(o, c);
#pragma unroll
            for (int i = 0; i < EMB_VEC; ++i) acc[i] = (float)old[i] + scale * acc[i];
            if (stream) store_row<TINY, true>(o, c, acc);
            else store_row<TINY>(o, c, acc);
        }
#pragma unroll
        for (int i = 0; i < EMB_VEC; ++i) acc[i] = 0.f;
        ++row;
    };

    int item_pos = 0, item_row = rows;                  // this lane's item of the current batch of `lanes` items
    auto fetch = [&](int j, vec8<T>(&w)[4]) {
#pragma unroll
        for (int u = 0; u < 4; ++u)                     // (behind the list: token 0, not used)
            w[u] = load_row<TINY, true>(dy + (int64_t)__shfl(item_pos, j + u, lanes) * ld, c);
    };
    for (int base = 0; base < total; base += lanes) {
        // lane l: item base + l of the list, its row by counting the rows that end before it
        const int it = base + in_group;
        int rr = 0;
        for (int k = 0; k < rows; ++k) rr += __shfl(upto, k, lanes) <= it;
        const int rc = rr < rows ? rr : rows - 1;
        const uint32_t ordinal = it - (__shfl(upto, rc, lanes) - __shfl(singles, rc, lanes));
        const RowParts p = row_parts(__shfl(first, rc, lanes), __shfl(behind, rc, lanes), ch);
        const uint32_t at = ordinal < p.a1 - p.a ? p.a + ordinal : p.b1 + (ordinal - (p.a1 - p.a));
        item_row = it < total ? rr : rows;
        item_pos = it < total ? (int)pos[at] : 0;
        const int count = total - base < lanes ? total - base : lanes;
        vec8<T> v[4], w[4];
        fetch(0, v);
        for (int j = 0; j < count; j += 4) {
            if (j + 4 < count) fetch(j + 4, w);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (j + u < count) {
                    const int to = __shfl(item_row, j + u, lanes);
                    while (row < to) finish();
                    add_row<T>(acc, v[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = w[u];
        }
    }
    while (row < rows) finish();
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
    const Chunks ch = chunks_of(n);
    w.part1 = (float *)take((size_t)(n >> ch.lg1) * D * 4);
    w.part2 = (float *)take((size_t)(n >> ch.lg2) * D * 4);
    w.bytes = o;
    return w;
}

extern "C" size_t ddg_embedding_grad_workspace_bytes(int64_t n, int D) {
    if (n < 0 || n > 0x7FFFFFFF || D < 1 || D > EMB_MAX_D) return 0;
    size_t most = emb_carve(nullptr, n, D).bytes;       // fewer tokens may need more: larger chunks begin behind these
    for (const int64_t last : {CHUNKS_SMALL, CHUNKS_MIDDLE}) {
        const size_t bytes = emb_carve(nullptr, n < last ? n : last, D).bytes;
        most = bytes > most ? bytes : most;
    }
    return most;
}

extern "C" int ddg_embedding_grad(const void *ids, int ids_64, int64_t n, const void *dy, int dy_type, int64_t ld_dy, int64_t V,
                                  int D, float scale, int64_t padding_idx, int accumulate, void *out, int out_type, int64_t ld_out,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    if (n < 0 || V < 1 || D < 1 || D > EMB_MAX_D || ld_dy < D || ld_out < D || !ddg_type_ok(dy_type) || !ddg_type_ok(out_type) ||
        (ids_64 != 0 && ids_64 != 1) || !out)
        return DDG_E_ARG;
    if (n > 0x7FFFFFFF || V > 0x7FFFFFFE) return DDG_E_UNSUPPORTED;
    if (n == 0 && accumulate) return DDG_OK;
    if (n > 0 && (!ids || !dy)) return DDG_E_ARG;
    if (!workspace || workspace_bytes < emb_carve(nullptr, n, D).bytes) return DDG_E_WORKSPACE;
    if ((uintptr_t)workspace & 15) return DDG_E_ARG;
    const Chunks ch = chunks_of(n);
    const int lg = emb_lg_tpr(D), rpb = EMB_NT >> lg;
    const int slabs = (D + (EMB_VEC << lg) - 1) / (EMB_VEC << lg);
    // k_embg_rows: groups of 8 to 64 lanes, and as many rows per group (16 at most, 32 per wave) as leave about 8 192 waves
    const int rlg = lg < 3 ? 3 : lg > 6 ? 6 : lg, groups = 64 >> rlg;
    const int64_t rslabs = ceil_div64(D, EMB_VEC << rlg);
    int64_t rows = V * rslabs / ((int64_t)groups * 8192);
    const int most = ROWS_MAX / groups < 16 ? ROWS_MAX / groups : 16;
    rows = rows < 1 ? 1 : rows > most ? most : rows;
    const int64_t rgrid = ceil_div64(V, EMB_NT / 64 * groups * rows);
    if (rgrid * rslabs > ddg_max_grid(EMB_NT) || ceil_div64(n >> ch.lg1, rpb) > ddg_max_grid(EMB_NT)) return DDG_E_UNSUPPORTED;
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
    return ddg_with_type(dy_type, [&](auto ti) {
        using TI = decltype(ti);
        auto sums = [&](auto tiny) {
            constexpr bool TINY = decltype(tiny)::value;
            const int64_t c1 = n >> ch.lg1, c2 = n >> ch.lg2;
            if (c1)
                k_embg_part<TI, 1, TINY><<<dim3((unsigned)ceil_div64(c1, rpb), slabs), EMB_NT, 0, s>>>(
                    w.key[cur], w.pos[cur], c1, ch, (uint32_t)V, (const TI *)dy, ld_dy, D, w.part1, lg);
            if (c2)
                k_embg_part<float, 2, TINY><<<dim3((unsigned)ceil_div64(c2, rpb), slabs), EMB_NT, 0, s>>>(
                    w.key[cur], w.pos[cur], c2, ch, (uint32_t)V, w.part1, D, D, w.part2, lg);
            return ddg_with_type(out_type, [&](auto to) {
                using TO = decltype(to);
                k_embg_rows<TI, TO, TINY><<<(unsigned)(rgrid * rslabs), EMB_NT, 0, s>>>(
                    w.key[cur], w.pos[cur], n, ch, V, (const TI *)dy, ld_dy, D, w.part1, w.part2, scale, accumulate, (TO *)out, ld_out,
                    rlg, (int)rows, (int)rslabs, V * D > EMB_STREAM);
                DDG_CHECK_LAUNCH();
                return (int)DDG_OK;
            });
        };
        return D < EMB_VEC ? sums(std::true_type()) : sums(std::false_type());
    });
}
