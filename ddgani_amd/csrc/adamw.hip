// AdamW over many tensors at once, states in 32 or in 8 bits, gradients clipped by their global norm on the device.
//
//     |g| = sqrt(sum over all tensors of g^2)         c = min(1, max_norm / (|g| + 1e-6))       g' = c g
//     m <- m + (1 - b1)(g' - m)        v <- b2 v + (1 - b2) g'^2
//     w <- w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by HBM traffic: fp32 parameters, gradients and states move 28 bytes an element, 8-bit states with 16-bit gradients
// and fp32 masters behind 16-bit parameters 16 bytes; the norm reads the gradients once more.  All tensors go through one
// launch (the table of at most 64 tensors travels in the kernel arguments, so a captured graph holds it); the step number,
// the bias corrections and the clip factor live in device memory, so a replayed graph advances them.
//
// 8-bit states: blocks of 256 consecutive elements share an fp32 scale s = max / 448 and keep e4m3 codes.  What is kept of v is its
// root r: the root halves the exponent range a block has to span, 2^-9 ... 448 = 2^17.8 in r is 2^35 in v.  Both averages are slow:
// where a step changes one by less than half a code, rounding to nearest puts the code back that was there, in every step.  b2
// close to 1 does that to r everywhere, so r is rounded up where its fraction plus a dither number passes one.  The number is a Weyl
// sequence over (element, step): it needs no random generator and no memory, and over the steps it is equally often above as below
// any fraction.  A positive r is never stored as 0, so that no element divides by eps alone.
// m must not keep its code either once its gradient stops: r goes on falling beside it, and the weight would walk on m / r for ever
// (b1 0.9, b2 0.95, half of every block without a gradient: 2 000 steps moved that half by 686 lr where 32 bits move it by 2.5).
// In e4m3's normal range half a code is 1/16 of the value at most, so that up to b1 = 0.93 a decay of 1 - b1 always reaches the next
// code and nearest, which is less noise than a dither, is kept there; in the linear range below 2^-6 (codes under 8: 0.9 x 4 = 3.6 is 4
// again) m is rounded by a dither of its own, as r is but down to 0, and above b1 = 0.93 everywhere.  The same half: moved by 2.5 lr, and
// then it rests.  What nearest still costs is the last half code of a gradient that stays the same: m comes to a stop up to half a
// code / (1 - b1) from it.
#include <math.h>
#include <type_traits>
#include "types.h"

#define ADW_NT 256
#define ADW_BLOCK DDG_ADAMW_BLOCK                 // elements that share a scale = one wave x 4 elements
#define ADW_VEC 4
#define ADW_WIDE 4                                // state blocks per wave in the wide variant (1 in the other)
#define ADW_TABLE 64
#define ADW_FEW 1024                              // workgroups that sum all partial norms themselves, at most
#define ADW_NORM_GRID 2048                        // workgroups of the norm per launch: eight per CU, 16 KB of partial sums
#define ADW_NEAREST_B1 0.93                       // 1 - b1 above half a code, 1/16 of a value, with room for the roundings of m / s
#define ADW_LINEAR 0.015625f                      // 2^-6: codes below are multiples of 2^-9
#define ADW_TINY 7.888609052210118e-31f           // 2^-100: blocks below are stored as zeros (448 / max stays finite)

struct AdwEntry {
    void *p;
    const void *g;
    int64_t n, off;
    float keep;                                   // 1 - lr wd
    int32_t chunk0;                               // first workgroup
};
struct AdwTable {
    AdwEntry t[ADW_TABLE];                        // behind `count`: chunk0 = INT32_MAX
    int count;
};
static_assert(ADW_TABLE == 64, "one lane looks at one entry");

struct AdwScalars {
    float step_size, root2;                       // lr / (1 - b1^t), sqrt(1 - b2^t)
    uint32_t dither_m, dither_r;                  // of the step
};
// device side of the handle (DDG_ADAMW_CONTROL_BYTES)
struct AdwControl {
    int64_t step;                                 // steps done
    float norm, clip;                             // of the last step
    AdwScalars sc;
    int32_t skip;                                 // 1: the norm is not finite, nothing moves
    int64_t next;                                 // step + 1, while a step without k_adamw_begin runs
};
struct AdwHyper {
    double lr, b1, b2;
    float max_norm;                               // <= 0: no clip
    bool dither_all;                              // 8 bits: m is dithered everywhere, not in the linear range only
};

__device__ __forceinline__ double adw_power(double b, int64_t t) {
    double r = 1.0;
    for (; t; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}
// bias corrections in fp64, as a host would form them
__device__ __forceinline__ AdwScalars adw_scalars(const AdwHyper &h, int64_t t) {
    return {(float)(h.lr / (1.0 - adw_power(h.b1, t))), (float)sqrt(1.0 - adw_power(h.b2, t)), (uint32_t)t * 2447445413u,
            (uint32_t)t * 2246822507u};
}

// the tensor of a workgroup: the last entry whose chunk0 <= chunk, one entry per lane
__device__ __forceinline__ int adw_find(const AdwTable &tb, int chunk) {
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(tb.t[threadIdx.x & 63].chunk0 <= chunk)) - 1);
}

// the partial sums of squares -> norm and clip factor, in every thread of the workgroup; false: the norm is not finite
template <int NT>
__device__ __forceinline__ bool adw_clip(const double *__restrict__ part, int64_t parts, float max_norm, float &norm, float &clip) {
    __shared__ double w[NT / 64];
    double sum = 0;
    int64_t i = threadIdx.x;
    for (; i + 3 * NT < parts; i += 4 * NT) sum += (part[i] + part[i + NT]) + (part[i + 2 * NT] + part[i + 3 * NT]);
    for (; i < parts; i += NT) sum += part[i];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0;
    for (int k = 0; k < NT / 64; ++k) sum += w[k];
    norm = (float)sqrt(sum);
    clip = max_norm / (norm + 1e-6f);
    clip = clip < 1.f ? clip : 1.f;
    return norm <= 3.402823466e38f;                              // false for NaN and infinity
}

// step number, scalars and (max_norm > 0) the clip factor of the step
__global__ __launch_bounds__(1024) void k_adamw_begin(const double *__restrict__ part, int64_t parts, AdwHyper h, AdwControl *c) {
    float norm, clip = 1.f;
    bool ok = true;
    if (h.max_norm > 0.f) ok = adw_clip<1024>(part, parts, h.max_norm, norm, clip);
    if (threadIdx.x) return;
    if (h.max_norm > 0.f) c->norm = norm;
    c->skip = !ok;
    if (!ok) return;
    c->clip = clip;
    c->sc = adw_scalars(h, ++c->step);
}

// One fp64 partial per workgroup, which takes every gridDim-th chunk; four or eight squares at a time are added in fp32,
// everything above in fp64.  ctl (may be NULL): the first workgroup writes the number of the step that begins.
template <class G, int UNITS>
__global__ __launch_bounds__(ADW_NT) void k_adamw_sqsum(AdwTable tb, int chunks, double *__restrict__ part, AdwControl *ctl) {
    constexpr int V = UNITS == 1 ? 4 : 8, LOADS = ADW_VEC * UNITS / V;
    double sum = 0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const AdwEntry &e = tb.t[adw_find(tb, c)];
        const int64_t base = (int64_t)(c - e.chunk0) * (ADW_NT * ADW_VEC * UNITS) + threadIdx.x * V;
        float v[LOADS][V];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int64_t i = base + u * (ADW_NT * V), left = e.n - i;
            load_n<V>((const G *)e.g + i, left < 0 ? 0 : left > V ? V : (int)left, v[u]);
        }
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            float s = 0;
#pragma unroll
            for (int k = 0; k < V; ++k) s += v[u][k] * v[u][k];
            sum += s;
        }
    }
    __shared__ double w[ADW_NT / 64];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    part[blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
    if (ctl && blockIdx.x == 0) ctl->next = ctl->step + 1;
}

// maximum over the wave, in every lane
__device__ __forceinline__ float wave_max(float x) {
    x = row16_max(x);
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}

// a non-negative value (already divided by the scale) -> e4m3 code, u below 2^20.  The bits below the code's last are the fraction
// within the code's step; below 2^-6 the codes are linear, which adding 2^-6 turns into the same case.
__device__ __forceinline__ int code_dithered(float y, uint32_t u) {
    const bool small = y < ADW_LINEAR;
    return (int)((__builtin_bit_cast(uint32_t, small ? y + ADW_LINEAR : y) + u) >> 20) - (small ? 968 : 960);
}
__device__ __forceinline__ uint32_t encode_r(const float (&y)[ADW_VEC], uint32_t first, uint32_t dither) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < ADW_VEC; ++i) {
        int c = code_dithered(y[i], ((first + i) * 2654435769u + dither) >> 12);
        c = c < 1 ? 1 : c > 126 ? 126 : c;
        if (!(y[i] > 0.f)) c = y[i] == 0.f ? 0 : 127;             // NaN stays NaN
        w |= (uint32_t)c << (8 * i);
    }
    return w;
}
// was: the codes stored so far.  every: all are dithered, else those that are linear codes (no exponent) before and now, in a branch
// that most waves pass by (nearest alone 1 081 us for the step of 332 million elements, 1 102 so; every lane through it 1 112 and
// 1 138 on another card, and small steps 8 % longer).  (The Weyl steps of the two dithers have nothing in common: 2^32 times the
// inverse of the golden ratio and its like for x^3 = x + 1)
__device__ __forceinline__ uint32_t encode_m(const float (&y)[ADW_VEC], uint32_t was, bool every, uint32_t first, uint32_t dither) {
    uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)w, true);
    const uint32_t e = (was | w) & 0x78787878u;                   // a byte of zero: linear
    if (!__any(every || ((e - 0x01010101u) & ~e & 0x80808080u))) return w;
#pragma unroll
    for (int i = 0; i < ADW_VEC; ++i) {
        const float a = fabsf(y[i]);
        const int c = code_dithered(a, ((first + i) * 3242174889u + dither) >> 12);
        const uint32_t byte = (uint32_t)(c > 126 ? 126 : c) | (y[i] < 0.f ? 128u : 0u);
        if (a < INFINITY && (every || !(e >> (8 * i) & 0x78))) w = (w & ~(0xFFu << (8 * i))) | byte << (8 * i);
    }
    return w;
}
__device__ __forceinline__ void decode(uint32_t w, float scale, float (&y)[ADW_VEC]) {
    y[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale;
    y[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale;
    y[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale;
    y[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale;
}
template <bool STREAM> __device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int n) {
    if (n >= ADW_VEC) return STREAM ? __builtin_nontemporal_load((const uint32_t *)p) : *(const uint32_t *)p;
    uint32_t w = 0;
    for (int i = 0; i < n; ++i) w |= (uint32_t)p[i] << (8 * i);
    return w;
}
template <bool STREAM> __device__ __forceinline__ void store_codes(uint8_t *p, int n, uint32_t w) {
    if (n >= ADW_VEC && STREAM) __builtin_nontemporal_store(w, (uint32_t *)p);
    else if (n >= ADW_VEC) *(uint32_t *)p = w;
    else
        for (int i = 0; i < n; ++i) p[i] = (uint8_t)(w >> (8 * i));
}

struct AdwState {
    void *m, *v;
    float *ms, *vs, *master;
};

// A wave owns UNITS blocks of 256 elements, four consecutive elements per lane: every access is one contiguous piece per
// wave, and a block's maximum is one reduction over the wave.  All loads come first.  Workgroups take the table from its end:
// what the norm read last is still in the 256 MB cache, and in the wide variant everything but the gradients goes past it
// (332 million elements 1 185 -> 1 070 to 1 110 us, of which the norm takes 105).  SELF (with a clip, at most ADW_FEW workgroups in all): every workgroup
// adds up the partial norms and forms the step's scalars itself, which is quicker than a launch of its own for them.
// (One launch for norm and step, whose last workgroup to arrive goes on alone, is slower: an atomic that all XCDs share takes
// 85 ns a workgroup.)
// No contraction: the products round as the formulas read.
#pragma clang fp contract(off)
template <class P, class G, bool BITS8, bool MASTER, int UNITS, bool SELF>
__global__ __launch_bounds__(ADW_NT) void k_adamw(AdwTable tb, AdwState st, AdwControl *ctl, AdwHyper h, float one_m_b1, float b2,
                                                  float one_m_b2, float eps, const double *__restrict__ part, int parts) {
    constexpr bool WIDE = UNITS > 1;
    const int chunk = (int)(gridDim.x - 1 - blockIdx.x);
    const AdwEntry &e = tb.t[adw_find(tb, chunk)];
    P *__restrict__ const p = (P *)e.p;
    const G *__restrict__ const g = (const G *)e.g;
    const int lane = threadIdx.x & 63;
    const int64_t base = (int64_t)(chunk - e.chunk0) * (ADW_NT * ADW_VEC * UNITS) + (threadIdx.x >> 6) * (UNITS * ADW_BLOCK);
    float gv[UNITS][ADW_VEC], wv[UNITS][ADW_VEC], mv[UNITS][ADW_VEC], vv[UNITS][ADW_VEC], ms[UNITS], vs[UNITS];
    uint32_t mc[UNITS], vc[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int64_t b = base + u * ADW_BLOCK, i = b + lane * ADW_VEC, f = e.off + i;
        const int n = e.n - i >= ADW_VEC ? ADW_VEC : e.n > i ? (int)(e.n - i) : 0;
        load_n<ADW_VEC>(g + i, n, gv[u]);
        if (MASTER) load_n<ADW_VEC, WIDE>(st.master + f, n, wv[u]);
        else load_n<ADW_VEC, WIDE>(p + i, n, wv[u]);
        if (BITS8) {
            mc[u] = load_codes<WIDE>((const uint8_t *)st.m + f, n);
            vc[u] = load_codes<WIDE>((const uint8_t *)st.v + f, n);
            const int64_t blk = (e.off + b) / ADW_BLOCK;
            ms[u] = b < e.n ? st.ms[blk] : 0.f;
            vs[u] = b < e.n ? st.vs[blk] : 0.f;
        } else {
            load_n<ADW_VEC, WIDE>((const float *)st.m + f, n, mv[u]);
            load_n<ADW_VEC, WIDE>((const float *)st.v + f, n, vv[u]);
        }
    }
    AdwScalars sc;
    float clip;
    if constexpr (SELF) {
        float norm;
        const int64_t t = ctl->next;
        const bool ok = adw_clip<ADW_NT>(part, parts, h.max_norm, norm, clip);
        if (chunk == 0 && threadIdx.x == 0) {
            ctl->norm = norm;
            if (ok) ctl->step = t;                                // (nobody reads it in this launch)
        }
        if (!ok) return;
        sc = adw_scalars(h, t);
    } else {
        if (ctl->skip) return;
        sc = ctl->sc;
        clip = h.max_norm > 0.f ? ctl->clip : 1.f;
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int64_t b = base + u * ADW_BLOCK;                   // first element of the block, of this lane's four: i
        if (b >= e.n) break;
        const int64_t i = b + lane * ADW_VEC, f = e.off + i;
        const int n = e.n - i >= ADW_VEC ? ADW_VEC : e.n > i ? (int)(e.n - i) : 0;
        float w[ADW_VEC], m[ADW_VEC], v[ADW_VEC], r[ADW_VEC];
        if (BITS8) {
            decode(mc[u], ms[u], m);
            decode(vc[u], vs[u], v);
#pragma unroll
            for (int k = 0; k < ADW_VEC; ++k) v[k] = v[k] * v[k];
        }
        float top_m = 0.f, top_r = 0.f;
#pragma unroll
        for (int k = 0; k < ADW_VEC; ++k) {
            if (!BITS8) {
                m[k] = mv[u][k];
                v[k] = vv[u][k];
            }
            const float gg = gv[u][k] * clip;
            m[k] = m[k] + one_m_b1 * (gg - m[k]);
            v[k] = v[k] * b2 + one_m_b2 * gg * gg;
            r[k] = sqrtf(v[k]);
            w[k] = wv[u][k] * e.keep - sc.step_size * (m[k] / (r[k] / sc.root2 + eps));
            if (k < n) {
                top_m = fmaxf(top_m, fabsf(m[k]));
                top_r = fmaxf(top_r, r[k]);
            }
        }
        if (MASTER) store_n<ADW_VEC, WIDE>(st.master + f, n, w);
        store_n<ADW_VEC, WIDE>(p + i, n, w);
        if (BITS8) {
            const int64_t blk = (e.off + b) / ADW_BLOCK;
            top_m = wave_max(top_m);
            top_r = wave_max(top_r);
            const float im = top_m >= ADW_TINY ? (1.f / top_m) * 448.f : 0.f, ir = top_r >= ADW_TINY ? (1.f / top_r) * 448.f : 0.f;
#pragma unroll
            for (int k = 0; k < ADW_VEC; ++k) {
                m[k] = m[k] * im;
                r[k] = r[k] * ir;
            }
            // (a block that has no m yet, or one whose largest m grows by half in a step, holds no slow average)
            const bool young = !(ms[u] * im > 0.6667f);
            store_codes<WIDE>((uint8_t *)st.m + f, n,
                              encode_m(m, young ? 0x78787878u : mc[u], h.dither_all && !young, (uint32_t)f, sc.dither_m));
            store_codes<WIDE>((uint8_t *)st.v + f, n, encode_r(r, (uint32_t)f, sc.dither_r));
            if (lane == 0) {
                st.ms[blk] = top_m >= ADW_TINY ? top_m * (1.f / 448.f) : 0.f;
                st.vs[blk] = top_r >= ADW_TINY ? top_r * (1.f / 448.f) : 0.f;
            }
        } else {
            store_n<ADW_VEC, WIDE>((float *)st.m + f, n, m);
            store_n<ADW_VEC, WIDE>((float *)st.v + f, n, v);
        }
    }
}
#pragma clang fp contract(on)

static inline int64_t adw_chunk(bool wide) { return ADW_NT * ADW_VEC * (wide ? ADW_WIDE : 1); }
static int64_t adw_total(const ddg_adamw_tensor *t, int n_tensors, bool wide) {
    int64_t total = 0;
    for (int i = 0; i < n_tensors; ++i) total += t[i].numel > 0 ? ceil_div64(t[i].numel, adw_chunk(wide)) : 0;
    return total;
}

static int adw_check(const ddg_adamw_tensor *t, int n_tensors, int64_t state_len) {
    if (n_tensors < 0 || (n_tensors > 0 && !t) || state_len < 0) return DDG_E_ARG;
    int64_t chunks = 0;
    for (int i = 0; i < n_tensors; ++i) {
        if (t[i].numel < 0 || t[i].offset < 0 || t[i].offset % ADW_BLOCK || t[i].numel > state_len ||
            t[i].offset > state_len - t[i].numel || !(t[i].weight_decay >= 0) || !ddg_type_ok(t[i].param_type) || !ddg_type_ok(t[i].grad_type))
            return DDG_E_ARG;
        if (t[i].numel > 0 && (!t[i].param || !t[i].grad)) return DDG_E_ARG;
        chunks += ceil_div64(t[i].numel, adw_chunk(true));
        if (chunks > ddg_max_grid(ADW_NT)) return DDG_E_UNSUPPORTED;
    }
    return DDG_OK;
}

// One block per wave and workgroups of 1 024 elements while that gives at most ADW_FEW of them (a million elements: latency
// counts), else four blocks per wave
static inline bool adw_wide(const ddg_adamw_tensor *t, int n_tensors) { return adw_total(t, n_tensors, false) > ADW_FEW; }

static inline int64_t adw_parts(const ddg_adamw_tensor *t, int n_tensors) {
    const int64_t parts = adw_total(t, n_tensors, adw_wide(t, n_tensors));
    return parts > 0 ? parts : 1;
}
extern "C" size_t ddg_adamw_workspace_bytes(const ddg_adamw_tensor *tensors, int n_tensors) {
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return 0;
    const int64_t parts = adw_parts(tensors, n_tensors);
    return (size_t)(parts > ADW_FEW || !adw_wide(tensors, n_tensors) ? parts : ADW_FEW) * sizeof(double);     // (what fewer elements take)
}

// calls f(table, workgroups) for groups of at most ADW_TABLE non-empty tensors that `take` accepts, in their order
template <class Take, class F>
static int adw_groups(const ddg_adamw_tensor *t, int n_tensors, bool wide, double lr, const Take &take, const F &f) {
    AdwTable tb;
    tb.count = 0;
    int64_t chunks = 0;
    auto flush = [&]() {
        for (int i = tb.count; i < ADW_TABLE; ++i) tb.t[i].chunk0 = INT32_MAX;
        const int rc = tb.count ? f(tb, chunks) : (int)DDG_OK;
        tb.count = 0;
        chunks = 0;
        return rc;
    };
    for (int i = 0; i < n_tensors; ++i) {
        if (t[i].numel == 0 || !take(t[i])) continue;
        tb.t[tb.count++] = {t[i].param, t[i].grad, t[i].numel, t[i].offset, (float)(1.0 - lr * (double)t[i].weight_decay),
                            (int32_t)chunks};
        chunks += ceil_div64(t[i].numel, adw_chunk(wide));
        if (tb.count == ADW_TABLE) {
            const int rc = flush();
            if (rc) return rc;
        }
    }
    return flush();
}

extern "C" int ddg_adamw_step(const ddg_adamw_tensor *tensors, int n_tensors, int state_bits, void *exp_avg, void *exp_avg_sq,
                              float *exp_avg_scale, float *exp_avg_sq_scale, float *masters, int64_t state_len, double lr,
                              double beta1, double beta2, double eps, double max_norm, void *control, void *workspace,
                              size_t workspace_bytes, void *stream) {
    const int rc = adw_check(tensors, n_tensors, state_len);
    if (rc) return rc;
    if ((state_bits != 8 && state_bits != 32) || !control || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) ||
        !(eps >= 0) || !(lr >= 0) || max_norm != max_norm)
        return DDG_E_ARG;
    if (state_len > 0 && (!exp_avg || !exp_avg_sq || (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)))) return DDG_E_ARG;
    if (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq | (uintptr_t)control | (uintptr_t)workspace) & 7) return DDG_E_ARG;
    const hipStream_t s = (hipStream_t)stream;
    AdwControl *ctl = (AdwControl *)control;
    static_assert(sizeof(AdwControl) <= DDG_ADAMW_CONTROL_BYTES, "control block");
    double *part = (double *)workspace;
    // (a positive max_norm below the smallest fp32 number still clips)
    const float to_norm = max_norm > 0 ? fmaxf((float)max_norm, 1.401298464e-45f) : 0.f;
    const AdwHyper h = {lr, beta1, beta2, to_norm, beta1 > ADW_NEAREST_B1};
    const bool wide = adw_wide(tensors, n_tensors), clip = max_norm > 0;
    const int64_t total = adw_total(tensors, n_tensors, wide);
    const bool self = clip && !wide && total > 0;       // no k_adamw_begin
    int64_t parts = 0;
    uint32_t types = 0;                                 // the (parameter, gradient) types that occur
    for (int i = 0; i < n_tensors; ++i)
        if (tensors[i].numel > 0) types |= 1u << (tensors[i].param_type * 3 + tensors[i].grad_type);
    if (clip) {
        if (!workspace || workspace_bytes < adw_parts(tensors, n_tensors) * sizeof(double)) return DDG_E_WORKSPACE;
        for (int gt = DDG_F32; gt <= DDG_F16; ++gt) {
            if (!(types & (0x49u << gt))) continue;
            const int r = adw_groups(
                tensors, n_tensors, wide, lr, [&](const ddg_adamw_tensor &t) { return t.grad_type == gt; },
                [&](const AdwTable &tb, int64_t chunks) {
                    return ddg_with_type(gt, [&](auto g) {
                        using G = decltype(g);
                        const int64_t grid = chunks < ADW_NORM_GRID ? chunks : ADW_NORM_GRID;
                        if (wide) k_adamw_sqsum<G, ADW_WIDE><<<(unsigned)grid, ADW_NT, 0, s>>>(tb, (int)chunks, part + parts, nullptr);
                        else k_adamw_sqsum<G, 1><<<(unsigned)grid, ADW_NT, 0, s>>>(tb, (int)chunks, part + parts, parts == 0 ? ctl : nullptr);
                        DDG_CHECK_LAUNCH();
                        parts += grid;
                        return (int)DDG_OK;
                    });
                });
            if (r) return r;
        }
    }
    if (!self) {
        k_adamw_begin<<<1, clip ? 1024 : 64, 0, s>>>(part, parts, h, ctl);
        DDG_CHECK_LAUNCH();
    }
    const AdwState st = {exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, masters};
    for (int pt = DDG_F32; pt <= DDG_F16; ++pt)
        for (int gt = DDG_F32; gt <= DDG_F16; ++gt) {
            if (!(types >> (pt * 3 + gt) & 1)) continue;
            // (chunk 0 of every group writes the step's number and norm: the same values)
            const int r = adw_groups(
                tensors, n_tensors, wide, lr,
                [&](const ddg_adamw_tensor &t) { return t.param_type == pt && t.grad_type == gt; },
                [&](const AdwTable &tb, int64_t chunks) {
                    return ddg_with_type(pt, [&](auto p) {
                        return ddg_with_type(gt, [&](auto g) {
                            using P = decltype(p);
                            using G = decltype(g);
                            auto go = [&](auto bits8, auto master, auto units, auto fin) {
                                k_adamw<P, G, decltype(bits8)::value, decltype(master)::value, decltype(units)::value,
                                        decltype(fin)::value><<<(unsigned)chunks, ADW_NT, 0, s>>>(
                                    tb, st, ctl, h, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, part,
                                    (int)parts);
                            };
                            const std::true_type yes;
                            const std::false_type no;
                            const std::integral_constant<int, 1> one;
                            const std::integral_constant<int, ADW_WIDE> more;
                            auto size = [&](auto bits8, auto master) {
                                if (wide) go(bits8, master, more, no);
                                else if (self) go(bits8, master, one, yes);
                                else go(bits8, master, one, no);
                            };
                            if constexpr (sizeof(P) == 2) {           // (an fp32 parameter is its own master)
                                if (masters && state_bits == 8) size(yes, yes);
                                else if (masters) size(no, yes);
                            }
                            if (sizeof(P) == 4 || !masters) {
                                if (state_bits == 8) size(yes, no); else size(no, no);
                            }
                            DDG_CHECK_LAUNCH();
                            return (int)DDG_OK;
                        });
                    });
                });
            if (r) return r;
        }
    return DDG_OK;
}
