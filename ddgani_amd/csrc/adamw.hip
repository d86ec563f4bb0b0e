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
// 8-bit states: blocks of 256 consecutive elements share an fp32 scale s = max / 448 and keep e4m3 codes.  m is rounded to
// nearest.  What is kept of v is its root r: the root halves the exponent range a block has to span, 2^-9 ... 448 = 2^17.8
// in r is 2^35 in v.  b2 close to 1 changes r by less than half a code per step, which rounding to nearest would undo each
// time, so r is rounded up where its fraction plus a dither number passes one.  The number is a Weyl sequence over (element,
// step): it needs no random generator and no memory, and over the steps it is equally often above as below any fraction.
// A positive r is never stored as 0, so that no element divides by eps alone.
#include <math.h>
#include <type_traits>
#include "types.h"

#define ADW_NT 256
#define ADW_BLOCK DDG_ADAMW_BLOCK                 // elements that share a scale = one wave x 4 elements
#define ADW_VEC 4
#define ADW_UNITS 4                               // state blocks per wave
#define ADW_CHUNK (ADW_NT * ADW_VEC * ADW_UNITS)  // elements per workgroup
#define ADW_TABLE 64
#define ADW_TINY 7.888609052210118e-31f           // 2^-100: blocks below are stored as zeros (448 / max stays finite)

struct AdwEntry {
    void *p;
    const void *g;
    int64_t n, off;
    float keep;                                   // 1 - lr wd
    int32_t chunk0;                               // first workgroup
};
struct AdwTable {
    AdwEntry t[ADW_TABLE];
    int count;
};

// device side of the handle (DDG_ADAMW_CONTROL_BYTES)
struct AdwControl {
    int64_t step;                                 // steps done, the current one included
    float norm, clip;
    float step_size, root2;                       // lr / (1 - b1^t), sqrt(1 - b2^t)
    uint32_t dither;                              // of this step
    int32_t skip;                                 // 1: the norm is not finite, nothing moves
};

__device__ __forceinline__ int adw_find(const AdwTable &tb, int chunk) {      // the last tensor whose chunk0 <= chunk
    int a = 0, b = tb.count;
    while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (tb.t[mid].chunk0 <= chunk) a = mid; else b = mid;
    }
    return a;
}

// one fp64 partial per workgroup; eight squares at a time are added in fp32, everything above in fp64
template <class G> __global__ __launch_bounds__(ADW_NT) void k_adamw_sqsum(AdwTable tb, double *__restrict__ part) {
    const AdwEntry &e = tb.t[adw_find(tb, blockIdx.x)];
    const G *g = (const G *)e.g;
    const int64_t base = (int64_t)(blockIdx.x - e.chunk0) * ADW_CHUNK;
    double sum = 0;
#pragma unroll
    for (int u = 0; u < ADW_CHUNK / (ADW_NT * 8); ++u) {
        const int64_t i = base + (u * ADW_NT + threadIdx.x) * 8;
        float v[8];
        const int64_t left = e.n - i;
        load_n<8>(g + i, left < 0 ? 0 : left > 8 ? 8 : (int)left, v);
        float s = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += v[k] * v[k];
        sum += s;
    }
    __shared__ double w[ADW_NT / 64];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}

// the step's scalars: norm and clip factor (max_norm > 0), step number, bias corrections in fp64 as the host would form them
__global__ __launch_bounds__(1024) void k_adamw_begin(const double *__restrict__ part, int64_t parts, float max_norm, double lr,
                                                      double b1, double b2, AdwControl *c) {
    __shared__ double w[16];
    double sum = 0;
    for (int64_t i = threadIdx.x; i < parts; i += 1024) sum += part[i];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    float clip = 1.f;
    bool ok = true;
    if (max_norm > 0.f) {
        sum = 0;
        for (int i = 0; i < 16; ++i) sum += w[i];
        const float norm = (float)sqrt(sum);
        ok = norm <= 3.402823466e38f;                            // false for NaN and infinity
        clip = max_norm / (norm + 1e-6f);
        clip = clip < 1.f ? clip : 1.f;
        c->norm = norm;
    }
    c->skip = !ok;
    if (!ok) return;
    const int64_t t = c->step + 1;
    c->step = t;
    c->clip = clip;
    c->step_size = (float)(lr / (1.0 - pow(b1, (double)t)));
    c->root2 = (float)sqrt(1.0 - pow(b2, (double)t));
    c->dither = (uint32_t)t * 2246822507u;
}

// maximum over the wave, in every lane
__device__ __forceinline__ float wave_max(float x) {
    x = row16_max(x);
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}

// four non-negative values (already divided by the scale) -> e4m3 codes.  The bits below the code's last are the fraction
// within the code's step; below 2^-6 the codes are linear, which adding 2^-6 turns into the same case.
__device__ __forceinline__ uint32_t encode_dithered(const float (&y)[ADW_VEC], uint32_t first, uint32_t dither) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < ADW_VEC; ++i) {
        const bool small = y[i] < 0.015625f;
        const uint32_t u = ((first + i) * 2654435769u + dither) >> 12;
        int c = (int)((__builtin_bit_cast(uint32_t, small ? y[i] + 0.015625f : y[i]) + u) >> 20) - (small ? 968 : 960);
        c = c < 1 ? 1 : c > 126 ? 126 : c;
        if (!(y[i] > 0.f)) c = y[i] == 0.f ? 0 : 127;             // NaN stays NaN
        w |= (uint32_t)c << (8 * i);
    }
    return w;
}
__device__ __forceinline__ uint32_t encode_nearest(const float (&y)[ADW_VEC]) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
__device__ __forceinline__ void decode(uint32_t w, float scale, float (&y)[ADW_VEC]) {
    y[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale;
    y[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale;
    y[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale;
    y[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale;
}
__device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int n) {
    if (n >= ADW_VEC) return *(const uint32_t *)p;
    uint32_t w = 0;
    for (int i = 0; i < n; ++i) w |= (uint32_t)p[i] << (8 * i);
    return w;
}
__device__ __forceinline__ void store_codes(uint8_t *p, int n, uint32_t w) {
    if (n >= ADW_VEC)
        *(uint32_t *)p = w;
    else
        for (int i = 0; i < n; ++i) p[i] = (uint8_t)(w >> (8 * i));
}

struct AdwState {
    void *m, *v;
    float *ms, *vs, *master;
};

// A wave owns ADW_UNITS blocks of 256 elements, four consecutive elements per lane: every access is one contiguous piece
// per wave, and a block's maximum is one reduction over the wave.  No contraction: the products round as the formulas read.
#pragma clang fp contract(off)
template <class P, class G, bool BITS8, bool MASTER>
__global__ __launch_bounds__(ADW_NT) void k_adamw(AdwTable tb, AdwState st, const AdwControl *__restrict__ ctl, float one_m_b1,
                                                  float b2, float one_m_b2, float eps) {
    if (ctl->skip) return;
    const AdwEntry &e = tb.t[adw_find(tb, blockIdx.x)];
    const float clip = ctl->clip, step_size = ctl->step_size, root2 = ctl->root2, keep = e.keep;
    const uint32_t dither = ctl->dither;
    P *p = (P *)e.p;
    const G *g = (const G *)e.g;
    const int lane = threadIdx.x & 63;
    const int64_t base = (int64_t)(blockIdx.x - e.chunk0) * ADW_CHUNK + (threadIdx.x >> 6) * (ADW_UNITS * ADW_BLOCK);
#pragma unroll
    for (int u = 0; u < ADW_UNITS; ++u) {
        const int64_t b = base + u * ADW_BLOCK;                   // first element of the block, of this lane's four: i
        if (b >= e.n) return;
        const int64_t i = b + lane * ADW_VEC, f = e.off + i;
        const int n = e.n - i >= ADW_VEC ? ADW_VEC : e.n > i ? (int)(e.n - i) : 0;
        float gv[ADW_VEC], w[ADW_VEC], m[ADW_VEC], v[ADW_VEC], r[ADW_VEC];
        load_n<ADW_VEC>(g + i, n, gv);
        if (MASTER) load_n<ADW_VEC>(st.master + f, n, w);
        else load_n<ADW_VEC>(p + i, n, w);
        const int64_t blk = (e.off + b) / ADW_BLOCK;
        if (BITS8) {
            decode(load_codes((const uint8_t *)st.m + f, n), st.ms[blk], m);
            decode(load_codes((const uint8_t *)st.v + f, n), st.vs[blk], v);
#pragma unroll
            for (int k = 0; k < ADW_VEC; ++k) v[k] = v[k] * v[k];
        } else {
            load_n<ADW_VEC>((const float *)st.m + f, n, m);
            load_n<ADW_VEC>((const float *)st.v + f, n, v);
        }
        float top_m = 0.f, top_r = 0.f;
#pragma unroll
        for (int k = 0; k < ADW_VEC; ++k) {
            const float gg = gv[k] * clip;
            m[k] = m[k] + one_m_b1 * (gg - m[k]);
            v[k] = v[k] * b2 + one_m_b2 * gg * gg;
            r[k] = sqrtf(v[k]);
            w[k] = w[k] * keep - step_size * (m[k] / (r[k] / root2 + eps));
            if (k < n) {
                top_m = fmaxf(top_m, fabsf(m[k]));
                top_r = fmaxf(top_r, r[k]);
            }
        }
        if (MASTER) store_n<ADW_VEC>(st.master + f, n, w);
        store_n<ADW_VEC>(p + i, n, w);
        if (BITS8) {
            top_m = wave_max(top_m);
            top_r = wave_max(top_r);
            const float im = top_m >= ADW_TINY ? (1.f / top_m) * 448.f : 0.f, ir = top_r >= ADW_TINY ? (1.f / top_r) * 448.f : 0.f;
#pragma unroll
            for (int k = 0; k < ADW_VEC; ++k) {
                m[k] = m[k] * im;
                r[k] = r[k] * ir;
            }
            store_codes((uint8_t *)st.m + f, n, encode_nearest(m));
            store_codes((uint8_t *)st.v + f, n, encode_dithered(r, (uint32_t)f, dither));
            if (lane == 0) {
                st.ms[blk] = top_m >= ADW_TINY ? top_m * (1.f / 448.f) : 0.f;
                st.vs[blk] = top_r >= ADW_TINY ? top_r * (1.f / 448.f) : 0.f;
            }
        } else {
            store_n<ADW_VEC>((float *)st.m + f, n, m);
            store_n<ADW_VEC>((float *)st.v + f, n, v);
        }
    }
}
#pragma clang fp contract(on)

static inline int64_t adw_chunks(int64_t n) { return ceil_div64(n, ADW_CHUNK); }

static int adw_check(const ddg_adamw_tensor *t, int n_tensors, int64_t state_len) {
    if (n_tensors < 0 || (n_tensors > 0 && !t) || state_len < 0) return DDG_E_ARG;
    for (int i = 0; i < n_tensors; ++i) {
        if (t[i].numel < 0 || t[i].offset < 0 || t[i].offset % ADW_BLOCK || t[i].numel > state_len ||
            t[i].offset > state_len - t[i].numel || !ddg_type_ok(t[i].param_type) || !ddg_type_ok(t[i].grad_type))
            return DDG_E_ARG;
        if (t[i].numel > 0 && (!t[i].param || !t[i].grad)) return DDG_E_ARG;
        if (adw_chunks(t[i].numel) > 0x7FFFFFFF / ADW_TABLE) return DDG_E_UNSUPPORTED;
    }
    return DDG_OK;
}

extern "C" size_t ddg_adamw_workspace_bytes(const ddg_adamw_tensor *tensors, int n_tensors) {
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return 0;
    int64_t parts = 0;
    for (int i = 0; i < n_tensors; ++i) parts += tensors[i].numel > 0 ? adw_chunks(tensors[i].numel) : 0;
    return (size_t)(parts > 0 ? parts : 1) * sizeof(double);
}

// calls f(table, chunks) for groups of at most ADW_TABLE non-empty tensors that `take` accepts, in their order
template <class Take, class F>
static int adw_groups(const ddg_adamw_tensor *t, int n_tensors, double lr, const Take &take, const F &f) {
    AdwTable tb;
    tb.count = 0;
    int64_t chunks = 0;
    auto flush = [&]() {
        const int rc = tb.count ? f(tb, chunks) : (int)DDG_OK;
        tb.count = 0;
        chunks = 0;
        return rc;
    };
    for (int i = 0; i < n_tensors; ++i) {
        if (t[i].numel == 0 || !take(t[i])) continue;
        tb.t[tb.count++] = {t[i].param, t[i].grad, t[i].numel, t[i].offset, (float)(1.0 - lr * (double)t[i].weight_decay),
                            (int32_t)chunks};
        chunks += adw_chunks(t[i].numel);
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
    double *part = (double *)workspace;
    int64_t parts = 0;
    if (max_norm > 0) {
        if (!workspace || workspace_bytes < ddg_adamw_workspace_bytes(tensors, n_tensors)) return DDG_E_WORKSPACE;
        for (int gt = DDG_F32; gt <= DDG_F16; ++gt) {
            const int r = adw_groups(
                tensors, n_tensors, lr, [&](const ddg_adamw_tensor &t) { return t.grad_type == gt; },
                [&](const AdwTable &tb, int64_t chunks) {
                    return ddg_with_type(gt, [&](auto g) {
                        k_adamw_sqsum<decltype(g)><<<(unsigned)chunks, ADW_NT, 0, s>>>(tb, part + parts);
                        DDG_CHECK_LAUNCH();
                        parts += chunks;
                        return (int)DDG_OK;
                    });
                });
            if (r) return r;
        }
    }
    k_adamw_begin<<<1, 1024, 0, s>>>(part, parts, (float)max_norm, lr, beta1, beta2, ctl);
    DDG_CHECK_LAUNCH();
    const AdwState st = {exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, masters};
    for (int pt = DDG_F32; pt <= DDG_F16; ++pt)
        for (int gt = DDG_F32; gt <= DDG_F16; ++gt) {
            const int r = adw_groups(
                tensors, n_tensors, lr, [&](const ddg_adamw_tensor &t) { return t.param_type == pt && t.grad_type == gt; },
                [&](const AdwTable &tb, int64_t chunks) {
                    return ddg_with_type(pt, [&](auto p) {
                        return ddg_with_type(gt, [&](auto g) {
                            using P = decltype(p);
                            using G = decltype(g);
                            auto go = [&](auto bits8, auto master) {
                                k_adamw<P, G, decltype(bits8)::value, decltype(master)::value><<<(unsigned)chunks, ADW_NT, 0, s>>>(
                                    tb, st, ctl, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps);
                            };
                            const std::true_type yes;
                            const std::false_type no;
                            if constexpr (sizeof(P) == 2) {           // (an fp32 parameter is its own master)
                                if (masters && state_bits == 8) go(yes, yes);
                                else if (masters) go(no, yes);
                            }
                            if (sizeof(P) == 4 || !masters) {
                                if (state_bits == 8) go(yes, no); else go(no, no);
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
