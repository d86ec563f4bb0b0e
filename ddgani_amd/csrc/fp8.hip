// Dense layer in 8-bit floating point (e4m3) with one scale for each block of 128, and its gradients.
//
//     Y[m, n]  = sum over k of Q(X)[m, k] Q(W)[n, k] + b[n]            X in groups of 128 along k, W in 128 x 128 blocks
//     dX[m, k] = sum over n of Q(dY)[m, n] Q(W)[n, k]                  dY in groups along n, the same codes of W
//     dW[n, k] = sum over m of Q'(dY)[m, n] Q'(X)[m, k]                both in groups of 128 along m
//     db[n]    = sum over m of dY[m, n]                                not quantised, fp32
//
// Q keeps e4m3 codes x / s rounded to nearest even, s the smallest power of two that brings the block's largest magnitude
// to 448 or below.  A power of two costs at most one of the 17 binary orders that a block can span and no precision above
// them, and buys two things: x / s is exact, so a code never depends on how the division rounded, and the scaled matrix
// instruction (v_mfma_scale_f32_16x16x128_f8f6f4) applies both operands' scales itself.  A block of 128 is exactly one such
// instruction deep, so the whole sum stays in its fp32 accumulator with no vector instruction in between.
//
// The fp8 matrix instructions drop bits inside: they align a group of products to its largest before adding them, which
// leaves 1.4e-5 of a result's size for one block and, as the cuts add up, 2e-4 for a sum over 32 blocks (measured against
// exact sums of normal codes).  That is far below the rounding of a bf16 result (2e-3) but not below that of an fp16 or fp32
// one, so only bf16 results come from them; for the others the codes are expanded to bf16, which holds code x scale exactly,
// and multiplied by v_mfma_f32_16x16x32_bf16 (8e-9 on the same data) at half the rate.
//
// Packed operand of `rows` rows and a reduction of `cols`: codes [rows][colsp] (colsp = cols rounded up to 128, zeros
// behind cols), then from the next multiple of 256 bytes the scales as biased exponents (2^(e - 127)), four consecutive
// blocks in one word: word [block / 4][row], byte block % 4.  The 16 rows of a matrix tile are 16 consecutive words.
#include <type_traits>
#include "types.h"

#define F8_BLOCK 128
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

static __host__ __device__ __forceinline__ int64_t f8_pad(int64_t cols) { return (cols + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK; }
static __host__ __device__ __forceinline__ size_t f8_codes_bytes(int64_t rows, int64_t cols) {
    return ((size_t)rows * f8_pad(cols) + 255) & ~(size_t)255;
}
static inline size_t f8_scale_bytes(int64_t rows, int64_t cols) {
    return (((size_t)rows * ((f8_pad(cols) / F8_BLOCK + 3) / 4) * 4) + 255) & ~(size_t)255;
}
struct F8Operand {
    uint8_t *q, *s;
    int64_t rows, cols;
};
static inline F8Operand f8_operand(void *base, int64_t rows, int64_t cols) {
    return {(uint8_t *)base, (uint8_t *)base + f8_codes_bytes(rows, cols), rows, cols};
}

// biased exponent of the scale for a block whose largest magnitude is a: the smallest power of two with a / s <= 448 =
// 1.75 x 2^8, found on the bits (a mantissa above 1.75 carries into the exponent).  Blocks below 2^-100 get no scale: 0
// stands for "all codes are zero" and reads as 2^-127, which no zero feels.
__device__ __forceinline__ int f8_exponent(float a) {
    return a >= 7.888609052210118e-31f ? (int)((__builtin_bit_cast(uint32_t, a) + 0x1FFFFFu) >> 23) - 8 : 0;
}
// 1 / s, exact; 0 for a block without a scale
__device__ __forceinline__ float f8_inverse(int e) { return e ? __builtin_bit_cast(float, (uint32_t)(254 - e) << 23) : 0.f; }
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ void f8_put_scale(uint8_t *s, int64_t rows, int64_t row, int64_t block, int e) {
    s[((block >> 2) * rows + row) * 4 + (block & 3)] = (uint8_t)e;
}

// ---------------------------------------------------------------------------------------------
// packing
// ---------------------------------------------------------------------------------------------
// groups along the rows: 16 lanes x 8 elements hold a group, its maximum is a reduction over one DPP row
template <class T>
__global__ __launch_bounds__(256) void k_f8_pack_rows(const T *__restrict__ x, int64_t ld, int64_t rows, int64_t cols, uint8_t *q,
                                                      uint8_t *s) {
    const int64_t cp = f8_pad(cols), nb = cp / F8_BLOCK;
    const int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (g >= rows * nb) return;                         // (whole DPP rows leave together)
    const int64_t r = g / nb, b = g - r * nb, c = b * F8_BLOCK + (threadIdx.x & 15) * 8;
    float v[8], a = 0.f;
    load_n<8>(x + r * ld + c, cols - c >= 8 ? 8 : cols > c ? (int)(cols - c) : 0, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));
    const int e = f8_exponent(row16_max(a));
    const float inv = f8_inverse(e);
    uint2 w;
    w.x = f8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    w.y = f8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    *(uint2 *)(q + r * cp + c) = w;
    if ((threadIdx.x & 15) == 0) f8_put_scale(s, rows, r, b, e);
}

// 128 x 128 tiles in registers, 8 x 8 elements per thread.  MODE F8_COLS: groups along the columns, packed transposed (qt, st);
// F8_ROWS_COLS: those and groups along the rows (q, s); F8_TILE: one scale for the tile, packed both ways (qt may be NULL).
// sums (may be NULL): fp32 column sums of the tile, [row tile][cols].
enum { F8_COLS, F8_ROWS_COLS, F8_TILE };
template <class T, int MODE>
__global__ __launch_bounds__(256) void k_f8_pack_tile(const T *__restrict__ x, int64_t ld, int64_t rows, int64_t cols, uint8_t *q,
                                                      uint8_t *s, uint8_t *qt, uint8_t *st, float *sums) {
    __shared__ float red[16][F8_BLOCK];
    __shared__ uint8_t tr[F8_BLOCK][F8_BLOCK + 8];
    const int tc = threadIdx.x & 15, tr8 = (threadIdx.x >> 4) * 8;
    const int64_t cb = blockIdx.x, rb = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    const int64_t r0 = rb * F8_BLOCK, c0 = cb * F8_BLOCK, c = c0 + tc * 8;
    if (r0 >= rows) return;
    const int64_t cp = f8_pad(cols), rp = f8_pad(rows);
    const int nc = cols - c >= 8 ? 8 : cols > c ? (int)(cols - c) : 0;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) load_n<8>(x + (r0 + tr8 + i) * ld + c, r0 + tr8 + i < rows ? nc : 0, v[i]);

    if (sums) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) a += v[i][j];
            red[threadIdx.x >> 4][tc * 8 + j] = a;
        }
        __syncthreads();
        if (threadIdx.x < F8_BLOCK && c0 + threadIdx.x < cols) {
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) a += red[i][threadIdx.x];
            sums[rb * cols + c0 + threadIdx.x] = a;
        }
        __syncthreads();
    }
    // column maxima of the tile (their maximum in F8_TILE)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i][j]));
        red[threadIdx.x >> 4][tc * 8 + j] = a;
    }
    __syncthreads();
    float top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        top[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top[j] = fmaxf(top[j], red[i][tc * 8 + j]);
    }
    int e[8];
    if (MODE == F8_TILE) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) a = fmaxf(a, top[j]);
        const int et = f8_exponent(row16_max(a));
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = et;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = f8_exponent(top[j]);
    }
    if (MODE == F8_TILE || MODE == F8_ROWS_COLS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = r0 + tr8 + i;
            int er = e[0];
            if (MODE == F8_ROWS_COLS) {
                float a = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) a = fmaxf(a, fabsf(v[i][j]));
                er = f8_exponent(row16_max(a));
            }
            const float inv = f8_inverse(er);
            if (r < rows) {
                uint2 w;
                w.x = f8_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
                w.y = f8_pack4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
                *(uint2 *)(q + r * cp + c) = w;
                if (tc == 0) f8_put_scale(s, rows, r, cb, er);
            }
        }
        if (MODE == F8_TILE && !qt) return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float inv = f8_inverse(e[j]);
        uint2 w;
        w.x = f8_pack4(v[0][j] * inv, v[1][j] * inv, v[2][j] * inv, v[3][j] * inv);
        w.y = f8_pack4(v[4][j] * inv, v[5][j] * inv, v[6][j] * inv, v[7][j] * inv);
        *(uint2 *)&tr[tc * 8 + j][tr8] = w;
        if (tr8 == 0 && c + j < cols) f8_put_scale(st, cols, c + j, rb, e[j]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {                       // 8 lanes write the 128 bytes of a column
        const int col = i * 32 + (threadIdx.x >> 3), at = (threadIdx.x & 7) * 16;
        if (c0 + col < cols) {
            uint4 w;
            __builtin_memcpy(&w, &tr[col][at], 16);
            *(uint4 *)(qt + (c0 + col) * rp + r0 + at) = w;
        }
    }
}

__global__ __launch_bounds__(256) void k_f8_colsum(const float *__restrict__ part, int64_t tiles, int64_t cols, float *__restrict__ out) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float a = 0.f;
    for (int64_t t = 0; t < tiles; ++t) a += part[t * cols + c];
    out[c] = a;
}

// ---------------------------------------------------------------------------------------------
// product of two packed operands: C[m, n] = sum over k of A[m, k] B[n, k]
// ---------------------------------------------------------------------------------------------
// LDS image of a stage: rows of 128 bytes (one block of the reduction), whose eight 16-byte pieces are exchanged by
// piece ^ (row / 2 % 8): a quarter wave that reads one piece of 16 consecutive rows touches all 64 banks once.  The
// copy into LDS writes linearly, so the exchange is applied to the global address.
__device__ __forceinline__ int f8_piece(int row, int piece) { return piece ^ ((row >> 1) & 7); }

// 32 codes of a lane -> the operands of four bf16 instructions, multiplied by the scale of biased exponent e
__device__ __forceinline__ void f8_expand(const i32x8 &f, uint32_t e, bf16x8 (&o)[4]) {
    const float s = __builtin_bit_cast(float, (e & 0xFF) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[i], s, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[i], s, true);
        o[i >> 1][(i & 1) * 4] = lo[0];
        o[i >> 1][(i & 1) * 4 + 1] = lo[1];
        o[i >> 1][(i & 1) * 4 + 2] = hi[0];
        o[i >> 1][(i & 1) * 4 + 3] = hi[1];
    }
}

template <int BM, int BN, int WM, int WN, bool EXPAND, class TO>
__global__ __launch_bounds__(64 * WM * WN) void k_f8_gemm(const uint8_t *__restrict__ A, const uint32_t *__restrict__ As, int64_t M,
                                                          const uint8_t *__restrict__ B, const uint32_t *__restrict__ Bs, int64_t N,
                                                          int64_t kp, const float *__restrict__ bias, TO *__restrict__ C, int64_t ldc,
                                                          int64_t tiles_m) {
    constexpr int WAVES = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16, ROWS = BM + BN, LOADS = ROWS / 8 / WAVES;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][ROWS * F8_BLOCK];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tm = blockIdx.x % tiles_m, tn = blockIdx.x / tiles_m;
    const int64_t m0 = tm * BM, n0 = tn * BN;
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int nk = (int)(kp / F8_BLOCK);

    // this wave's copies: 8 rows each, rows behind the end repeat the last one
    const uint8_t *src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int row = (i * WAVES + wave) * 8 + (lane >> 3), piece = f8_piece(row, lane & 7);
        if (row < BM) {
            const int64_t r = m0 + row < M ? m0 + row : M - 1;
            src[i] = A + r * kp + piece * 16;
        } else {
            const int64_t r = n0 + row - BM < N ? n0 + row - BM : N - 1;
            src[i] = B + r * kp + piece * 16;
        }
    }
    auto copy = [&](int k, int buf) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src[i] + (int64_t)k * F8_BLOCK),
                                             (__attribute__((address_space(3))) void *)&lds[buf][(i * WAVES + wave) * 8 * F8_BLOCK],
                                             16, 0, 0);
    };
    // this lane's scale words: operand row lane % 16 of every 16-row tile
    const uint32_t *sa[MT], *sb[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t r = m0 + wm + i * 16 + (lane & 15);
        sa[i] = As + (r < M ? r : M - 1);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t r = n0 + wn + j * 16 + (lane & 15);
        sb[j] = Bs + (r < N ? r : N - 1);
    }
    uint32_t ea[MT], eb[NT];
    f32x4 acc[NT][MT] = {};
    auto frag = [&](const uint8_t *base, int row) {
        i32x8 f;
        const uint8_t *p = base + row * F8_BLOCK;
        const int4 lo = *(const int4 *)(p + f8_piece(row, (lane >> 4) * 2) * 16), hi = *(const int4 *)(p + f8_piece(row, (lane >> 4) * 2 + 1) * 16);
        f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
        f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
        return f;
    };
    copy(0, 0);
    for (int k = 0; k < nk; ++k) {
        __syncthreads();                                // stage k has landed, stage k - 1 has been read
        if (k + 1 < nk) copy(k + 1, (k + 1) & 1);
        if ((k & 3) == 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i) ea[i] = sa[i][(int64_t)(k >> 2) * M];
#pragma unroll
            for (int j = 0; j < NT; ++j) eb[j] = sb[j][(int64_t)(k >> 2) * N];
        }
        const uint8_t *la = lds[k & 1], *lb = lds[k & 1] + BM * F8_BLOCK;
        i32x8 fa[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[i] = frag(la, wm + i * 16 + (lane & 15));
        const int sh = (k & 3) * 8;
        // first operand of the instructions: rows of the result = n, so that a lane gets four consecutive n
        if constexpr (EXPAND) {
            bf16x8 xa[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i) f8_expand(fa[i], ea[i] >> sh, xa[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                bf16x8 xb[4];
                f8_expand(frag(lb, wn + j * 16 + (lane & 15)), eb[j] >> sh, xb);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[t], xa[i][t], acc[j][i], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const i32x8 fb = frag(lb, wn + j * 16 + (lane & 15));
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa[i], acc[j][i], 0, 0, 0,
                                                                                (int)(eb[j] >> sh), 0, (int)(ea[i] >> sh));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t n = n0 + wn + j * 16 + (lane >> 4) * 4;
        const int left = N - n >= 4 ? 4 : N > n ? (int)(N - n) : 0;
        float b[4] = {};
        if (bias) load_n<4>(bias + n, left, b);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int64_t m = m0 + wm + i * 16 + (lane & 15);
            if (m >= M) continue;
            float v[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = acc[j][i][t] + b[t];
            store_n<4>(C + m * ldc + n, left, v);
        }
    }
}

// At most 16 rows: bound by the bytes of B.  A workgroup owns 16 rows of B and its eight waves share the reduction; the
// rows of X are quantised on the way (each lane its 32 elements of a group), so one launch does the layer.  Every result
// type takes the expanded product here: the matrix unit is idle either way.
#define F8_SKINNY 16
#define F8_SKW 8
template <class TX, class TO>
__global__ __launch_bounds__(64 * F8_SKW) void k_f8_skinny(const TX *__restrict__ X, int64_t ldx, int M, int64_t K,
                                                           const uint8_t *__restrict__ B, const uint32_t *__restrict__ Bs, int64_t N,
                                                           int64_t kp, const float *__restrict__ bias, TO *__restrict__ C,
                                                           int64_t ldc) {
    __shared__ f32x4 part[F8_SKW][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * 16, nr = n0 + m < N ? n0 + m : N - 1;
    const int nk = (int)(kp / F8_BLOCK);
    f32x4 acc = {};
    for (int k = wave; k < nk; k += F8_SKW) {
        const int64_t c = (int64_t)k * F8_BLOCK + (lane >> 4) * 32;
        i32x8 fb;
        __builtin_memcpy(&fb, __builtin_assume_aligned(B + nr * kp + c, 32), 32);
        const uint32_t eb = Bs[(int64_t)(k >> 2) * N + nr] >> ((k & 3) * 8);
        float v[32], a = 0.f;
        load_n<32>(X + (m < M ? m : 0) * ldx + c, m >= M || c >= K ? 0 : K - c >= 32 ? 32 : (int)(K - c), v);
#pragma unroll
        for (int i = 0; i < 32; ++i) a = fmaxf(a, fabsf(v[i]));
        a = fmaxf(a, __shfl_xor(a, 16));
        a = fmaxf(a, __shfl_xor(a, 32));
        const int e = f8_exponent(a);
        const float inv = f8_inverse(e);
        i32x8 fa;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            fa[i] = (int)f8_pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
        bf16x8 xa[4], xb[4];
        f8_expand(fa, e, xa);
        f8_expand(fb, eb, xb);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[t], xa[t], acc, 0, 0, 0);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < F8_SKW; ++w) acc += part[w][lane];
    const int64_t n = n0 + (lane >> 4) * 4;
    const int left = N - n >= 4 ? 4 : N > n ? (int)(N - n) : 0;
    if (m >= M) return;
    float v[4], b[4] = {};
    if (bias) load_n<4>(bias + n, left, b);
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = acc[t] + b[t];
    store_n<4>(C + m * ldc + n, left, v);
}

// ---------------------------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------------------------
template <int N> using Int = std::integral_constant<int, N>;
static inline bool f8_dims_ok(int64_t a, int64_t b) { return a >= 0 && b >= 0 && a <= 0x3FFFFFFF && b <= 0x3FFFFFFF; }

extern "C" size_t ddg_fp8_operand_bytes(int64_t rows, int64_t cols) {
    if (!f8_dims_ok(rows, cols)) return 0;
    return f8_codes_bytes(rows, cols) + f8_scale_bytes(rows, cols);
}

static int f8_pack_rows(const void *x, int type, int64_t ld, const F8Operand &o, hipStream_t s) {
    const int64_t groups = o.rows * (f8_pad(o.cols) / F8_BLOCK), grid = ceil_div64(groups, 16);
    if (grid > 0x7FFFFFFF) return DDG_E_UNSUPPORTED;
    return ddg_with_type(type, [&](auto t) {
        using T = decltype(t);
        k_f8_pack_rows<T><<<(unsigned)grid, 256, 0, s>>>((const T *)x, ld, o.rows, o.cols, o.q, o.s);
        DDG_CHECK_LAUNCH();
        return (int)DDG_OK;
    });
}
// x [rows, cols] -> o (groups along rows, or tiles) and ot (its transpose); see k_f8_pack_tile
template <int MODE>
static int f8_pack_tile(const void *x, int type, int64_t ld, int64_t rows, int64_t cols, const F8Operand &o, const F8Operand &ot,
                        float *sums, hipStream_t s) {
    const int64_t rb = ceil_div64(rows, F8_BLOCK), cb = ceil_div64(cols, F8_BLOCK), gy = rb < 32768 ? rb : 32768;
    const dim3 grid((unsigned)cb, (unsigned)gy, (unsigned)ceil_div64(rb, gy));
    return ddg_with_type(type, [&](auto t) {
        using T = decltype(t);
        k_f8_pack_tile<T, MODE><<<grid, 256, 0, s>>>((const T *)x, ld, rows, cols, o.q, o.s, ot.q, ot.s, sums);
        DDG_CHECK_LAUNCH();
        return (int)DDG_OK;
    });
}

static int f8_gemm(const F8Operand &a, const F8Operand &b, const float *bias, void *c, int type, int64_t ldc, hipStream_t s) {
    return ddg_with_type(type, [&](auto t) {
        using TO = decltype(t);
        constexpr bool EXPAND = !std::is_same<TO, bf16_t>::value;
        auto go = [&](auto bm, auto bn, auto wm, auto wn) {
            constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
            const int64_t tm = ceil_div64(a.rows, BM), tn = ceil_div64(b.rows, BN);
            if (tm * tn > 0x7FFFFFFF) return (int)DDG_E_UNSUPPORTED;
            k_f8_gemm<BM, BN, WM, WN, EXPAND, TO><<<(unsigned)(tm * tn), 64 * WM * WN, 0, s>>>(
                a.q, (const uint32_t *)a.s, a.rows, b.q, (const uint32_t *)b.s, b.rows, f8_pad(a.cols), bias, (TO *)c, ldc, tm);
            DDG_CHECK_LAUNCH();
            return (int)DDG_OK;
        };
        if constexpr (EXPAND) {
            return go(Int<128>(), Int<128>(), Int<2>(), Int<2>());
        } else {
            if (ceil_div64(a.rows, 256) * ceil_div64(b.rows, 256) >= 192) return go(Int<256>(), Int<256>(), Int<2>(), Int<4>());
            return go(Int<128>(), Int<128>(), Int<2>(), Int<2>());
        }
    });
}

extern "C" int ddg_fp8_pack_weight(const void *W, int type, int64_t ld, int64_t out, int64_t in, void *packed, void *packed_t,
                                   void *stream) {
    if (!f8_dims_ok(out, in) || out < 1 || in < 1 || ld < in || !ddg_type_ok(type) || !W || !packed) return DDG_E_ARG;
    if (((uintptr_t)packed | (uintptr_t)packed_t) & 255) return DDG_E_ARG;
    F8Operand t = {};
    if (packed_t) t = f8_operand(packed_t, in, out);
    return f8_pack_tile<F8_TILE>(W, type, ld, out, in, f8_operand(packed, out, in), t, nullptr, (hipStream_t)stream);
}

extern "C" size_t ddg_fp8_linear_workspace_bytes(int64_t rows, int64_t in) {
    if (!f8_dims_ok(rows, in) || in < 1) return 0;
    return rows <= F8_SKINNY ? 0 : ddg_fp8_operand_bytes(rows, in);
}

extern "C" int ddg_fp8_linear(const void *x, int x_type, int64_t ld_x, int64_t rows, const void *packed_w, int64_t out, int64_t in,
                              const float *bias, void *y, int y_type, int64_t ld_y, void *workspace, size_t workspace_bytes,
                              void *stream) {
    if (!f8_dims_ok(rows, in) || !f8_dims_ok(out, 0) || out < 1 || in < 1 || ld_x < in || ld_y < out || !ddg_type_ok(x_type) ||
        !ddg_type_ok(y_type) || !packed_w || ((uintptr_t)packed_w & 255))
        return DDG_E_ARG;
    if (rows == 0) return DDG_OK;
    if (!x || !y) return DDG_E_ARG;
    const F8Operand w = f8_operand((void *)packed_w, out, in);
    const hipStream_t s = (hipStream_t)stream;
    if (rows <= F8_SKINNY)
        return ddg_with_type(x_type, [&](auto tx) {
            return ddg_with_type(y_type, [&](auto to) {
                using TX = decltype(tx);
                using TO = decltype(to);
                k_f8_skinny<TX, TO><<<(unsigned)ceil_div64(out, 16), 64 * F8_SKW, 0, s>>>(
                    (const TX *)x, ld_x, (int)rows, in, w.q, (const uint32_t *)w.s, out, f8_pad(in), bias, (TO *)y, ld_y);
                DDG_CHECK_LAUNCH();
                return (int)DDG_OK;
            });
        });
    if (!workspace || workspace_bytes < ddg_fp8_linear_workspace_bytes(rows, in)) return DDG_E_WORKSPACE;
    if ((uintptr_t)workspace & 255) return DDG_E_ARG;
    const F8Operand a = f8_operand(workspace, rows, in);
    const int rc = f8_pack_rows(x, x_type, ld_x, a, s);
    return rc ? rc : f8_gemm(a, w, bias, y, y_type, ld_y, s);
}

struct F8GradWs {
    void *dy, *dyt, *xt;
    float *sums;
    size_t bytes;
};
static inline F8GradWs f8_grad_carve(void *base, int64_t rows, int64_t out, int64_t in) {
    char *p = (char *)base;
    size_t o = 0;
    auto take = [&](size_t b) {
        char *q = p ? p + o : nullptr;
        o += (b + 255) & ~(size_t)255;
        return q;
    };
    F8GradWs w;
    w.dy = take(ddg_fp8_operand_bytes(rows, out));
    w.dyt = take(ddg_fp8_operand_bytes(out, rows));
    w.xt = take(ddg_fp8_operand_bytes(in, rows));
    w.sums = (float *)take((size_t)ceil_div64(rows, F8_BLOCK) * out * 4);
    w.bytes = o;
    return w;
}
extern "C" size_t ddg_fp8_linear_grads_workspace_bytes(int64_t rows, int64_t out, int64_t in) {
    if (!f8_dims_ok(rows, in) || !f8_dims_ok(out, 0) || out < 1 || in < 1) return 0;
    return f8_grad_carve(nullptr, rows, out, in).bytes;
}

extern "C" int ddg_fp8_linear_grads(const void *dy, int dy_type, int64_t ld_dy, const void *x, int x_type, int64_t ld_x,
                                    int64_t rows, const void *packed_wt, int64_t out, int64_t in, void *dx, int dx_type,
                                    int64_t ld_dx, float *dw, float *db, void *workspace, size_t workspace_bytes, void *stream) {
    if (!f8_dims_ok(rows, in) || !f8_dims_ok(out, 0) || rows < 1 || out < 1 || in < 1 || ld_dy < out || ld_x < in || ld_dx < in ||
        !ddg_type_ok(dy_type) || !ddg_type_ok(x_type) || !ddg_type_ok(dx_type) || !dy || !x || !packed_wt || !dx || !dw ||
        ((uintptr_t)packed_wt & 255))
        return DDG_E_ARG;
    if (!workspace || workspace_bytes < ddg_fp8_linear_grads_workspace_bytes(rows, out, in)) return DDG_E_WORKSPACE;
    if ((uintptr_t)workspace & 255) return DDG_E_ARG;
    const F8GradWs w = f8_grad_carve(workspace, rows, out, in);
    const hipStream_t s = (hipStream_t)stream;
    const F8Operand gy = f8_operand(w.dy, rows, out), gyt = f8_operand(w.dyt, out, rows), xt = f8_operand(w.xt, in, rows);
    int rc = f8_pack_tile<F8_ROWS_COLS>(dy, dy_type, ld_dy, rows, out, gy, gyt, db ? w.sums : nullptr, s);
    if (rc) return rc;
    if (db) {
        k_f8_colsum<<<(unsigned)ceil_div64(out, 256), 256, 0, s>>>(w.sums, ceil_div64(rows, F8_BLOCK), out, db);
        DDG_CHECK_LAUNCH();
    }
    rc = f8_pack_tile<F8_COLS>(x, x_type, ld_x, rows, in, F8Operand{}, xt, nullptr, s);
    if (rc) return rc;
    rc = f8_gemm(gy, f8_operand((void *)packed_wt, in, out), nullptr, dx, dx_type, ld_dx, s);
    return rc ? rc : f8_gemm(gyt, xt, nullptr, dw, DDG_F32, in, s);
}
