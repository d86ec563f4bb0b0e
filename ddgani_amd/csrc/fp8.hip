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
// one, so only bf16 results come from them (where large products of a
// block cancel, what is dropped can be more than the small result's rounding: another result type avoids it); for the others the codes are expanded to bf16, which holds code x scale exactly,
// and multiplied by v_mfma_f32_16x16x32_bf16 (8e-9 on the same data) at half the rate.
//
// Packed operand of `rows` rows and a reduction of `cols`: codes of colsp columns (cols rounded up to 128, zeros behind cols),
// for the product's first operand row by row; for its second (weights, and X in dW) in pieces of 16 rows x 128 columns,
// [row / 16][column / 128], as the matrix instruction takes them: lane r + 16 g holds codes 32 g to 32 g + 31 of row r, and the
// first 16 of all lanes come first.  A wave loads such a piece as 2 KB in a row.  (Rows up to the next multiple of 16 are zeros.)
// Then, from the next multiple of 256 bytes, the scales as biased exponents (2^(e - 127)), four consecutive blocks in one word:
// word [block / 4][row], byte block % 4.  The 16 rows of a matrix tile are 16 consecutive words.  1 KB behind the scales belongs
// to the operand too: a workgroup reads whole 256-row pieces of them.
#include <type_traits>
#include "types.h"

#define F8_BLOCK 128
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

static __host__ __device__ __forceinline__ int64_t f8_pad(int64_t cols) { return (cols + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK; }
static __host__ __device__ __forceinline__ size_t f8_codes_bytes(int64_t rows, int64_t cols) {
    return ((size_t)(rows + 15) / 16 * 16 * f8_pad(cols) + 255) & ~(size_t)255;
}
static inline size_t f8_scale_bytes(int64_t rows, int64_t cols) {
    return (((size_t)rows * ((f8_pad(cols) / F8_BLOCK + 3) / 4) * 4) + 1024 + 255) & ~(size_t)255;
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
// groups along the rows: 16 lanes x 8 elements hold a group, its maximum is a reduction over one DPP row.  Bound by HBM: 200 000 x
// 176 fp32 37 us, 5.2 TB/s
template <class T>
__global__ __launch_bounds__(256) void k_f8_pack_rows(const T *__restrict__ x, int64_t ld, int64_t rows, int64_t cols, uint8_t *q,
                                                      uint8_t *s) {
    const int64_t cp = f8_pad(cols), nb = cp / F8_BLOCK;
    const int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (g >= rows * nb) return;                         // (whole DPP rows leave together)
    const int64_t r = g / nb, b = g - r * nb, c = b * F8_BLOCK + (threadIdx.x & 15) * 8;
    float v[8], a = 0.f;
    load_n<8, true>(x + r * ld + c, cols - c >= 8 ? 8 : cols > c ? (int)(cols - c) : 0, v);
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
// F8_ROWS_COLS packs a first operand (of either product), the others second operands.
// sums (may be NULL): fp32 column sums of the tile, [row tile][cols].  Bound by HBM once there are a few tiles per CU (operands of
// the gradients of 4001 x 2048 x 5000 in bf16 25 us, 4.2 TB/s), by latency below (128 x 176 x 352 7 us): hence all loads in front of
// the first use, and the whole tile in registers.
enum { F8_COLS, F8_ROWS_COLS, F8_TILE };
struct F8Pack {
    const void *x;
    int64_t ld, rows, cols;
    uint8_t *q, *s, *qt, *st;
    float *sums;
};
template <class T, int MODE> __device__ __forceinline__ void f8_pack_one(const F8Pack &p, int64_t tile) {
    const T *const x = (const T *)p.x;
    const int64_t ld = p.ld, rows = p.rows, cols = p.cols;
    uint8_t *const q = p.q, *const s = p.s, *const qt = p.qt, *const st = p.st;
    float *const sums = p.sums;
    __shared__ float red[2][4][F8_BLOCK];
    __shared__ uint8_t tr[F8_BLOCK][F8_BLOCK + 8];
    const int tc = threadIdx.x & 15, tr8 = (threadIdx.x >> 4) * 8;
    const int64_t tiles_c = (cols + F8_BLOCK - 1) / F8_BLOCK, rb = tile / tiles_c, cb = tile - rb * tiles_c;
    const int64_t r0 = rb * F8_BLOCK, c0 = cb * F8_BLOCK, c = c0 + tc * 8;
    const int64_t cp = f8_pad(cols), rp = f8_pad(rows);
    const int nc = cols - c >= 8 ? 8 : cols > c ? (int)(cols - c) : 0;
    float v[8][8];
    if (cols % 8 == 0) {                                // a thread's eight columns exist or not, together: no branch between loads
        vec8<T> t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = load_whole(x + (r0 + tr8 + i < rows ? r0 + tr8 + i : rows - 1) * ld + (nc ? c : 0));
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = nc && r0 + tr8 + i < rows ? (float)t[i][j] : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_n<8>(x + (r0 + tr8 + i) * ld + c, r0 + tr8 + i < rows ? nc : 0, v[i]);
    }

    // column maxima (and sums) of the tile: over the thread's eight rows, the four row groups of a wave, the four waves
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i][j]));
        a = fmaxf(a, __shfl_xor(a, 16));
        a = fmaxf(a, __shfl_xor(a, 32));
        if (lane < 16) red[0][wave][tc * 8 + j] = a;
    }
    if (sums) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) a += v[i][j];
            a += __shfl_xor(a, 16);
            a += __shfl_xor(a, 32);
            if (lane < 16) red[1][wave][tc * 8 + j] = a;
        }
    }
    __syncthreads();
    if (sums && threadIdx.x < F8_BLOCK && c0 + threadIdx.x < cols) {
        const int t = threadIdx.x;
        sums[rb * cols + c0 + t] = (red[1][0][t] + red[1][1][t]) + (red[1][2][t] + red[1][3][t]);
    }
    float top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
        top[j] = fmaxf(fmaxf(red[0][0][tc * 8 + j], red[0][1][tc * 8 + j]), fmaxf(red[0][2][tc * 8 + j], red[0][3][tc * 8 + j]));
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
    // the codes in tr as a second operand: rows from row0 on of n, block `block` of `blocks`; 2 KB at a time
    auto put_pieces = [&](uint8_t *to, int64_t row0, int64_t n, int64_t block, int64_t blocks) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tile = i * 2 + (threadIdx.x >> 7), part = threadIdx.x & 127;
            if (row0 + tile * 16 < n) {
                uint4 w;
                __builtin_memcpy(&w, &tr[tile * 16 + (part & 15)][((part >> 4) & 3) * 32 + (part >> 6) * 16], 16);
                *(uint4 *)(to + ((row0 / 16 + tile) * blocks + block) * (16 * F8_BLOCK) + part * 16) = w;
            }
        }
    };
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
            uint2 w;
            w.x = f8_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
            w.y = f8_pack4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
            if (MODE == F8_TILE) *(uint2 *)&tr[tr8 + i][tc * 8] = w;
            else if (r < rows) *(uint2 *)(q + r * cp + c) = w;
            if (tc == 0 && r < rows) f8_put_scale(s, rows, r, cb, er);
        }
        if (MODE == F8_TILE) {
            put_pieces(q, r0, rows, cb, cp / F8_BLOCK);
            if (!qt) return;
            __syncthreads();
        }
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
    if (MODE != F8_ROWS_COLS) {
        put_pieces(qt, c0, cols, rb, rp / F8_BLOCK);
        return;
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

template <class T> __global__ __launch_bounds__(256, 4) void k_f8_pack_weight(F8Pack w) { f8_pack_one<T, F8_TILE>(w, blockIdx.x); }

// the operands of both gradients in one launch: tiles of dy, then tiles of x (either may be none)
template <class T> __global__ __launch_bounds__(256, 4) void k_f8_pack_grads(F8Pack dy, uint32_t tiles_dy, F8Pack x) {
    if (blockIdx.x < tiles_dy) f8_pack_one<T, F8_ROWS_COLS>(dy, blockIdx.x);
    else f8_pack_one<T, F8_COLS>(x, blockIdx.x - tiles_dy);
}

// column sums from those of the row tiles: 64 columns per workgroup, its four waves share the tiles (lds: 1 KB)
struct F8Colsum {
    const float *part;
    int64_t tiles, cols;
    float *out;
};
__device__ __forceinline__ void f8_colsum(const F8Colsum &s, uint32_t block, float *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)block * 64 + lane;
    float a = 0.f;
    if (c < s.cols) {
#pragma unroll 8
        for (int64_t t = wave; t < s.tiles; t += 4) a += s.part[t * s.cols + c];
    }
    lds[wave * 64 + lane] = a;
    __syncthreads();
    if (wave == 0 && c < s.cols) s.out[c] = (lds[lane] + lds[64 + lane]) + (lds[128 + lane] + lds[192 + lane]);
}
__global__ __launch_bounds__(256) void k_f8_colsum(F8Colsum s) {
    __shared__ float lds[256];
    f8_colsum(s, blockIdx.x, lds);
}

// ---------------------------------------------------------------------------------------------
// product of two packed operands: C[m, n] = sum over k of A[m, k] B[n, k]
// ---------------------------------------------------------------------------------------------
// A workgroup owns BM x BN of the result, a wave MT x NT tiles of 16 x 16; one block of the reduction is a stage.  256 x 256, 8192 x
// 4096 x 8192: 205 us and 2.7 PFLOP/s in a long run (225 us in the first ten calls, while the clock settles).  Of a stage's 3 290
// cycles the matrix unit is at work for 2 048, the LDS for 1 070 with reads (24 KB a wave; conflicts 50) and for some 1 000 with
// copies (64 KB), by counters; larger tiles do not fit the registers (four waves of 128 x 128: 271 us then against 257).
//
// LDS image of a stage: B's pieces as they are packed, read by consecutive lanes at consecutive addresses.  A: rows of 128
// bytes, whose eight 16-byte pieces are exchanged by f8_swap(row).  A 16-byte read is served
// in groups of 16 lanes, 0-3 + 12-15 + 20-27 and so on; with a fragment's lanes (row lane % 16, pieces lane / 16 * 2 and + 1) such a
// group asks for one piece of eight rows and for another one of the other eight, and f8_swap puts all 16 into different
// banks.  (row / 2 % 8 alone, right for 16 consecutive lanes, had every read take twice its time.)  The copy from global
// memory straight to LDS writes linearly, so the exchange is applied to the global address.  The scale words of four stages
// lie behind the two stages.
//
// One barrier per stage, towards its end: by then every fragment of stage k has been read, so its buffer takes stage k + 2,
// and stage k + 1 has landed, whose fragments are read between the matrix instructions behind the barrier.  Codes: the wave holds
// its NT fragments of B and takes those of A one after the other, two steps of NT instructions behind the barrier (the other
// way round, 18 reads of 16 bytes fall into a quarter of the stage, more than the LDS delivers: 8192 x 4096 x 8192 with the
// codes of X 234 us against 226).  Expanded: it holds A and takes B, one column behind the barrier, so that B is expanded bit by bit
// (8192 x 4096 x 4096 235 us; the other way round 253).  The copies of a stage are issued one by one between the matrix
// instructions: issued in a row they hold up the instructions behind them, as a CU takes about 64 bytes of them a cycle.
template <int MT, int NT, int WM, int WN> struct F8Shape {
    static constexpr int WAVES = WM * WN, BM = MT * 16 * WM, BN = NT * 16 * WN, ROWS = BM + BN, LOADS = ROWS / 8 / WAVES,
                         LOADS_A = BM / 8 / WAVES, STAGE = ROWS * F8_BLOCK, STAGES = 2 * STAGE + 2 * ROWS * 4;
    // the finished tile of a wave: rows of NT * 16 elements and 16 bytes, so that rows start in different banks
    static constexpr int PITCH(int bytes) { return NT * 16 * bytes + 16; }
    static constexpr int OUT(int bytes) { return MT * 16 * PITCH(bytes); }
    static constexpr int LDS(int bytes) { return STAGES > WAVES * OUT(bytes) ? STAGES : WAVES * OUT(bytes); }
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && ROWS % 64 == 0 && ROWS <= 64 * WAVES && BM % 64 == 0,
                  "whole copies: eight rows of codes, 64 rows of scale words per wave");
};

__device__ __forceinline__ int f8_swap(int row) { return ((row >> 1) & 7) ^ ((((row >> 2) ^ (row >> 3)) & 1) << 1); }

// 32 codes of a lane -> the operands of four bf16 instructions, multiplied by the scale of biased exponent e
__device__ __forceinline__ void f8_expand(const i32x8 &f, uint32_t e, bf16x8 (&o)[4]) {
    const float s = __builtin_bit_cast(float, e << 23);
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

// copies 16 (4) bytes per lane from base + off to LDS address dst + lane * 16 (4).  The compiler does not wait for these
// copies in front of the LDS reads below (the address goes through an integer, and the reads are of plain vector types):
// the barriers do
__device__ __forceinline__ void f8_copy16(const void *base, uint32_t off, uint32_t dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)((const char *)base + off),
                                     (__attribute__((address_space(3))) void *)(uintptr_t)dst, 16, 0, 0);
}
__device__ __forceinline__ void f8_copy4(const void *base, uint32_t off, uint32_t dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)((const char *)base + off),
                                     (__attribute__((address_space(3))) void *)(uintptr_t)dst, 4, 0, 0);
}

struct F8Gemm {
    const uint8_t *A;
    const uint32_t *As;
    int64_t M;
    const uint8_t *B;
    const uint32_t *Bs;
    int64_t N, kp;
    const float *bias;
    void *C;
    int64_t ldc;
    uint32_t tiles_m, tiles_n;
    uint32_t splits, blocks;            // the reduction in `splits` parts of `blocks` (a multiple of 4) blocks; part s goes to
                                        // C + s * M * N (fp32, dense), k_f8_join adds the parts
};

// tile `id` of the product
template <int MT, int NT, int WM, int WN, bool EXPAND, class TO> __device__ __forceinline__ void f8_gemm_tile(const F8Gemm &g, uint32_t id) {
    const uint32_t tiles_m = g.tiles_m, tiles_n = g.tiles_n, split = id / (tiles_m * tiles_n);
    id -= split * tiles_m * tiles_n;
    const int64_t M = g.M, N = g.N, kp = g.kp, ldc = g.ldc, k0 = (int64_t)split * g.blocks;
    const uint8_t *const A = g.A + k0 * F8_BLOCK, *const B = g.B + k0 * (16 * F8_BLOCK);
    const uint32_t *const As = g.As + k0 / 4 * M, *const Bs = g.Bs + k0 / 4 * N;
    const float *const bias = g.bias;
    TO *const C = (TO *)g.C + split * M * N;
    using S = F8Shape<MT, NT, WM, WN>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Tiles in bands of 8 along m, and every XCD (workgroups go round the eight XCDs) a consecutive run of them: the 32 or
    // more workgroups that share an L2 work on a few rows and columns of tiles
    const uint32_t tiles = tiles_m * tiles_n, q = tiles / 8, rest = tiles % 8, xcd = id % 8;
    const uint32_t t = xcd * q + (xcd < rest ? xcd : rest) + id / 8;
    const uint32_t band = t / (8 * tiles_n), in_band = t - band * 8 * tiles_n;
    const uint32_t height = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
    const int64_t m0 = (int64_t)(band * 8 + in_band % height) * S::BM, n0 = (int64_t)(in_band / height) * S::BN;
    const int wm = (wave % WM) * (MT * 16), wn = (wave / WM) * (NT * 16);
    const int nk = (int)(kp / F8_BLOCK - k0 < g.blocks ? kp / F8_BLOCK - k0 : g.blocks);

    const uint8_t *const a0 = A + m0 * kp, *const b0 = B + n0 * kp;
    const int64_t last_a = M - m0 - 1, last_b = (N - n0 - 1) / 16;      // last row of A, last 16 rows of B
    uint32_t off[S::LOADS];                             // rows behind the end repeat the last ones
#pragma unroll
    for (int i = 0; i < S::LOADS; ++i) {
        const int eight = i * S::WAVES + wave, row = eight * 8 + (lane >> 3), tile = (eight - S::BM / 8) / 2;
        off[i] = i < S::LOADS_A ? (uint32_t)(row < last_a ? row : last_a) * (uint32_t)kp + (((lane & 7) ^ f8_swap(row)) * 16)
                                : (uint32_t)(tile < last_b ? tile : last_b) * (uint32_t)kp * 16 + (eight & 1) * 1024 + lane * 16;
    }
    const int srow = (wave < S::ROWS / 64 ? wave : S::ROWS / 64 - 1) * 64;        // (further waves copy the last piece again)
    const bool scale_a = srow < S::BM;
    const uint32_t *const s0 = scale_a ? As + m0 + srow : Bs + n0 + (srow - S::BM);
    const int64_t s_rows = scale_a ? M : N;
    // piece i of stage k to buffer buf; the scale words are piece LOADS, copied with each of their four stages (the same bytes
    // over themselves).  No branches around here: the compiler would move matrix instructions across them
    auto copy = [&](int k, int buf, int i) {
        if (i < S::LOADS) {
            const uint8_t *base = i < S::LOADS_A ? a0 + (int64_t)k * F8_BLOCK : b0 + (int64_t)k * (16 * F8_BLOCK);
            uint32_t o = off[i];
            asm("" : "+s"(base), "+v"(o));              // scalar base and 32-bit offset: one register per copy and lane
            f8_copy16(base, o, lds0 + buf * S::STAGE + (i * S::WAVES + wave) * 8 * F8_BLOCK);
        } else {                                        // (an operand's scales are followed by 1 KB that may be read)
            const uint32_t *base = s0 + (k >> 2) * s_rows;
            asm("" : "+s"(base));
            f8_copy4(base, lane * 4, lds0 + 2 * S::STAGE + ((k >> 2) & 1) * (S::ROWS * 4) + srow * 4);
        }
    };
    // this lane's two pieces of a fragment (row lane % 16 of a tile, 32 codes of the block) and its scale, for the wave's
    // first tile of either operand; the other tiles lie at constant distances
    const int r16 = lane & 15, swap = f8_swap(r16), g2 = (lane >> 4) * 2;
    const uint8_t *const lo_a = lds + (wm + r16) * F8_BLOCK + (g2 ^ swap) * 16, *const hi_a = lds + (wm + r16) * F8_BLOCK + ((g2 + 1) ^ swap) * 16;
    const uint8_t *const lo_b = lds + (S::BM + wn) * F8_BLOCK + lane * 16, *const hi_b = lo_b + 1024;
    const uint8_t *const sc_a = lds + 2 * S::STAGE + (wm + r16) * 4, *const sc_b = sc_a + (S::BM + wn - wm) * 4;
    auto frag = [&](const uint8_t *lo, const uint8_t *hi, int k, int tile) {
        const i32x4 x = *(const i32x4 *)(lo + (k & 1) * S::STAGE + tile * (16 * F8_BLOCK));
        const i32x4 y = *(const i32x4 *)(hi + (k & 1) * S::STAGE + tile * (16 * F8_BLOCK));
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto scale = [&](const uint8_t *sc, int k, int tile) -> uint32_t {
        return *(sc + (((k >> 2) & 1) * (S::ROWS * 4) + (k & 3)) + tile * 64);
    };

    f32x4 acc[NT][MT] = {};
    constexpr int HALF = S::LOADS / 2;
    static_assert(S::LOADS % 2 == 0, "half a stage's copies at a time");
#pragma unroll
    for (int i = 0; i <= S::LOADS; ++i) copy(0, 0, i);
#pragma unroll
    for (int i = 0; i < HALF; ++i) copy(nk > 1 ? 1 : 0, 1, i);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    // copy number `slot` of `slots` places, in the last steps of stage k (the first half of stage k + 2) and in the first ones
    // (the second half of stage k + 1, and its scale words)
    auto copy_last = [&](int k, int slot, int slots) {
        const int every = slots / HALF;
        if (slot % every == every - 1 && slot / every < HALF) copy(k + 2 < nk ? k + 2 : nk - 1, k & 1, slot / every);
    };
    auto copy_first = [&](int k, int slot, int slots) {
        const int every = slots / HALF, to = k + 1 < nk ? k + 1 : nk - 1;
        if (slot % every == every - 1 && slot / every < HALF) copy(to, (k + 1) & 1, HALF + slot / every);
        if (slot == slots - 1) copy(to, (k + 1) & 1, S::LOADS);
    };
    // The matrix instructions' first operand: rows of the result = n, so that a lane gets four consecutive n.  The order of the
    // statements is the schedule: nothing moves across the sched_barriers.  (Behind the last stage: read and not used.)
    if constexpr (EXPAND) {
        i32x8 fa[MT], fb;
        uint32_t ea[MT], eb;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            fa[i] = frag(lo_a, hi_a, 0, i);
            ea[i] = scale(sc_a, 0, i);
        }
        fb = frag(lo_b, hi_b, 0, 0);
        eb = scale(sc_b, 0, 0);
        for (int k = 0; k < nk; ++k) {
            bf16x8 xa[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i) f8_expand(fa[i], ea[i], xa[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                bf16x8 xb[4];
                f8_expand(fb, eb, xb);
                if (j + 1 == NT) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                fb = frag(lo_b, hi_b, j + 1 < NT ? k : k + 1, j + 1 < NT ? j + 1 : 0);
                eb = scale(sc_b, j + 1 < NT ? k : k + 1, j + 1 < NT ? j + 1 : 0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[u], xa[i][u], acc[j][i], 0, 0, 0);
                    if (j + 1 == NT) {
                        fa[i] = frag(lo_a, hi_a, k + 1, i);
                        ea[i] = scale(sc_a, k + 1, i);
                        copy_last(k, i, MT);
                        __builtin_amdgcn_sched_barrier(0);
                    } else if (j == 0) {
                        copy_first(k, i, MT);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    } else {
        constexpr int WALL = MT - 2;                    // the barrier stands before this step
        i32x8 fb0[NT], fb1[NT], next_a;                 // fragments that a stage begins with, and their scales
        uint32_t e0[NT], e1[NT], next_ea;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            fb0[j] = frag(lo_b, hi_b, 0, j);
            e0[j] = scale(sc_b, 0, j);
        }
        next_a = frag(lo_a, hi_a, 0, 0);
        next_ea = scale(sc_a, 0, 0);
        auto stage = [&](int k, const i32x8(&b)[NT], const uint32_t(&e)[NT], i32x8(&bn)[NT], uint32_t(&en)[NT]) {
            i32x8 a[MT];
            uint32_t ea[MT];
            a[0] = next_a;
            ea[0] = next_ea;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (i == WALL) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
                for (int r = 0; r < MT; ++r)            // one step ahead; the last two of them before the barrier
                    if (r == i + 1 ? r < WALL : r == WALL ? i == WALL - 2 : r == WALL + 1 && i == WALL - 1) {
                        a[r] = frag(lo_a, hi_a, k, r);
                        ea[r] = scale(sc_a, k, r);
                    }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], a[i], acc[j][i], 0, 0, 0, (int)e[j], 0,
                                                                                (int)ea[i]);
                    const int slot = (i < WALL ? i : i - WALL) * NT + j;
                    if (i >= WALL) {
                        if (slot % 2 == 0) {
                            bn[slot / 2] = frag(lo_b, hi_b, k + 1, slot / 2);
                            en[slot / 2] = scale(sc_b, k + 1, slot / 2);
                        }
                        if (slot == 2 * NT - 1) {
                            next_a = frag(lo_a, hi_a, k + 1, 0);
                            next_ea = scale(sc_a, k + 1, 0);
                        }
                        copy_last(k, slot, 2 * NT);
                    } else if (i < 2) {
                        copy_first(k, slot, 2 * NT);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        for (int k = 0;; k += 2) {
            stage(k, fb0, e0, fb1, e1);
            if (k + 1 >= nk) break;
            stage(k + 1, fb1, e1, fb0, e0);
            if (k + 2 >= nk) break;
        }
    }
    // The copies behind the last stage end here, and the stages' memory becomes the waves' own: a wave turns its tile around in
    // LDS, so that it is written in whole rows of NT * 16 elements (128 bytes and more), not in pieces of four
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    uint8_t *const own = lds + wave * S::OUT(sizeof(TO));
    constexpr int PITCH = S::PITCH(sizeof(TO)), VEC = 16 / sizeof(TO), LPR = NT * 16 / VEC, RPI = 64 / LPR;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t n = n0 + wn + j * 16 + (lane >> 4) * 4;
        float b[4] = {};
        if (bias) load_n<4>(bias + n, N - n >= 4 ? 4 : N > n ? (int)(N - n) : 0, b);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            typedef TO out4 __attribute__((ext_vector_type(4)));
            out4 v;
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = (TO)(acc[j][i][u] + b[u]);
            *(out4 *)(own + (i * 16 + r16) * PITCH + (j * 16 + (lane >> 4) * 4) * sizeof(TO)) = v;
        }
    }
    __builtin_amdgcn_wave_barrier();                    // (a wave's LDS accesses stay in order)
    const int64_t n = n0 + wn + (lane % LPR) * VEC;
    const int left = N - n >= VEC ? VEC : N > n ? (int)(N - n) : 0;
#pragma unroll 4
    for (int i = 0; i < MT * 16; i += RPI) {
        const int row = i + lane / LPR;
        const int64_t m = m0 + wm + row;
        if (m >= M) continue;
        TO v[VEC];
        __builtin_memcpy(v, __builtin_assume_aligned(own + row * PITCH + (lane % LPR) * 16, 16), 16);
        TO *o = C + m * ldc + n;
        if (left == VEC) {
            // (past the caches where a wave writes whole lines of them: 4 to 12 % less time; not 64 columns of 16 bits, 10 % more)
            if (MT * NT * sizeof(TO) >= 32) store16_streaming(o, v);
            else __builtin_memcpy(o, v, 16);
        } else {
#pragma unroll
            for (int u = 0; u < VEC; ++u)
                if (u < left) o[u] = v[u];
        }
    }
}

template <int MT, int NT, int WM, int WN, bool EXPAND, class TO>
__global__ __launch_bounds__(64 * WM * WN, MT * NT <= 8 ? 3 : 2) void k_f8_gemm(F8Gemm g) {
    f8_gemm_tile<MT, NT, WM, WN, EXPAND, TO>(g, blockIdx.x);
}
// dW (fp32) and dX of one layer, and db, in one launch: neither product has the tiles for whole rounds of the CUs.  db's
// workgroups (`sums`, may be none) first, then those of the product whose workgroups take longer
template <int NT, bool EXPAND, class TO>
__global__ __launch_bounds__(256, NT == 2 ? 3 : 2) void k_f8_gemm_grads(F8Gemm dw, F8Gemm dx, F8Colsum db, uint32_t sums) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t nw = dw.tiles_m * dw.tiles_n * dw.splits, nx = dx.tiles_m * dx.tiles_n * dx.splits, id = blockIdx.x - sums;
    const bool dx_first = dx.blocks * (EXPAND ? 2 : 1) > dw.blocks * 2;         // (codes: half the time for a block)
    if (blockIdx.x < sums) f8_colsum(db, blockIdx.x, (float *)lds);
    else if (dx_first ? id >= nx : id < nw) f8_gemm_tile<4, NT, 2, 2, true, float>(dw, dx_first ? id - nx : id);
    else f8_gemm_tile<4, NT, 2, 2, EXPAND, TO>(dx, dx_first ? id : id - nw);
}

// C = bias + sum of the parts, four columns per lane, in an order that the number of parts decides.  Up to eight parts: all of them
// in flight, bound by HBM, 3.2 TB/s.  More: latency, so the waves of a workgroup share them (79 parts of 64 x 64 4.6 us, a
// wave alone 9).
#define F8_JOIN_ALONE 8
struct F8Join {
    const float *part;
    int64_t M, N;
    uint32_t splits;
    const float *bias;
    void *C;
    int64_t ldc;
};
template <class TO> __device__ __forceinline__ void f8_join(const F8Join &j, int64_t block, f32x4 (&lds)[4][64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool alone = j.splits <= F8_JOIN_ALONE;
    const int first = alone ? 0 : wave, step = alone ? 1 : 4;
    const int64_t units = (j.N + 3) / 4, i = alone ? block * 256 + threadIdx.x : block * 64 + lane, m = i / units, n = (i - m * units) * 4;
    const int left = m >= j.M ? 0 : j.N - n < 4 ? (int)(j.N - n) : 4;
    const float *const part = j.part + (left ? m * j.N + n : 0);
    f32x4 sum = {};
    if (left == 4) {                                    // eight parts in flight (behind the end: the last one, not added)
        for (uint32_t s = first; s < j.splits; s += 8 * step) {
            float p[8][4];
#pragma unroll
            for (int t = 0; t < 8; ++t) load_n<4>(part + (s + t * step < j.splits ? s + t * step : j.splits - 1) * j.M * j.N, 4, p[t]);
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (s + t * step < j.splits) sum += f32x4{p[t][0], p[t][1], p[t][2], p[t][3]};
        }
    } else {
        for (uint32_t s = first; s < j.splits; s += step)
#pragma unroll
            for (int u = 0; u < 3; ++u)
                if (u < left) sum[u] += part[s * j.M * j.N + u];
    }
    if (!alone) {
        lds[wave][lane] = sum;
        __syncthreads();
        if (wave) return;
        sum = (lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]);
    }
    if (!left) return;
    float v[4] = {};
    if (j.bias) load_n<4>(j.bias + n, left, v);
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] += sum[u];
    store_n<4>((TO *)j.C + m * j.ldc + n, left, v);
}
// a: of type TO, `first` workgroups; b: fp32 (either may be none)
template <class TO> __global__ __launch_bounds__(256) void k_f8_join(F8Join a, uint32_t first, F8Join b) {
    __shared__ f32x4 lds[4][64];
    if (blockIdx.x < first) f8_join<TO>(a, blockIdx.x, lds);
    else f8_join<float>(b, blockIdx.x - first, lds);
}

// Few rows, 16 at most (f8_skinny): bound by the bytes of B and by latency, so one launch does the layer.  A workgroup owns 16
// rows of B; its W waves share the reduction, and their first codes of B are on the way while the workgroup quantises X into LDS,
// each element once: quantised by the lanes that multiply it, 16 rows at a time whatever their number, X took longer than B.
// Every result type takes the expanded product here: the matrix unit is idle either way.  One row of 4096 x 4096 in bf16: 5.1 us,
// 3.3 TB/s (6.7 us with B row by row, where neighbouring lanes read different rows); 28672 x 8192 38 us, 6.1 TB/s.
#define F8_SKINNY 16
#define F8_SKINNY_LDS (140 * 1024)
template <class TX, class TO, int W>
__global__ __launch_bounds__(64 * W) void k_f8_skinny(const TX *__restrict__ X, int64_t ldx, int M, int64_t K, const uint8_t *__restrict__ B,
                                                      const uint32_t *__restrict__ Bs, int64_t N, int64_t kp,
                                                      const float *__restrict__ bias, TO *__restrict__ C, int64_t ldc) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];       // [M][pitch] codes, [M][nk] exponents, [W][64] sums
    constexpr int U = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * 16, nr = n0 + m < N ? n0 + m : N - 1;
    const int nk = (int)(kp / F8_BLOCK), pitch = nk * F8_BLOCK + 16, groups = M * nk;
    uint8_t *const ex = lds + M * pitch;
    const uint8_t *const brow = B + n0 * kp + lane * 16;
    f32x4 acc = {};
    i32x8 fb[U];
    uint32_t eb[U];
    auto load = [&](int k0) {                           // blocks k0, k0 + W, ... (behind the end: the last block, not used)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * W < nk ? k0 + u * W : nk - 1;
            const uint8_t *const b = brow + (int64_t)k * (16 * F8_BLOCK);
            fb[u] = __builtin_shufflevector(*(const i32x4 *)b, *(const i32x4 *)(b + 1024), 0, 1, 2, 3, 4, 5, 6, 7);
            eb[u] = Bs[(int64_t)(k >> 2) * N + nr] >> ((k & 3) * 8);
        }
    };
    load(wave);
    const float per_row = 1.f / (float)nk;
    auto quantise = [&](auto in_flight) {               // groups of 128 of this lane's 16, that many loaded at a time
        constexpr int Q = decltype(in_flight)::value;
        for (int g0 = threadIdx.x >> 4; g0 < groups; g0 += W * 4 * Q) {
            vec8<TX> v[Q];
            int row[Q], k[Q];
#pragma unroll
            for (int u = 0; u < Q; ++u) {
                const int g = g0 + u * W * 4 < groups ? g0 + u * W * 4 : groups - 1;
                row[u] = (int)(((float)g + 0.5f) * per_row);            // g / nk: g < 2^11, half a unit is more than the rounding
                k[u] = g - row[u] * nk;
                const int64_t c = (int64_t)k[u] * F8_BLOCK + m * 8;
                const TX *const p = X + row[u] * ldx;
                if (K >= 8) v[u] = load_whole(p + (c + 8 <= K ? c : 0));
                if (K % 8 && c < K && c + 8 > K) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[u][i] = c + i < K ? p[c + i] : (TX)0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < Q; ++u) {
                if (g0 + u * W * 4 >= groups) break;    // (whole groups of 16 lanes leave)
                const bool live = (int64_t)k[u] * F8_BLOCK + m * 8 < K;
                float f[8], a = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[i] = live ? (float)v[u][i] : 0.f;
                    a = fmaxf(a, fabsf(f[i]));
                }
                const int e = f8_exponent(row16_max(a));
                const float inv = f8_inverse(e);
                uint2 w;
                w.x = f8_pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
                w.y = f8_pack4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
                *(uint2 *)(lds + row[u] * pitch + k[u] * F8_BLOCK + m * 8) = w;
                if (m == 0) ex[row[u] * nk + k[u]] = (uint8_t)e;
            }
        }
    };
    if (groups <= W * 4) quantise(std::integral_constant<int, 1>());
    else if (groups <= W * 8) quantise(std::integral_constant<int, 2>());
    else quantise(std::integral_constant<int, 4>());
    __syncthreads();
    const uint8_t *const arow = lds + (m < M ? m : 0) * pitch + (lane >> 4) * 32, *const erow = ex + (m < M ? m : 0) * nk;
    for (int k0 = wave; k0 < nk; k0 += U * W) {
        if (k0 != wave) load(k0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * W;
            if (k >= nk) break;
            const i32x4 x = *(const i32x4 *)(arow + k * F8_BLOCK), y = *(const i32x4 *)(arow + k * F8_BLOCK + 16);
            bf16x8 xa[4], xb[4];
            f8_expand(__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7), erow[k], xa);
            f8_expand(fb[u], eb[u] & 0xFF, xb);
#pragma unroll
            for (int t = 0; t < 4; ++t) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[t], xa[t], acc, 0, 0, 0);
        }
    }
    f32x4 *const part = (f32x4 *)(lds + ((M * (pitch + nk) + 15) & ~15));
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < W; ++w) acc += part[w * 64 + lane];
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
    if (grid > ddg_max_grid(256)) return DDG_E_UNSUPPORTED;
    return ddg_with_type(type, [&](auto t) {
        using T = decltype(t);
        k_f8_pack_rows<T><<<(unsigned)grid, 256, 0, s>>>((const T *)x, ld, o.rows, o.cols, o.q, o.s);
        DDG_CHECK_LAUNCH();
        return (int)DDG_OK;
    });
}
static inline int64_t f8_tiles(int64_t rows, int64_t cols) { return ceil_div64(rows, F8_BLOCK) * ceil_div64(cols, F8_BLOCK); }

#define F8_WORKGROUPS 512                               // two per CU
// Reductions are addressed with 32-bit offsets within a workgroup's 256 rows; both gradients' tiles and db's workgroups (at
// most two for a tile of dW) fit one launch of 256 threads each.  Tiles of 128 x 64 are at most twice as many: 2^23 for a product on its
// own, and both gradients take them only below eight stages for each of F8_WORKGROUPS; splits are of products of up to 256 tiles.
// Checked in front of an entry point's first launch.
#define F8_MAX_REDUCTION ((int64_t)1 << 24)
static inline bool f8_product_ok(int64_t rows_a, int64_t rows_b, int64_t cols) {
    return f8_pad(cols) < F8_MAX_REDUCTION && ceil_div64(rows_a, 128) * ceil_div64(rows_b, 128) < (1 << 22);
}

// Tiles are 256 x 256 (bf16 results only) once there are three quarters of a CU's worth of them and their rounds (one per CU)
// cost less than those of 128 x 128 tiles (two per CU, two thirds of the time a round: 40 000 x 176 x 352 30.8 us with 256 x 256,
// 25.3 with 128 x 128; 8192 x 4096 x 8192 is four rounds and eight); else 128 x 128, or 128 x 64 while
// all tiles together have fewer than eight stages for each of 512 workgroups: there the time is latency.  Not where 128 x 128 tiles
// come near one for each of those and cover no more columns (20 000 x 176 x 352 19.4 us with 128 x 64, 18.5 with 128 x 128); where
// they cover more, 128 x 64 for fp32 results of short reductions and any number of rows (100 000 x 176 x 176 44.9 us and 48.9,
// 100 000 x 1000 x 64 121 and 130, but 100 000 x 4096 x 64 506 and 494; 100 000 x 352 x 320 in bf16 67 and 56).  A tile whose reduction
// takes twice its share of all stages and more is split into parts of about that share (a whole number of scale words, so
// four stages at least), which are added afterwards, where that saves more (0.6 us a stage) than it costs (a launch, 3 us, and
// the parts written and read, 3.2 TB/s); all figures measured.  17 x 8192 x 1000 in fp32 53 -> 12.7 us, 128 x 4096 x 4096
// 36 -> 21.5 us; 256 x 1000 x 8192 is left whole, 15 us.
static inline bool f8_wide(int64_t rows_a, int64_t rows_b) {
    const int64_t wide = ceil_div64(rows_a, 256) * ceil_div64(rows_b, 256), small = ceil_div64(rows_a, 128) * ceil_div64(rows_b, 128);
    return wide >= 192 && ceil_div64(wide, 256) * 3 < ceil_div64(small, F8_WORKGROUPS) * 2;
}
static inline int64_t f8_stages(int64_t rows_a, int64_t rows_b, int64_t cols, int bn) {
    return ceil_div64(rows_a, 128) * ceil_div64(rows_b, bn) * (f8_pad(cols) / F8_BLOCK);
}
static inline bool f8_narrow(int64_t rows_a, int64_t rows_b, int64_t cols, bool f32) {
    const bool latency = f8_stages(rows_a, rows_b, cols, 128) < 8 * F8_WORKGROUPS;
    if (ceil_div64(rows_b, 128) * 2 != ceil_div64(rows_b, 64)) return latency || (f32 && f8_pad(cols) <= 8 * F8_BLOCK);
    return latency && ceil_div64(rows_a, 128) * ceil_div64(rows_b, 128) < 400;
}
struct F8Split {
    int64_t splits, blocks;
};
static inline F8Split f8_share(int64_t cols, int64_t all_stages) {
    const int64_t share = ceil_div64(ceil_div64(all_stages, F8_WORKGROUPS), 4) * 4;
    return {ceil_div64(f8_pad(cols) / F8_BLOCK, share), share};
}
// the largest m whose split saves more than it costs (0: none)
static inline int64_t f8_split_most(int64_t n, int64_t cols, const F8Split &sp) {
    const int64_t nk = f8_pad(cols) / F8_BLOCK, saved = (nk - sp.blocks) * 600 - 3000;         // ns
    return nk < 2 * sp.blocks || saved < 0 ? 0 : ((saved + 1) * 800 - 1) / (sp.splits * n);
}
static inline F8Split f8_split(int64_t m, int64_t n, int64_t cols, int64_t all_stages) {
    const F8Split sp = f8_share(cols, all_stages);
    if (m > f8_split_most(n, cols, sp)) return {1, ceil_div64(f8_pad(cols) / F8_BLOCK, 4) * 4};
    return sp;
}
// stages and split of a product on its own (short reductions are not split in either tile)
static inline int64_t f8_stages_one(int64_t rows_a, int64_t rows_b, int64_t cols) {
    return f8_stages(rows_a, rows_b, cols, f8_narrow(rows_a, rows_b, cols, false) ? 64 : 128);
}
static inline F8Split f8_split_one(int64_t rows_a, int64_t rows_b, int64_t cols, bool bf16) {
    if (bf16 && f8_wide(rows_a, rows_b)) return {1, ceil_div64(f8_pad(cols) / F8_BLOCK, 4) * 4};
    return f8_split(rows_a, rows_b, cols, f8_stages_one(rows_a, rows_b, cols));
}
static inline size_t f8_parts_bytes(const F8Split &sp, int64_t m, int64_t n) {
    return sp.splits > 1 ? ((size_t)sp.splits * m * n * 4 + 255) & ~(size_t)255 : 0;
}
// The most that the parts of a product with up to m rows take: stages(rows) depends on the number of row tiles alone, so that for each
// number the largest m that is split counts.  None is split above 256 tiles (two shares would be more than the reduction)
template <class Stages> static inline size_t f8_parts_most(int64_t m, int64_t n, int64_t cols, const Stages &stages) {
    size_t most = 0;
    for (int64_t t = 1; (t - 1) * 128 < m && t * ceil_div64(n, 128) <= 256; ++t) {
        const int64_t rows = t * 128 < m ? t * 128 : m;
        const F8Split sp = f8_share(cols, stages(rows));
        const int64_t split = f8_split_most(n, cols, sp), last = rows < split ? rows : split;
        if (last <= (t - 1) * 128) continue;
        const size_t bytes = f8_parts_bytes(sp, last, n);
        most = bytes > most ? bytes : most;
    }
    return most;
}

template <class S>
static F8Gemm f8_problem(const F8Operand &a, const F8Operand &b, const float *bias, void *c, int64_t ldc, const F8Split &sp,
                         float *parts) {
    const bool split = sp.splits > 1;
    return {a.q, (const uint32_t *)a.s, a.rows, b.q, (const uint32_t *)b.s, b.rows, f8_pad(a.cols), split ? nullptr : bias,
            split ? parts : c, split ? b.rows : ldc, (uint32_t)ceil_div64(a.rows, S::BM), (uint32_t)ceil_div64(b.rows, S::BN),
            (uint32_t)sp.splits, (uint32_t)sp.blocks};
}
template <class K> static int f8_lds(K kernel, int bytes) {        // more than 64 KB has to be asked for
    if (bytes <= 65536) return DDG_OK;
    return hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess ? DDG_OK
                                                                                                                 : DDG_E_LAUNCH;
}
static F8Join f8_joined(const F8Operand &a, const F8Operand &b, const F8Split &sp, const float *parts, const float *bias, void *c,
                        int64_t ldc) {
    return {parts, a.rows, b.rows, (uint32_t)sp.splits, bias, c, ldc};
}
static inline int64_t f8_join_grid(const F8Join &j) { return j.splits > 1 ? ceil_div64(j.M * ((j.N + 3) / 4), j.splits > F8_JOIN_ALONE ? 64 : 256) : 0; }
// whichever of the two was split (b: fp32)
static int f8_join_parts(const F8Join &a, int type, const F8Join &b, hipStream_t s) {
    const int64_t ga = f8_join_grid(a), gb = f8_join_grid(b);
    if (ga + gb == 0) return DDG_OK;
    return ddg_with_type(type, [&](auto t) {
        k_f8_join<decltype(t)><<<(unsigned)(ga + gb), 256, 0, s>>>(a, (uint32_t)ga, b);
        DDG_CHECK_LAUNCH();
        return (int)DDG_OK;
    });
}

static int f8_gemm(const F8Operand &a, const F8Operand &b, const float *bias, void *c, int type, int64_t ldc, float *parts, hipStream_t s) {
    const F8Split sp = f8_split_one(a.rows, b.rows, a.cols, type == DDG_BF16);
    const bool narrow = f8_narrow(a.rows, b.rows, a.cols, type == DDG_F32);
    auto go = [&](auto mt, auto nt, auto wm, auto wn, auto expand, auto to) {
        using TO = decltype(to);
        constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
        using S = F8Shape<MT, NT, WM, WN>;
        const F8Gemm g = f8_problem<S>(a, b, bias, c, ldc, sp, parts);
        const auto kernel = k_f8_gemm<MT, NT, WM, WN, decltype(expand)::value, TO>;
        const int rc = f8_lds(kernel, S::LDS(sizeof(TO)));
        if (rc) return rc;
        kernel<<<g.tiles_m * g.tiles_n * g.splits, 64 * WM * WN, S::LDS(sizeof(TO)), s>>>(g);
        DDG_CHECK_LAUNCH();
        return (int)DDG_OK;
    };
    const std::true_type yes;
    const std::false_type no;
    auto tiles = [&](auto expand, auto to) {
        return narrow ? go(Int<4>(), Int<2>(), Int<2>(), Int<2>(), expand, to) : go(Int<4>(), Int<4>(), Int<2>(), Int<2>(), expand, to);
    };
    int rc;
    if (sp.splits > 1) rc = type == DDG_BF16 ? tiles(no, float()) : tiles(yes, float());
    else if (type == DDG_BF16 && f8_wide(a.rows, b.rows)) rc = go(Int<8>(), Int<4>(), Int<2>(), Int<4>(), no, bf16_t());
    else rc = type == DDG_BF16 ? tiles(no, bf16_t()) : type == DDG_F16 ? tiles(yes, f16_t()) : tiles(yes, float());
    return rc ? rc : f8_join_parts(f8_joined(a, b, sp, parts, bias, c, ldc), type, F8Join{nullptr, 0, 0, 1, nullptr, nullptr, 0}, s);
}

// The gradients' products: dx [rows, in] over out, dw [out, in] over rows.  Two launches, dx in 256 x 256 tiles, where there are
// enough of those, dw's tiles fill three quarters of their rounds of two per CU, and dx's reduction is not short; in one launch
// dx's tiles fill the rounds.  Measured at 20 000 rows, apart and together: 8192 x 8192 3 200 and 3 470 us, 6000 x 6000 1 879 and
// 1 977, 3000 x 3000 (0.56 of its rounds) 653 and 563, 2048 x 5000 (in x out) 663 and 632, 5000 x 2048 730 and 632; 8192 x 1000 567
// and 570, but 131 and 120 at 4 001 rows.
struct F8GradSplits {
    bool apart, narrow;                 // two launches (dx in 256 x 256 tiles); 128 x 64 tiles
    F8Split dx, dw;
};
static inline int64_t f8_grad_stages(int64_t rows, int64_t out, int64_t in, int bn) {
    return f8_stages(rows, in, out, bn) + f8_stages(out, in, rows, bn);
}
static inline bool f8_grad_narrow(int64_t rows, int64_t out, int64_t in) { return f8_grad_stages(rows, out, in, 128) < 8 * F8_WORKGROUPS; }
static inline F8GradSplits f8_grad_splits(int64_t rows, int64_t out, int64_t in, bool bf16) {
    F8GradSplits g;
    const int64_t tw = ceil_div64(out, 128) * ceil_div64(in, 128);
    g.apart = bf16 && f8_wide(rows, in) && out > 1024 && tw * 4 >= ceil_div64(tw, F8_WORKGROUPS) * F8_WORKGROUPS * 3;
    g.narrow = f8_grad_narrow(rows, out, in);
    const int64_t all = f8_grad_stages(rows, out, in, g.narrow ? 64 : 128);
    g.dx = g.apart ? f8_split_one(rows, in, out, bf16) : f8_split(rows, in, out, all);
    g.dw = g.apart ? f8_split_one(out, in, rows, false) : f8_split(out, in, rows, all);
    return g;
}
// dx = gy wt, dw = gyt xt
static int f8_gemm_grads(const F8Operand &gy, const F8Operand &wt, void *dx, int dx_type, int64_t ld_dx, float *parts_dx,
                         const F8Operand &gyt, const F8Operand &xt, float *dw, float *parts_dw, const F8Colsum &db, hipStream_t s) {
    const F8GradSplits sp = f8_grad_splits(gy.rows, gy.cols, wt.rows, dx_type == DDG_BF16);
    const uint32_t sums = db.out ? (uint32_t)ceil_div64(db.cols, 64) : 0;
    if (sp.apart) {
        if (sums) {
            k_f8_colsum<<<sums, 256, 0, s>>>(db);
            DDG_CHECK_LAUNCH();
        }
        const int rc = f8_gemm(gy, wt, nullptr, dx, dx_type, ld_dx, parts_dx, s);
        return rc ? rc : f8_gemm(gyt, xt, nullptr, dw, DDG_F32, xt.rows, parts_dw, s);
    }
    auto go = [&](auto nt, auto expand, auto to) {
        using S = F8Shape<4, decltype(nt)::value, 2, 2>;
        const F8Gemm gw = f8_problem<S>(gyt, xt, nullptr, dw, xt.rows, sp.dw, parts_dw);
        const F8Gemm gx = f8_problem<S>(gy, wt, nullptr, dx, ld_dx, sp.dx, parts_dx);
        const auto kernel = k_f8_gemm_grads<decltype(nt)::value, decltype(expand)::value, decltype(to)>;
        const int rc = f8_lds(kernel, S::LDS(4));
        if (rc) return rc;
        kernel<<<sums + gw.tiles_m * gw.tiles_n * gw.splits + gx.tiles_m * gx.tiles_n * gx.splits, 256, S::LDS(4), s>>>(gw, gx, db, sums);
        DDG_CHECK_LAUNCH();
        return (int)DDG_OK;
    };
    const std::true_type yes;
    const std::false_type no;
    auto tiles = [&](auto expand, auto to) { return sp.narrow ? go(Int<2>(), expand, to) : go(Int<4>(), expand, to); };
    int rc;
    if (sp.dx.splits > 1) rc = dx_type == DDG_BF16 ? tiles(no, float()) : tiles(yes, float());
    else rc = dx_type == DDG_BF16 ? tiles(no, bf16_t()) : dx_type == DDG_F16 ? tiles(yes, f16_t()) : tiles(yes, float());
    return rc ? rc : f8_join_parts(f8_joined(gy, wt, sp.dx, parts_dx, nullptr, dx, ld_dx), dx_type,
                                   f8_joined(gyt, xt, sp.dw, parts_dw, nullptr, dw, xt.rows), s);
}

extern "C" int ddg_fp8_pack_weight(const void *W, int type, int64_t ld, int64_t out, int64_t in, void *packed, void *packed_t,
                                   void *stream) {
    if (!f8_dims_ok(out, in) || out < 1 || in < 1 || ld < in || !ddg_type_ok(type) || !W || !packed) return DDG_E_ARG;
    if (((uintptr_t)packed | (uintptr_t)packed_t) & 255) return DDG_E_ARG;
    F8Operand t = {};
    if (packed_t) t = f8_operand(packed_t, in, out);
    const F8Operand o = f8_operand(packed, out, in);
    const int64_t tiles = f8_tiles(out, in);
    if (tiles > ddg_max_grid(256)) return DDG_E_UNSUPPORTED;
    return ddg_with_type(type, [&](auto ty) {
        k_f8_pack_weight<decltype(ty)><<<(unsigned)tiles, 256, 0, (hipStream_t)stream>>>(
            F8Pack{W, ld, out, in, o.q, o.s, t.q, t.s, nullptr});
        DDG_CHECK_LAUNCH();
        return (int)DDG_OK;
    });
}

// k_f8_skinny: X fits the LDS, and its quantisation by every workgroup (13 elements a ns, and 3 us a workgroup besides; one
// workgroup per CU at a time) takes less than the detour over packed X and tiles, 18 us and with another result than bf16
// 22 us.  Rows from which the tiles were quicker (bf16, in x out): 2048 x 2048 and 4096 x 4096 none, 8192 x 8192 nine, 14336 x 4096
// thirteen, 4096 x 14336 six, 4096 x 32000 one; 16 rows through 8192 x 8192 32 us here and 24 us there, through 4096 x 4096 10 and 14.
static inline bool f8_skinny(int64_t rows, int64_t out, int64_t in, bool bf16) {
    const int64_t nk = f8_pad(in) / F8_BLOCK;
    return rows <= F8_SKINNY && rows * (nk * (F8_BLOCK + 1) + 16) <= F8_SKINNY_LDS &&
           (rows * in / 13 + 3000) * (out > 4096 ? out : 4096) <= (int64_t)(bf16 ? 18000 : 22000) * 4096;
}

extern "C" size_t ddg_fp8_linear_workspace_bytes(int64_t rows, int64_t out, int64_t in) {
    if (!f8_dims_ok(rows, in) || !f8_dims_ok(out, 0) || in < 1 || out < 1) return 0;
    if (f8_skinny(rows, out, in, true)) return 0;
    // (the result's type decides about more rows there, and about 256 x 256 tiles, which are not split: room for either)
    return ddg_fp8_operand_bytes(rows, in) + f8_parts_most(rows, out, in, [&](int64_t m) { return f8_stages_one(m, out, in); });
}

extern "C" int ddg_fp8_linear(const void *x, int x_type, int64_t ld_x, int64_t rows, const void *packed_w, int64_t out, int64_t in,
                              const float *bias, void *y, int y_type, int64_t ld_y, void *workspace, size_t workspace_bytes,
                              void *stream) {
    if (!f8_dims_ok(rows, in) || !f8_dims_ok(out, 0) || out < 1 || in < 1 || ld_x < in || ld_y < out || !ddg_type_ok(x_type) ||
        !ddg_type_ok(y_type) || !packed_w || ((uintptr_t)packed_w & 255))
        return DDG_E_ARG;
    if (rows == 0) return DDG_OK;
    if (!x || !y) return DDG_E_ARG;
    if (!f8_product_ok(rows, out, in)) return DDG_E_UNSUPPORTED;
    const F8Operand w = f8_operand((void *)packed_w, out, in);
    const hipStream_t s = (hipStream_t)stream;
    if (f8_skinny(rows, out, in, y_type == DDG_BF16))
        return ddg_with_type(x_type, [&](auto tx) {
            return ddg_with_type(y_type, [&](auto to) {
                using TX = decltype(tx);
                using TO = decltype(to);
                const int nk = (int)(f8_pad(in) / F8_BLOCK);
                auto go = [&](auto waves) {
                    constexpr int W = decltype(waves)::value;
                    const int bytes = (((int)rows * (nk * (F8_BLOCK + 1) + 16) + 15) & ~15) + W * 64 * 16;
                    const auto kernel = k_f8_skinny<TX, TO, W>;
                    const int rc = f8_lds(kernel, bytes);
                    if (rc) return rc;
                    kernel<<<(unsigned)ceil_div64(out, 16), 64 * W, bytes, s>>>((const TX *)x, ld_x, (int)rows, in, w.q,
                                                                               (const uint32_t *)w.s, out, f8_pad(in), bias, (TO *)y,
                                                                               ld_y);
                    DDG_CHECK_LAUNCH();
                    return (int)DDG_OK;
                };
                return nk > 8 ? go(Int<16>()) : go(Int<8>());
            });
        });
    const size_t parts = f8_parts_bytes(f8_split_one(rows, out, in, y_type == DDG_BF16), rows, out);
    if (!workspace || workspace_bytes < ddg_fp8_operand_bytes(rows, in) + parts) return DDG_E_WORKSPACE;
    if ((uintptr_t)workspace & 255) return DDG_E_ARG;
    const F8Operand a = f8_operand(workspace, rows, in);
    const int rc = f8_pack_rows(x, x_type, ld_x, a, s);
    return rc ? rc : f8_gemm(a, w, bias, y, y_type, ld_y, (float *)((char *)workspace + ddg_fp8_operand_bytes(rows, in)), s);
}

struct F8GradWs {
    void *dy, *dyt, *xt;
    float *sums, *parts_dx, *parts_dw;
    size_t bytes;
};
// parts_dx, parts_dw: bytes of the parts of the two products
static inline F8GradWs f8_grad_carve(void *base, int64_t rows, int64_t out, int64_t in, size_t parts_dx, size_t parts_dw) {
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
    w.parts_dx = (float *)take(parts_dx);
    w.parts_dw = (float *)take(parts_dw);
    w.bytes = o;
    return w;
}
extern "C" size_t ddg_fp8_linear_grads_workspace_bytes(int64_t rows, int64_t out, int64_t in) {
    if (!f8_dims_ok(rows, in) || !f8_dims_ok(out, 0) || in < 1 || out < 1) return 0;
    // Where the products go apart nothing is split: dX is 256 x 256 tiles, and two shares of dW's 384 tiles and more are longer than
    // its reduction.  Together both have the same number of stages, so that dW's share is 1 / 256 of them at least
    const size_t dx = f8_parts_most(rows, in, out, [&](int64_t m) { return f8_grad_stages(m, out, in, f8_grad_narrow(m, out, in) ? 64 : 128); });
    const int64_t nk = ceil_div64(rows, F8_BLOCK), tw = f8_tiles(out, in), few = ceil_div64(nk, 4), share = ceil_div64(256, tw);
    const size_t dw = nk < 8 || tw > 128 ? 0 : f8_parts_bytes({few < share ? few : share, 4}, out, in);
    return f8_grad_carve(nullptr, rows, out, in, dx, dw).bytes;
}

extern "C" int ddg_fp8_linear_grads(const void *dy, int dy_type, int64_t ld_dy, const void *x, int x_type, int64_t ld_x,
                                    int64_t rows, const void *packed_wt, int64_t out, int64_t in, void *dx, int dx_type,
                                    int64_t ld_dx, float *dw, float *db, void *workspace, size_t workspace_bytes, void *stream) {
    if (!f8_dims_ok(rows, in) || !f8_dims_ok(out, 0) || rows < 1 || out < 1 || in < 1 || ld_dy < out || ld_x < in || ld_dx < in ||
        !ddg_type_ok(dy_type) || !ddg_type_ok(x_type) || !ddg_type_ok(dx_type) || !dy || !x || !packed_wt || !dx || !dw ||
        ((uintptr_t)packed_wt & 255))
        return DDG_E_ARG;
    if (!f8_product_ok(rows, in, out) || !f8_product_ok(out, in, rows)) return DDG_E_UNSUPPORTED;
    const F8GradSplits sp = f8_grad_splits(rows, out, in, dx_type == DDG_BF16);
    const F8GradWs w = f8_grad_carve(workspace, rows, out, in, f8_parts_bytes(sp.dx, rows, in), f8_parts_bytes(sp.dw, out, in));
    if (!workspace || workspace_bytes < w.bytes) return DDG_E_WORKSPACE;
    if ((uintptr_t)workspace & 255) return DDG_E_ARG;
    const hipStream_t s = (hipStream_t)stream;
    const F8Operand gy = f8_operand(w.dy, rows, out), gyt = f8_operand(w.dyt, out, rows), xt = f8_operand(w.xt, in, rows);
    const int64_t tiles_dy = f8_tiles(rows, out), tiles_x = f8_tiles(rows, in), row_tiles = ceil_div64(rows, F8_BLOCK);
    if (tiles_dy + tiles_x > ddg_max_grid(256)) return DDG_E_UNSUPPORTED;
    // (one row tile: its column sums are the result)
    const F8Pack pd = {dy, ld_dy, rows, out, gy.q, gy.s, gyt.q, gyt.s, !db ? nullptr : row_tiles == 1 ? db : w.sums};
    const F8Pack px = {x, ld_x, rows, in, nullptr, nullptr, xt.q, xt.s, nullptr};
    auto pack = [&](int type, int64_t td, int64_t tx) {
        return ddg_with_type(type, [&](auto t) {
            k_f8_pack_grads<decltype(t)><<<(unsigned)(td + tx), 256, 0, s>>>(pd, (uint32_t)td, px);
            DDG_CHECK_LAUNCH();
            return (int)DDG_OK;
        });
    };
    int rc = pack(dy_type, tiles_dy, x_type == dy_type ? tiles_x : 0);
    if (!rc && x_type != dy_type) rc = pack(x_type, 0, tiles_x);
    if (rc) return rc;
    const F8Colsum sum = {w.sums, row_tiles, out, db && row_tiles > 1 ? db : nullptr};
    return f8_gemm_grads(gy, f8_operand((void *)packed_wt, in, out), dx, dx_type, ld_dx, w.parts_dx, gyt, xt, dw, w.parts_dw, sum, s);
}
