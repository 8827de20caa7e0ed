// smelter_amd/csrc/kernels/linear.hpp — what the linear-layer kernels (linear.hip) share: element types, the MX4 block format, group lookup, epilogue.
//
//     y[s, n] = act(bias[e, n] + sum_k x[r(s), k] * w[e, n, k])          e = the group slot s lies in: offsets[e] <= s < offsets[e + 1];  r(s) = rows ? rows[s] : s
//     gated:  y[s, n] = silu(z[s, n]) * z[s, N + n],  z = the product (with bias) over 2 N weight rows
//
// Operand kinds: fp16 / bf16 (2 bytes), MX4 = blocks of 32 e2m1 elements along K (16 bytes, even element in the low nibble) with one e8m0 scale byte 2^(b - 127) each (255 = NaN).
#pragma once
#include "common.hpp"

typedef __bf16 bf16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef int intx4_t __attribute__((ext_vector_type(4)));
typedef int intx8_t __attribute__((ext_vector_type(8)));
typedef float floatx2_t __attribute__((ext_vector_type(2)));

#define LIN_MARKED (-(1 << 30))
struct LinearParams {
    const char* x; const unsigned char* xs;         // x rows; scales of an MX4 x
    const char* w; const unsigned char* ws;
    const float* bias; void* y;
    const int* offsets; const int* rows;
    long long x_ld, xs_ld;                          // BYTES per x row / per scale row
    long long w_ld, ws_ld, w_es, ws_es;             // BYTES per weight row, scale row, expert
    long long y_ld, M, T;                           // y row stride in elements; slots; x rows
    int N, K, E, act; float slope;
    int gated, y_type, y_vec, w_rows;               // y_vec: eight consecutive outputs may be stored as 16-byte words;  w_rows = N or 2 N
    float* part; long long part_ld; int splits;     // fp32 sums [splits][M][part_ld] of a product whose K is cut into `splits` runs (1: none)
    int parts;                                      // (lin_join_kernel) not 0: the sums are [M][parts][part_ld], of the parts of fp32 rows
    const int* power;                               // fp32 rows in fp16 parts: the power of two of each slot's row, or LIN_MARKED: multiplied in fp32
    long long m_tiles; int n_tiles;                 // launch grid: a bound on the row tiles (the real number is known on the device only) x column tiles
};

__device__ __forceinline__ float lin_act(float v, int act, float slope) {
    if (act == SM_ACT_NONE) return v;
    if (act == SM_ACT_RELU) return v < 0.f ? 0.f : v;
    if (act == SM_ACT_PRELU) return v < 0.f ? v * slope : v;
    return sm_act_other(v, act, slope);
}
// v / (1 + e^-v) by the hardware's reciprocal: a division costs ten instructions a value, 11 us of the 94 of 8192 x 4096 gated columns with K = 2048 in MX4.  What it is off by, relative to the result:
// the reciprocal 2^-23, the product 2^-24, and 2^-24 |v| of the exponential's argument (v log2(e) rounded once; e^-v is that sensitive to the rounding of v itself).  Below v = -87.3 the result is 0
// (there |silu| < 2^-119), as the reciprocal of more than 2^126 is.
__device__ __forceinline__ float lin_silu(float v) { return v * __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// one rounding to the output type (nearest even)
__device__ __forceinline__ void lin_store1(void* y, long long i, float v, int type) {
    if (type == SM_F16) ((half_t*)y)[i] = (half_t)v;
    else if (type == SM_BF16) ((bf16_t*)y)[i] = (bf16_t)v;
    else ((float*)y)[i] = v;
}
__device__ __forceinline__ void lin_store4(void* y, long long i, const float* v, int type) {
    if (type == SM_F16) { half4_t h; for (int q = 0; q < 4; q++) h[q] = (half_t)v[q]; *(half4_t*)((half_t*)y + i) = h; }
    else if (type == SM_BF16) { bf16x4_t h; for (int q = 0; q < 4; q++) h[q] = (bf16_t)v[q]; *(bf16x4_t*)((bf16_t*)y + i) = h; }
    else *(floatx4*)((float*)y + i) = floatx4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ void lin_store8(void* y, long long i, const float* v, int type) {
    if (type == SM_F16) { half8_t h; for (int q = 0; q < 8; q++) h[q] = (half_t)v[q]; *(half8_t*)((half_t*)y + i) = h; }
    else if (type == SM_BF16) { bf16x8_t h; for (int q = 0; q < 8; q++) h[q] = (bf16_t)v[q]; *(bf16x8_t*)((bf16_t*)y + i) = h; }
    else { *(floatx4*)((float*)y + i) = floatx4{v[0], v[1], v[2], v[3]}; *(floatx4*)((float*)y + i + 4) = floatx4{v[4], v[5], v[6], v[7]}; }
}

// a bound on the row tiles of BM slots: the sum of ceil(rows / BM) over at most min(E, M) non-empty groups
inline long long lin_row_tiles(const LinearParams& p, int BM) {
    const long long groups = p.offsets ? (p.M < p.E ? p.M : p.E) : 1;
    return (p.M + (BM - 1ll) * groups) / BM;
}
inline bool lin_one_launch(long long blocks, int threads) { return blocks < (1ll << 32) / threads; }   // a launch counts its threads in 32 bits
// the tile kernels hold byte offsets inside an expert's weights, and inside x (gathered rows) or the rows of a tile, in 32 bits
inline bool lin_tile_fits(const LinearParams& p) { return p.w_es < (1ll << 32) && (p.rows ? p.T * p.x_ld : 256 * p.x_ld) < (1ll << 32); }
// linear_tile.hip: the tile kernels; shape 0 = 128 x 128, 1 = 256 x 256, 2 = 128 columns x 64 slots;  dma = both operands have rows of whole, 16-byte aligned chunks
int lin_tile_launch(const LinearParams& p, int x_kind, int w_kind, int shape, bool dma, hipStream_t s);
// linear_deep.hip: the kernel for few tiles, shapes 0 and 2 of whole chunks; > 0: not enough LDS for the scales of so long a row
int lin_deep_launch(const LinearParams& p, int x_kind, int w_kind, int shape, hipStream_t s);
int lin_join_launch(const LinearParams& p, hipStream_t s);

struct LinTile { int e; long long row0; int rows; long long total; };            // group, first slot, rows of the tile (<= BM); number of row tiles

// Row tile `t` of the group list.  Every group is cut into tiles of BM slots; the offsets live on the device, so each wave counts the tiles of 64 groups at a time (prefix sum over the
// lanes) until it has passed `t`.  Offsets are clamped to 0 .. M, a group that ends before it begins is empty: nothing outside the M slots is ever addressed, whatever they hold.
// rows = 0: there is no such tile.  Wave-uniform.
__device__ __forceinline__ long long lin_clamp(long long v, long long hi) { return v < 0 ? 0 : (v > hi ? hi : v); }
__device__ __forceinline__ long long lin_uniform(long long v) {                     // a wave-uniform value into scalar registers
    return ((long long)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ LinTile lin_find_tile(const LinearParams& p, int BM, long long t, bool want_total) {
    LinTile r; r.e = 0; r.row0 = 0; r.rows = 0; r.total = 0;
    if (!p.offsets) {
        r.total = (p.M + BM - 1) / BM;
        if (t < r.total) { r.row0 = t * BM; long long left = p.M - r.row0; r.rows = (int)(left < BM ? left : BM); }
        return r;
    }
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < p.E; base += 64) {
        int e = base + lane;
        long long lo = 0, hi = 0;
        if (e < p.E) { lo = lin_clamp(p.offsets[e], p.M); hi = lin_clamp(p.offsets[e + 1], p.M); }
        int n = hi > lo ? (int)((hi - lo + BM - 1) / BM) : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { int up = __shfl_up(sum, d); if (lane >= d) sum += up; }
        const int all = __builtin_amdgcn_readlane(sum, 63);
        if (r.rows == 0 && t < r.total + all) {
            const unsigned long long past = __ballot(r.total + sum > t);
            const int at = __builtin_ctzll(past);
            const long long tl = t - r.total - (__shfl(sum, at) - __shfl(n, at));
            const long long l = __shfl(lo, at), h = __shfl(hi, at);
            const long long row0 = l + tl * BM, left = tl < 0 ? 0 : h - row0;         // (offsets that do not ascend may count more tiles than 32 bits hold)
            r.e = base + at; r.row0 = lin_uniform(row0); r.rows = __builtin_amdgcn_readfirstlane((int)(left < 0 ? 0 : left < BM ? left : BM));
            if (!want_total) return r;
        }
        r.total += all;
    }
    return r;
}

// eight consecutive 16-bit elements k .. k + 7 of a row of K, zero behind its end (any alignment: the compiler's unaligned 16-byte load)
__device__ __forceinline__ intx4_t lin_load8(const char* row, int k, int K) {
    intx4_t v = {0, 0, 0, 0};
    if (k + 8 <= K) __builtin_memcpy(&v, row + 2ll * k, 16);
    else if (k < K) {
        unsigned h[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) if (k + i < K) { unsigned short q; __builtin_memcpy(&q, row + 2ll * (k + i), 2); h[i >> 1] |= (unsigned)q << (16 * (i & 1)); }
        v = intx4_t{(int)h[0], (int)h[1], (int)h[2], (int)h[3]};
    }
    return v;
}

// eight MX4 elements (one dword of codes) as 16-bit values times the power of two `scale` (exact while the result is in the type's range; a NaN scale gives NaN)
template <int KIND> __device__ __forceinline__ intx4_t mx4_to16(int codes, float scale) {
    intx4_t r;
    if constexpr (KIND == SM_F16) {
        r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)); r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1));
        r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)); r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3));
    } else {
        r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)); r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
        r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)); r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    }
    return r;
}
__device__ __forceinline__ float mx4_scale(int byte) { return __builtin_bit_cast(float, byte << 23); }   // as an operand of the MX4 conversions, which read the exponent field alone (0 = 2^-127)

// fp16 x on MX4 weights: a weight as an fp16 operand of the matrix instruction is taken relative to the largest scale `top` of its row (or run), which becomes 2^13: 6 * 2^13 is below 65504, and the
// code .5 is exact down to 2^-24, so that scales 2^36 apart are exact together.  The sum is multiplied by lin_top_scale.  Where a row holds a block further below (and not all of it 0) the rows
// of its fragments are multiplied by lin_exact_blocks.  top >= 14.
#define LIN_REACH 36
__device__ __forceinline__ int lin_relative(int byte, int top) { const int d = byte - top + 140; return byte == 255 ? 255 : d > 0 ? d : 0; }
__device__ __forceinline__ float lin_top_scale(int top) { return mx4_scale(top - 13); }
__device__ __forceinline__ int lin_top_of(int top, int byte) { return byte != 255 && byte > top ? byte : top; }       // (a NaN block is one under every scale)

// largest and smallest of scale bytes, four at a time (lin_top_of takes three instructions a byte: 4 us of the 49 of 1024 x 4096 x 4096)
typedef unsigned short ushortx2_t __attribute__((ext_vector_type(2)));
struct LinSpread {
    ushortx2_t hi = {0, 0}, lo = {255, 255};
    __device__ __forceinline__ void look(unsigned v) {
        const ushortx2_t a = __builtin_bit_cast(ushortx2_t, v & 0x00ff00ffu), b = __builtin_bit_cast(ushortx2_t, v >> 8 & 0x00ff00ffu);
        hi = __builtin_elementwise_max(hi, __builtin_elementwise_max(a, b)); lo = __builtin_elementwise_min(lo, __builtin_elementwise_min(a, b));
    }
    __device__ __forceinline__ int top() const { return hi[0] > hi[1] ? hi[0] : hi[1]; }
    __device__ __forceinline__ int low() const { return lo[0] < lo[1] ? lo[0] : lo[1]; }
};

// eight fp16 values as sums of two bf16 ones: eight bits cut off, three left (an infinity, a NaN: once)
__device__ __forceinline__ void lin_halves(intx4_t v, intx4_t& hi, intx4_t& lo) {
    const half8_t h = __builtin_bit_cast(half8_t, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned a[2], b[2];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const float f = (float)h[2 * i + q];
            a[q] = __builtin_bit_cast(unsigned, f) >> 16;
            const float left = __builtin_fabsf(f) < __builtin_inff() ? f - __builtin_bit_cast(float, a[q] << 16) : 0.f;
            b[q] = __builtin_bit_cast(unsigned, left) >> 16;
        }
        hi[i] = (int)(a[0] | a[1] << 16); lo[i] = (int)(b[0] | b[1] << 16);
    }
}

// 16 x 16 x 32 product of 16-bit fragments: lane l holds row l & 15, k = 8 (l >> 4) .. + 7 of either operand; result rows (first operand) 4 (l >> 4) + i, column l & 15
template <int KIND> __device__ __forceinline__ floatx4 lin_mma16(intx4_t a, intx4_t b, floatx4 c) {
    if constexpr (KIND == SM_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// 32 x 32 x 16: lane l holds row l & 31, k = 8 (l >> 5) .. + 7; result rows 8 (i / 4) + 4 (l >> 5) + i % 4, column l & 31
template <int KIND> __device__ __forceinline__ floatx16 lin_mma16(intx4_t a, intx4_t b, floatx16 c) {
    if constexpr (KIND == SM_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// 16 x 16 x 4 product of fp32 elements: lane l holds row l & 15 and one k, l >> 4; the result lies as that of 16 x 16 x 32
__device__ __forceinline__ floatx4 lin_mma32(float a, float b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// 16 x 16 x 128 (32 x 32 x 64) product of MX4 fragments: lane l holds row l % 16 (32) and one block of 32, with its scale in byte SEL of sa, in the low byte of sb
template <int SEL> __device__ __forceinline__ floatx4 lin_mma4(intx4_t a, int sa, intx4_t b, int sb, floatx4 c) {
    const intx8_t va = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), vb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);   // (a 4-bit operand is four registers)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, SEL, sa, 0, sb);
}
template <int SEL> __device__ __forceinline__ floatx16 lin_mma4(intx4_t a, int sa, intx4_t b, int sb, floatx16 c) {
    const intx8_t va = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), vb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, c, 4, 4, SEL, sa, 0, sb);
}

// fp16 x on MX4 weights with bf16 instructions, straight from memory: any scale is exact there, x becomes two bf16 fragments.  For the rare fragments whose rows hold scales more than 2^36 apart,
// where it is right and slow (us with such a row in every fragment: 5 rows of 16384 x 8192 140 against 20, 512 of 4096 x 4096 210 / 29, 4001 of 8192 x 4096 3446 / 210); the blocks first .. last - 1 of one fragment of FR weight rows.  w, scales, x[b] = this lane's rows, xk[b] = K, or 0: none;  add(b, w, x): the product,
// raise(): the sums so far times 2^128.  Blocks at the upper end of the range come first, 2^128 smaller, so that no weight is an infinity in bf16 (a second part that is 0 times it: a NaN).
template <int FR, int FM, class F, class R>
__device__ __forceinline__ void lin_exact_blocks(const char* w, const unsigned char* scales, const char* const (&x)[FM], const int (&xk)[FM], int first, int last, F add, R raise) {
    const int g = (threadIdx.x & 63) / FR;
    auto high = [](int byte) { return byte >= 200 && byte != 255; };
    bool upper = false;
    for (int block = first; block < last; block++) upper |= high(scales[block]);
#pragma unroll 1
    for (int pass = __any(upper) ? 0 : 1; pass < 2; pass++) {
#pragma unroll 1
        for (int block = first; block < last; block++)
#pragma unroll 1
            for (int h = 0; h < FR / 16; h++) {
                const int q = h * (64 / FR) + g, byte = scales[block];               // a lane's eight k of the block
                const bool now = high(byte) == (pass == 0);
                int code; __builtin_memcpy(&code, w + 16ll * block + 4 * q, 4);
                const intx4_t wf = mx4_to16<SM_BF16>(now ? code : 0, mx4_scale(now ? byte - (pass == 0 ? 128 : 0) : 127));
#pragma unroll
                for (int b = 0; b < FM; b++) {
                    intx4_t hi, lo; lin_halves(lin_load8(x[b], 32 * block + 8 * q, xk[b]), hi, lo);
                    add(b, wf, hi); add(b, wf, lo);
                }
            }
        if (pass == 0) raise();
    }
}
