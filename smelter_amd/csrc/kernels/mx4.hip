// smelter_amd/csrc/kernels/mx4.hip — MX4 tensors: blocks of 32 e2m1 elements with one e8m0 scale (the OCP microscaling format), packing and reading back.
//
//     scale = 2^(floor(log2 amax) - 2)  (2 = the largest exponent of e2m1; clamped below at 2^-127)      code = nearest of {0, .5, 1, 1.5, 2, 3, 4, 6} to |v| / scale, ties to the even code
//
// |v| / scale lies below 8; what lies above 6 becomes 6 (the format's own rule: the scale is not raised).  Division by a power of two is exact, so the code of every value is decided without a
// rounding before it.  A block that holds a NaN or an infinity gets scale byte 255 (NaN) and codes 0; a block of zeros scale byte 0.  The sign of a value that becomes zero is kept.
// Both directions are bound by memory: 2 + 17/32 bytes per 16-bit element.  65536 x 4096 bf16: packed in 156 us (4.4 TB/s), read back in 117 (5.8 TB/s; a copy of 1 GiB: 5.1).  A thread packs a whole
// block, so that no maximum crosses lanes; it reads back eight elements, so that it stores 16 bytes.
#include "linear.hpp"

template <int KIND> struct Mx4In;      // the 32 elements of one block in registers, and their largest magnitude as fp32 bits (>= 0x7f800000: an infinity or a NaN)
template <> struct Mx4In<SM_F32> {
    static constexpr int ES = 4; float f[32];
    __device__ __forceinline__ unsigned top() const { unsigned m = 0; for (int i = 0; i < 32; i++) { unsigned b = __builtin_bit_cast(unsigned, f[i]) & 0x7fffffffu; m = m > b ? m : b; } return m; }
    __device__ __forceinline__ int pack8(int q, float s) const {
        unsigned c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[8 * q], f[8 * q + 1], s, 0); c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[8 * q + 2], f[8 * q + 3], s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[8 * q + 4], f[8 * q + 5], s, 2); return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[8 * q + 6], f[8 * q + 7], s, 3);
    }
};
template <int KIND> struct Mx4In16 {
    static constexpr int ES = 2; unsigned f[16];
    __device__ __forceinline__ unsigned top() const {
        unsigned lo = 0, hi = 0;
        for (int i = 0; i < 16; i++) { unsigned a = f[i] & 0x7fffu, b = f[i] & 0x7fff0000u; lo = lo > a ? lo : a; hi = hi > b ? hi : b; }
        const unsigned m = lo > (hi >> 16) ? lo : (hi >> 16);
        if (KIND == SM_BF16) return m << 16;
        return m >= 0x7c00u ? 0x7f800000u : __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(half_t, (unsigned short)m));
    }
    __device__ __forceinline__ int pack8(int q, float s) const {
        unsigned c = 0;
        if constexpr (KIND == SM_F16) {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(half2_t, f[4 * q]), s, 0); c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(half2_t, f[4 * q + 1]), s, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(half2_t, f[4 * q + 2]), s, 2); return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(half2_t, f[4 * q + 3]), s, 3);
        } else {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, f[4 * q]), s, 0); c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, f[4 * q + 1]), s, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, f[4 * q + 2]), s, 2); return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, f[4 * q + 3]), s, 3);
        }
    }
};
template <> struct Mx4In<SM_F16> : Mx4In16<SM_F16> {};
template <> struct Mx4In<SM_BF16> : Mx4In16<SM_BF16> {};

__device__ __forceinline__ void mx4_split(long long u, int per, long long* row, int* at) {       // u = row * per + at
    if (u < 0x7fffffffll) { const unsigned q = (unsigned)u / (unsigned)per; *row = q; *at = (int)((unsigned)u - q * (unsigned)per); }
    else { *row = u / per; *at = (int)(u - *row * per); }
}

// one thread per block
template <int KIND> __global__ void mx4_quantize_kernel(const char* x, long long units, int nb, int K, long long x_ld, unsigned char* codes, unsigned char* scales) {
    for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < units; u += (long long)gridDim.x * blockDim.x) {
        long long row; int b; mx4_split(u, nb, &row, &b);
        Mx4In<KIND> v; constexpr int ES = Mx4In<KIND>::ES;
        const char* src = x + row * x_ld + 32ll * ES * b;
        const int left = K - 32 * b;
        if (left >= 32) __builtin_memcpy(v.f, src, 32 * ES);
        else {
            if constexpr (ES == 4) { for (int i = 0; i < 32; i++) { v.f[i] = 0.f; if (i < left) __builtin_memcpy(&v.f[i], src + 4 * i, 4); } }
            else for (int i = 0; i < 16; i++) {
                unsigned short a = 0, c = 0;
                if (2 * i < left) __builtin_memcpy(&a, src + 4 * i, 2);
                if (2 * i + 1 < left) __builtin_memcpy(&c, src + 4 * i + 2, 2);
                v.f[i] = a | (unsigned)c << 16;
            }
        }
        const unsigned top = v.top();
        const bool bad = top >= 0x7f800000u;
        int byte = (int)(top >> 23) - 2; if (byte < 0) byte = 0; if (bad) byte = 255;
        const float s = mx4_scale(byte);
        intx4_t c;
        for (int q = 0; q < 4; q++) c[q] = bad ? 0 : v.pack8(q, s);
        *(intx4_t*)(codes + 16 * u) = c;
        scales[u] = (unsigned char)byte;
    }
}

// one thread per eight elements
template <int KIND> __global__ void mx4_dequantize_kernel(const unsigned char* codes, const unsigned char* scales, long long units, int nb, int K, void* y, long long y_ld, int vec) {
    for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < units; u += (long long)gridDim.x * blockDim.x) {
        long long row; int q; mx4_split(u, 4 * nb, &row, &q);
        const int c = *(const int*)(codes + 4 * u);
        const float s = mx4_scale(scales[u >> 2]);
        const long long at = row * y_ld + 8ll * q;
        const int left = K - 8 * q;
        if constexpr (KIND == SM_F32) {
            float v[8]; floatx2_t t;
            t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0); v[0] = t[0]; v[1] = t[1]; t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1); v[2] = t[0]; v[3] = t[1];
            t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2); v[4] = t[0]; v[5] = t[1]; t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3); v[6] = t[0]; v[7] = t[1];
            float* dst = (float*)y + at;
            if (left >= 8 && vec) { *(floatx4*)dst = floatx4{v[0], v[1], v[2], v[3]}; *(floatx4*)(dst + 4) = floatx4{v[4], v[5], v[6], v[7]}; }
            else for (int i = 0; i < 8; i++) if (i < left) dst[i] = v[i];
        } else {
            const intx4_t v = mx4_to16<KIND>(c, s);
            unsigned short* dst = (unsigned short*)y + at;
            if (left >= 8 && vec) *(intx4_t*)dst = v;
            else for (int i = 0; i < 8; i++) if (i < left) dst[i] = (unsigned short)((unsigned)v[i >> 1] >> (16 * (i & 1)));
        }
    }
}

static int mx4_grid(long long units, int block) { const long long b = (units + block - 1) / block, cap = (long long)SM_NUM_CU * 32; return (int)(b < cap ? b : cap); }

extern "C" int sm_mx4_quantize(const void* x, int32_t x_type, int64_t rows, int32_t K, int64_t x_ld, void* codes, void* scales, sm_stream_t stream) {
    SM_REQUIRE(x_type == SM_F16 || x_type == SM_BF16 || x_type == SM_F32, "mx4_quantize: type %d is not fp16, bf16 or fp32", x_type);
    SM_REQUIRE(rows >= 0 && K >= 0, "mx4_quantize: negative size (%lld x %d)", (long long)rows, K);
    if (rows == 0 || K == 0) return SM_OK;
    const int nb = K / 32 + (K % 32 != 0);
    SM_REQUIRE(x && codes && scales, "mx4_quantize: null operand");
    SM_REQUIRE(rows <= (1ll << 40) / nb, "mx4_quantize: %lld x %d elements", (long long)rows, K);
    SM_REQUIRE(rows == 1 || x_ld >= K, "mx4_quantize: row stride %lld below the %d columns", (long long)x_ld, K);
    const int es = x_type == SM_F32 ? 4 : 2;
    SM_REQUIRE(((size_t)x % es) == 0 && ((size_t)codes & 15) == 0, "mx4_quantize: codes need 16-byte alignment, x its type's");
    const long long units = rows * nb;
    const dim3 grid(mx4_grid(units, 256));
    if (x_type == SM_F32) mx4_quantize_kernel<SM_F32><<<grid, 256, 0, sm_s(stream)>>>((const char*)x, units, nb, K, x_ld * es, (unsigned char*)codes, (unsigned char*)scales);
    else if (x_type == SM_F16) mx4_quantize_kernel<SM_F16><<<grid, 256, 0, sm_s(stream)>>>((const char*)x, units, nb, K, x_ld * es, (unsigned char*)codes, (unsigned char*)scales);
    else mx4_quantize_kernel<SM_BF16><<<grid, 256, 0, sm_s(stream)>>>((const char*)x, units, nb, K, x_ld * es, (unsigned char*)codes, (unsigned char*)scales);
    SM_LAUNCH_CHECK();
    return SM_OK;
}

extern "C" int sm_mx4_dequantize(const void* codes, const void* scales, int64_t rows, int32_t K, void* y, int32_t y_type, int64_t y_ld, sm_stream_t stream) {
    SM_REQUIRE(y_type == SM_F16 || y_type == SM_BF16 || y_type == SM_F32, "mx4_dequantize: type %d is not fp16, bf16 or fp32", y_type);
    SM_REQUIRE(rows >= 0 && K >= 0, "mx4_dequantize: negative size (%lld x %d)", (long long)rows, K);
    if (rows == 0 || K == 0) return SM_OK;
    const int nb = K / 32 + (K % 32 != 0);
    SM_REQUIRE(y && codes && scales, "mx4_dequantize: null operand");
    SM_REQUIRE(rows <= (1ll << 40) / nb, "mx4_dequantize: %lld x %d elements", (long long)rows, K);
    SM_REQUIRE(rows == 1 || y_ld >= K, "mx4_dequantize: row stride %lld below the %d columns", (long long)y_ld, K);
    const int es = y_type == SM_F32 ? 4 : 2;
    SM_REQUIRE(((size_t)y % es) == 0 && ((size_t)codes & 15) == 0, "mx4_dequantize: codes need 16-byte alignment, y its type's");
    const long long units = rows * nb * 4;
    const int vec = ((size_t)y & 15) == 0 && (rows == 1 || (y_ld * es) % 16 == 0);
    const dim3 grid(mx4_grid(units, 256));
    if (y_type == SM_F32) mx4_dequantize_kernel<SM_F32><<<grid, 256, 0, sm_s(stream)>>>((const unsigned char*)codes, (const unsigned char*)scales, units, nb, K, y, y_ld, vec);
    else if (y_type == SM_F16) mx4_dequantize_kernel<SM_F16><<<grid, 256, 0, sm_s(stream)>>>((const unsigned char*)codes, (const unsigned char*)scales, units, nb, K, y, y_ld, vec);
    else mx4_dequantize_kernel<SM_BF16><<<grid, 256, 0, sm_s(stream)>>>((const unsigned char*)codes, (const unsigned char*)scales, units, nb, K, y, y_ld, vec);
    SM_LAUNCH_CHECK();
    return SM_OK;
}
