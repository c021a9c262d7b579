// Device helpers of the microscaled (MX) formats: 32 consecutive values of a row share the scale 2^(byte - 127).
//   fmt 8: e4m3 values (largest 448), fmt 4: e2m1 values (largest 6), two to a byte, the even one in the low nibble
//   byte = biased exponent of the block's largest magnitude - exponent of the format's largest power of two, at least 0;
//   byte 255: the block held an infinity or a NaN, its codes are zero and every value of it stands for NaN
// Rows are padded with zero codes to MX_PAD values, so that a product needs no test inside its k loop.
#pragma once
#include "common.h"

// 16 bytes at any element's address.  Global memory takes unaligned vector accesses, so rows of odd length cost an extra cache
// line here and there instead of an instruction per value (1001 x 1283 x 1024 with an fp32 result: 18.7 us with scalar stores,
// 13 so).
typedef u32x4 u32x4_any __attribute__((aligned(2)));
__device__ __forceinline__ u32x4 load16_any(const void* p) { return *static_cast<const u32x4_any*>(p); }
__device__ __forceinline__ void store16_any(void* p, const u32x4& v) { *static_cast<u32x4_any*>(p) = v; }

constexpr int MX_BLOCK = 32;
constexpr int MX_PAD = 128;

__host__ __device__ constexpr int mx_emax(int fmt) { return fmt == 8 ? 8 : 2; }
__host__ __device__ constexpr int mx_bytes(int fmt, int values) { return fmt == 8 ? values : values / 2; }
__host__ __device__ constexpr int mx_padded(int k) { return (k + MX_PAD - 1) / MX_PAD * MX_PAD; }

// Largest magnitude of N values; NaN if one of them is (v_maximum3_f32 passes a NaN on, v_max_f32 would drop it).
template <int N> __device__ __forceinline__ float mx_largest(const float* v) {
    float top = __builtin_fabsf(v[0]);
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2) top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(v[i]), __builtin_fabsf(v[i + 1])), top);
    if constexpr (N % 2 == 0) top = __builtin_elementwise_maximum(top, __builtin_fabsf(v[N - 1]));
    return top;
}
template <int FMT> __device__ __forceinline__ uint32_t mx_scale_byte(float top) {
    const uint32_t e = __float_as_uint(top) >> 23;  // biased (the sign is 0); 0 for zero and subnormals, whose scale is the smallest anyway
    return (e & 255u) == 255u ? 255u : (e > (uint32_t)mx_emax(FMT) ? e - mx_emax(FMT) : 0u);
}
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : (byte == 0u ? 0x00400000u : byte << 23));
}

// Eight values -> eight codes in W words (W = 2: e4m3, 1: e2m1) under the scale 2^(byte - 127); to nearest even, saturated; zeros
// under byte 255.  The conversions divide by the scale themselves (exactly, a power of two; 2^-127 included) and the 4-bit one
// saturates; the 8-bit one makes NaN of what is too large, hence the clamp.
template <int FMT> struct MxCodes {
    static constexpr int W = FMT == 8 ? 2 : 1;
    uint32_t w[W];
};
template <int FMT> __device__ __forceinline__ MxCodes<FMT> mx_encode8(const float* v, uint32_t byte) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const float scale = mx_scale(byte);
    MxCodes<FMT> c;
    if constexpr (FMT == 8) {
        const float most = 448.f * scale;
        float u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = __builtin_amdgcn_fmed3f(v[i], -most, most);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s16x2 w = {0, 0};
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, u[4 * h], u[4 * h + 1], scale, false);
            c.w[h] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, u[4 * h + 2], u[4 * h + 3], scale, true));
        }
    } else {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
        c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    }
#pragma unroll
    for (int i = 0; i < MxCodes<FMT>::W; ++i) c.w[i] = byte == 255u ? 0u : c.w[i];
    return c;
}
template <int FMT> __device__ __forceinline__ void mx_decode8(const uint32_t* w, float scale, float* v) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    f2 p[4];
    if constexpr (FMT == 8) {
        p[0] = __builtin_amdgcn_cvt_pk_f32_fp8(w[0], false);
        p[1] = __builtin_amdgcn_cvt_pk_f32_fp8(w[0], true);
        p[2] = __builtin_amdgcn_cvt_pk_f32_fp8(w[1], false);
        p[3] = __builtin_amdgcn_cvt_pk_f32_fp8(w[1], true);
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 0);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 1);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 2);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 3);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = p[i][0] * scale;
        v[2 * i + 1] = p[i][1] * scale;
    }
}
// largest of the four lanes of a quad (the 32 values of a block when every lane holds eight)
__device__ __forceinline__ float mx_quad_largest(float v) {
    v = __builtin_elementwise_maximum(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true)));  // quad_perm 1 0 3 2
    return __builtin_elementwise_maximum(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, true)));  // 2 3 0 1
}
// A quad's 32 values -> codes and (first lane) scale.  `codes` points at this lane's eight codes, `scale` at the block's byte.
template <int FMT> __device__ __forceinline__ void mx_store_quad(const float* v, unsigned char* codes, unsigned char* scale, int lane) {
    const uint32_t byte = mx_scale_byte<FMT>(mx_quad_largest(mx_largest<8>(v)));
    const MxCodes<FMT> c = mx_encode8<FMT>(v, byte);
    if constexpr (FMT == 8) *reinterpret_cast<u32x2*>(codes) = u32x2{c.w[0], c.w[1]};
    else *reinterpret_cast<uint32_t*>(codes) = c.w[0];
    if ((lane & 3) == 0) *scale = (unsigned char)byte;
}
