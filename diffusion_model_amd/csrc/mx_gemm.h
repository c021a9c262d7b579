// Shared by the two kernels of dm_mx_gemm: C = act(X W^T + bias) + r on microscaled (MX) matrices.
#pragma once
#include <type_traits>

#include "dm_hip.h"
#include "mx.h"

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
// a lane's share of a 32-row operand of one matrix instruction: 32 values
template <int F> struct MxFragment { typedef typename std::conditional<F == 8, i32x8, i32x4>::type type; };
typedef __attribute__((ext_vector_type(16))) float f32x16;

struct MxArgs {
    const unsigned char *x, *xs, *w, *ws;
    long ldx, ld_xs, ldw, ld_ws;
    int m, n_out, n_pad;  // rows of C; columns of C; columns to write (MX results: padded, the padding as zeros)
    int nkt;              // k-tiles of 128 values
    int last_blocks;      // blocks of 32 in the last of them that hold values: 1 to 4
    int tiles_m, tiles_n;
    const float* bias;
    const void* r;
    void* c;
    unsigned char* cs;
    long ldr, ldc, ld_cs;
    int epi, c_type;
    int k;                // X as plain rows: values of a row
};

// F32: kernels for fp32 results, and others for bf16 and MX ones, so that no kernel holds an epilogue that it is not launched for (65536 x
// 2560 x 320 with GEGLU, 4 bits to 8: 87.5 us with the fp32 activations beside it, 81.5 without).  With an e4m3 operand fp32
// results come from the operands decoded to bf16 (EXACT).
constexpr bool mx_exact(int xf, int wf, bool f32) { return f32 && (xf == 8 || wf == 8); }

__device__ __forceinline__ i32x8 widen(const i32x8& v) { return v; }
__device__ __forceinline__ i32x8 widen(const i32x4& v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }  // the instruction reads four registers
// Also waits for this wave's LDS reads: what follows is the barrier behind which other waves refill what they read.
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
// at most min(young, MAXY) k-tiles of LOADS requests each may still be outstanding
template <int LOADS, int MAXY> __device__ __forceinline__ void wait_young(int young) {
    if constexpr (MAXY == 0) {
        wait_vm<0>();
    } else {
        if (young >= MAXY) wait_vm<MAXY * LOADS>();
        else wait_young<LOADS, MAXY - 1>(young);
    }
}
__device__ __forceinline__ void to_lds16(const unsigned char* src, unsigned char* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const unsigned char* src, unsigned char* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}

// A k-tile of a row in LDS: 128 values in 128 (e4m3) or 64 (e2m1) bytes, as 16-byte chunks that the XOR below spreads over the
// banks.  A 16-byte read takes four passes of 16 lanes, 0-3, 12-15, 20-27 of each 32 and then the others, and has no conflict when a
// pass's chunks fill 256 bytes.  A fragment of 32 rows has one chunk number in a pass, one of 16 rows has two that differ in their
// last bit.  (Counted at 8192^3, 4 bits: with the second form in both, 60 % of the LDS' cycles were conflicts.)
// Requests fill LDS lane by lane, so it is the chunk they fetch that is permuted.
template <int F, int ROWS> __device__ __forceinline__ int swizzle(int row, int chunk) {
    if constexpr (ROWS == 32) return F == 8 ? chunk ^ ((row >> 1) & 7) : chunk ^ ((row >> 2) & 3);
    else return F == 8 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3);
}
template <int F, int ROWS> __device__ __forceinline__ i32x4 lds_chunk(const unsigned char* base, int row, int chunk) {
    return *reinterpret_cast<const i32x4*>(base + row * mx_bytes(F, MX_PAD) + swizzle<F, ROWS>(row, chunk) * 16);
}
// A block's 32 values as bf16 with the scale applied (exact: at most four significant bits), in four groups of eight.
template <int F> __device__ __forceinline__ void decode_block(const typename MxFragment<F>::type& c, float scale, u32x4* out) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if constexpr (F == 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = (uint32_t)c[2 * q + e / 2];
                out[q][e] = __builtin_bit_cast(uint32_t, e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)
                                                               : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
            }
        } else {
            const uint32_t w = (uint32_t)c[q];
            out[q][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
            out[q][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
            out[q][2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
            out[q][3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
        }
    }
}
// Activations of fp32 results, right to a few units of the result where it is small, too.  An exponential's argument is rounded by
// up to 2^-24 of itself, the exponential by that times the argument, so what the rounding dropped is multiplied on behind it.  Both begin
// from the negative side's value, e or Phi(-|x|), which a sum with 1 would have swallowed: 1 + erff loses 2e-4 of the result at a
// gate of -4, 4 % at -5 and all of it from -5.5 on.  Finite bounds, where the exponential is 0 already, keep infinity - infinity
// out; the product with x then gives what IEEE arithmetic says.  Cost against erff and the fast exponential: 4096 x 10240 x 1280 GEGLU
// 116 -> 125 us, 4096 x 5120 x 1280 QuickGELU 71 -> 75.
__device__ __forceinline__ float quick_gelu_f32(float v) {
    constexpr float rate = 1.702f, rate_rest = (float)(1.702 - (double)1.702f);
    const float t = fminf(fabsf(v), 128.f), a = rate * t, rest = fmaf(rate_rest, t, fmaf(rate, t, -a));
    float e = expf(-a);
    e = fmaf(-e, rest, e);
    return v * (v < 0.f ? e : 1.f) / (1.f + e);
}
// x Phi(x), Phi(-t) = exp(-t^2 / 2) erfcx(t / sqrt 2) / 2
__device__ __forceinline__ float gelu_f32(float x) {
    const float t = fminf(fabsf(x), 20.f), a = t * t, rest = fmaf(t, t, -a);
    float e = expf(-0.5f * a);
    e = fmaf(-0.5f * e, rest, e);
    const float q = 0.5f * e * erfcxf(t * 0.70710678118654752440f);
    return x * (x < 0.f ? q : 1.f - q);
}
// GELU(erf) = x Phi(x) for results of 16 bits and fewer: Phi(-t) = 2^P(t), P of degree 9, fitted on 0 <= t <= 13 to log2 of it.  Evaluated
// in fp32 it is within 6e-6 of the result up to t = 3 and 6e-5 up to 13, a 60th of bf16's rounding; behind 13, where
// Phi leaves the normal range, P falls on to -infinity.  (A polynomial for Phi itself, three instructions and the exponential less, is
// within 1.4e-5 |x|, which is 0.4 % of the result at -3 and 30 % at -4.  It is 4 to 7 % faster at 65536 x 2560 x 320 with GEGLU for
// e4m3 x e2m1, 6 % for 4-bit and 14 % for 8-bit pairs.)
__device__ __forceinline__ float gelu_exp2_f(float x) {
    const float t = fabsf(x);
    float p = -2.1005828187981024e-09f;
    p = fmaf(p, t, 1.5147142562454974e-07f);
    p = fmaf(p, t, -4.794749202119419e-06f);
    p = fmaf(p, t, 8.823825919535011e-05f);
    p = fmaf(p, t, -0.0010582347167655826f);
    p = fmaf(p, t, 0.00884547084569931f);
    p = fmaf(p, t, -0.05443787947297096f);
    p = fmaf(p, t, -0.45813828706741333f);
    p = fmaf(p, t, -1.1513338088989258f);
    p = fmaf(p, t, -0.9999920725822449f);
    const float q = __builtin_amdgcn_exp2f(p);
    return x * (x < 0.f ? q : 1.f - q);
}

// A launch holds fewer than 2^32 threads.
inline bool mx_grid_ok(long blocks, int threads) { return blocks * threads < (1L << 32); }

// Launches the split kernel on tiles of 16 fm rows by 16 fn rows of W; fm, fn = 1 x 1, 1 x 2, 1 x 4, 2 x 2, 2 x 4 or 4 x 4 (1 x .. where X is
// plain rows), fn even for GEGLU, whole MX blocks of columns for an MX result.
int dm_mx_split_launch(const MxArgs& p, int x_fmt, int w_fmt, bool f32, int x_src, int fm, int fn, hipStream_t stream);
