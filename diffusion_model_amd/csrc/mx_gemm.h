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
    int tiles_m, tiles_n;
    const float* bias;
    const void* r;
    void* c;
    unsigned char* cs;
    long ldr, ldc, ld_cs;
    int epi, c_type;
    bool vec;             // rows of C and r may be accessed 16 bytes at a time
    bool xvec;            // X as plain rows: so may they
    int k;                // X as plain rows: values of a row
};

__device__ __forceinline__ i32x8 widen(const i32x8& v) { return v; }
__device__ __forceinline__ i32x8 widen(const i32x4& v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }  // the instruction reads four registers
// A block's 32 values as bf16 with the scale applied (exact: at most four significant bits), in four groups of eight.
template <int F> __device__ __forceinline__ void decode_block(const typename MxFragment<F>::type& c, float scale, u32x4* out) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float v[8];
        const uint32_t w[2] = {(uint32_t)c[F == 8 ? 2 * q : q], (uint32_t)c[F == 8 ? 2 * q + 1 : q]};
        mx_decode8<F>(w, scale, v);
        out[q] = f32_to_chunk<bf16_t>(v);
    }
}
// Launches the split kernel on tiles of 16 fm rows by 16 fn rows of W; fm, fn = 1 x 1, 1 x 2, 1 x 4, 2 x 2 or 2 x 4 (1 x .. where X is
// plain rows), fn even for GEGLU, whole MX blocks of columns for an MX result.
int dm_mx_split_launch(const MxArgs& p, int x_fmt, int w_fmt, bool exact, int x_src, int fm, int fn, hipStream_t stream);
