// Quantisation to the microscaled (MX) formats and back, and the row norms (RMS / layer norm with the residual's addition)
// that write them.  All of it is bound by HBM: every value is read once, with 16-byte accesses whatever the rows' alignment.
#include "dm_hip.h"
#include "mx.h"

namespace {

constexpr int THREADS = 256;

// Eight consecutive values at p, of which those below `left` exist (the others read as zero).  The conversion from bf16 stands
// in the branch on `left`, so a bf16 load is waited for before the next one is issued; fp32 loads of several groups are in flight together.
template <typename T> __device__ __forceinline__ void load8(const T* p, int left, float* v) {
    constexpr int EPC = ElemTraits<T>::EPC;
    if (left >= 8) {
#pragma unroll
        for (int c = 0; c < 8 / EPC; ++c) chunk_to_f32<T>(load16_any(p + c * EPC), v + c * EPC);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? ElemTraits<T>::load(p + i) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int left, const float* v) {
    constexpr int EPC = ElemTraits<T>::EPC;
    if (left >= 8) {
#pragma unroll
        for (int c = 0; c < 8 / EPC; ++c) store16_any(p + c * EPC, f32_to_chunk<T>(v + c * EPC));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) ElemTraits<T>::store(p + i, v[i]);
    }
}

// ---- quantise / dequantise ------------------------------------------------------------------------------------------
// A lane holds eight values, a quad the 32 of a block.  `gpr` = groups of eight per padded row (a multiple of 16), so a
// quad never straddles rows; a block sweeps UNROLL x 256 consecutive groups with all its loads ahead of the arithmetic (fp32 and
// dequantisation; bf16 rows: one 16-byte load at a time per lane, see load8).  Bound by HBM: 65536 x 1280 bf16 to 4 bits 50 us
// (212 MB, 4.2 TB/s; a large copy reaches 5.1 here), back 32 us (6.6 TB/s, what was just written is still cached); 1003 x 1283 fp32
// 3.2 us, of which 2.5 are the launch.
struct Groups {
    int gpr;
    uint32_t magic;  // ceil(2^32 / gpr)
    double inverse;  // 1 / gpr
    long total;
    // group `first` as (row, group of the row); the estimate is off by one row at most
    __device__ __forceinline__ void split(long first, long& row, int& g) const {
        row = (long)((double)first * inverse);
        long rest = first - row * gpr;
        if (rest < 0) { --row; rest += gpr; }
        if (rest >= gpr) { ++row; rest -= gpr; }
        g = (int)rest;
    }
    // at / gpr for at < gpr + 1024 * UNROLL: multiplied while at * gpr < 2^32 makes that exact
    __device__ __forceinline__ uint32_t rows_in(uint32_t at) const {
        return gpr < 16384 ? __umulhi(at, magic) : (at >= (uint32_t)gpr);
    }
};

template <typename T, int FMT, int UNROLL>
__global__ __launch_bounds__(THREADS) void mx_quantize_kernel(const T* __restrict__ x, long ldx, Groups n, int k,
                                                               unsigned char* __restrict__ codes, long ldc,
                                                               unsigned char* __restrict__ scales, long lds) {
    const long first = (long)blockIdx.x * (THREADS * UNROLL);
    long row0;
    int g0;
    n.split(first, row0, g0);
    float v[UNROLL][8];
    long row[UNROLL];
    int g[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const unsigned at = g0 + u * THREADS + threadIdx.x;
        const unsigned r = n.rows_in(at);
        row[u] = row0 + r;
        g[u] = at - r * n.gpr;
        if (first + u * THREADS + threadIdx.x < n.total) load8<T>(x + row[u] * ldx + g[u] * 8, k - g[u] * 8, v[u]);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
        if (first + u * THREADS + threadIdx.x < n.total)
            mx_store_quad<FMT>(v[u], codes + row[u] * ldc + g[u] * mx_bytes(FMT, 8), scales + row[u] * lds + (g[u] >> 2), threadIdx.x);
}

template <typename T, int FMT, int UNROLL>
__global__ __launch_bounds__(THREADS) void mx_dequantize_kernel(const unsigned char* __restrict__ codes, long ldc,
                                                                 const unsigned char* __restrict__ scales, long lds, Groups n,
                                                                 int k, T* __restrict__ y, long ldy) {
    const long first = (long)blockIdx.x * (THREADS * UNROLL);
    long row0;
    int g0;
    n.split(first, row0, g0);
    uint32_t w[UNROLL][2], s[UNROLL];
    long row[UNROLL];
    int g[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const unsigned at = g0 + u * THREADS + threadIdx.x;
        const unsigned r = n.rows_in(at);
        row[u] = row0 + r;
        g[u] = at - r * n.gpr;
        if (first + u * THREADS + threadIdx.x < n.total) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(codes + row[u] * ldc + g[u] * mx_bytes(FMT, 8));
            if constexpr (FMT == 8) {
                const u32x2 t = *reinterpret_cast<const u32x2*>(p);
                w[u][0] = t[0];
                w[u][1] = t[1];
            } else {
                w[u][0] = p[0];
            }
            s[u] = scales[row[u] * lds + (g[u] >> 2)];
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
        if (first + u * THREADS + threadIdx.x < n.total) {
            float v[8];
            mx_decode8<FMT>(w[u], mx_scale(s[u]), v);
            store8<T>(y + row[u] * ldy + g[u] * 8, k - g[u] * 8, v);
        }
}

// ---- norms ----------------------------------------------------------------------------------------------------------
struct NormArgs {
    const void* x;
    const void* r;  // residual or NULL
    void* h;        // x + r (with r)
    const float* gamma;
    const float* beta;  // layer norm; NULL = none
    void* y;            // T rows, or codes
    unsigned char* ys;  // scales
    long ldx, ldr, ldh, ldy, ldys;
    long rows, first;  // rows of the matrix; row of the launch's first block
    int c, layer;
    float eps;
    double inverse;  // 1 / c
};

// Sum over the TPR threads that share a row, in a fixed order: every one of them gets it.  By DPP and lane swaps (a shuffle
// through LDS takes an order of magnitude longer, and short rows are bound by this chain).  In 64 bits like the threads' own
// sums, which hold any square and add equal terms without drifting; fp32 sums cost a constant row of 1000.1 a mean that is off by 11
// units at 8192 values, and a row of 2^24 values 2.6e-4 of its RMS.
template <int CTRL> __device__ __forceinline__ double dpp_add(double v) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    const u32x2 o = {(uint32_t)__builtin_amdgcn_mov_dpp((int)w[0], CTRL, 0xF, 0xF, true), (uint32_t)__builtin_amdgcn_mov_dpp((int)w[1], CTRL, 0xF, 0xF, true)};
    return v + __builtin_bit_cast(double, o);
}
// v plus the other 16 lanes' of 32 (W = 16) or the other half wave's (W = 32): the swap leaves one half's values in the first word
// of every lane and the other's in the second.
template <int W> __device__ __forceinline__ double swap_add(double v) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    u32x2 a, b;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto t = W == 16 ? __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false) : __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false);
        a[i] = t[0];
        b[i] = t[1];
    }
    return __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b);
}
template <int TPR> __device__ __forceinline__ double row_sum(double v, double* red) {
    v = dpp_add<0xB1>(v);   // quad_perm 1 0 3 2
    v = dpp_add<0x4E>(v);   // quad_perm 2 3 0 1
    v = dpp_add<0x141>(v);  // row_half_mirror: the other quad of eight lanes
    v = dpp_add<0x140>(v);  // row_mirror: the other eight of sixteen
    v = swap_add<16>(v);
    v = swap_add<32>(v);
    if constexpr (TPR > 64) {
        __syncthreads();  // the previous sum has been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v += red[i];
    }
    return v;
}
// Eight values on top of a thread's sum for the mean (layer) or the mean square, in two chains.
__device__ __forceinline__ double add8(double s, const float* v, bool layer) {
    double a = 0., b = 0.;
    if (layer) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) { a += v[i]; b += v[i + 1]; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) { a = fma((double)v[i], (double)v[i], a); b = fma((double)v[i + 1], (double)v[i + 1], b); }
    }
    return s + (a + b);
}
// A mean as two fp32 numbers: v - mean keeps its bits where the row lies far from zero.
struct Mean {
    float high = 0.f, low = 0.f;
    __device__ __forceinline__ Mean() {}
    __device__ __forceinline__ explicit Mean(double m) : high((float)m), low((float)(m - high)) {}
    __device__ __forceinline__ float distance(float v) const { return (v - high) - low; }
};
// Eight values become their distances from the mean (0 from `left` on), whose squares go on top of a thread's sum.
__device__ __forceinline__ double add8_squares(double s, float* v, const Mean& mean, int left) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? mean.distance(v[i]) : 0.f;
    return add8(s, v, false);
}
// eight values of h = x + r, rounded to the storage type (the norm is that of the stored row)
template <typename T> __device__ __forceinline__ void load_h(const NormArgs& p, long row, int at, float* v) {
    load8<T>(static_cast<const T*>(p.x) + row * p.ldx + at, p.c - at, v);
    if (p.r) {
        float r[8];
        load8<T>(static_cast<const T*>(p.r) + row * p.ldr + at, p.c - at, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] += r[i];
            if constexpr (sizeof(T) == 2) v[i] = bf16_to_f32(f32_to_bf16(v[i]));
        }
    }
}
__device__ __forceinline__ void load_affine(const NormArgs& p, int at, float* gamma, float* beta) {
    load8<float>(p.gamma + at, p.c - at, gamma);
    if (p.beta) load8<float>(p.beta + at, p.c - at, beta);
}
// v / sqrt(s), rounded once: the product with the reciprocal is corrected by its remainder.  (The product alone is off by up to
// 1.5 units, for a whole row at once, and values next to a code's border change sides.)  Both sides are scaled by the power of two
// that brings the root next to 1, so that the steps between stay in fp32's normal range for every s.
struct Root {
    float scale, root, inverse;
    bool plain;  // no remainder where the root is 0, infinite or NaN
    __device__ __forceinline__ explicit Root(double s) {
        const int e = ((int)((__builtin_bit_cast(u32x2, s)[1] >> 20) & 2047u) - 1023) >> 1;
        const int by = -min(max(e, -126), 126);
        scale = __uint_as_float((uint32_t)(by + 127) << 23);
        root = sqrtf((float)__builtin_ldexp(s, 2 * by));
        inverse = 1.f / root;
        plain = !(inverse > 0.f && inverse < INFINITY);
    }
    __device__ __forceinline__ float divide(float v) const {
        const float u = v * scale, q = u * inverse;
        return plain ? q : fmaf(fmaf(-q, root, u), inverse, q);
    }
};
template <typename T, int OUT>
__device__ __forceinline__ void norm_store(const NormArgs& p, long row, int at, const float* v, const Root& root, const float* gamma, const float* beta) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = root.divide(v[i]) * gamma[i];
    if (p.beta) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] += beta[i];
    }
    if constexpr (OUT == 0) {
        store8<T>(static_cast<T*>(p.y) + row * p.ldy + at, p.c - at, o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = at + i < p.c ? o[i] : 0.f;
        mx_store_quad<OUT>(o, static_cast<unsigned char*>(p.y) + row * p.ldy + mx_bytes(OUT, at), p.ys + row * p.ldys + (at >> 5), threadIdx.x);
    }
}

// The row stays in registers: TPR threads of NV groups of eight values, so x and the residual are read once, and the layer
// norm's variance is a second sum over registers, not a difference of moments.  Bound by HBM: 16384 x 8192 bf16 with residual to
// e4m3 180 to 199 us (944 MB, 4.7 to 5.2 TB/s; a large copy reaches 5.1), LayerNorm 205 to 208; short ones by the chain load - sum - store:
// 1 x 1280 2.8 us, 1024 x 1280 fp32 6.1 us (21 MB).  Sums in 64 bits cost 65536 x 1280 LayerNorm to e2m1 7 to 9 % (164 us in
// 32), the others at most 3 %.  A wave per row up to 1024 values needs no barrier; longer rows are spread over four, so that no
// lane has more than 64.
template <typename T, int OUT, int TPR, int NV>
__global__ __launch_bounds__(THREADS) void row_norm_kernel(NormArgs p) {
    __shared__ double red[TPR / 64];
    const int t = threadIdx.x % TPR;
    const long row = p.first + (long)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
    if (row >= p.rows) return;  // whole waves; TPR > 64 has one row per block
    const int cp = OUT ? mx_padded(p.c) : p.c;
    float v[NV][8];
#pragma unroll
    for (int n = 0; n < NV; ++n) load_h<T>(p, row, (n * TPR + t) * 8, v[n]);
    // short rows: the scale is on its way while the row is summed; long ones have other rows to wait with
    constexpr bool EARLY = NV <= 2;
    float gamma[EARLY ? NV : 1][8], beta[EARLY ? NV : 1][8];
    if constexpr (EARLY) {
#pragma unroll
        for (int n = 0; n < NV; ++n) load_affine(p, (n * TPR + t) * 8, gamma[n], beta[n]);
    }
    double s = 0.;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int at = (n * TPR + t) * 8;
        if (p.r) store8<T>(static_cast<T*>(p.h) + row * p.ldh + at, p.c - at, v[n]);
        s = add8(s, v[n], p.layer);
    }
    double m = row_sum<TPR>(s, red) * p.inverse;
    if (p.layer) {
        const Mean mean(m);
        s = 0.;
#pragma unroll
        for (int n = 0; n < NV; ++n) s = add8_squares(s, v[n], mean, p.c - (n * TPR + t) * 8);
        m = row_sum<TPR>(s, red) * p.inverse;
    }
    const Root root(m + p.eps);
#pragma unroll
    for (int n = 0; n < NV; ++n)
        if ((n * TPR + t) * 8 < cp) {
            if constexpr (!EARLY) load_affine(p, (n * TPR + t) * 8, gamma[0], beta[0]);
            norm_store<T, OUT>(p, row, (n * TPR + t) * 8, v[n], root, gamma[EARLY ? n : 0], beta[EARLY ? n : 0]);
        }
}

// Rows too long for registers: one block per row sweeps it once per sum and once for the output; the sweeps behind the
// first are served by the caches.  With a residual they read the stored h (each thread what it wrote itself), so h may be x
// or the residual itself here as in the kernel above.  1024 x 32768 bf16 with residual: RMS norm 60 us, LayerNorm 72 (268 MB, 4.5 and 3.7 TB/s).
template <typename T, int OUT> __global__ __launch_bounds__(THREADS) void row_norm_loop_kernel(NormArgs p) {
    __shared__ double red[THREADS / 64];
    const long row = p.first + blockIdx.x;
    const int cp = OUT ? mx_padded(p.c) : p.c;
    const T* stored = p.r ? static_cast<const T*>(p.h) + row * p.ldh : static_cast<const T*>(p.x) + row * p.ldx;
    double s = 0.;
    Mean mean;
    for (int at = threadIdx.x * 8; at < p.c; at += THREADS * 8) {
        float v[8];
        load_h<T>(p, row, at, v);
        if (p.r) store8<T>(static_cast<T*>(p.h) + row * p.ldh + at, p.c - at, v);
        s = add8(s, v, p.layer);
    }
    double m = row_sum<THREADS>(s, red) * p.inverse;
    if (p.layer) {
        mean = Mean(m);
        s = 0.;
        for (int at = threadIdx.x * 8; at < p.c; at += THREADS * 8) {
            float v[8];
            load8<T>(stored + at, p.c - at, v);
            s = add8_squares(s, v, mean, p.c - at);
        }
        m = row_sum<THREADS>(s, red) * p.inverse;
    }
    const Root root(m + p.eps);
    for (int at = threadIdx.x * 8; at < cp; at += THREADS * 8) {
        float v[8];
        load8<T>(stored + at, p.c - at, v);
        float gamma[8], beta[8];
        load_affine(p, at, gamma, beta);
        if (p.layer) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = mean.distance(v[i]);
        }
        norm_store<T, OUT>(p, row, at, v, root, gamma, beta);
    }
}

// A launch holds fewer than 2^32 threads: longer matrices take several.
constexpr long MAX_BLOCKS = 1L << 23;
template <typename T, int OUT, int TPR, int NV> int launch_row_norm(NormArgs p, hipStream_t s) {
    constexpr int ROWS = THREADS / TPR;  // per block
    for (p.first = 0; p.first < p.rows; p.first += MAX_BLOCKS * ROWS) {
        const long blocks = (p.rows - p.first + ROWS - 1) / ROWS;
        const dim3 grid((unsigned)(blocks < MAX_BLOCKS ? blocks : MAX_BLOCKS));
        if constexpr (NV > 0) row_norm_kernel<T, OUT, TPR, NV><<<grid, THREADS, 0, s>>>(p);
        else row_norm_loop_kernel<T, OUT><<<grid, THREADS, 0, s>>>(p);
        if (const int rc = dm_check_launch()) return rc;
    }
    return DM_OK;
}
template <typename T, int OUT> int launch_norm(const NormArgs& p, hipStream_t s) {
    if (p.c <= 512) return launch_row_norm<T, OUT, 64, 1>(p, s);
    if (p.c <= 1024) return launch_row_norm<T, OUT, 64, 2>(p, s);
    if (p.c <= 2048) return launch_row_norm<T, OUT, 256, 1>(p, s);
    if (p.c <= 4096) return launch_row_norm<T, OUT, 256, 2>(p, s);
    if (p.c <= 8192) return launch_row_norm<T, OUT, 256, 4>(p, s);
    if (p.c <= 16384) return launch_row_norm<T, OUT, 256, 8>(p, s);
    return launch_row_norm<T, OUT, 256, 0>(p, s);
}

bool mx_fmt_ok(int fmt) { return fmt == DM_MXFP8 || fmt == DM_MXFP4; }
bool dtype_ok(int dtype) { return dtype == DM_F32 || dtype == DM_BF16; }
// codes / scales of `rows` rows of k values: 0 or an error code
int mx_layout(const void* codes, long ldc, const void* scales, long lds, int k, int fmt) {
    if (!codes || !scales || !mx_fmt_ok(fmt)) return DM_ERR_ARG;
    const int kp = mx_padded(k);
    if (ldc < mx_bytes(fmt, kp) || lds < kp / MX_BLOCK) return DM_ERR_ARG;
    if (!dm_aligned16(codes) || ldc % 16 || (reinterpret_cast<uintptr_t>(scales) & 3u) || lds % 4) return DM_ERR_ALIGN;
    return DM_OK;
}
constexpr int MAX_K = 1 << 24;       // values of a row: 32-bit offsets inside a row
constexpr long MAX_ROWS = 1L << 40;  // products of rows and groups stay inside 64 bits
constexpr long MAX_GROUPS = (1L << 32) - 1024;  // of eight values, a thread each at least: a launch holds fewer than 2^32 threads
Groups groups_of(long rows, int k) {
    Groups n;
    n.gpr = mx_padded(k) / 8;
    n.magic = (uint32_t)((0x100000000ULL + n.gpr - 1) / n.gpr);
    n.inverse = 1.0 / n.gpr;
    n.total = rows * n.gpr;
    return n;
}
// Four groups per thread once that leaves eight blocks per CU; fewer values are spread over more CUs.
int unroll_of(long total) { return total >= 2048L * THREADS * 4 ? 4 : 1; }

}  // namespace

extern "C" int dm_mx_quantize(const void* x, long ldx, long rows, int k, int dtype, int fmt, unsigned char* codes, long ldc,
                              unsigned char* scales, long lds, hipStream_t stream) {
    if (rows < 0 || rows > MAX_ROWS || k < 1 || k > MAX_K || !dtype_ok(dtype) || !mx_fmt_ok(fmt)) return DM_ERR_ARG;
    if (rows == 0) return DM_OK;
    if (!x || ldx < k) return DM_ERR_ARG;
    if (const int rc = mx_layout(codes, ldc, scales, lds, k, fmt)) return rc;
    const Groups n = groups_of(rows, k);
    if (n.total / unroll_of(n.total) > MAX_GROUPS) return DM_ERR_ARG;
    const int unroll = unroll_of(n.total);
    const dim3 grid((unsigned)((n.total + THREADS * unroll - 1) / (THREADS * unroll)));
#define DM_MX_Q(T, F)                                                                                                                   \
    (unroll == 1 ? mx_quantize_kernel<T, F, 1><<<grid, THREADS, 0, stream>>>(static_cast<const T*>(x), ldx, n, k, codes, ldc, scales, lds) \
                 : mx_quantize_kernel<T, F, 4><<<grid, THREADS, 0, stream>>>(static_cast<const T*>(x), ldx, n, k, codes, ldc, scales, lds))
    if (dtype == DM_F32) { if (fmt == DM_MXFP8) DM_MX_Q(float, 8); else DM_MX_Q(float, 4); }
    else { if (fmt == DM_MXFP8) DM_MX_Q(bf16_t, 8); else DM_MX_Q(bf16_t, 4); }
#undef DM_MX_Q
    return dm_check_launch();
}

extern "C" int dm_mx_dequantize(const unsigned char* codes, long ldc, const unsigned char* scales, long lds, long rows, int k, int fmt,
                                void* y, long ldy, int dtype, hipStream_t stream) {
    if (rows < 0 || rows > MAX_ROWS || k < 1 || k > MAX_K || !dtype_ok(dtype) || !mx_fmt_ok(fmt)) return DM_ERR_ARG;
    if (rows == 0) return DM_OK;
    if (!y || ldy < k) return DM_ERR_ARG;
    if (const int rc = mx_layout(codes, ldc, scales, lds, k, fmt)) return rc;
    const Groups n = groups_of(rows, k);
    if (n.total / unroll_of(n.total) > MAX_GROUPS) return DM_ERR_ARG;
    const int unroll = unroll_of(n.total);
    const dim3 grid((unsigned)((n.total + THREADS * unroll - 1) / (THREADS * unroll)));
#define DM_MX_D(T, F)                                                                                                                     \
    (unroll == 1 ? mx_dequantize_kernel<T, F, 1><<<grid, THREADS, 0, stream>>>(codes, ldc, scales, lds, n, k, static_cast<T*>(y), ldy) \
                 : mx_dequantize_kernel<T, F, 4><<<grid, THREADS, 0, stream>>>(codes, ldc, scales, lds, n, k, static_cast<T*>(y), ldy))
    if (dtype == DM_F32) { if (fmt == DM_MXFP8) DM_MX_D(float, 8); else DM_MX_D(float, 4); }
    else { if (fmt == DM_MXFP8) DM_MX_D(bf16_t, 8); else DM_MX_D(bf16_t, 4); }
#undef DM_MX_D
    return dm_check_launch();
}

extern "C" int dm_row_norm(const DmRowNormDesc* d, hipStream_t stream) {
    if (!d || d->rows < 0 || d->rows > MAX_ROWS || d->c < 1 || d->c > MAX_K || !dtype_ok(d->dtype) || (d->kind != DM_NORM_RMS && d->kind != DM_NORM_LAYER) ||
        (d->out_fmt != 0 && !mx_fmt_ok(d->out_fmt)))
        return DM_ERR_ARG;
    if (d->rows == 0) return DM_OK;
    if (!d->x || !d->gamma || !d->y || (d->r == nullptr) != (d->h == nullptr)) return DM_ERR_ARG;
    if (d->ldx < d->c || (d->r && (d->ldr < d->c || d->ldh < d->c))) return DM_ERR_ARG;
    if (d->out_fmt) {
        if (const int rc = mx_layout(d->y, d->ldy, d->y_scales, d->ldys, d->c, d->out_fmt)) return rc;
    } else if (d->ldy < d->c) {
        return DM_ERR_ARG;
    }
    NormArgs p;
    p.x = d->x; p.r = d->r; p.h = d->h; p.gamma = d->gamma; p.beta = d->beta; p.y = d->y; p.ys = d->y_scales;
    p.ldx = d->ldx; p.ldr = d->ldr; p.ldh = d->ldh; p.ldy = d->ldy; p.ldys = d->ldys;
    p.rows = d->rows; p.c = d->c; p.layer = d->kind == DM_NORM_LAYER; p.eps = d->eps;
    p.inverse = 1. / d->c;
#define DM_NORM(T) \
    (d->out_fmt == 0 ? launch_norm<T, 0>(p, stream) : d->out_fmt == DM_MXFP8 ? launch_norm<T, 8>(p, stream) : launch_norm<T, 4>(p, stream))
    return d->dtype == DM_F32 ? DM_NORM(float) : DM_NORM(bf16_t);
#undef DM_NORM
}
