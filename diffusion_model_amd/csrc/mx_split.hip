// dm_mx_gemm for few output tiles, and for X in plain rows: one block per tile, its k axis divided between the waves.
#include "mx_gemm.h"

namespace {

// ---- split kernel ----------------------------------------------------------------------------------------------------
// Few output tiles: the eight waves of a block share one tile of 16 FM rows by 16 FN rows of W; every eighth k-tile is a wave's, so
// that their reads of a row lie side by side.  Nothing is
// shared before the end, so operands go from memory straight to registers, UNIT k-tiles at once and without a barrier, and the
// eight partial sums meet in LDS in a fixed order.  What bounds it is how many cache lines the loads touch, so it uses the
// 16-row instruction: four lanes read 64 bytes of a row where the 32-row one's two lanes read 32, and the scales of four
// k-tiles come as 16 bytes of a row by its four lanes, which hand them round (16 x 8192 x 8192: x us against y).
// XSRC: 0 = X is an MX matrix, 1 / 2 = X is bf16 / fp32 rows that every block quantises as it reads them, to the codes that
// dm_mx_quantize gives: a block's 32 values are in one lane or in a pair of them.
constexpr int SPLIT_WAVES = 8;

// N values from p on, those at `left` and behind as zeros
template <typename T, int N> __device__ __forceinline__ void load_values(const T* p, int left, float* v) {
    constexpr int EPC = ElemTraits<T>::EPC;
    if (left >= N) {
#pragma unroll
        for (int c = 0; c < N / EPC; ++c) chunk_to_f32<T>(load16_any(p + c * EPC), v + c * EPC);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < left ? ElemTraits<T>::load(p + i) : 0.f;
    }
}
// A lane's share of a 16-row operand of one instruction (128 values per row, four lanes g to a row).  e2m1, or EXACT: block g;
// e4m3: 16 values from 16 g (registers 0-3) and from 64 + 16 g on.  Its scale operand is that of block g either way.
template <int F, bool EXACT> __device__ __forceinline__ typename MxFragment<F>::type load_fragment16(const unsigned char* at, int g) {
    if constexpr (F == 8) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(at + (EXACT ? 32 * g : 16 * g));
        const i32x4 hi = *reinterpret_cast<const i32x4*>(at + (EXACT ? 32 * g + 16 : 64 + 16 * g));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return *reinterpret_cast<const i32x4*>(at + 16 * g);
    }
}
template <int F, bool EXACT, typename T>
__device__ __forceinline__ typename MxFragment<F>::type quantize_fragment16(const T* row, int k, int kt, int lane, int& scale) {
    const int g = lane >> 4;
    typename MxFragment<F>::type out;
    float v[32];
    uint32_t byte[2];
    if constexpr (F == 8 && !EXACT) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {  // half a block each; the other half is in lane l ^ 16
            const int at = kt * MX_PAD + 64 * b + 16 * g;
            load_values<T, 16>(row + at, k - at, v + 16 * b);
            float top = mx_largest<16>(v + 16 * b);
            top = __builtin_elementwise_maximum(top, __shfl_xor(top, 16));
            byte[b] = mx_scale_byte<8>(top);  // of block 2 b + g / 2
        }
        const int from = (lane & 15) + 32 * (g & 1);  // a lane that holds the byte of block g
        const int lo = __shfl((int)byte[0], from), hi = __shfl((int)byte[1], from);
        scale = g < 2 ? lo : hi;
    } else {
        const int at = kt * MX_PAD + 32 * g;
        load_values<T, 32>(row + at, k - at, v);
        byte[0] = byte[1] = mx_scale_byte<F>(mx_largest<32>(v));
        scale = (int)byte[0];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const MxCodes<F> c = mx_encode8<F>(v + 8 * q, byte[q >> 1]);
#pragma unroll
        for (int e = 0; e < MxCodes<F>::W; ++e) out[q * MxCodes<F>::W + e] = (int)c.w[e];
    }
    return out;
}
template <int XF, int WF, bool EXACT>
__device__ __forceinline__ void mma16(f32x4& acc, const typename MxFragment<XF>::type& x, const typename MxFragment<WF>::type& w, int sx, int sw) {
    if constexpr (!EXACT) {
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(w), widen(x), acc, WF == 8 ? 0 : 4, XF == 8 ? 0 : 4, 0, sw, 0, sx);
    } else {
        u32x4 xb[4], wb[4];
        decode_block<XF>(x, mx_scale(sx & 255), xb);
        decode_block<WF>(w, mx_scale(sw & 255), wb);
#pragma unroll
        for (int q = 0; q < 4; ++q) Mma16<bf16_t>::mma(acc, wb[q], xb[q]);
    }
}
// Columns col .. col + 7 of row m; the four lanes of a quad hold the 32 columns of an MX block.
__device__ __forceinline__ void store8(const MxArgs& p, long m, int col, float* v, int lane) {
    if (p.c_type == DM_MXFP8 || p.c_type == DM_MXFP4) {
        if (col >= p.n_pad) return;  // whole quads
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = col + e < p.n_out ? v[e] : 0.f;
        unsigned char *codes = static_cast<unsigned char*>(p.c) + m * p.ldc, *scale = p.cs + m * p.ld_cs + (col >> 5);
        if (p.c_type == DM_MXFP8) mx_store_quad<8>(v, codes + col, scale, lane);
        else mx_store_quad<4>(v, codes + (col >> 1), scale, lane);
        return;
    }
    const int left = p.n_out - col;
    if (p.c_type == DM_BF16) {
        bf16_t* dst = static_cast<bf16_t*>(p.c) + m * p.ldc + col;
        float r[8] = {};
        if (p.r) load_values<bf16_t, 8>(static_cast<const bf16_t*>(p.r) + m * p.ldr + col, left, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
        if (left >= 8) {
            store16_any(dst, f32_to_chunk<bf16_t>(v));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) dst[e] = f32_to_bf16(v[e]);
        }
    } else {
        float* dst = static_cast<float*>(p.c) + m * p.ldc + col;
        float r[8] = {};
        if (p.r) load_values<float, 8>(static_cast<const float*>(p.r) + m * p.ldr + col, left, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
        if (left >= 8) {
            store16_any(dst, f32_to_chunk<float>(v));
            store16_any(dst + 4, f32_to_chunk<float>(v + 4));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) dst[e] = v[e];
        }
    }
}

template <int XF, int WF, bool EXACT, int XSRC, int FM, int FN>
__global__ __launch_bounds__(64 * SPLIT_WAVES) void mx_split_kernel(MxArgs p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, g = lane >> 4, fr = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool geglu = p.epi == DM_EPI_GEGLU;
    constexpr int UNIT = FM * FN <= 2 ? 4 : 2;  // k-tiles whose operands are on their way together
    const int tile_m = blockIdx.x / p.tiles_n, tile_n = blockIdx.x % p.tiles_n;
    const int m0 = tile_m * 16 * FM, col0 = tile_n * (geglu ? FN * 8 : FN * 16);

    // rows that do not exist are read from the last one
    const unsigned char *xrow[FM], *xsrow[FM], *wrow[FN], *wsrow[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const long row = min(m0 + i * 16 + fr, p.m - 1);
        xrow[i] = p.x + row * p.ldx;
        xsrow[i] = XSRC == 0 ? p.xs + row * p.ld_xs : nullptr;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {  // GEGLU: fragments 0, 2, .. are values, 1, 3, .. their gates
        const long row = min(col0 + (geglu ? j >> 1 : j) * 16 + fr, p.n_out - 1) + (geglu && (j & 1) ? p.n_out : 0);
        wrow[j] = p.w + row * p.ldw;
        wsrow[j] = p.ws + row * p.ld_ws;
    }
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{};

    auto process = [&](int kt, auto count) {
        constexpr int N = decltype(count)::value;  // k-tiles kt, kt + 8, .. of this wave
        typename MxFragment<XF>::type x[N][FM];
        typename MxFragment<WF>::type w[N][FN];
        int sx[N][FM], sw[N][FN], sxw[FM], sww[FN];
        // lane g: the four scale bytes of k-tile g (mod N) of its row
        const long sat = 4L * (kt + SPLIT_WAVES * (g % N));
#pragma unroll
        for (int j = 0; j < FN; ++j) sww[j] = *reinterpret_cast<const int*>(wsrow[j] + sat);
#pragma unroll
        for (int i = 0; i < FM; ++i)
            if constexpr (XSRC == 0) sxw[i] = *reinterpret_cast<const int*>(xsrow[i] + sat);
#pragma unroll
        for (int u = 0; u < N; ++u) {
#pragma unroll
            for (int j = 0; j < FN; ++j) w[u][j] = load_fragment16<WF, EXACT>(wrow[j] + (long)(kt + SPLIT_WAVES * u) * mx_bytes(WF, MX_PAD), g);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                if constexpr (XSRC == 0) x[u][i] = load_fragment16<XF, EXACT>(xrow[i] + (long)(kt + SPLIT_WAVES * u) * mx_bytes(XF, MX_PAD), g);
                if constexpr (XSRC == 1) x[u][i] = quantize_fragment16<XF, EXACT>(reinterpret_cast<const bf16_t*>(xrow[i]), p.k, kt + SPLIT_WAVES * u, lane, sx[u][i]);
                if constexpr (XSRC == 2) x[u][i] = quantize_fragment16<XF, EXACT>(reinterpret_cast<const float*>(xrow[i]), p.k, kt + SPLIT_WAVES * u, lane, sx[u][i]);
            }
        }
#pragma unroll
        for (int u = 0; u < N; ++u) {  // byte g of the word that lane u of the row holds
#pragma unroll
            for (int j = 0; j < FN; ++j) sw[u][j] = (N == 1 ? sww[j] : __shfl(sww[j], u * 16 + fr)) >> (8 * g);
#pragma unroll
            for (int i = 0; i < FM; ++i)
                if constexpr (XSRC == 0) sx[u][i] = (N == 1 ? sxw[i] : __shfl(sxw[i], u * 16 + fr)) >> (8 * g);
        }
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) mma16<XF, WF, EXACT>(acc[i][j], x[u][i], w[u][j], sx[u][i], sw[u][j]);
    };
    int kt = wave;
    for (; kt + SPLIT_WAVES * (UNIT - 1) < p.nkt; kt += SPLIT_WAVES * UNIT) process(kt, std::integral_constant<int, UNIT>());
    if constexpr (UNIT == 4)
        if (kt + SPLIT_WAVES < p.nkt) {
            process(kt, std::integral_constant<int, 2>());
            kt += 2 * SPLIT_WAVES;
        }
    if (kt < p.nkt) process(kt, std::integral_constant<int, 1>());

    // ---- partial sums [wave][fragment][lane]; lane (q, m) of a fragment holds columns 4 q .. 4 q + 3 of row m.  A thread then
    // sums eight columns of one row: four threads to 32 columns.
    f32x4* const red = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) red[((wave * FM + i) * FN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    const int per_row = geglu ? FN : FN * 2;  // threads
    const int row = threadIdx.x / per_row, c8 = threadIdx.x % per_row;
    if (row >= 16 * FM || m0 + row >= p.m) return;  // a quad has one row (MX results: FN a multiple of 2, GEGLU 4)
    const int col = col0 + c8 * 8;
    auto total = [&](int frag, int bias_at, float* v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p.bias && col + e < p.n_out ? p.bias[bias_at + e] : 0.f;
#pragma unroll
        for (int s = 0; s < SPLIT_WAVES; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 t = red[((s * FM + row / 16) * FN + frag) * 64 + (2 * (c8 & 1) + h) * 16 + row % 16];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * h + e] += t[e];
            }
    };
    float v[8];
    total(geglu ? 2 * (c8 >> 1) : c8 >> 1, col, v);
    if (geglu) {
        float gate[8];
        total(2 * (c8 >> 1) + 1, p.n_out + col, gate);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= p.c_type == DM_F32 ? gelu_erf_f(gate[e]) : gelu_poly_f(gate[e]);
    } else if (p.epi == DM_EPI_QUICKGELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] / (1.f + __expf(-1.702f * v[e]));
    }
    store8(p, m0 + row, col, v, threadIdx.x);
}

template <int XF, int WF, bool EXACT, int XSRC, int FM, int FN> int launch_split(MxArgs p, hipStream_t s) {
    constexpr int LDS = SPLIT_WAVES * FM * FN * 1024;
    static_assert(32 * FM * FN <= 64 * SPLIT_WAVES && LDS <= 64 * 1024, "one thread per eight columns");
    const int bo = p.epi == DM_EPI_GEGLU ? FN * 8 : FN * 16;
    p.tiles_m = (p.m + 16 * FM - 1) / (16 * FM);
    p.tiles_n = (p.n_pad + bo - 1) / bo;
    if ((long)p.tiles_m * p.tiles_n > 0x7fffffffL) return DM_ERR_ARG;
    mx_split_kernel<XF, WF, EXACT, XSRC, FM, FN><<<dim3((unsigned)(p.tiles_m * p.tiles_n)), 64 * SPLIT_WAVES, LDS, s>>>(p);
    return dm_check_launch();
}

template <int XF, int WF, bool EXACT, int XSRC> int launch_tile(const MxArgs& p, int fm, int fn, hipStream_t s) {
    if (fm == 1) {
        if (fn == 1) return launch_split<XF, WF, EXACT, XSRC, 1, 1>(p, s);
        if (fn == 2) return launch_split<XF, WF, EXACT, XSRC, 1, 2>(p, s);
        if (fn == 4) return launch_split<XF, WF, EXACT, XSRC, 1, 4>(p, s);
    }
    if constexpr (XSRC == DM_X_MX) {
        if (fm == 2 && fn == 2) return launch_split<XF, WF, EXACT, XSRC, 2, 2>(p, s);
        if (fm == 2 && fn == 4) return launch_split<XF, WF, EXACT, XSRC, 2, 4>(p, s);
    }
    return DM_ERR_ARG;
}
template <int XF, int WF, bool EXACT> int launch_src(const MxArgs& p, int x_src, int fm, int fn, hipStream_t s) {
    if (x_src == DM_X_BF16) return launch_tile<XF, WF, EXACT, DM_X_BF16>(p, fm, fn, s);
    if (x_src == DM_X_F32) return launch_tile<XF, WF, EXACT, DM_X_F32>(p, fm, fn, s);
    return launch_tile<XF, WF, EXACT, DM_X_MX>(p, fm, fn, s);
}
template <int XF, int WF> int launch_exact(const MxArgs& p, bool exact, int x_src, int fm, int fn, hipStream_t s) {
    if constexpr (XF == 8 || WF == 8)
        if (exact) return launch_src<XF, WF, true>(p, x_src, fm, fn, s);
    return launch_src<XF, WF, false>(p, x_src, fm, fn, s);
}

}  // namespace

int dm_mx_split_launch(const MxArgs& p, int x_fmt, int w_fmt, bool exact, int x_src, int fm, int fn, hipStream_t stream) {
    if (x_fmt == DM_MXFP8)
        return w_fmt == DM_MXFP8 ? launch_exact<8, 8>(p, exact, x_src, fm, fn, stream) : launch_exact<8, 4>(p, exact, x_src, fm, fn, stream);
    return w_fmt == DM_MXFP8 ? launch_exact<4, 8>(p, exact, x_src, fm, fn, stream) : launch_exact<4, 4>(p, exact, x_src, fm, fn, stream);
}
