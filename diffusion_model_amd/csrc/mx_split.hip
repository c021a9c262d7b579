// dm_mx_gemm for few output tiles, and for X in plain rows: one block per tile, its k axis divided between the waves.
#include "mx_gemm.h"

namespace {

// Few output tiles: the eight waves of a block share one tile of 16 FM rows by 16 FN rows of W; every eighth k-tile is a wave's, so
// that their reads of a row lie side by side, and the eight partial sums meet in LDS in a fixed order.  Until then nothing is
// shared: each wave keeps a ring of DEPTH k-tiles in LDS of its own and waits for nobody.
// Fragments are not loaded straight to registers: the instruction wants 16 rows in 16 neighbouring lanes, and such a load
// costs a pass per row and quarter wave (measured 61 cycles for 1 KB; 16 x 8192 x 8192 took 11.2 us so, at 14 bytes per cycle and CU
// whatever cache held them).  A request with four or eight lanes to a row does not: 7.6 us through LDS, 36 MB at 4.8 TB/s with the
// launch's 2.5 us in it; 77 x 1280 x 5120 5.4 us against 8.2 (and 14.4 for the 64 x 64 tile).
// x_src: X is an MX matrix, or bf16 / fp32 rows that every block quantises as it reads them, a block of 32 values per lane, to
// the codes that dm_mx_quantize gives.  Loads of plain rows stand behind the requests for W of up to DEPTH k-tiles and are waited for with
// them, so the ring drains at every k-tile: 1 x 1280 x 1280, at most two k-tiles per wave, takes 4.7 us, but 1 x 8192 x 8192 13
// against 6.6 from an MX row, and 1 x 1283 x 1279, whose last block is loaded value by value, 6.6 against 3.6.
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
// A lane's share of a 16-row operand of one instruction (128 values per row, four lanes g to a row), from the row in LDS.  e2m1, or
// EXACT: block g; e4m3: 16 values from 16 g (registers 0-3) and from 64 + 16 g on.  Its scale operand is that of block g either way.
template <int F, bool EXACT> __device__ __forceinline__ typename MxFragment<F>::type lds_fragment16(const unsigned char* base, int row, int g) {
    if constexpr (F == 8) {
        const i32x4 lo = lds_chunk<8, 16>(base, row, EXACT ? 2 * g : g);
        const i32x4 hi = lds_chunk<8, 16>(base, row, EXACT ? 2 * g + 1 : 4 + g);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return lds_chunk<4, 16>(base, row, g);
    }
}
// One k-tile of 16 plain rows -> codes [16][k-tile] and scales (byte `word` * 4 + block of [16][16]) in LDS: lane (row, block)
template <int F, typename T>
__device__ __forceinline__ void quantize_tile16(const T* row, int k, int kt, int lane, unsigned char* codes, unsigned char* scales, int word) {
    const int r = lane >> 2, block = lane & 3, at = kt * MX_PAD + 32 * block;
    float v[32];
    load_values<T, 32>(row + at, k - at, v);
    const uint32_t byte = mx_scale_byte<F>(mx_largest<32>(v));
    uint32_t w[4 * MxCodes<F>::W];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const MxCodes<F> c = mx_encode8<F>(v + 8 * q, byte);
#pragma unroll
        for (int e = 0; e < MxCodes<F>::W; ++e) w[q * MxCodes<F>::W + e] = c.w[e];
    }
#pragma unroll
    for (int c = 0; c < MxCodes<F>::W; ++c)
        *reinterpret_cast<u32x4*>(codes + r * mx_bytes(F, MX_PAD) + swizzle<F, 16>(r, block * MxCodes<F>::W + c) * 16) = u32x4{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
    scales[r * 16 + word * 4 + block] = (unsigned char)byte;
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
template <bool F32> __device__ __forceinline__ void store8(const MxArgs& p, long m, int col, float* v, int lane) {
    if (!F32 && p.c_type != DM_BF16) {
        if (col >= p.n_pad) return;  // whole quads
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = col + e < p.n_out ? v[e] : 0.f;
        unsigned char *codes = static_cast<unsigned char*>(p.c) + m * p.ldc, *scale = p.cs + m * p.ld_cs + (col >> 5);
        if (p.c_type == DM_MXFP8) mx_store_quad<8>(v, codes + col, scale, lane);
        else mx_store_quad<4>(v, codes + (col >> 1), scale, lane);
        return;
    }
    const int left = p.n_out - col;
    if (!F32) {
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

template <int XF, int WF, int FM, int FN> struct SplitRing {
    static constexpr int XB = mx_bytes(XF, MX_PAD), WB = mx_bytes(WF, MX_PAD);
    static constexpr int TILE = 16 * (FM * XB + FN * WB);  // bytes of a k-tile
    static constexpr int DEPTH = SPLIT_WAVES * TILE * 4 <= 128 * 1024 ? 4 : SPLIT_WAVES * TILE * 2 <= 128 * 1024 ? 2 : 1;
    static constexpr int GROUP = 16 * (FM + FN) * 16;  // scales of four k-tiles: [row][16 bytes]; two such buffers
    static constexpr int WAVE = DEPTH * TILE + 2 * GROUP;
    static constexpr int LDS = SPLIT_WAVES * (WAVE > FM * FN * 1024 ? WAVE : FM * FN * 1024);  // the partial sums reuse it
    static constexpr int XN = XB / 64, WN = WB / 64;  // requests per fragment: 8 or 16 rows each
    static_assert(LDS <= 160 * 1024, "LDS of a CU");
};

template <int XF, int WF, bool F32, int XSRC, int FM, int FN>
__global__ __launch_bounds__(64 * SPLIT_WAVES) void mx_split_kernel(MxArgs p) {
    typedef SplitRing<XF, WF, FM, FN> G;
    constexpr bool EXACT = mx_exact(XF, WF, F32);
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, g = lane >> 4, fr = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool geglu = p.epi == DM_EPI_GEGLU;
    const int tile_m = blockIdx.x / p.tiles_n, tile_n = blockIdx.x % p.tiles_n;
    const int m0 = tile_m * 16 * FM, col0 = tile_n * (geglu ? FN * 8 : FN * 16);

    // ---- sources: 16-byte pieces of rows by eight (e4m3) or four lanes, scale words by four.  Rows that do not exist are read
    // from the last one.
    auto x_row = [&](int r) { return (long)min(m0 + r, p.m - 1); };
    auto w_row = [&](int j, int r) {  // GEGLU: fragments 0, 2, .. are values, 1, 3, .. their gates
        return (long)min(col0 + (geglu ? j >> 1 : j) * 16 + r, p.n_out - 1) + (geglu && (j & 1) ? p.n_out : 0);
    };
    const unsigned char *xp[FM][G::XN], *wp[FN][G::WN], *xsp[FM], *wsp[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        if constexpr (XSRC == DM_X_MX) {
#pragma unroll
            for (int e = 0; e < G::XN; ++e) {
                const int r = e * (16 / G::XN) + lane / (G::XB / 16), pos = lane % (G::XB / 16);
                xp[i][e] = p.x + x_row(i * 16 + r) * p.ldx + swizzle<XF, 16>(r, pos) * 16;
            }
            xsp[i] = p.xs + x_row(i * 16 + (lane >> 2)) * p.ld_xs;
        } else {
            xp[i][0] = p.x + x_row(i * 16 + (lane >> 2)) * p.ldx;
        }
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
#pragma unroll
        for (int e = 0; e < G::WN; ++e) {
            const int r = e * (16 / G::WN) + lane / (G::WB / 16), pos = lane % (G::WB / 16);
            wp[j][e] = p.w + w_row(j, r) * p.ldw + swizzle<WF, 16>(r, pos) * 16;
        }
        wsp[j] = p.ws + w_row(j, lane >> 2) * p.ld_ws;
    }
    const int count = (p.nkt - wave + SPLIT_WAVES - 1) / SPLIT_WAVES;  // this wave's k-tiles: wave, wave + 8, ..
    unsigned char* const ring = smem + wave * G::WAVE;
    unsigned char* const groups = ring + G::DEPTH * G::TILE;
    auto request = [&](int s, int slot) {
        const int kt = wave + SPLIT_WAVES * s;
        unsigned char* const group = groups + ((s >> 2) & 1) * G::GROUP;
        if ((s & 3) == 0) {  // scale words of this k-tile and the wave's next three (the last one repeated)
            const int at = 4 * (wave + SPLIT_WAVES * min(s + (lane & 3), count - 1));
#pragma unroll
            for (int j = 0; j < FN; ++j) to_lds4(wsp[j] + at, group + (FM + j) * 256);
            if constexpr (XSRC == DM_X_MX) {
#pragma unroll
                for (int i = 0; i < FM; ++i) to_lds4(xsp[i] + at, group + i * 256);
            }
        }
        unsigned char* const to = ring + slot * G::TILE;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < G::WN; ++e) to_lds16(wp[j][e] + (long)kt * G::WB, to + FM * 16 * G::XB + (j * G::WN + e) * 1024);
        if constexpr (XSRC == DM_X_MX) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int e = 0; e < G::XN; ++e) to_lds16(xp[i][e] + (long)kt * G::XB, to + (i * G::XN + e) * 1024);
        }
    };
    constexpr int LOADS = FN * G::WN + (XSRC == DM_X_MX ? FM * G::XN : 0);  // per k-tile; scale words on top only lengthen a wait

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{};
#pragma unroll
    for (int s = 0; s < G::DEPTH; ++s)
        if (s < count) request(s, s);
    int slot = 0;
    for (int s = 0; s < count; ++s) {
        unsigned char* const at = ring + slot * G::TILE;
        unsigned char* const group = groups + ((s >> 2) & 1) * G::GROUP;
        if constexpr (XSRC != DM_X_MX) {
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                typedef typename std::conditional<XSRC == DM_X_F32, float, bf16_t>::type T;
                quantize_tile16<XF, T>(reinterpret_cast<const T*>(xp[i][0]), p.k, wave + SPLIT_WAVES * s, lane, at + i * 16 * G::XB, group + i * 256, s & 3);
            }
        }
        wait_young<LOADS, G::DEPTH - 1>(count - 1 - s);  // k-tile s has landed; nobody else reads or writes this ring
        typename MxFragment<XF>::type x[FM];
        typename MxFragment<WF>::type w[FN];
        int sx[FM], sw[FN];
        // a lane's scale bytes are those of block g; behind the last block they belong to nothing: 2^-127 for its zero codes
        const int held = wave + SPLIT_WAVES * s < p.nkt - 1 || g < p.last_blocks ? 0xff : 0;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            x[i] = lds_fragment16<XF, EXACT>(at + i * 16 * G::XB, fr, g);
            sx[i] = group[i * 256 + fr * 16 + (s & 3) * 4 + g] & held;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            w[j] = lds_fragment16<WF, EXACT>(at + FM * 16 * G::XB + j * 16 * G::WB, fr, g);
            sw[j] = group[(FM + j) * 256 + fr * 16 + (s & 3) * 4 + g] & held;
        }
        if (s + G::DEPTH < count) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the fragments are in registers: the slot may be refilled
            request(s + G::DEPTH, slot);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) mma16<XF, WF, EXACT>(acc[i][j], x[i], w[j], sx[i], sw[j]);
        if (++slot == G::DEPTH) slot = 0;
    }
    __syncthreads();  // the rings are done with

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
        for (int e = 0; e < 8; ++e) v[e] *= F32 ? gelu_f32(gate[e]) : gelu_exp2_f(gate[e]);
    } else if (p.epi == DM_EPI_QUICKGELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = F32 ? quick_gelu_f32(v[e]) : v[e] / (1.f + __expf(-1.702f * v[e]));
    }
    store8<F32>(p, m0 + row, col, v, threadIdx.x);
}

template <int XF, int WF, bool F32, int XSRC, int FM, int FN> int launch_split(MxArgs p, hipStream_t s) {
    constexpr int LDS = SplitRing<XF, WF, FM, FN>::LDS;
    static_assert(32 * FM * FN <= 64 * SPLIT_WAVES, "one thread per eight columns");
    const int bo = p.epi == DM_EPI_GEGLU ? FN * 8 : FN * 16;
    p.tiles_m = (p.m + 16 * FM - 1) / (16 * FM);
    p.tiles_n = (p.n_pad + bo - 1) / bo;
    if (!mx_grid_ok((long)p.tiles_m * p.tiles_n, 64 * SPLIT_WAVES)) return DM_ERR_ARG;
    static DmLdsAttr attr;
    if (LDS > 64 * 1024)
        if (const int rc = dm_set_lds_attr(reinterpret_cast<const void*>(&mx_split_kernel<XF, WF, F32, XSRC, FM, FN>), attr, LDS)) return rc;
    mx_split_kernel<XF, WF, F32, XSRC, FM, FN><<<dim3((unsigned)(p.tiles_m * p.tiles_n)), 64 * SPLIT_WAVES, LDS, s>>>(p);
    return dm_check_launch();
}

template <int XF, int WF, bool F32, int XSRC> int launch_tile(const MxArgs& p, int fm, int fn, hipStream_t s) {
    if (fm == 1) {
        if (fn == 1) return launch_split<XF, WF, F32, XSRC, 1, 1>(p, s);
        if (fn == 2) return launch_split<XF, WF, F32, XSRC, 1, 2>(p, s);
        if (fn == 4) return launch_split<XF, WF, F32, XSRC, 1, 4>(p, s);
    }
    if constexpr (XSRC == DM_X_MX) {
        if (fm == 2 && fn == 2) return launch_split<XF, WF, F32, XSRC, 2, 2>(p, s);
        if (fm == 2 && fn == 4) return launch_split<XF, WF, F32, XSRC, 2, 4>(p, s);
        if (fm == 4 && fn == 4) return launch_split<XF, WF, F32, XSRC, 4, 4>(p, s);
    }
    return DM_ERR_ARG;
}
template <int XF, int WF, bool F32> int launch_src(const MxArgs& p, int x_src, int fm, int fn, hipStream_t s) {
    if (x_src == DM_X_BF16) return launch_tile<XF, WF, F32, DM_X_BF16>(p, fm, fn, s);
    if (x_src == DM_X_F32) return launch_tile<XF, WF, F32, DM_X_F32>(p, fm, fn, s);
    return launch_tile<XF, WF, F32, DM_X_MX>(p, fm, fn, s);
}
template <int XF, int WF> int launch_result(const MxArgs& p, bool f32, int x_src, int fm, int fn, hipStream_t s) {
    return f32 ? launch_src<XF, WF, true>(p, x_src, fm, fn, s) : launch_src<XF, WF, false>(p, x_src, fm, fn, s);
}

}  // namespace

int dm_mx_split_launch(const MxArgs& p, int x_fmt, int w_fmt, bool f32, int x_src, int fm, int fn, hipStream_t stream) {
    if (x_fmt == DM_MXFP8)
        return w_fmt == DM_MXFP8 ? launch_result<8, 8>(p, f32, x_src, fm, fn, stream) : launch_result<8, 4>(p, f32, x_src, fm, fn, stream);
    return w_fmt == DM_MXFP8 ? launch_result<4, 8>(p, f32, x_src, fm, fn, stream) : launch_result<4, 4>(p, f32, x_src, fm, fn, stream);
}
