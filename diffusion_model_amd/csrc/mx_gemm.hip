// Products of microscaled (MX) matrices on the scaled matrix instructions: C = act(X W^T + bias) + r.
//
// v_mfma_scale_f32_32x32x64 multiplies e4m3 / e2m1 operands as they lie in memory and applies the two operands' block scales
// itself, so a k-tile costs no arithmetic besides the instruction: 4 bits run at twice the rate of 8 bits on either side.
// W is the instruction's first operand, so that a lane holds 16 columns of C for one row; the rows of a 32-row W fragment are
// permuted when they are brought to LDS such that those 16 columns follow each other (and lanes l, l + 32 hold the 32 columns of
// an MX block of C).
#include "dm_hip.h"
#include "mx.h"

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
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
};

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

// ---- one k-tile of a 32-row operand fragment -------------------------------------------------------------------------
// A k-tile is 128 values = blocks 0..3 of a row: 128 bytes (e4m3) or 64 (e2m1), in 16-byte chunks that the XOR below spreads
// over the LDS banks (any eight consecutive rows then occupy eight different 16-byte columns of a 128-byte line).  Instruction
// j = 0, 1 of a k-tile multiplies two blocks, one per lane half g = lane / 32: block 2 g + j, so that a lane's two scale bytes
// are neighbours (one 16-bit read; the instruction selects byte j).  An e2m1 lane holds its whole block; an e4m3 lane holds
// half g of both blocks (registers 0-3: the block of lanes 0-31).
template <int F> __device__ __forceinline__ int swizzle(int row, int chunk) {
    return F == 8 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3);
}
template <int F> __device__ __forceinline__ u32x4 lds_chunk(const unsigned char* base, int row, int chunk) {
    return *reinterpret_cast<const u32x4*>(base + row * mx_bytes(F, MX_PAD) + swizzle<F>(row, chunk) * 16);
}
template <int F> __device__ __forceinline__ i32x8 lds_fragment(const unsigned char* base, int row, int g, int j) {
    u32x4 lo, hi = {0u, 0u, 0u, 0u};
    if constexpr (F == 8) {
        lo = lds_chunk<8>(base, row, 2 * j + g);
        hi = lds_chunk<8>(base, row, 2 * (2 + j) + g);
    } else {
        lo = lds_chunk<4>(base, row, 2 * g + j);
    }
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// The same block, decoded to bf16 with its scale applied (exact: at most four significant bits): 32 values in four chunks.
template <int F> __device__ __forceinline__ void lds_fragment_bf16(const unsigned char* base, int row, int g, int j, float scale, u32x4* out) {
    if constexpr (F == 8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 c = lds_chunk<8>(base, row, 2 * (2 * g + j) + h);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float v[8];
                const uint32_t w[2] = {c[2 * q], c[2 * q + 1]};
                mx_decode8<8>(w, scale, v);
                out[2 * h + q] = f32_to_chunk<bf16_t>(v);
            }
        }
    } else {
        const u32x4 c = lds_chunk<4>(base, row, 2 * g + j);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float v[8];
            const uint32_t w[1] = {c[q]};
            mx_decode8<4>(w, scale, v);
            out[q] = f32_to_chunk<bf16_t>(v);
        }
    }
}
template <int WF, int XF, int J> __device__ __forceinline__ f32x16 mma_scaled(const i32x8& w, const i32x8& x, const f32x16& acc, int sw, int sx) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, acc, WF == 8 ? 0 : 4, XF == 8 ? 0 : 4, J, sw, J, sx);
}

// ---- epilogue --------------------------------------------------------------------------------------------------------
// 16 consecutive columns of row m from column `col` on (values past n_out are zeros already) in the result's type.
__device__ __forceinline__ void store16(const MxArgs& p, long m, int col, float* v, int lane) {
    if (p.c_type == DM_MXFP8 || p.c_type == DM_MXFP4) {
        // lanes l and l + 32 hold the two halves of a block
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, mx_abs_bits(v[i]));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        if (m >= p.m || col >= p.n_pad) return;
        const uint32_t byte = p.c_type == DM_MXFP8 ? mx_scale_byte<8>(top) : mx_scale_byte<4>(top);
        const float inv = mx_inverse_scale(byte);
        if (p.c_type == DM_MXFP8) {
            const MxCodes<8> a = mx_encode8<8>(v, inv, byte != 255u), b = mx_encode8<8>(v + 8, inv, byte != 255u);
            *reinterpret_cast<u32x4*>(static_cast<unsigned char*>(p.c) + m * p.ldc + col) = u32x4{a.w[0], a.w[1], b.w[0], b.w[1]};
        } else {
            const MxCodes<4> a = mx_encode8<4>(v, inv, byte != 255u), b = mx_encode8<4>(v + 8, inv, byte != 255u);
            *reinterpret_cast<u32x2*>(static_cast<unsigned char*>(p.c) + m * p.ldc + (col >> 1)) = u32x2{a.w[0], b.w[0]};
        }
        if (lane < 32) p.cs[m * p.ld_cs + (col >> 5)] = (unsigned char)byte;
        return;
    }
    if (m >= p.m || col >= p.n_out) return;
    const int left = p.n_out - col;
    const bool whole = p.vec && left >= 16;
    if (p.c_type == DM_BF16) {
        bf16_t* dst = static_cast<bf16_t*>(p.c) + m * p.ldc + col;
        const bf16_t* res = static_cast<const bf16_t*>(p.r) + m * p.ldr + col;
        if (whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (p.r) {
                    float f[8];
                    chunk_to_f32<bf16_t>(*reinterpret_cast<const u32x4*>(res + 8 * h), f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[8 * h + i] += f[i];
                }
                *reinterpret_cast<u32x4*>(dst + 8 * h) = f32_to_chunk<bf16_t>(v + 8 * h);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < left) dst[i] = f32_to_bf16(p.r ? v[i] + bf16_to_f32(res[i]) : v[i]);
        }
    } else {
        float* dst = static_cast<float*>(p.c) + m * p.ldc + col;
        const float* res = static_cast<const float*>(p.r) + m * p.ldr + col;
        if (whole) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                f32x4 o = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
                if (p.r) o += *reinterpret_cast<const f32x4*>(res + 4 * h);
                *reinterpret_cast<f32x4*>(dst + 4 * h) = o;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < left) dst[i] = p.r ? v[i] + res[i] : v[i];
        }
    }
}
__device__ __forceinline__ void load_bias16(const MxArgs& p, int at, int left, float* b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = p.bias && i < left ? p.bias[at + i] : 0.f;
}

// ---- tile kernel -----------------------------------------------------------------------------------------------------
// BM rows of X by BN rows of W per block, one WM x WN piece per wave; a ring of STAGES k-tiles in LDS, filled by loads that
// bypass the registers.  EXACT: the operands are decoded to bf16 and multiplied there (see dm_mx_gemm).
template <int XF, int WF, bool EXACT, int BM, int BN, int WM, int WN, int STAGES> struct MxTile {
    static constexpr int XB = mx_bytes(XF, MX_PAD), WB = mx_bytes(WF, MX_PAD);
    static constexpr int WAVES = (BM / WM) * (BN / WN);
    static constexpr int STAGE = BM * XB + BN * WB + (BM + BN) * 4;  // bytes
    static constexpr int NX = BM * XB / 1024, NW = BN * WB / 1024, NS = (BM + BN) / 64;  // requests of a wave's 64 lanes per k-tile
    static constexpr int PX = (NX + WAVES - 1) / WAVES, PW = (NW + WAVES - 1) / WAVES, PS = (NS + WAVES - 1) / WAVES;
    static constexpr int LOADS = PX + PW + PS;  // per wave; where a kind does not divide, waves repeat a request (same bytes)
    static_assert(BM % 64 == 0 && BN % 64 == 0 && WM % 32 == 0 && WN % 32 == 0, "whole requests and fragments");
    static_assert(WN % 64 == 0, "a wave holds both the values and the gates of its columns");
    static_assert((STAGES - 1) * LOADS <= 63, "vmcnt counts to 63");
};

template <int XF, int WF, bool EXACT, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__((64 * MxTile<XF, WF, EXACT, BM, BN, WM, WN, STAGES>::WAVES)) void mx_gemm_kernel(MxArgs p) {
    typedef MxTile<XF, WF, EXACT, BM, BN, WM, WN, STAGES> G;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, g = lane >> 5, fr = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % (BM / WM), wn = wave / (BM / WM);
    const bool geglu = p.epi == DM_EPI_GEGLU;

    const int tile_m = blockIdx.x % p.tiles_m, tile_n = blockIdx.x / p.tiles_m;
    const int m0 = tile_m * BM;
    const int col0 = tile_n * (geglu ? BN / 2 : BN);  // first column of C

    // ---- sources of this wave's requests.  Rows that do not exist are read from row m - 1 / the last row and not stored.
    const unsigned char *xp[G::PX], *wp[G::PW], *sp[G::PS];
    int xd[G::PX], wd[G::PW], sd[G::PS];
    auto w_row = [&](int rho) {  // row of W behind LDS row rho of the tile
        const int f = rho >> 5, i = rho & 31;
        const int col = 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
        const int o = col0 + (geglu ? (f >> 1) : f) * 32 + col;
        return (long)min(o, p.n_out - 1) + (geglu && (f & 1) ? p.n_out : 0);
    };
#pragma unroll
    for (int i = 0; i < G::PX; ++i) {
        const int slot = (wave + i * G::WAVES) % G::NX;
        const int row = slot * (1024 / G::XB) + lane / (G::XB / 16), pos = lane % (G::XB / 16);
        xp[i] = p.x + (long)min(m0 + row, p.m - 1) * p.ldx + swizzle<XF>(row, pos) * 16;
        xd[i] = slot * 1024;
    }
#pragma unroll
    for (int i = 0; i < G::PW; ++i) {
        const int slot = (wave + i * G::WAVES) % G::NW;
        const int row = slot * (1024 / G::WB) + lane / (G::WB / 16), pos = lane % (G::WB / 16);
        wp[i] = p.w + w_row(row) * p.ldw + swizzle<WF>(row, pos) * 16;
        wd[i] = BM * G::XB + slot * 1024;
    }
#pragma unroll
    for (int i = 0; i < G::PS; ++i) {
        const int slot = (wave + i * G::WAVES) % G::NS;
        const int row = slot * 64 + lane;
        sp[i] = row < BM ? p.xs + (long)min(m0 + row, p.m - 1) * p.ld_xs : p.ws + w_row(row - BM) * p.ld_ws;
        sd[i] = BM * G::XB + BN * G::WB + slot * 256;
    }
    auto request = [&](int stage) {
        unsigned char* base = smem + stage * G::STAGE;
#pragma unroll
        for (int i = 0; i < G::PX; ++i) { to_lds16(xp[i], base + xd[i]); xp[i] += G::XB; }
#pragma unroll
        for (int i = 0; i < G::PW; ++i) { to_lds16(wp[i], base + wd[i]); wp[i] += G::WB; }
#pragma unroll
        for (int i = 0; i < G::PS; ++i) { to_lds4(sp[i], base + sd[i]); sp[i] += 4; }
    };

    constexpr int FM = WM / 32, FN = WN / 32;
    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};

#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < p.nkt) request(s);
    int stage = 0;
    for (int kt = 0; kt < p.nkt; ++kt) {
        // k-tile kt has landed once only younger requests are outstanding; behind the barrier it is visible to all waves and
        // all reads of the stage that is refilled next are done
        wait_young<G::LOADS, STAGES - 2>(p.nkt - 1 - kt);
        __builtin_amdgcn_s_barrier();
        if (kt + STAGES - 1 < p.nkt) request(stage == 0 ? STAGES - 1 : stage - 1);
        const unsigned char* xb = smem + stage * G::STAGE;
        const unsigned char* wb = xb + BM * G::XB;
        const unsigned char* sb = wb + BN * G::WB;
        int sx[FM], sw[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) sx[i] = *reinterpret_cast<const uint16_t*>(sb + (wm * WM + i * 32 + fr) * 4 + 2 * g);
#pragma unroll
        for (int j = 0; j < FN; ++j) sw[j] = *reinterpret_cast<const uint16_t*>(sb + (BM + wn * WN + j * 32 + fr) * 4 + 2 * g);
        if constexpr (!EXACT) {
#define MX_HALF(J)                                                                                                              \
    {                                                                                                                           \
        i32x8 xf[FM], wf[FN];                                                                                                   \
        _Pragma("unroll") for (int i = 0; i < FM; ++i) xf[i] = lds_fragment<XF>(xb, wm * WM + i * 32 + fr, g, J);                \
        _Pragma("unroll") for (int j = 0; j < FN; ++j) wf[j] = lds_fragment<WF>(wb, wn * WN + j * 32 + fr, g, J);                \
        _Pragma("unroll") for (int i = 0; i < FM; ++i)                                                                          \
            _Pragma("unroll") for (int j = 0; j < FN; ++j) acc[i][j] = mma_scaled<WF, XF, J>(wf[j], xf[i], acc[i][j], sw[j], sx[i]); \
    }
            MX_HALF(0)
            MX_HALF(1)
#undef MX_HALF
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 xf[FM][4], wf[FN][4];
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    lds_fragment_bf16<XF>(xb, wm * WM + i * 32 + fr, g, h, mx_scale((sx[i] >> (8 * h)) & 255), xf[i]);
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    lds_fragment_bf16<WF>(wb, wn * WN + j * 32 + fr, g, h, mx_scale((sw[j] >> (8 * h)) & 255), wf[j]);
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, wf[j][q]),
                                                                                __builtin_bit_cast(bf16x8, xf[i][q]), acc[i][j], 0, 0, 0);
            }
        }
        if (++stage == STAGES) stage = 0;
    }

    // ---- epilogue: lane holds row m0 + .. + fr, 16 columns per fragment
    if (geglu) {
#pragma unroll
        for (int j = 0; j < FN / 2; ++j) {
            const int col = col0 + wn * (WN / 2) + j * 32 + 16 * g, left = p.n_out - col;
            float bv[16], bg[16];
            load_bias16(p, col, left, bv);
            load_bias16(p, p.n_out + col, left, bg);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float gate = acc[i][2 * j + 1][e] + bg[e];
                    const float o = (acc[i][2 * j][e] + bv[e]) * (p.c_type == DM_F32 ? gelu_erf_f(gate) : gelu_erf_fast_f(gate));
                    v[e] = e < left ? o : 0.f;
                }
                store16(p, m0 + wm * WM + i * 32 + fr, col, v, lane);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int col = col0 + wn * WN + j * 32 + 16 * g, left = p.n_out - col;
            float b[16];
            load_bias16(p, col, left, b);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float o = acc[i][j][e] + b[e];
                    if (p.epi == DM_EPI_QUICKGELU) o = o / (1.f + __expf(-1.702f * o));
                    v[e] = e < left ? o : 0.f;
                }
                store16(p, m0 + wm * WM + i * 32 + fr, col, v, lane);
            }
        }
    }
}

template <int XF, int WF, bool EXACT, int BM, int BN, int WM, int WN, int STAGES> int launch(MxArgs p, hipStream_t s) {
    typedef MxTile<XF, WF, EXACT, BM, BN, WM, WN, STAGES> G;
    constexpr int LDS = STAGES * G::STAGE;
    static DmLdsAttr attr;
    const void* fn = reinterpret_cast<const void*>(&mx_gemm_kernel<XF, WF, EXACT, BM, BN, WM, WN, STAGES>);
    if (LDS > 64 * 1024)
        if (const int rc = dm_set_lds_attr(fn, attr, LDS)) return rc;
    const int bo = p.epi == DM_EPI_GEGLU ? BN / 2 : BN;
    p.tiles_m = (p.m + BM - 1) / BM;
    p.tiles_n = (p.n_pad + bo - 1) / bo;
    if ((long)p.tiles_m * p.tiles_n > 0x7fffffffL) return DM_ERR_ARG;
    mx_gemm_kernel<XF, WF, EXACT, BM, BN, WM, WN, STAGES><<<dim3((unsigned)(p.tiles_m * p.tiles_n)), 64 * G::WAVES, LDS, s>>>(p);
    return dm_check_launch();
}
template <int XF, int WF, bool EXACT> int launch_fmt(const MxArgs& p, hipStream_t s) {
    return launch<XF, WF, EXACT, 64, 64, 32, 64, 3>(p, s);
}
template <int XF, int WF> int launch_type(const MxArgs& p, hipStream_t s) {
    if constexpr (XF == 8 || WF == 8)
        if (p.c_type == DM_F32) return launch_fmt<XF, WF, true>(p, s);
    return launch_fmt<XF, WF, false>(p, s);
}

bool fmt_ok(int fmt) { return fmt == DM_MXFP8 || fmt == DM_MXFP4; }
int operand(const void* codes, long ld, const void* scales, long lds, int kp, int fmt) {
    if (!codes || !scales || ld < mx_bytes(fmt, kp) || lds < kp / MX_BLOCK) return DM_ERR_ARG;
    return dm_aligned16(codes) && ld % 16 == 0 && !(reinterpret_cast<uintptr_t>(scales) & 3u) && lds % 4 == 0 ? DM_OK : DM_ERR_ALIGN;
}

}  // namespace

extern "C" int dm_mx_gemm(const DmMxGemmDesc* d, hipStream_t stream) {
    if (!d || d->m < 0 || d->n < 1 || d->k < 1 || d->k > (1 << 24) || d->n > (1 << 24) || !fmt_ok(d->x_fmt) || !fmt_ok(d->w_fmt)) return DM_ERR_ARG;
    if (d->epi != DM_EPI_PLAIN && d->epi != DM_EPI_GEGLU && d->epi != DM_EPI_QUICKGELU) return DM_ERR_ARG;
    if (d->epi == DM_EPI_GEGLU && d->n % 2) return DM_ERR_ARG;
    if (d->c_type != DM_F32 && d->c_type != DM_BF16 && !fmt_ok(d->c_type)) return DM_ERR_ARG;
    if (d->m == 0) return DM_OK;
    const int kp = mx_padded(d->k);
    if (const int rc = operand(d->x, d->ldx, d->x_scales, d->ld_xs, kp, d->x_fmt)) return rc;
    if (const int rc = operand(d->w, d->ldw, d->w_scales, d->ld_ws, kp, d->w_fmt)) return rc;
    MxArgs p = {};
    p.x = d->x; p.xs = d->x_scales; p.w = d->w; p.ws = d->w_scales;
    p.ldx = d->ldx; p.ld_xs = d->ld_xs; p.ldw = d->ldw; p.ld_ws = d->ld_ws;
    p.m = d->m; p.n_out = d->epi == DM_EPI_GEGLU ? d->n / 2 : d->n; p.n_pad = p.n_out;
    p.nkt = kp / MX_PAD;
    p.bias = d->bias; p.r = d->r; p.ldr = d->ldr; p.c = d->c; p.ldc = d->ldc; p.cs = d->c_scales; p.ld_cs = d->ld_cs;
    p.epi = d->epi; p.c_type = d->c_type;
    if (fmt_ok(d->c_type)) {
        if (d->r) return DM_ERR_ARG;
        p.n_pad = mx_padded(p.n_out);
        if (const int rc = operand(d->c, d->ldc, d->c_scales, d->ld_cs, p.n_pad, d->c_type)) return rc;
    } else {
        const int esz = d->c_type == DM_F32 ? 4 : 2;
        if (!d->c || d->ldc < p.n_out || (d->r && d->ldr < p.n_out)) return DM_ERR_ARG;
        p.vec = dm_aligned16(d->c) && (d->ldc * esz) % 16 == 0 && (!d->r || (dm_aligned16(d->r) && (d->ldr * esz) % 16 == 0));
    }
    if (d->x_fmt == DM_MXFP8) return d->w_fmt == DM_MXFP8 ? launch_type<8, 8>(p, stream) : launch_type<8, 4>(p, stream);
    return d->w_fmt == DM_MXFP8 ? launch_type<4, 8>(p, stream) : launch_type<4, 4>(p, stream);
}
