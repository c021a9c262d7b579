// Products of microscaled (MX) matrices on the scaled matrix instructions: C = act(X W^T + bias) + r.
//
// v_mfma_scale_f32_32x32x64 multiplies e4m3 / e2m1 operands as they lie in memory and applies the two operands' block scales
// itself, so a k-tile costs no arithmetic besides the instruction: 4 bits run at twice the rate of 8 bits on either side.
// W is the instruction's first operand, so that a lane holds 16 columns of C for one row; the rows of a 32-row W fragment are
// permuted when they are brought to LDS such that those 16 columns follow each other (and lanes l, l + 32 hold the 32 columns of
// an MX block of C).
#include "mx_gemm.h"

namespace {

// ---- one k-tile of a 32-row operand fragment -------------------------------------------------------------------------
// Instruction j = 0, 1 of a k-tile (blocks 0..3 of a row) multiplies two blocks, one per lane half g = lane / 32: block 2 g + j, so
// that a lane's two scale bytes are neighbours (one 16-bit read; the instruction selects byte j).  An e2m1 lane holds its whole
// block; an e4m3 lane holds half g of both blocks (registers 0-3: the block of lanes 0-31).
// EXACT: both formats as the plain block 2 g + j, for products in bf16.
template <int F, bool EXACT> __device__ __forceinline__ typename MxFragment<F>::type lds_fragment(const unsigned char* base, int row, int g, int j) {
    if constexpr (F == 8) {
        const i32x4 lo = lds_chunk<8, 32>(base, row, EXACT ? 2 * (2 * g + j) : 2 * j + g);
        const i32x4 hi = lds_chunk<8, 32>(base, row, EXACT ? 2 * (2 * g + j) + 1 : 2 * (2 + j) + g);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return lds_chunk<4, 32>(base, row, 2 * g + j);
    }
}
// Half J of a k-tile: one X fragment with every W fragment.
template <int XF, int WF, bool EXACT, int J, int FN>
__device__ __forceinline__ void mma_row(f32x16 (&acc)[FN], const typename MxFragment<XF>::type& x, const typename MxFragment<WF>::type (&w)[FN],
                                        int sx, const int (&sw)[FN]) {
    if constexpr (!EXACT) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(w[j]), widen(x), acc[j], WF == 8 ? 0 : 4, XF == 8 ? 0 : 4, J, sw[j], J, sx);
    } else {
        u32x4 xb[4];
        decode_block<XF>(x, mx_scale((sx >> (8 * J)) & 255), xb);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            u32x4 wb[4];
            decode_block<WF>(w[j], mx_scale((sw[j] >> (8 * J)) & 255), wb);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, wb[q]), __builtin_bit_cast(bf16x8, xb[q]), acc[j], 0, 0, 0);
        }
    }
}

// ---- epilogue --------------------------------------------------------------------------------------------------------
// 16 consecutive columns of row m from column `col` on, in the result's type CT; `edge`: some of the block's are past n_out.
template <int CT> __device__ __forceinline__ void store16(const MxArgs& p, long m, int col, float* v, int lane, bool edge) {
    if constexpr (CT == DM_MXFP8 || CT == DM_MXFP4) {
        if (edge) {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = col + e < p.n_out ? v[e] : 0.f;
        }
        // lanes l and l + 32 hold the two halves of a block
        float top = mx_largest<16>(v);
        top = __builtin_elementwise_maximum(top, __shfl_xor(top, 32));
        if (m >= p.m || col >= p.n_pad) return;
        const uint32_t byte = mx_scale_byte<CT>(top);
        const MxCodes<CT> a = mx_encode8<CT>(v, byte), b = mx_encode8<CT>(v + 8, byte);
        unsigned char* dst = static_cast<unsigned char*>(p.c) + m * p.ldc + mx_bytes(CT, col);
        if constexpr (CT == DM_MXFP8) *reinterpret_cast<u32x4*>(dst) = u32x4{a.w[0], a.w[1], b.w[0], b.w[1]};
        else *reinterpret_cast<u32x2*>(dst) = u32x2{a.w[0], b.w[0]};
        if (lane < 32) p.cs[m * p.ld_cs + (col >> 5)] = (unsigned char)byte;
    } else {
        typedef typename std::conditional<CT == DM_F32, float, bf16_t>::type T;
        constexpr int EPC = ElemTraits<T>::EPC;
        if (m >= p.m || col >= p.n_out) return;
        T* dst = static_cast<T*>(p.c) + m * p.ldc + col;
        const T* res = static_cast<const T*>(p.r) + m * p.ldr + col;
        const int left = p.n_out - col;
        if (!edge || left >= 16) {
#pragma unroll
            for (int h = 0; h < 16 / EPC; ++h) {
                if (p.r) {
                    float f[EPC];
                    chunk_to_f32<T>(load16_any(res + EPC * h), f);
#pragma unroll
                    for (int i = 0; i < EPC; ++i) v[EPC * h + i] += f[i];
                }
                store16_any(dst + EPC * h, f32_to_chunk<T>(v + EPC * h));
            }
        } else {
            for (int i = 0; i < 16; ++i)
                if (i < left) ElemTraits<T>::store(dst + i, p.r ? v[i] + ElemTraits<T>::load(res + i) : v[i]);
        }
    }
}
// A wave's fragments.  One instance per activation and type: with the choices inside, every fragment's code holds all of them
// and the instruction cache (64 KB for two CUs) sees the epilogue anew with each tile.
template <int EPI, int CT, int FM, int FN, typename Row, typename Column>
__device__ __forceinline__ void store_fragments(const MxArgs& p, const f32x16 (&acc)[FM][FN], Row row, Column column, int lane, bool edge) {
    constexpr int STEP = EPI == DM_EPI_GEGLU ? 2 : 1;
#pragma unroll
    for (int j = 0; j < FN; j += STEP)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float o = acc[i][j][e];
                if constexpr (EPI == DM_EPI_GEGLU) {
                    const float gate = acc[i][j + STEP - 1][e];
                    v[e] = o * (CT == DM_F32 ? gelu_f32(gate) : gelu_exp2_f(gate));
                } else if constexpr (EPI == DM_EPI_QUICKGELU) {
                    v[e] = CT == DM_F32 ? quick_gelu_f32(o) : o / (1.f + __expf(-1.702f * o));
                } else {
                    v[e] = o;
                }
            }
            store16<CT>(p, row(i), column(j), v, lane, edge);
        }
}
template <int EPI, bool F32, int FM, int FN, typename Row, typename Column>
__device__ __forceinline__ void store_typed(const MxArgs& p, const f32x16 (&acc)[FM][FN], Row row, Column column, int lane, bool edge) {
    if constexpr (F32) store_fragments<EPI, DM_F32>(p, acc, row, column, lane, edge);
    else if (p.c_type == DM_BF16) store_fragments<EPI, DM_BF16>(p, acc, row, column, lane, edge);
    else if (p.c_type == DM_MXFP8) store_fragments<EPI, DM_MXFP8>(p, acc, row, column, lane, edge);
    else store_fragments<EPI, DM_MXFP4>(p, acc, row, column, lane, edge);
}

// ---- tile kernel -----------------------------------------------------------------------------------------------------
// BM rows of X by BN rows of W per block, one WM x WN piece per wave; a ring of STAGES k-tiles in LDS, filled by loads that
// bypass the registers.  EXACT: the operands are decoded to bf16 and multiplied there (see dm_mx_gemm).
//
// Scales would cost a request as many cache lines as it has lanes if they were fetched per k-tile (four bytes of every row; measured
// at 8192^3, 4 bits: a fifth of the kernel's time).  They are fetched for a group of four k-tiles, 16 bytes of a row, a
// quarter of the tile's rows with every k-tile: "quarter" q = 4 group + c is requested with k-tile q - 3 and is used with k-tile 4
// group at the earliest, when every request up to that k-tile's has landed.
template <int XF, int WF, bool F32, int BM, int BN, int WM, int WN, int STAGES> struct MxTile {
    static constexpr int XB = mx_bytes(XF, MX_PAD), WB = mx_bytes(WF, MX_PAD);
    static constexpr int WAVES = (BM / WM) * (BN / WN);
    static constexpr int STAGE = BM * XB + BN * WB;  // bytes
    // A group's first quarter is requested STAGES + 3 k-tiles ahead of the group; with two stages the group two before it has
    // been read by then, with more the third before it.
    static constexpr int GROUPS = STAGES > 2 ? 3 : 2, GROUP = (BM + BN) * 16;
    static constexpr int LDS = STAGES * STAGE + GROUPS * GROUP;
    static constexpr int PX = BM * XB / 1024 / WAVES, PW = BN * WB / 1024 / WAVES;  // requests of a wave's 64 lanes per k-tile
    static constexpr int LOADS = PX + PW + 1;
    static constexpr int BLOCKS = 160 * 1024 / LDS >= 2 ? 2 : 1;  // per CU, by LDS: leave registers for as many
    static_assert(BM % 64 == 0 && BN % 64 == 0 && WM % 32 == 0 && WN % 32 == 0, "whole requests and fragments");
    static_assert(PX * WAVES * 1024 == BM * XB && PW * WAVES * 1024 == BN * WB && (BM + BN) / 64 <= WAVES, "every wave requests the same");
    static_assert(WN % 64 == 0, "a wave holds both the values and the gates of its columns");
    static_assert((STAGES - 1) * LOADS <= 63 && (STAGES == 2 || STAGES == 3), "vmcnt counts to 63; the tail of the k loop");
};

template <int XF, int WF, bool F32, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__((64 * MxTile<XF, WF, F32, BM, BN, WM, WN, STAGES>::WAVES), (MxTile<XF, WF, F32, BM, BN, WM, WN, STAGES>::WAVES * MxTile<XF, WF, F32, BM, BN, WM, WN, STAGES>::BLOCKS + 3) / 4) void mx_gemm_kernel(MxArgs p) {
    typedef MxTile<XF, WF, F32, BM, BN, WM, WN, STAGES> G;
    constexpr bool EXACT = mx_exact(XF, WF, F32);
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, g = lane >> 5, fr = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % (BM / WM), wn = wave / (BM / WM);
    const bool geglu = p.epi == DM_EPI_GEGLU;

    // Blocks go to the 8 XCDs in turn and each XCD has its own L2: give an XCD a run of neighbouring tiles, walked down
    // GROUP_M tile rows before the next tile column, so that its 32 CUs share a patch of 8 x 4 tiles' operands.
    int tile_m, tile_n;
    {
        constexpr int XCDS = 8, GROUP_M = 8;
        const int nb = gridDim.x, xcd = blockIdx.x % XCDS, per = nb / XCDS, more = nb % XCDS;
        const int t = xcd * per + min(xcd, more) + blockIdx.x / XCDS;
        const int in_group = GROUP_M * p.tiles_n, group = t / in_group, rest = t - group * in_group;
        const int rows = min(GROUP_M, p.tiles_m - group * GROUP_M);
        tile_m = group * GROUP_M + rest % rows;
        tile_n = rest / rows;
    }
    const int m0 = tile_m * BM;
    const int col0 = tile_n * (geglu ? BN / 2 : BN);  // first column of C

    // ---- sources of this wave's requests: a scalar base that moves on by a k-tile, and each lane's offset from it.  A request
    // lies inside one 32-row W fragment, so values and gates have bases of their own and no offset spans the matrix.  Rows
    // that do not exist are read from the last one and their products not stored.
    const unsigned char* xbase = p.x + (long)m0 * p.ldx;
    const int first = min(col0, p.n_out - 1);  // col0 can lie in the padding of an MX result
    const unsigned char* wbase = p.w + (long)first * p.ldw;
    const long gate_bytes = geglu ? p.n_out * p.ldw : 0;
    const int rows_left = p.m - 1 - m0, cols_left = p.n_out - 1 - first;
    uint32_t xo[G::PX], wo[G::PW];
    auto w_col = [&](int rho) {  // column of the tile behind LDS row rho
        const int f = rho >> 5, i = rho & 31;
        return (geglu ? f >> 1 : f) * 32 + 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
    };
    auto gate = [&](int rho) { return geglu && ((rho >> 5) & 1); };
#pragma unroll
    for (int i = 0; i < G::PX; ++i) {
        const int row = (wave + i * G::WAVES) * (1024 / G::XB) + lane / (G::XB / 16), pos = lane % (G::XB / 16);
        xo[i] = (uint32_t)min(row, rows_left) * (uint32_t)p.ldx + swizzle<XF, 32>(row, pos) * 16;
    }
#pragma unroll
    for (int i = 0; i < G::PW; ++i) {
        const int row = (wave + i * G::WAVES) * (1024 / G::WB) + lane / (G::WB / 16), pos = lane % (G::WB / 16);
        wo[i] = (uint32_t)min(w_col(row), cols_left) * (uint32_t)p.ldw + swizzle<WF, 32>(row, pos) * 16;
    }
    // scalar base + 32-bit lane offset in every request: hidden from the optimiser, which would make each a 64-bit address of its
    // own, carried and advanced in two more registers
    auto lane_offset = [](uint32_t o) { asm volatile("" : "+v"(o)); return o; };
    // requests [from, to) of a k-tile's; the last one moves the sources on
    constexpr int REQUESTS = G::PX + G::PW;
    auto request = [&](int stage, int from, int to) {
        unsigned char* base = smem + stage * G::STAGE;
#pragma unroll
        for (int i = 0; i < G::PX; ++i)
            if (i >= from && i < to) to_lds16(xbase + lane_offset(xo[i]), base + (wave + i * G::WAVES) * 1024);
#pragma unroll
        for (int i = 0; i < G::PW; ++i) {
            const int slot = wave + i * G::WAVES;
            if (G::PX + i >= from && G::PX + i < to) to_lds16(wbase + (gate(slot * (1024 / G::WB)) ? gate_bytes : 0) + lane_offset(wo[i]), base + BM * G::XB + slot * 1024);
        }
        if (to == REQUESTS) {
            xbase += G::XB;
            wbase += G::WB;
        }
    };

    // quarter q = 4 group + c: of every wave's 64 rows of X or of W those that are c modulo 4, four lanes per row (waves past the
    // last rows repeat others').  So a lane's row moves on by one with c, within its 32-row fragment and in W's permuted order as
    // well, and one address per lane does for all four.  The rows lie in the group's buffer as they come, [row / 64][c][row / 4]
    // [16 bytes], word w of a row at w ^ c: the same word of 32 rows fills the 32 banks then (with the words in order: 4 passes).
    // Computed without a branch or an indexed register: the loop below is one block.
    unsigned char* const scales = smem + STAGES * G::STAGE;
    const int taker = wave % ((BM + BN) / 64);
    const bool take_x = taker * 64 < BM;
    const uint32_t take_ld = (uint32_t)(take_x ? p.ld_xs : p.ld_ws);
    const unsigned char* take;
    uint32_t take_span;  // bytes to the last of the next three rows that exists: below 2^26, whatever the matrix spans
    {
        const int row0 = taker * 64 + (lane & ~3), left = take_x ? rows_left : cols_left;
        const int row = min(take_x ? row0 : w_col(row0 - BM), left);
        take = take_x ? p.xs + m0 * p.ld_xs : p.ws + (first + (gate(row0 - BM) ? p.n_out : 0)) * p.ld_ws;
        take += row * (long)take_ld;
        take_span = (uint32_t)min(left - row, 3) * take_ld;
    }
    int quarter = 0, fill = 0;  // next quarter to request and its group's buffer
    const int last_kt = p.nkt - 1;
    auto request_scales = [&]() {
        const int c = quarter & 3;
        const uint32_t at = 4 * min((quarter & ~3) + ((lane & 3) ^ c), last_kt);  // quarters behind the last k-tile repeat it, unread
        to_lds4(take + min(c * take_ld, take_span) + at, scales + fill * G::GROUP + taker * 1024 + c * 256);
        if ((++quarter & 3) == 0) fill = fill + 1 == G::GROUPS ? 0 : fill + 1;
    };

    constexpr int FM = WM / 32, FN = WN / 32;
    // a lane's 16 columns of W fragment j begin at `col`; the sums start from the bias
    f32x16 acc[FM][FN];
    auto column = [&](int j) { return geglu ? col0 + wn * (WN / 2) + (j >> 1) * 32 + 16 * g : col0 + wn * WN + j * 32 + 16 * g; };
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        f32x16 b = {};
        if (p.bias) {
            const int col = column(j), left = p.n_out - col;
            const float* src = p.bias + (geglu && (j & 1) ? p.n_out : 0) + col;
            if (col0 + (geglu ? BN / 2 : BN) <= p.n_out) {
#pragma unroll
                for (int e = 0; e < 16; ++e) b[e] = src[e];
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) b[e] = e < left ? src[e] : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[i][j] = b;
    }

    // ---- k loop.  A k-tile is two halves of FM x FN matrix instructions.  X fragment i of the next half is read from LDS as
    // soon as the instructions on X fragment i of this one have been issued; W fragments, which all of them use, have two sets.
    // The wait and the barrier for the next k-tile stand behind the first instructions of the second half: every wave has read
    // all of this k-tile by then, so its stage is refilled, a few requests behind each row of instructions (all at once they
    // cost 8192^3 2 to 4 %: both waves of a SIMD issue them at the same time, and the matrix pipe waits).
    typename MxFragment<XF>::type x[FM];
    typename MxFragment<WF>::type w[2][FN];
    int sx[FM], sw[FN], sx_next[FM], sw_next[FN];
    const int xrow = wm * WM + fr, wrow = wn * WN + fr;
    auto read_x = [&](int stage, int half, int i) { x[i] = lds_fragment<XF, EXACT>(smem + stage * G::STAGE, xrow + i * 32, g, half); };
    auto read_w = [&](int stage, int half) {
#pragma unroll
        for (int j = 0; j < FN; ++j) w[half][j] = lds_fragment<WF, EXACT>(smem + stage * G::STAGE + BM * G::XB, wrow + j * 32, g, half);
    };
    int next = 0, drain = 0;  // k-tile whose scales are read next and its group's buffer
    auto read_scales = [&]() {
        const unsigned char* sb = scales + drain * G::GROUP + (fr & 3) * 256 + (fr >> 2) * 16 + ((next ^ fr) & 3) * 4 + 2 * g;
        auto fragment = [&](int f) { return *reinterpret_cast<const uint16_t*>(sb + (f >> 1) * 1024 + (f & 1) * 128); };
#pragma unroll
        for (int i = 0; i < FM; ++i) sx_next[i] = fragment(wm * FM + i);
#pragma unroll
        for (int j = 0; j < FN; ++j) sw_next[j] = fragment(BM / 32 + wn * FN + j);
        if ((++next & 3) == 0) drain = drain + 1 == G::GROUPS ? 0 : drain + 1;
    };

    for (int q = 0; q < STAGES + 3; ++q) request_scales();
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
        if (s < p.nkt) request(s, 0, REQUESTS);
    wait_young<G::LOADS - 1, STAGES - 1>(p.nkt - 1);
    __builtin_amdgcn_s_barrier();
    read_scales();
    read_w(0, 0);
#pragma unroll
    for (int i = 0; i < FM; ++i) read_x(0, 0, i);
    int stage = 0;
    // LEFT: k-tiles behind this one that have been requested, STAGES - 1 at most; MORE: one more is requested into this one's
    // stage.  Both are constants and the body has no branch, so the order below is the order of issue.
    auto k_tile = [&](auto left, auto more) {
        constexpr int LEFT = decltype(left)::value;
        constexpr bool MORE = decltype(more)::value;
        const int here = stage;
        if (++stage == STAGES) stage = 0;
        // scale bytes behind the last block belong to nothing: 2^-127 for their zero codes
        const int blocks = LEFT > 0 ? 2 : p.last_blocks - 2 * g, held = blocks >= 2 ? 0xffff : blocks == 1 ? 0xff : 0;
#pragma unroll
        for (int i = 0; i < FM; ++i) sx[i] = LEFT > 0 ? sx_next[i] : sx_next[i] & held;
#pragma unroll
        for (int j = 0; j < FN; ++j) sw[j] = LEFT > 0 ? sw_next[j] : sw_next[j] & held;
        read_w(here, 1);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            mma_row<XF, WF, EXACT, 0>(acc[i], x[i], w[0], sx[i], sw);
            read_x(here, 1, i);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            mma_row<XF, WF, EXACT, 1>(acc[i], x[i], w[1], sx[i], sw);
            if constexpr (LEFT > 0) {
                if (i == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    wait_vm<(LEFT - 1) * (G::LOADS - 1)>();  // requests of scales among the younger ones only make it wait for more
                    __builtin_amdgcn_s_barrier();
                    read_scales();
                    read_w(stage, 0);
                }
                read_x(stage, 0, i);
                if constexpr (MORE) {
                    request(here, i * REQUESTS / FM, (i + 1) * REQUESTS / FM);
                    if (i == FM - 1) request_scales();
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int left = p.nkt - 1;
    for (; left >= STAGES; --left) k_tile(std::integral_constant<int, STAGES - 1>(), std::true_type());
    if constexpr (STAGES > 2)
        if (left >= 2) { k_tile(std::integral_constant<int, 2>(), std::false_type()); --left; }
    if (left >= 1) k_tile(std::integral_constant<int, 1>(), std::false_type());
    k_tile(std::integral_constant<int, 0>(), std::false_type());

    // ---- epilogue: a lane holds row .. + fr and 16 columns per fragment
    const bool edge = col0 + (geglu ? BN / 2 : BN) > p.n_out;
    auto row = [&](int i) { return (long)(m0 + wm * WM + i * 32 + fr); };
    if (geglu) store_typed<DM_EPI_GEGLU, F32>(p, acc, row, column, lane, edge);
    else if (p.epi == DM_EPI_QUICKGELU) store_typed<DM_EPI_QUICKGELU, F32>(p, acc, row, column, lane, edge);
    else store_typed<DM_EPI_PLAIN, F32>(p, acc, row, column, lane, edge);
}

template <int XF, int WF, bool F32, int BM, int BN, int WM, int WN, int STAGES> int launch(MxArgs p, hipStream_t s) {
    typedef MxTile<XF, WF, F32, BM, BN, WM, WN, STAGES> G;
    constexpr int LDS = G::LDS;
    const int bo = p.epi == DM_EPI_GEGLU ? BN / 2 : BN;
    p.tiles_m = (p.m + BM - 1) / BM;
    p.tiles_n = (p.n_pad + bo - 1) / bo;
    if (!mx_grid_ok((long)p.tiles_m * p.tiles_n, 64 * G::WAVES)) return DM_ERR_ARG;
    static DmLdsAttr attr;
    const void* fn = reinterpret_cast<const void*>(&mx_gemm_kernel<XF, WF, F32, BM, BN, WM, WN, STAGES>);
    if (LDS > 64 * 1024)
        if (const int rc = dm_set_lds_attr(fn, attr, LDS)) return rc;
    mx_gemm_kernel<XF, WF, F32, BM, BN, WM, WN, STAGES><<<dim3((unsigned)(p.tiles_m * p.tiles_n)), 64 * G::WAVES, LDS, s>>>(p);
    return dm_check_launch();
}
// Which tile, by measurement on a warm card (e4m3 x e2m1 and a bf16 result where nothing else is said):
//   256 x 256  one block per CU.  Where its rounds over the 256 CUs are full and k is long: 8192^3 in 279 us against 342 for
//              the next (4 bits), 386 against 424 (e4m3 x e2m1); 16384 x 5120 x 5120: 313 against 342
//   128 x 256  two blocks per CU, so that one's epilogue runs beside the other's k loop; W in 4 bits only, whose four
//              fragments per wave fit the 128 registers that leaves (16384 x 5120 x 320: 50 us against 54 for 256 x 256 and 54 for
//              128 x 128; 65536 x 2560 x 320 with GEGLU: 93, 103, 101; at k = 1280 it is level with 256 x 256: 65536 x 2560 233 and 232,
//              16384 x 5120 108 and 105)
//   128 x 128  two blocks per CU, once there is one for each (4096 x 1280 x 1280: 12.2 us against 12.4 for 64 x 64; x 5120: 32.4
//              against 38.8)
//   64 x 64    the rest (1024 x 1280 x 1280: 7.2 us against 7.6; x 5120: 18.8 against 28.3; a short k is the exception, 512 x 1280 x 320
//              4.9 to 6.0 against 4.8)
template <int XF, int WF, bool F32> int launch_fmt(const MxArgs& p, hipStream_t s) {
    const int wide = p.epi == DM_EPI_GEGLU ? 2 * p.n_pad : p.n_pad;
    auto tiles = [&](int bm, int bn) { return (long)((p.m + bm - 1) / bm) * ((wide + bn - 1) / bn); };
    if constexpr (!mx_exact(XF, WF, F32)) {
        const long t256 = tiles(256, 256), rounds = (t256 + 255) / 256;
        if (t256 * 5 >= rounds * 256 * 4 && (WF == 8 || p.nkt >= 32))
            return launch<XF, WF, F32, 256, 256, 128, 64, XF == 4 && WF == 4 ? 3 : 2>(p, s);
        if constexpr (WF == 4)
            if (tiles(128, 256) >= 512) return launch<XF, WF, F32, 128, 256, 32, 128, 2>(p, s);
    }
    if (tiles(128, 128) >= 256) return launch<XF, WF, F32, 128, 128, 64, 64, 2>(p, s);
    return launch<XF, WF, F32, 64, 64, 32, 64, 2>(p, s);
}
template <int XF, int WF> int launch_tile(const MxArgs& p, bool f32, hipStream_t s) {
    return f32 ? launch_fmt<XF, WF, true>(p, s) : launch_fmt<XF, WF, false>(p, s);
}
// The split kernel's tile: the smallest that needs at most one block per CU, since blocks read their operands anew
// (77 x 1280 x 5120: 7.7 us in 400 blocks, 5.4 in 200, the 64 x 64 tile 14.4; 128 x 8192 x 8192 with the largest 17.3 against 31.2;
// 256 x 8192 x 8192 in 512 of those 32.2 against 32.2, 1024 x 1280 x 5120 in 320 of them 23 against 18.8).  The largest is slower than
// the 64 x 64 tile on a short k (512 x 1280 x 1280: 6.0 us against 5.8; x 5120: 9.8 against 14.6).  Up to 16 rows a tile of 16 x 64 is
// taken at any size: W is read once then, and that is all there is to do.
bool split_tile(const MxArgs& p, int* fm, int* fn) {
    static const int shapes[][2] = {{1, 1}, {1, 2}, {2, 2}, {1, 4}, {2, 4}, {4, 4}};
    const bool geglu = p.epi == DM_EPI_GEGLU, mx = p.c_type == DM_MXFP8 || p.c_type == DM_MXFP4;
    for (const auto& t : shapes) {
        const int cols = geglu ? t[1] * 8 : t[1] * 16;
        if ((geglu && t[1] % 2) || (mx && cols % MX_BLOCK) || (t[0] > 1 && p.m <= 16) || (t[0] == 4 && p.nkt < 16)) continue;
        const long blocks = (long)((p.m + 16 * t[0] - 1) / (16 * t[0])) * ((p.n_pad + cols - 1) / cols);
        if (blocks <= 256 || (p.m <= 16 && t[1] == 4)) {
            *fm = t[0];
            *fn = t[1];
            return true;
        }
    }
    return false;
}

constexpr long MAX_LD = 1L << 24;  // bytes of a row: 32-bit offsets inside the rows of a tile
bool fmt_ok(int fmt) { return fmt == DM_MXFP8 || fmt == DM_MXFP4; }
int operand(const void* codes, long ld, const void* scales, long lds, int kp, int fmt) {
    if (!codes || !scales || ld < mx_bytes(fmt, kp) || lds < kp / MX_BLOCK) return DM_ERR_ARG;
    if (ld > MAX_LD || lds > MAX_LD) return DM_ERR_ARG;
    return dm_aligned16(codes) && ld % 16 == 0 && !(reinterpret_cast<uintptr_t>(scales) & 3u) && lds % 4 == 0 ? DM_OK : DM_ERR_ALIGN;
}

}  // namespace

extern "C" int dm_mx_gemm(const DmMxGemmDesc* d, hipStream_t stream) {
    if (!d || d->m < 0 || d->m > (1 << 30) || d->n < 1 || d->k < 1 || d->k > (1 << 24) || d->n > (1 << 24) || !fmt_ok(d->x_fmt) || !fmt_ok(d->w_fmt)) return DM_ERR_ARG;
    if (d->epi != DM_EPI_PLAIN && d->epi != DM_EPI_GEGLU && d->epi != DM_EPI_QUICKGELU) return DM_ERR_ARG;
    if (d->epi == DM_EPI_GEGLU && d->n % 2) return DM_ERR_ARG;
    if (d->c_type != DM_F32 && d->c_type != DM_BF16 && !fmt_ok(d->c_type)) return DM_ERR_ARG;
    if (d->m == 0) return DM_OK;
    const int kp = mx_padded(d->k);
    if (d->x_src == DM_X_MX) {
        if (const int rc = operand(d->x, d->ldx, d->x_scales, d->ld_xs, kp, d->x_fmt)) return rc;
    } else if (!d->x || d->ldx < d->k || d->m > DM_X_ROWS_MAX_M || (d->x_src != DM_X_BF16 && d->x_src != DM_X_F32)) {
        return DM_ERR_ARG;
    }
    if (const int rc = operand(d->w, d->ldw, d->w_scales, d->ld_ws, kp, d->w_fmt)) return rc;
    MxArgs p = {};
    p.x = static_cast<const unsigned char*>(d->x); p.xs = d->x_scales; p.w = d->w; p.ws = d->w_scales;
    p.ldx = d->ldx; p.ld_xs = d->ld_xs; p.ldw = d->ldw; p.ld_ws = d->ld_ws;
    p.m = d->m; p.n_out = d->epi == DM_EPI_GEGLU ? d->n / 2 : d->n; p.n_pad = p.n_out;
    p.nkt = kp / MX_PAD;
    p.last_blocks = (d->k + MX_BLOCK - 1) / MX_BLOCK - (p.nkt - 1) * (MX_PAD / MX_BLOCK);
    p.bias = d->bias; p.r = d->r; p.ldr = d->ldr; p.c = d->c; p.ldc = d->ldc; p.cs = d->c_scales; p.ld_cs = d->ld_cs;
    p.epi = d->epi; p.c_type = d->c_type;
    if (fmt_ok(d->c_type)) {
        if (d->r) return DM_ERR_ARG;
        p.n_pad = mx_padded(p.n_out);
        if (const int rc = operand(d->c, d->ldc, d->c_scales, d->ld_cs, p.n_pad, d->c_type)) return rc;
    } else {
        if (!d->c || d->ldc < p.n_out || (d->r && d->ldr < p.n_out)) return DM_ERR_ARG;
    }
    if (d->x_src != DM_X_MX) {
        p.ldx = d->ldx * (d->x_src == DM_X_F32 ? 4 : 2);  // bytes, as for codes
        p.k = d->k;
    }
    const bool f32 = d->c_type == DM_F32;
    int fm, fn;
    if (split_tile(p, &fm, &fn)) return dm_mx_split_launch(p, d->x_fmt, d->w_fmt, f32, d->x_src, fm, fn, stream);
    if (d->x_fmt == DM_MXFP8) return d->w_fmt == DM_MXFP8 ? launch_tile<8, 8>(p, f32, stream) : launch_tile<8, 4>(p, f32, stream);
    return d->w_fmt == DM_MXFP8 ? launch_tile<4, 8>(p, f32, stream) : launch_tile<4, 4>(p, f32, stream);
}
