// 4-bit product of an MoE layer's experts over ragged row segments (gfx950):
//   D[r, n] = sum_k (A[r, k] 2^ea[r, k / 32]) (B[g, n, k] 2^eb[g, n, k / 32]),  g = group of row r,
// A and B e2m1 (two a byte, element 2i in the low nibble), one power-of-two scale (UE8M0, four
// to an int32 word) for 32 elements of a row; segments as in dg_ragged.hpp. The matrix
// instruction v_mfma_scale_f32_32x32x64_f8f6f4 takes the scales: products of e2m1 values and powers of two are
// exact in FP32 and summed there; the sum is rounded once, to D's type.
//
// 256 elements are a step: 128 bytes of a row, as 64 BF16 values are, so that a step of the 4-bit
// operands is one of the BF16 products' K-major operands, and is loaded, laid out in LDS and
// read like it. A row has two words of scales a step.
//
// 16384 rows over 8 groups, n 4096, k 7168: 275 to 285 us, 3.4 to 3.5 PFLOP/s. 8192 x 4096 x 32768 reaches 4.3
// PFLOP/s of random values and 5.6 of zeros, the clock that the matrix load leaves; what the shorter axis
// loses to that are a tile's first loads and stores and the last, partial round (36 to 42 us for 6% of the
// tiles). k 2048, n 7168 163 us; 32 rows over 32 groups, 4096 x 7168 90 us, 5.5 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "dg_internal.hpp"
#include "dg_ragged.hpp"

namespace dgm {
namespace {

using namespace dev;

constexpr int kFmtE2M1 = 4;   // operand format of the matrix instruction

// The scales of 32 rows of a tile (a slab), WORDS words a row at a time (2: a step's, 4: those of
// two steps): word q of row r goes to (r * WORDS + q) * 4. Neighbouring lanes load neighbouring words
// of a row, 64 / WORDS rows a wave load; rows past the tile's read its last row's.
template <int WORDS>
struct ScaleSlab {
    static constexpr int kBytes = 32 * WORDS * 4, kLoads = WORDS / 2;   // wave loads
    const uint8_t* base;    // the first row's words to be issued next
    uint32_t row[kLoads];   // byte offsets of this lane's rows
    uint32_t word;          // of its word
    int64_t step;           // bytes to the next words
    int left;               // words from there on

    __device__ __forceinline__ void init(const uint32_t* at, int64_t sr, int64_t sk, int first_row, int rows, int words, int lane) {
        base = reinterpret_cast<const uint8_t*>(at);
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            row[i] = (uint32_t)(min(first_row + i * (64 / WORDS) + lane / WORDS, rows - 1) * (int)sr * 4);
        word = (uint32_t)(lane % WORDS) * (uint32_t)sk * 4u;   // (up to 3 GiB)
        step = sk * 4 * WORDS;
        left = words;
    }
    __device__ __forceinline__ void issue(uint32_t lds, int lane) {
        const uint32_t w = lane % WORDS < left ? word : 0u;   // (past the last word: the first again)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) dma4_saddr(base, row[i] + w, lds + i * 256);
        const bool more = left > WORDS;   // (past the end: the last ones again)
        base += more ? step : 0;
        left -= more ? WORDS : 0;
    }
};

// The scales of one step for this lane's row of a slab: two words as they lie in LDS, then byte
// (ks & 1) * 2 of word ks >> 1 the exponent of the lane's 32 elements of the ks-th matrix
// instruction. What is past the end counts as 2^0 (its codes are zeros, which a NaN scale would
// not leave zeros). left: scales from the step's first one on.
struct StepScales {
    uint32_t m0, m1;
    __device__ __forceinline__ explicit StepScales(int left) {
        m0 = left >= 4 ? ~0u : (1u << (8 * max(left, 0))) - 1u;
        m1 = left >= 8 ? ~0u : (1u << (8 * max(left - 4, 0))) - 1u;
    }
    // WORDS: of a row in LDS; first: the step's first of them
    template <int WORDS>
    __device__ __forceinline__ static void read(const uint8_t* slab, int lane, uint32_t first, uint32_t (&words)[2]) {
        const uint2 w = *reinterpret_cast<const uint2*>(slab + (lane & 31) * (WORDS * 4) + first * 4);
        words[0] = w.x, words[1] = w.y;
    }
    __device__ __forceinline__ void get(const uint32_t (&words)[2], int lane, int (&out)[2]) const {
        const uint32_t ones = 0x7F7F7F7Fu;
        const int shift = lane >> 5 << 3;
        out[0] = (int)(((words[0] & m0) | (ones & ~m0)) >> shift);
        out[1] = (int)(((words[1] & m1) | (ones & ~m1)) >> shift);
    }
};

// acc += B fragment x A fragment of 64 elements, the ks-th of a step.
__device__ __forceinline__ f32x16 mfma4(int ks, const bf16x8& b, const bf16x8& a, const f32x16& acc, const int (&sb)[2],
                                        const int (&sa)[2]) {
    const i32x4 b4 = __builtin_bit_cast(i32x4, b), a4 = __builtin_bit_cast(i32x4, a);
    const i32x8 b8{b4[0], b4[1], b4[2], b4[3], 0, 0, 0, 0}, a8{a4[0], a4[1], a4[2], a4[3], 0, 0, 0, 0};
    // (the byte is an immediate)
    return ks & 1 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b8, a8, acc, kFmtE2M1, kFmtE2M1, 2, sb[ks >> 1], 2, sa[ks >> 1])
                  : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b8, a8, acc, kFmtE2M1, kFmtE2M1, 0, sb[ks >> 1], 0, sa[ks >> 1]);
}

// One workgroup per BM x BN tile: 256 x 256 on eight waves (128 x 64 each), one workgroup on a
// CU, or 128 x 128 on four (64 x 64), two on a CU; PART 2: 128 x 128 quarters of 256 x 256 tiles
// (dg_ragged.hpp). Two steps of A and of B in LDS, and four of the scales; A's by slices (the
// 32-row slabs that the waves multiply at a time, side by side), a wave load for each wave. Two
// barriers a step, at which places are handed on and arrivals certified: before its last
// slice (every wave holds the slices up to the last; slices of the first half, B and the scales of
// the next step have arrived, and are read under the last slice), and at the start of its
// second half (every wave holds B and the first half's slices; the second half's have arrived).
// So a load is issued 1.5 steps before it is waited for.
template <int BM, int BN, int WGM, int WGN, int PART>
__global__ void __launch_bounds__(WGM * WGN * 64, WGM * WGN == 4 ? 2 : 1) fp4_tile_kernel(const RaggedFp4Args p, const RaggedLaunch l) {
    constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, SM = WM / 32, SN = WN / 32, KS = 4;
    constexpr int A_STEP = BM * BK * 2, B_STEP = BN * BK * 2;   // bytes of a step
    constexpr int SLAB = ScaleSlab<4>::kBytes, S_PAIR = (BM + BN) / 32 * SLAB, S_SLOTS = 3;   // scales of two steps
    constexpr int B_AT = 2 * A_STEP, S_AT = B_AT + 2 * B_STEP;
    static_assert(SM % 2 == 0 && BM / 32 == NW && BN / 32 == NW, "a slab of A's and of B's scales for each wave");
    static_assert(128 * BN * 4 <= S_AT, "the epilogue's rows fit");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[S_AT + S_SLOTS * S_PAIR];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    constexpr int LIST_BM = PART == 2 ? 2 * BM : BM, LIST_BN = PART == 2 ? 2 * BN : BN;
    RaggedTile t{};
    if (!locate_rows<LIST_BM, LIST_BN, PART>(p.g, l, t)) return;
    const int m0 = t.m0, n0 = t.n0, m_end = t.m_end;
    // this workgroup's piece of the reduced axis, in whole steps (none: it writes zeros)
    const int piece = ((p.g.k + BK - 1) / BK + l.splits - 1) / l.splits * BK;
    const int k0 = min((int)blockIdx.y * piece, p.g.k);
    const int reduced = min(piece, p.g.k - k0), words = (reduced + 31) / 32;
    const int a_rows = min(BM, m_end - m0), b_rows = min(BN, p.g.n - n0);

    Operand<BM, 1, NW> oa;
    Operand<BN, 1, NW> ob;
    ScaleSlab<4> sa, sb;
    oa.init(p.g.a + (int64_t)m0 * p.g.lda + k0, p.g.lda, a_rows, reduced, wave, lane);
    ob.init(static_cast<const uint16_t*>(p.g.b) + (int64_t)t.g * p.g.b_gs + (int64_t)n0 * p.g.ldb + k0, p.g.ldb, b_rows, reduced,
            wave, lane);
    sa.init(p.a_sf + (int64_t)m0 * p.a_sr + (int64_t)(k0 / 32) * p.a_sk, p.a_sr, p.a_sk, wave * 32, a_rows, words, lane);
    sb.init(p.b_sf + (int64_t)t.g * p.b_sg + (int64_t)n0 * p.b_sr + (int64_t)(k0 / 32) * p.b_sk, p.b_sr, p.b_sk, wave * 32, b_rows,
            words, lane);

    f32x16 acc[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem));
    Fragments<BM, 1, SM> fa;
    Fragments<BN, 1, SN> fb;
    fa.init(wm * WM, lane);
    fb.init(wn * WN, lane);
    bf16x8 op_b[SN][KS], op_a[2][KS];
    uint32_t wa[2][2], wb[SN][2];
    // words of a slab's rows for a step: pair, the place of its two steps' scales; odd, which of them it is
    auto read_a_scales = [&](uint32_t pair, uint32_t odd, int slab, uint32_t (&to)[2]) {
        StepScales::read<4>(smem + pair + (wm * SM + slab) * SLAB, lane, odd * 2, to);
    };
    auto read_b_scales = [&](uint32_t pair, uint32_t odd, int slab, uint32_t (&to)[2]) {
        StepScales::read<4>(smem + pair + (NW + wn * SN + slab) * SLAB, lane, odd * 2, to);
    };

    const int steps = (reduced + BK - 1) / BK;
    // Loads of a wave for a step: HALF of A at the hand-off of its last slice, TOP_LOADS (scales, A's
    // first half, B) at the other one; in flight at either: those of the step after the next.
    constexpr int HALF = decltype(oa)::kInstr / 2, B_LOADS = decltype(ob)::kInstr, S_LOADS = decltype(sa)::kLoads;
    constexpr int TOP_LOADS = S_LOADS + HALF + B_LOADS;
    constexpr int IN_FLIGHT = TOP_LOADS + HALF, PER_SLICE = HALF * 2 / SM;   // loads of a slice
    // The q-th load of a step of A: pieces of 8 rows of its slice, four of each wave row. (Offsets
    // worked out where they are used, from few scalars: kept, they would fill the scalar registers.)
    const uint32_t wave_lds = lds0 + wave * 1024;
    const int wave_piece = NW == 8 ? (wave >> 2) * (SM * 4) + (wave & 3) : wave;
    auto load_a = [&](const typename decltype(oa)::Step& s, int q, uint32_t at) {
        static_assert(NW == 4 || NW == 8, "pieces of one wave row or of both by each load");
        const int piece = q % PER_SLICE * (SM * 4) + q / PER_SLICE * 4;   // (+ wave_piece)
        int apart = decltype(oa)::kRows * (int)oa.pitch, mine = wave_piece;
        uint32_t lds = lds0 + at;
        asm volatile("" : "+s"(apart), "+s"(lds), "+s"(mine));
        dma16_buffer(s.rsrc, s.v + (uint32_t)((piece + mine) * apart), lds + (piece + mine) * 1024);
    };
    auto load_b = [&](const typename decltype(ob)::Step& s, int q, uint32_t at) {
        int apart = decltype(ob)::kRows * (int)ob.pitch;
        uint32_t lds = wave_lds + at;
        asm volatile("" : "+s"(apart), "+s"(lds));
        dma16_buffer(s.rsrc, s.v + (uint32_t)((q * NW + wave) * apart), lds + q * (NW * 1024));
    };
    // Scales come two steps at a time: A's of the pair after the next in even steps, B's in odd ones,
    // to the place after the next pair's (three places).
    uint32_t s_cur = S_AT, s_next = S_AT + S_PAIR, s_last = S_AT + 2 * S_PAIR;
    auto issue_scales = [&](bool b, uint32_t pair) {
        ScaleSlab<4> s = sa;
        s.base = b ? sb.base : sa.base, s.left = b ? sb.left : sa.left, s.step = b ? sb.step : sa.step;
        s.word = b ? sb.word : sa.word;
#pragma unroll
        for (int i = 0; i < S_LOADS; ++i) s.row[i] = b ? sb.row[i] : sa.row[i];
        s.issue(lds0 + pair + (wave + (b ? NW : 0)) * SLAB, lane);
        (b ? sb.base : sa.base) = s.base, (b ? sb.left : sa.left) = s.left;
    };
    auto next_pair = [&](int kb) {   // after an odd step
        const uint32_t done = s_cur;
        s_cur = kb & 1 ? s_next : s_cur, s_next = kb & 1 ? s_last : s_next, s_last = kb & 1 ? done : s_last;
    };
    if (steps > 0) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const auto s = oa.next();
            issue_scales(false, S_AT + kb * S_PAIR);
            issue_scales(true, S_AT + kb * S_PAIR);
#pragma unroll
            for (int q = 0; q < HALF; ++q) load_a(s, q, kb * A_STEP);
            ob.issue(lds0 + B_AT + kb * B_STEP, wave);
#pragma unroll
            for (int q = HALF; q < 2 * HALF; ++q) load_a(s, q, kb * A_STEP);
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt_barrier<HALF + S_LOADS + IN_FLIGHT>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) op_a[0][ks] = fa.read(smem, 0, ks);
        read_a_scales(s_cur, 0, 0, wa[0]);
#pragma unroll
        for (int j = 0; j < SN; ++j) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) op_b[j][ks] = fb.read(smem + B_AT, j, ks);
            read_b_scales(s_cur, 0, j, wb[j]);
        }
    }
    const bool computes = m0 + wm * WM < m_end;   // else a wave of rows past the group's: it loads and synchronises only
    if (!computes) {
        for (int kb = 0; kb < steps; ++kb) {
            wait_vmcnt_barrier<IN_FLIGHT>();
            const auto s = oa.next();
            issue_scales(kb & 1, s_last);
            next_pair(kb);
#pragma unroll
            for (int q = 0; q < HALF; ++q) load_a(s, q, (kb & 1) * A_STEP);
            ob.issue(lds0 + B_AT + (kb & 1) * B_STEP, wave);
            wait_vmcnt_barrier<IN_FLIGHT>();
#pragma unroll
            for (int q = HALF; q < 2 * HALF; ++q) load_a(s, q, (kb & 1) * A_STEP);
        }
    } else
    for (int kb = 0; kb < steps; ++kb) {
        const uint32_t odd = kb & 1, a_cur = odd * A_STEP, a_next = (odd ^ 1) * A_STEP;
        const uint32_t b_cur = B_AT + odd * B_STEP, b_next = B_AT + (odd ^ 1) * B_STEP;
        const uint32_t s_ahead = odd ? s_next : s_cur;   // the next step's
        const StepScales scales(reduced / 8 - kb * 8);
        int eb[SN][2];
        typename decltype(oa)::Step step_a;
        typename decltype(ob)::Step step_b;
        // A slice's matrix instructions with the LDS reads and loads of the steps to come set
        // between them one by one (as the BF16 products').
        constexpr int N = SN * KS, TOP = SM / 2 - 1;
#pragma unroll
        for (int i = 0; i < SM; ++i) {
            const bool last = i + 1 == SM;
            __builtin_amdgcn_sched_barrier(0);
            if (i == TOP) {
                wait_vmcnt_barrier<IN_FLIGHT>();
                step_a = oa.next();
                step_b = ob.next();
            }
            if (last) wait_vmcnt_barrier<IN_FLIGHT>();
            int ea[2];
            scales.get(wa[i & 1], lane, ea);
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < SN; ++j) scales.get(wb[j], lane, eb[j]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                // (the last slice by columns of fragments, whose registers are then free)
                const int j = last ? n / KS : n % SN, ks = last ? n % KS : n / SN;
                acc[i][j] = mfma4(ks, op_b[j][ks], op_a[i & 1][ks], acc[i][j], eb[j], ea);
                __builtin_amdgcn_sched_barrier(0);
                if (n < KS) {
                    if (last) op_a[0][n] = fa.read(smem + a_next, 0, n);
                    else op_a[(i + 1) & 1][n] = fa.read(smem + a_cur, i + 1, n);
                }
                if (n == 0) read_a_scales(last ? s_ahead : s_cur, last ? odd ^ 1 : odd, last ? 0 : i + 1, wa[last ? 0 : (i + 1) & 1]);
                if (last && n > 0 && n <= SN) read_b_scales(s_ahead, odd ^ 1, n - 1, wb[n - 1]);
                if (last && n >= KS) op_b[n / KS - 1][n % KS] = fb.read(smem + b_next, n / KS - 1, n % KS);
                if (i == TOP) {
                    if (n == 0) issue_scales(odd, s_last);
#pragma unroll
                    for (int q = n * (HALF + B_LOADS) / N; q < (n + 1) * (HALF + B_LOADS) / N; ++q) {
                        if (q < HALF) load_a(step_a, q, a_cur);
                        else load_b(step_b, q - HALF, b_cur);
                    }
                }
                if (last) {
#pragma unroll
                    for (int q = n * HALF / N; q < (n + 1) * HALF / N; ++q) load_a(step_a, HALF + q, a_cur);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (last) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) op_b[SN - 1][ks] = fb.read(smem + b_next, SN - 1, ks);
            }
        }
        next_pair(kb);
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt_barrier<0>();   // (loads of steps past the end wrote zeros to LDS)
    __builtin_amdgcn_sched_barrier(0);
    if (p.g.out_f32) store_tile<1, BM, BN, WGM, WGN>(p.g, acc, smem, 0, m0, m_end, n0, wave, lane, l.vec);
    else store_tile<0, BM, BN, WGM, WGN>(p.g, acc, smem, 0, m0, m_end, n0, wave, lane, l.vec);
}

// Few rows a group (decode): 32 x 128 or 64 x 128 tiles on four waves of 32 columns, two
// workgroups on a CU, which stream the weights from HBM. Three steps of 21 or 26 KB in LDS and one
// barrier a step: it certifies the next step's loads and frees this one's place, whose
// fragments every wave holds. (A slab of A's scales is loaded by more than one wave, to one place.)
template <int SM>
__global__ void __launch_bounds__(256, 2) fp4_few_rows_kernel(const RaggedFp4Args p, const RaggedLaunch l) {
    constexpr int BM = SM * 32, BN = 128, NW = 4, KS = 4, SLOTS = 3, SLAB = ScaleSlab<2>::kBytes;
    constexpr int A_STEP = BM * BK * 2, B_STEP = BN * BK * 2, S_AT = A_STEP + B_STEP, STEP = S_AT + (SM + NW) * SLAB;
    static_assert(NW % SM == 0 && BM * BN * 4 <= SLOTS * STEP, "whole slabs; the epilogue's rows fit");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[SLOTS * STEP];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    RaggedTile t{};
    if (!locate_rows<BM, BN, 0>(p.g, l, t)) return;
    const int piece = ((p.g.k + BK - 1) / BK + l.splits - 1) / l.splits * BK;   // (as in the tile kernel)
    const int k0 = min((int)blockIdx.y * piece, p.g.k);
    const int reduced = min(piece, p.g.k - k0), words = (reduced + 31) / 32;

    Operand<BM, 1, NW> oa;
    Operand<BN, 1, NW> ob;
    ScaleSlab<2> sa, sb;
    const int a_rows = min(BM, t.m_end - t.m0), b_rows = min(BN, p.g.n - t.n0);
    oa.init(p.g.a + (int64_t)t.m0 * p.g.lda + k0, p.g.lda, a_rows, reduced, wave, lane);
    ob.init(static_cast<const uint16_t*>(p.g.b) + (int64_t)t.g * p.g.b_gs + (int64_t)t.n0 * p.g.ldb + k0, p.g.ldb, b_rows, reduced,
            wave, lane);
    sa.init(p.a_sf + (int64_t)t.m0 * p.a_sr + (int64_t)(k0 / 32) * p.a_sk, p.a_sr, p.a_sk, wave % SM * 32, a_rows, words, lane);
    sb.init(p.b_sf + (int64_t)t.g * p.b_sg + (int64_t)t.n0 * p.b_sr + (int64_t)(k0 / 32) * p.b_sk, p.b_sr, p.b_sk, wave * 32, b_rows,
            words, lane);
    constexpr int LOADS = decltype(oa)::kInstr + decltype(ob)::kInstr + 2;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem));
    auto issue = [&](int slot) {
        const uint32_t at = lds0 + slot * STEP;
        oa.issue(at, wave);
        ob.issue(at + A_STEP, wave);
        sa.issue(at + S_AT + wave % SM * SLAB, lane);
        sb.issue(at + S_AT + (SM + wave) * SLAB, lane);
    };
    Fragments<BM, 1, SM> fa;
    Fragments<BN, 1, 1> fb;
    fa.init(0, lane);
    fb.init(wave * 32, lane);
    bf16x8 op_a[2][SM][KS], op_b[2][KS];
    uint32_t wa[2][SM][2], wb[2][2];
    auto read = [&](int to, int slot) {
        const uint8_t* at = smem + slot * STEP;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            op_b[to][ks] = fb.read(at + A_STEP, 0, ks);
#pragma unroll
            for (int i = 0; i < SM; ++i) op_a[to][i][ks] = fa.read(at, i, ks);
        }
        StepScales::read<2>(at + S_AT + (SM + wave) * SLAB, lane, 0, wb[to]);
#pragma unroll
        for (int i = 0; i < SM; ++i) StepScales::read<2>(at + S_AT + i * SLAB, lane, 0, wa[to][i]);
    };
    f32x16 acc[SM][1];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][0][e] = 0.f;

    const int steps = (reduced + BK - 1) / BK;
    if (steps > 0) {   // (no reduced elements: no scales to read)
#pragma unroll
        for (int st = 0; st < SLOTS; ++st) issue(st);
        wait_vmcnt_barrier<(SLOTS - 1) * LOADS>();
        read(0, 0);
    }
    for (int kb = 0, slot = 0; kb < steps; kb += 2) {   // (a step past an odd end: zeros)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wait_vmcnt_barrier<(SLOTS - 2) * LOADS>();
            issue(slot);
            slot = slot + 1 == SLOTS ? 0 : slot + 1;
            read(h ^ 1, slot);
            const StepScales scales(reduced / 8 - (kb + h) * 8);
            int ea[SM][2], eb[2];
            scales.get(wb[h], lane, eb);
#pragma unroll
            for (int i = 0; i < SM; ++i) scales.get(wa[h][i], lane, ea[i]);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < SM; ++i) acc[i][0] = mfma4(ks, op_b[h][ks], op_a[h][i][ks], acc[i][0], eb, ea[i]);
        }
    }
    wait_vmcnt_barrier<0>();   // (loads of steps past the end wrote zeros to LDS)
    if (p.g.out_f32) store_tile<1, BM, BN, 1, NW>(p.g, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
    else store_tile<0, BM, BN, 1, NW>(p.g, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
}

}  // namespace

// Tiles and pieces of the reduced axis by a model of the time, in us: a step (256 elements) of a
// tile on a CU takes 0.38, 0.5 and 0.7 (32, 64 and 128 rows) alone and 0.88, 0.98 and 1.35 beside another,
// 1.9 of 256 x 256; a tile's start and end 2 (256 x 256: 10); a split call 3.5 more and its sums'
// two ways at 2 TB/s. Row blocks of a group that has rows: as many as its average, and half a one,
// at least one. Both sides measured (us; NT, groups x (rows in all), n, k):
// 256 x 256 and 128 x 128: 8 x 16384, 4096, 7168 286 and 331; 8 x 8192, 7168, 2048 99 and 113; 8 x 2048, 4096,
//   7168 61 and 66; 32 x 2048, 4096, 2048 42 and 32; 1 x 4096, 4096, 1024 22.1 and 20.7.
// Where 128 x 128 tiles fill three quarters of the CUs, smaller ones only read weights again: 128,
//   64 and 32 rows at 8 x 256, 4096, 7168 30, 48 and 45; 32 x 512, 4096, 7168 97, 107 and 112; 32 x 32, 4096, 7168 90, 95
//   and 94, 5120 68, 73 and 71. But for up to 8 rows a group and a short reduced axis, where a tile's end
//   counts. 128 and 32 rows, weights from HBM, 32 groups of n 4096: 2, 8, 12, 16 and 24 rows each, 2048 31.9/30.8, 31.9/31.4,
//   32.0/31.9, 32.3/32.5 and 32.4/33.6; 3584 49.2/49.5, 49.9/51.1, 50.2/51.7, 50.7/53.1 and 51.7/54.7; 1024 21.2/19.5,
//   21.2/19.5, 21.3/19.9, 21.6/20.4 and 21.8/21.2. 8 groups, 2048: 8 and 16 rows 11.4/10.7 and 11.5/10.9.
// The rows are the buffer's, padding and what no group has with it, as the ends are on the device: 8 routed rows over 64
//   groups, 2048, 7168 take 17.2 back to back, 22.0 where they lie 16 apart and 26.0 where they lie 128 apart.
// Where they do not: 1 x 512, 4096, 7168 22, 19 and 27; 1 x 256, 2112, 7168 22, 18 and 16; 2 x 128, 4096, 4096 14.7, 12.6
//   and 11.4.
// Whole, in 2, 4 and 8 pieces, 32 rows: 1 x 64, 2112, 7168 15.4, 13.9, 12.3, 14.3; 1 x 256, 2112, 7168 15.6, 20.2, 22.7, 23.1.
RaggedPlan plan_ragged_fp4(const RaggedFp4Args& a, int slots, int block, int splits) {
    const double used = (double)std::max<int64_t>(1, std::min<int64_t>(a.g.groups, a.g.rows));   // groups with rows, at most
    const double steps = (double)ceil_div(a.g.k, BK), rows = (double)a.g.rows;
    auto tiles = [&](int b) {   // expected
        return std::max(used, rows / b + (rows > used ? 0.5 * used : 0.0)) * (double)ceil_div(a.g.n, b == 256 ? 256 : 128);
    };
    auto us = [&](int b, double t, double n) {   // t tiles of n steps, two of which fit a CU
        const double alone = b == 32 ? 0.38 : b == 64 ? 0.5 : 0.7, both = b == 32 ? 0.88 : b == 64 ? 0.98 : 1.35, ends = 2.0;
        const double per_cu = t / slots, whole = std::floor(per_cu / 2), rest = per_cu - 2 * whole;
        return whole * (n * both + ends) +
               (rest > 0 ? n * (alone + (both - alone) * std::max(0.0, rest - 1)) + ends * std::min(rest, 1.0) : 0.0);
    };
    if (block == 0) {
        const double t128 = tiles(128), t256 = tiles(256);
        if (t256 * 128 >= slots * 75 && std::max(1.0, t256 / slots) * (steps * 1.9 + 10) < 1.1 * us(128, t128, steps)) {
            block = 256;
        } else {
            block = t128 * 4 >= slots * 3 && rows <= 8 * used && steps <= 12 ? kFewRows : 128;
            for (int b : {64, 32})   // (the larger of two that are about as fast)
                if (t128 * 4 < slots * 3 && us(b, tiles(b), steps) < 0.95 * us(block, tiles(block), steps)) block = b;
        }
    }
    RaggedPlan plan{block, 1, 0};
    if (block == 256) return plan;
    const double sums = rows * a.g.n * 4;   // bytes of a piece's
    double best = 1e300;
    for (int s = 1; s <= 32; ++s) {
        if (splits > 0 ? s != splits : (s > 1 && steps < 4 * s)) continue;
        const double t = us(block, tiles(block) * s, std::ceil(steps / s)) + (s > 1 ? 3.5 + 2 * sums * s / 2e6 : 0.0);
        if (t < best) best = t, plan.splits = s;
    }
    if (plan.splits > 1) plan.workspace_bytes = (int64_t)a.g.rows * ceil_div(a.g.n, 4) * 16 * plan.splits;
    return plan;
}

void check_ragged_fp4_launches(const RaggedFp4Args& a, const RaggedPlan& plan) {
    if (plan.block <= 2 * kFewRows) {
        DG_CHECK_GRID(row_blocks(kRaggedNT, a.g, plan.block) * ceil_div(a.g.n, 128), 256);
    } else {
        DG_CHECK_GRID(tile_blocks(kRaggedNT, a.g, plan.block, false, 1), plan.block * 2);
    }
    if (plan.splits > 1) DG_CHECK_GRID(join_blocks(kRaggedNT, a.g), 256);
}

namespace {

template <int BM, int BN, int WGM, int WGN, int PART>
void launch_fp4_tiles(const RaggedFp4Args& a, int slots, int splits, hipStream_t stream) {
    constexpr int LIST = PART == 2 ? 2 : 1;
    const int64_t mb = row_blocks(kRaggedNT, a.g, LIST * BM), nb = ceil_div(a.g.n, LIST * BN);
    const int64_t blocks = tile_blocks(kRaggedNT, a.g, LIST * BM, PART == 2, slots);
    const RaggedLaunch l{(int)mb, (int)nb, slots, splits, takes_vectors(a.g)};
    hipLaunchKernelGGL((fp4_tile_kernel<BM, BN, WGM, WGN, PART>), dim3((unsigned)blocks, (unsigned)splits), dim3(WGM * WGN * 64), 0,
                       stream, a, l);
    DG_HIP_CHECK(hipGetLastError());
}

template <int SM>
void launch_fp4_few_rows(const RaggedFp4Args& a, int slots, int splits, hipStream_t stream) {
    const int64_t mb = row_blocks(kRaggedNT, a.g, SM * 32), nb = ceil_div(a.g.n, 128);
    const RaggedLaunch l{(int)mb, (int)nb, slots, splits, takes_vectors(a.g)};
    hipLaunchKernelGGL(fp4_few_rows_kernel<SM>, dim3((unsigned)(mb * nb), (unsigned)splits), dim3(256), 0, stream, a, l);
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace

void launch_ragged_fp4(const RaggedFp4Args& a, const RaggedPlan& plan, float* ws, int slots, hipStream_t stream) {
    DG_CHECK(plan.splits == 1 || ws != nullptr);
    if (plan.block == 256) {
        launch_fp4_tiles<256, 256, 2, 4, 1>(a, slots, 1, stream);
        launch_fp4_tiles<128, 128, 2, 2, 2>(a, slots, 1, stream);
        return;
    }
    auto launch = [&](const RaggedFp4Args& args) {
        if (plan.block == kFewRows) launch_fp4_few_rows<1>(args, slots, plan.splits, stream);
        else if (plan.block == 2 * kFewRows) launch_fp4_few_rows<2>(args, slots, plan.splits, stream);
        else launch_fp4_tiles<128, 128, 2, 2, 0>(args, slots, plan.splits, stream);
    };
    if (plan.splits == 1) return launch(a);
    const int64_t ld = ceil_div(a.g.n, 4) * 4;
    RaggedFp4Args part = a;
    part.g.d = ws, part.g.ldd = ld, part.g.d_split = a.g.rows * ld, part.g.out_f32 = 1;
    launch(part);
    RaggedGemmArgs whole = a.g;
    whole.d_split = part.g.d_split;
    hipLaunchKernelGGL(ragged_join_kernel<kRaggedNT>, dim3((unsigned)join_blocks(kRaggedNT, a.g)), dim3(256), 0, stream, whole,
                       (const float*)ws, ld, plan.splits, (int)ceil_div(a.g.n, 1024));
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
