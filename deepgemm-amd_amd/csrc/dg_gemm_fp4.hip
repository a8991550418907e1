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
#include <hip/hip_runtime.h>

#include <algorithm>

#include "dg_internal.hpp"
#include "dg_ragged.hpp"

namespace dgm {
namespace {

using namespace dev;

constexpr int kFmtE2M1 = 4;   // operand format of the matrix instruction

// The scales of 32 rows of a tile, two words a row for each step: word q of row r goes to
// (q * 32 + r) * 4. One wave load; rows past the tile's read its last row's.
struct ScaleSlab {
    const uint8_t* base;   // the first row's words of the step to be issued next
    uint32_t row, word;    // byte offsets of this lane's row, and of its word
    int64_t step;          // bytes between steps
    int left;              // words from there on

    __device__ __forceinline__ void init(const uint32_t* at, int64_t sr, int64_t sk, int first_row, int rows, int words, int lane) {
        base = reinterpret_cast<const uint8_t*>(at);
        row = (uint32_t)(min(first_row + (lane & 31), rows - 1) * (int)sr * 4);
        word = (uint32_t)((lane >> 5) * (int)sk * 4);
        step = sk * 8;
        left = words;
    }
    __device__ __forceinline__ void issue(uint32_t lds) {
        dma4_saddr(base, row + (left > 1 ? word : 0u), lds);   // (an odd last word: twice)
        base += left > 2 ? step : 0;                            // (steps past the end read the last one again)
        left -= left > 2 ? 2 : 0;
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
    __device__ __forceinline__ static void read(const uint8_t* slab, int lane, uint32_t (&words)[2]) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(slab) + (lane & 31);
        words[0] = w[0], words[1] = w[32];
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
// (dg_ragged.hpp). Two steps of A, of B and of the scales in LDS, and two barriers a step: the
// hand-off before a step's last 32-row slice (the next step's loads have arrived, and every
// wave has read A's last slice and the scales, whose places the step after the next takes), and
// another one a slice after the step's start, when every wave holds its B fragments, whose
// place is handed on.
template <int BM, int BN, int WGM, int WGN, int PART>
__global__ void __launch_bounds__(WGM * WGN * 64, WGM * WGN == 4 ? 2 : 1) fp4_tile_kernel(const RaggedFp4Args p, const RaggedLaunch l) {
    constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, SM = WM / 32, SN = WN / 32, KS = 4;
    constexpr int A_STEP = BM * BK * 2, B_STEP = BN * BK * 2, S_STEP = (BM + BN) / 32 * 256;   // bytes of a step
    constexpr int B_AT = 2 * A_STEP, S_AT = B_AT + 2 * B_STEP;
    static_assert(SM % 2 == 0 && BM / 32 == NW && BN / 32 == NW, "a slab of A's and of B's scales for each wave");
    static_assert(128 * BN * 4 <= S_AT, "the epilogue's rows fit");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[S_AT + 2 * S_STEP];

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
    ScaleSlab sa, sb;
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
    auto a_scales = [&](uint32_t step, int slab) { return smem + S_AT + step + (wm * SM + slab) * 256; };
    auto b_scales = [&](uint32_t step, int slab) { return smem + S_AT + step + (NW + wn * SN + slab) * 256; };
    auto issue_scales = [&](uint32_t s) {
        sa.issue(lds0 + S_AT + s + wave * 256);
        sb.issue(lds0 + S_AT + s + (NW + wave) * 256);
    };

    const int steps = (reduced + BK - 1) / BK;
    constexpr int A_LOADS = decltype(oa)::kInstr, B_LOADS = decltype(ob)::kInstr;
    constexpr int IN_FLIGHT = B_LOADS;   // at a hand-off: B of the step after the next
    if (steps > 0) {
        oa.issue(lds0, wave);
        ob.issue(lds0 + B_AT, wave);
        issue_scales(0);
        oa.issue(lds0 + A_STEP, wave);
        ob.issue(lds0 + B_AT + B_STEP, wave);
        issue_scales(S_STEP);
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt_barrier<A_LOADS + B_LOADS + 2>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) op_a[0][ks] = fa.read(smem, 0, ks);
        StepScales::read(a_scales(0, 0), lane, wa[0]);
#pragma unroll
        for (int j = 0; j < SN; ++j) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) op_b[j][ks] = fb.read(smem + B_AT, j, ks);
            StepScales::read(b_scales(0, j), lane, wb[j]);
        }
    }
    const bool computes = m0 + wm * WM < m_end;   // else a wave of rows past the group's: it loads and synchronises only
    if (!computes) {
        for (int kb = 0; kb < steps; ++kb) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            ob.issue(lds0 + B_AT + (kb & 1) * B_STEP, wave);
            wait_vmcnt_barrier<IN_FLIGHT>();
            oa.issue(lds0 + (kb & 1) * A_STEP, wave);
            issue_scales((kb & 1) * S_STEP);
        }
    } else
    for (int kb = 0; kb < steps; ++kb) {
        const uint32_t odd = kb & 1, a_cur = odd * A_STEP, a_next = (odd ^ 1) * A_STEP;
        const uint32_t b_cur = B_AT + odd * B_STEP, b_next = B_AT + (odd ^ 1) * B_STEP, s_cur = odd * S_STEP, s_next = (odd ^ 1) * S_STEP;
        const StepScales scales(reduced / 8 - kb * 8);
        int eb[SN][2];
        // A slice's matrix instructions with the LDS reads and loads of the steps to come set
        // between them one by one (as the BF16 products').
        constexpr int N = SN * KS, TOP = SM > 2 ? 1 : 0;
#pragma unroll
        for (int i = 0; i < SM; ++i) {
            const bool last = i + 1 == SM;
            typename decltype(oa)::Step step_a;
            typename decltype(ob)::Step step_b;
            __builtin_amdgcn_sched_barrier(0);
            if (i == TOP) {
                // every wave holds its B fragments and B's scales of this step, and A's up to slice TOP
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                step_b = ob.next();
            }
            if (last) {
                wait_vmcnt_barrier<IN_FLIGHT>();
                step_a = oa.next();
            }
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
                if (n == 0) StepScales::read(last ? a_scales(s_next, 0) : a_scales(s_cur, i + 1), lane, wa[last ? 0 : (i + 1) & 1]);
                if (last && n > 0 && n <= SN) StepScales::read(b_scales(s_next, n - 1), lane, wb[n - 1]);
                if (last && n >= KS) op_b[n / KS - 1][n % KS] = fb.read(smem + b_next, n / KS - 1, n % KS);
                if (i == TOP) {
#pragma unroll
                    for (int q = n * B_LOADS / N; q < (n + 1) * B_LOADS / N; ++q) ob.load(step_b, q, lds0 + b_cur, wave);
                }
                if (last) {
#pragma unroll
                    for (int q = n * A_LOADS / N; q < (n + 1) * A_LOADS / N; ++q) oa.load(step_a, q, lds0 + a_cur, wave);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (last) {
                issue_scales(s_cur);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) op_b[SN - 1][ks] = fb.read(smem + b_next, SN - 1, ks);
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt_barrier<0>();   // (loads of steps past the end wrote zeros to LDS)
    __builtin_amdgcn_sched_barrier(0);
    if (p.g.out_f32) store_tile<1, BM, BN, WGM, WGN>(p.g, acc, smem, 0, m0, m_end, n0, wave, lane, l.vec);
    else store_tile<0, BM, BN, WGM, WGN>(p.g, acc, smem, 0, m0, m_end, n0, wave, lane, l.vec);
}

// 32 x 128 tiles on four waves of 32 x 32, two workgroups on a CU.
__global__ void __launch_bounds__(256, 2) fp4_few_rows_kernel(const RaggedFp4Args p, const RaggedLaunch l) {
    constexpr int BM = kFewRows, BN = 128, NW = 4, KS = 4, SLOTS = 3;
    constexpr int A_STEP = BM * BK * 2, B_STEP = BN * BK * 2, S_AT = A_STEP + B_STEP, STEP = S_AT + NW * 512;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[SLOTS * STEP];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    RaggedTile t{};
    if (!locate_rows<BM, BN, 0>(p.g, l, t)) return;
    const int reduced = p.g.k, words = (reduced + 31) / 32;

    Operand<BM, 1, NW> oa;
    Operand<BN, 1, NW> ob;
    ScaleSlab sa, sb;
    const int a_rows = min(BM, t.m_end - t.m0), b_rows = min(BN, p.g.n - t.n0);
    oa.init(p.g.a + (int64_t)t.m0 * p.g.lda, p.g.lda, a_rows, reduced, wave, lane);
    ob.init(static_cast<const uint16_t*>(p.g.b) + (int64_t)t.g * p.g.b_gs + (int64_t)t.n0 * p.g.ldb, p.g.ldb, b_rows, reduced,
            wave, lane);
    sa.init(p.a_sf + (int64_t)t.m0 * p.a_sr, p.a_sr, p.a_sk, 0, a_rows, words, lane);
    sb.init(p.b_sf + (int64_t)t.g * p.b_sg + (int64_t)t.n0 * p.b_sr, p.b_sr, p.b_sk, wave * 32, b_rows, words, lane);
    constexpr int LOADS = decltype(oa)::kInstr + decltype(ob)::kInstr + 2;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem));
    auto issue = [&](int slot) {
        const uint32_t at = lds0 + slot * STEP;
        oa.issue(at, wave);
        ob.issue(at + A_STEP, wave);
        sa.issue(at + S_AT + wave * 512);
        sb.issue(at + S_AT + wave * 512 + 256);
    };
    Fragments<BM, 1, 1> fa;
    Fragments<BN, 1, 1> fb;
    fa.init(0, lane);
    fb.init(wave * 32, lane);
    f32x16 acc[1][1];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][0][e] = 0.f;

    const int steps = (reduced + BK - 1) / BK;
    if (steps > 0) {   // (no reduced elements: no scales to read)
#pragma unroll
        for (int st = 0; st < SLOTS; ++st) issue(st);
    }
    for (int kb = 0, slot = 0; kb < steps; ++kb) {
        wait_vmcnt_barrier<(SLOTS - 1) * LOADS>();
        const uint8_t* at = smem + slot * STEP;
        bf16x8 a[KS], b[KS];
        uint32_t wa[2], wb[2];
        int ea[2], eb[2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            a[ks] = fa.read(at, 0, ks);
            b[ks] = fb.read(at + A_STEP, 0, ks);
        }
        const StepScales scales(reduced / 8 - kb * 8);
        scales.read(at + S_AT + wave * 512, lane, wa);
        scales.read(at + S_AT + wave * 512 + 256, lane, wb);
        scales.get(wa, lane, ea), scales.get(wb, lane, eb);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc[0][0] = mfma4(ks, b[ks], a[ks], acc[0][0], eb, ea);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // every wave has read this step
        issue(slot);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
    }
    wait_vmcnt_barrier<0>();   // (loads of steps past the end wrote zeros to LDS)
    if (p.g.out_f32) store_tile<1, BM, BN, 1, NW>(p.g, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
    else store_tile<0, BM, BN, 1, NW>(p.g, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
}

}  // namespace

RaggedPlan plan_ragged_fp4(const RaggedFp4Args& a, int slots, int block, int) {
    if (block) return RaggedPlan{block, 1, 0};
    const int64_t used = std::max<int64_t>(1, std::min<int64_t>(a.g.groups, a.g.rows));
    if (a.g.rows <= kFewRows * used) return RaggedPlan{kFewRows, 1, 0};
    return RaggedPlan{(a.g.rows / 256 + 0.5 * used) * ceil_div(a.g.n, 256) * 128 >= slots * 75 ? 256 : 128, 1, 0};
}

void check_ragged_fp4_launches(const RaggedFp4Args& a, const RaggedPlan& plan) {
    if (plan.block == kFewRows) {
        DG_CHECK_GRID(row_blocks(kRaggedNT, a.g, kFewRows) * ceil_div(a.g.n, 128), 256);
    } else {
        DG_CHECK_GRID(tile_blocks(kRaggedNT, a.g, plan.block, false, 1), plan.block * 2);
    }
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

}  // namespace

void launch_ragged_fp4(const RaggedFp4Args& a, const RaggedPlan& plan, float*, int slots, hipStream_t stream) {
    if (plan.block == 256) {
        launch_fp4_tiles<256, 256, 2, 4, 1>(a, slots, 1, stream);
        launch_fp4_tiles<128, 128, 2, 2, 2>(a, slots, 1, stream);
        return;
    }
    if (plan.block == 128) return launch_fp4_tiles<128, 128, 2, 2, 0>(a, slots, 1, stream);
    const int64_t mb = row_blocks(kRaggedNT, a.g, kFewRows), nb = ceil_div(a.g.n, 128);
    const RaggedLaunch l{(int)mb, (int)nb, slots, 1, takes_vectors(a.g)};
    hipLaunchKernelGGL(fp4_few_rows_kernel, dim3((unsigned)(mb * nb)), dim3(256), 0, stream, a, l);
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
