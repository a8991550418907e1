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

// The scales of one step for this lane's row of a slab, byte (ks & 1) * 2 of word ks >> 1 the
// exponent of its 32 elements of the ks-th matrix instruction. What is past the end counts
// as 2^0 (its codes are zeros, which a NaN scale would not leave zeros). left: scales from
// the step's first one on.
struct StepScales {
    uint32_t m0, m1;
    __device__ __forceinline__ explicit StepScales(int left) {
        m0 = left >= 4 ? ~0u : (1u << (8 * max(left, 0))) - 1u;
        m1 = left >= 8 ? ~0u : (1u << (8 * max(left - 4, 0))) - 1u;
    }
    __device__ __forceinline__ void read(const uint8_t* slab, int lane, int (&out)[2]) const {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(slab) + (lane & 31);
        const uint32_t ones = 0x7F7F7F7Fu;
        const int shift = lane >> 5 << 3;
        out[0] = (int)(((w[0] & m0) | (ones & ~m0)) >> shift);
        out[1] = (int)(((w[32] & m1) | (ones & ~m1)) >> shift);
    }
};

// acc += B fragment x A fragment of 64 elements, the ks-th of a step.
template <int KS>
__device__ __forceinline__ f32x16 mfma4(const i32x4& b, const i32x4& a, const f32x16& acc, const int (&sb)[2], const int (&sa)[2]) {
    const i32x8 bb{b[0], b[1], b[2], b[3], 0, 0, 0, 0}, aa{a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(bb, aa, acc, kFmtE2M1, kFmtE2M1, (KS & 1) * 2, sb[KS >> 1],
                                                           (KS & 1) * 2, sa[KS >> 1]);
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
        i32x4 a[KS], b[KS];
        int wa[2], wb[2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            a[ks] = __builtin_bit_cast(i32x4, fa.read(at, 0, ks));
            b[ks] = __builtin_bit_cast(i32x4, fb.read(at + A_STEP, 0, ks));
        }
        const StepScales scales(reduced / 8 - kb * 8);
        scales.read(at + S_AT + wave * 512, lane, wa);
        scales.read(at + S_AT + wave * 512 + 256, lane, wb);
        acc[0][0] = mfma4<0>(b[0], a[0], acc[0][0], wb, wa);
        acc[0][0] = mfma4<1>(b[1], a[1], acc[0][0], wb, wa);
        acc[0][0] = mfma4<2>(b[2], a[2], acc[0][0], wb, wa);
        acc[0][0] = mfma4<3>(b[3], a[3], acc[0][0], wb, wa);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // every wave has read this step
        issue(slot);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
    }
    wait_vmcnt_barrier<0>();   // (loads of steps past the end wrote zeros to LDS)
    if (p.g.out_f32) store_tile<1, BM, BN, 1, NW>(p.g, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
    else store_tile<0, BM, BN, 1, NW>(p.g, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
}

}  // namespace

RaggedPlan plan_ragged_fp4(const RaggedFp4Args&, int, int, int) { return RaggedPlan{kFewRows, 1, 0}; }

void check_ragged_fp4_launches(const RaggedFp4Args& a, const RaggedPlan&) {
    DG_CHECK_GRID(row_blocks(kRaggedNT, a.g, kFewRows) * ceil_div(a.g.n, 128), 256);
}

void launch_ragged_fp4(const RaggedFp4Args& a, const RaggedPlan&, float*, int slots, hipStream_t stream) {
    const int64_t mb = row_blocks(kRaggedNT, a.g, kFewRows), nb = ceil_div(a.g.n, 128);
    const RaggedLaunch l{(int)mb, (int)nb, slots, 1, takes_vectors(a.g)};
    hipLaunchKernelGGL(fp4_few_rows_kernel, dim3((unsigned)(mb * nb)), dim3(256), 0, stream, a, l);
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
