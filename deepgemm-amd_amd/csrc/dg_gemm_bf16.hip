// BF16 products of an MoE layer's experts over ragged row segments (gfx950).
//
// Group g owns rows [s_g, e_g) of the token-major operands, e_g = group_ends[g] and
// s_g = align(e_{g-1}, alignment) (s_0 = 0): segments of any length, with alignment 1
// back to back, with 16 or 128 the psum layout of the MoE dispatch. Three products:
//   NT  D[r, n] = sum_k A[r, k] B[g, n, k]            (forward)
//   NN  D[r, n] = sum_k A[r, k] B[g, k, n]            (gradient of the input)
//   TN  D[g, m, n] = C[g, m, n] + sum_r A[r, m] B[r, n]   (gradient of the weight; B BF16
//       or e4m3 with an FP32 scale per row and 128 columns, an 8-bit activation checkpoint)
// BF16 products are exact in FP32 and summed there by v_mfma_f32_32x32x16_bf16; the sum
// (with C added in FP32) is rounded once, to D's type. A checkpoint value is rounded to
// BF16 after its scale, which is exact where the scale is a power of two.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "dg_internal.hpp"
#include "dg_kernel_common.hpp"

namespace dgm {
namespace {

using namespace dev;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Rows [start, end) of group g, inside the `rows` that exist whatever group_ends holds.
__device__ __forceinline__ void group_rows(const int32_t* ends, int g, int rows, int alignment, int& start, int& end) {
    const int prev = g > 0 ? min(max(ends[g - 1], 0), rows) : 0;
    start = min(align_up(prev, alignment), rows);
    end = max(start, min(ends[g], rows));
}

// The row block `blk` (of BM rows each) of the launch's blocks, groups in order: its group,
// first row and the group's end; false past the last one. A wave looks at 64 groups at a
// time: every lane counts one group's blocks, a prefix sum over the lanes places them.
template <int BM>
__device__ __forceinline__ bool find_block(const int32_t* ends, int groups, int rows, int alignment, int64_t blk, int& g,
                                           int& m0, int& row_end) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int g0 = 0; g0 < groups; g0 += 64) {
        int start = 0, end = 0;
        if (g0 + lane < groups) group_rows(ends, g0 + lane, rows, alignment, start, end);
        const int mine = (end - start + BM - 1) / BM;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            incl += lane >= o ? v : 0;
        }
        const int total = __shfl(incl, 63);
        if (blk < base + total) {
            const int at = __ffsll((unsigned long long)__ballot(base + incl > blk)) - 1;
            g = g0 + at;
            m0 = __shfl(start, at) + (int)(blk - base - __shfl(incl - mine, at)) * BM;
            row_end = __shfl(end, at);
            return true;
        }
        base += total;
    }
    return false;
}

constexpr int kBM = 128, kBN = 128, kBK = 32, kPitch = kBK + 8;

__device__ __forceinline__ uint16_t load_b(const RaggedGemmArgs& p, int64_t row, int col, const uint16_t* b) {
    if (!p.b_sf) return b[row * p.ldb + col];
    const uint8_t q = reinterpret_cast<const uint8_t*>(b)[row * p.ldb + col];
    const float v = __builtin_amdgcn_cvt_f32_fp8(q, 0) * p.b_sf[row * p.sf_sr + (int64_t)(col >> 7) * p.sf_sc];
    return bf16_bits(v);
}

template <int KIND>
__global__ void __launch_bounds__(256) ragged_gemm_kernel(const RaggedGemmArgs p, const int nb) {
    __shared__ __attribute__((aligned(16))) uint16_t s_a[kBM * kPitch], s_b[kBN * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int g, m0, m_end, k0 = 0, k_end = p.k;   // output rows [m0, m_end), reduced over [k0, k_end)
    const int64_t blk = blockIdx.x / nb;
    const int n0 = (int)(blockIdx.x % nb) * kBN;
    if constexpr (KIND == kRaggedTN) {
        const int mb = (p.m + kBM - 1) / kBM;
        g = (int)(blk / mb);
        m0 = (int)(blk % mb) * kBM;
        m_end = p.m;
        group_rows(p.ends, g, p.rows, p.alignment, k0, k_end);
    } else {
        if (!find_block<kBM>(p.ends, p.groups, p.rows, p.alignment, blk, g, m0, m_end)) return;
    }
    const uint16_t* b = static_cast<const uint16_t*>(p.b) + (KIND == kRaggedTN ? 0 : (int64_t)g * p.b_gs);

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    for (int kk = k0; kk < k_end; kk += kBK) {
        __syncthreads();
        for (int i = tid; i < kBM * kBK; i += 256) {
            const int r = KIND == kRaggedTN ? i % kBM : i / kBK, k = KIND == kRaggedTN ? i / kBM : i % kBK;
            const bool in = m0 + r < m_end && kk + k < k_end;
            s_a[r * kPitch + k] =
                !in ? (uint16_t)0
                    : KIND == kRaggedTN ? p.a[(int64_t)(kk + k) * p.lda + m0 + r] : p.a[(int64_t)(m0 + r) * p.lda + kk + k];
        }
        for (int i = tid; i < kBN * kBK; i += 256) {
            const int c = KIND == kRaggedNT ? i / kBK : i % kBN, k = KIND == kRaggedNT ? i % kBK : i / kBN;
            const bool in = n0 + c < p.n && kk + k < k_end;
            s_b[c * kPitch + k] = !in                 ? (uint16_t)0
                                  : KIND == kRaggedNT ? b[(int64_t)(n0 + c) * p.ldb + kk + k]
                                                      : load_b(p, kk + k, n0 + c, b);
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < kBK / 16; ++ks) {
            const int off = ks * 16 + (lane >> 5) * 8;
            bf16x8 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const bf16x8*>(&s_a[(wm + i * 32 + (lane & 31)) * kPitch + off]);
                fb[i] = *reinterpret_cast<const bf16x8*>(&s_b[(wn + i * 32 + (lane & 31)) * kPitch + off]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
        }
    }
    // lane: row lane & 31 of D, columns 8 (e / 4) + 4 (lane >> 5) + e % 4
    const int64_t d_off = KIND == kRaggedTN ? (int64_t)g * p.d_gs : 0, c_off = (int64_t)g * p.c_gs;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = m0 + wm + i * 32 + (lane & 31), c = n0 + wn + j * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                if (r >= m_end || c >= p.n) continue;
                float v = acc[i][j][e];
                const int64_t at = c_off + (int64_t)r * p.ldc + c;
                if (p.c) v += p.out_f32 ? static_cast<const float*>(p.c)[at] : bf16_to_f32(static_cast<const uint16_t*>(p.c)[at]);
                const int64_t to = d_off + (int64_t)r * p.ldd + c;
                if (p.out_f32) static_cast<float*>(p.d)[to] = v;
                else static_cast<uint16_t*>(p.d)[to] = bf16_bits(v);
            }
}

}  // namespace

void launch_ragged_gemm(RaggedKind kind, const RaggedGemmArgs& a, hipStream_t stream) {
    const int64_t nb = (a.n + kBN - 1) / kBN;
    // (row blocks at most: whole ones, and one partial block for each group that has rows)
    const int64_t mb = kind == kRaggedTN ? (int64_t)a.groups * ((a.m + kBM - 1) / kBM)
                                         : a.rows / kBM + std::min<int64_t>(a.groups, a.rows);
    DG_CHECK(mb * nb < ((int64_t)1 << 31));
    const dim3 grid((unsigned)(mb * nb)), block(256);
    switch (kind) {
        case kRaggedNT: hipLaunchKernelGGL(ragged_gemm_kernel<kRaggedNT>, grid, block, 0, stream, a, (int)nb); break;
        case kRaggedNN: hipLaunchKernelGGL(ragged_gemm_kernel<kRaggedNN>, grid, block, 0, stream, a, (int)nb); break;
        case kRaggedTN: hipLaunchKernelGGL(ragged_gemm_kernel<kRaggedTN>, grid, block, 0, stream, a, (int)nb); break;
    }
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
