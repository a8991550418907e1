// Gradients of an MoE layer's dispatch and combination (gfx950).
//
// pos[t, j] is the row of token t's slot j (-1: not routed, skipped).
//   Dispatch     a[pos[t, j]] = x[t], row_w[pos[t, j]] = w[t, j]:
//     dx[t] = sum over j of drows[pos[t, j]] (FP32, in the slots' order, rounded once),
//     dw[t, j] = drow_w[pos[t, j]].
//   Combination  out[t] = sum over j of w[t, j] y[pos[t, j]]:
//     dy[pos[t, j]] = w[t, j] dout[t] (rounded once; copied without w),
//     dw[t, j] = sum over the columns of dout[t] y[pos[t, j]] (FP32).
// Both are bound by HBM: every routed row is read once (dispatch), or read and written once
// (combination), beside a row for each token. A lane owns 8 columns (16 bytes); the rows of
// up to 8 slots are on their way at a time.
#include <hip/hip_runtime.h>

#include "dg_internal.hpp"
#include "dg_kernel_common.hpp"

namespace dgm {
namespace {

using namespace dev;
constexpr int kBatch = 8;   // slots whose rows are loaded at a time

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return uint4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

__device__ __forceinline__ int64_t row_at(int r, int max_m, int64_t ld, int64_t gs) {
    return max_m ? (int64_t)(r / max_m) * gs + (int64_t)(r % max_m) * ld : (int64_t)r * ld;
}

// Lane j < k: the row of the token's slot j, or -1 (also for what is no row).
__device__ __forceinline__ int lane_row(const MoeGradArgs& p, int64_t t, int lane) {
    const int r = lane < p.k ? p.pos[t * p.k + lane] : -1;
    return r < p.rows ? r : -1;
}

// One wave per (token, 512 columns).
__global__ void __launch_bounds__(256) dispatch_backward_kernel(const MoeGradArgs p, int slices) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tb = blockIdx.x / slices, slice = blockIdx.x - tb * slices;
    const int64_t t = (int64_t)tb * 4 + wave;
    if (t >= p.t) return;   // wave-uniform
    const int row = lane_row(p, t, lane);
    if (slice == 0 && p.dw && lane < p.k) p.dw[t * p.k + lane] = row >= 0 ? p.w[row] : 0.f;
    const int col = slice * 512 + lane * 8;
    if (col >= p.n) return;
    float acc[8] = {};
    for (int j = 0; j < p.k; j += kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const int r = __builtin_amdgcn_readlane(row, j + q);   // (lanes from k on hold -1)
            v[q] = uint4{0, 0, 0, 0};
            if (r >= 0) v[q] = *reinterpret_cast<const uint4*>(p.rows_in + row_at(r, p.max_m, p.ld_in, p.gs_in) + col);
        }
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            float x[8];
            unpack8(v[q], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += x[e];
        }
    }
    *reinterpret_cast<uint4*>(p.tokens + t * p.ldt + col) = pack8(acc);
}

// WPT waves per token (1, 2 or 4, one for each 512 columns up to four). dw: each lane's
// columns in order, then the lanes of a wave, then the waves, always in the same order.
template <int WPT>
__global__ void __launch_bounds__(256) combine_backward_kernel(const MoeGradArgs p) {
    __shared__ float s_dw[4][kMoeMaxTopk];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = (int64_t)blockIdx.x * (4 / WPT) + wave / WPT;
    const bool live = t < p.t;
    if (live) {
        const int row = lane_row(p, t, lane);
        const float weight = p.w && lane < p.k ? p.w[t * p.w_st + lane * p.w_sk] : 1.f;
        for (int j = 0; j < p.k; j += kBatch) {
            float dot[kBatch] = {};
            for (int col = (wave % WPT) * 512 + lane * 8; col < p.n; col += WPT * 512) {
                const uint4 raw = *reinterpret_cast<const uint4*>(p.tokens + t * p.ldt + col);
                uint4 v[kBatch];
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    const int r = __builtin_amdgcn_readlane(row, j + q);
                    if (p.w && r >= 0) v[q] = *reinterpret_cast<const uint4*>(p.rows_in + row_at(r, p.max_m, p.ld_in, p.gs_in) + col);
                }
                float d[8];
                unpack8(raw, d);
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    const int r = __builtin_amdgcn_readlane(row, j + q);
                    if (r < 0) continue;   // wave-uniform
                    uint16_t* to = p.rows_out + row_at(r, p.max_m, p.ld_out, p.gs_out) + col;
                    if (!p.w) {
                        *reinterpret_cast<uint4*>(to) = raw;
                        continue;
                    }
                    const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), j + q));
                    float y[8], o[8];
                    unpack8(v[q], y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot[q] += d[e] * y[e], o[e] = w * d[e];
                    *reinterpret_cast<uint4*>(to) = pack8(o);
                }
            }
            if (!p.dw) continue;
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) dot[q] += __shfl_xor(dot[q], o);
                if (lane == 0 && j + q < p.k) s_dw[wave][j + q] = dot[q];
            }
        }
    }
    if (!p.dw) return;   // uniform over the launch
    __syncthreads();
    if (live && wave % WPT == 0 && lane < p.k) {
        float sum = s_dw[wave][lane];
#pragma unroll
        for (int i = 1; i < WPT; ++i) sum += s_dw[wave + i][lane];
        p.dw[t * p.k + lane] = sum;
    }
}

}  // namespace

void launch_dispatch_backward(const MoeGradArgs& a, hipStream_t stream) {
    if (a.t == 0) return;
    const int64_t slices = a.n > 0 ? (a.n + 511) / 512 : 1, blocks = dispatch_backward_blocks(a.t, a.n);
    DG_CHECK_GRID(blocks, 256);
    hipLaunchKernelGGL(dispatch_backward_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a, (int)slices);
    DG_HIP_CHECK(hipGetLastError());
}

void launch_combine_backward(const MoeGradArgs& a, hipStream_t stream) {
    if (a.t == 0) return;
    const int64_t blocks = combine_backward_blocks(a.t, a.n);
    DG_CHECK_GRID(blocks, 256);
    const dim3 grid((unsigned)blocks), block(256);
    switch (moe_grad_waves(a.n)) {
        case 1: hipLaunchKernelGGL(combine_backward_kernel<1>, grid, block, 0, stream, a); break;
        case 2: hipLaunchKernelGGL(combine_backward_kernel<2>, grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL(combine_backward_kernel<4>, grid, block, 0, stream, a); break;
    }
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
