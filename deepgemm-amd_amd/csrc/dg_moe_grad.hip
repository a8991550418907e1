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
// up to 8 slots are on their way at a time. 8192 tokens x 8 slots of 7168 columns: 179 us (5.9 TB/s)
// and 395 us (5.0 TB/s; a copy 5.1); 33 x 8 of 1024 2.9 and 5.5 us in a graph.
#include <hip/hip_runtime.h>

#include "dg_internal.hpp"
#include "dg_kernel_common.hpp"

namespace dgm {
namespace {

using namespace dev;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
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

// 8 values of a row. STREAM: past the caches' usual order, for what is read once; see stream_rows.
template <bool STREAM>
__device__ __forceinline__ uint4 load8(const uint16_t* from) {
    if constexpr (STREAM) {
        const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from));
        return uint4{v.x, v.y, v.z, v.w};
    } else {
        return *reinterpret_cast<const uint4*>(from);
    }
}
__device__ __forceinline__ void store8(uint16_t* to, const uint4& v) {
    __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(to));
}

// Lane j < k: the row of the token's slot j, or -1 (also for what is no row).
__device__ __forceinline__ int lane_row(const MoeGradArgs& p, int64_t t, int lane) {
    const int r = lane < p.k ? p.pos[t * p.k + lane] : -1;
    return r < p.rows ? r : -1;
}

// One wave per (token, 512 columns).
template <bool STREAM>
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
            if (r >= 0) v[q] = load8<STREAM>(p.rows_in + row_at(r, p.max_m, p.ld_in, p.gs_in) + col);
        }
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            float x[8];
            unpack8(v[q], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += x[e];
        }
    }
    store8(p.tokens + t * p.ldt + col, pack8(acc));
}

// WPT waves per token: one for each 512 columns, up to four, or, for few tokens, up to 16. dw: each
// lane's columns in order, then the lanes of a wave, then the waves, always in the same order.
template <int WPT, bool STREAM>
__global__ void __launch_bounds__(WPT > 4 ? WPT * 64 : 256) combine_backward_kernel(const MoeGradArgs p) {
    constexpr int NW = WPT > 4 ? WPT : 4;
    __shared__ float s_dw[NW][kMoeMaxTopk];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = (int64_t)blockIdx.x * (NW / WPT) + wave / WPT;
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
                    if (p.w && r >= 0) v[q] = load8<STREAM>(p.rows_in + row_at(r, p.max_m, p.ld_in, p.gs_in) + col);
                }
                float d[8];
                unpack8(raw, d);
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    const int r = __builtin_amdgcn_readlane(row, j + q);
                    if (r < 0) continue;   // wave-uniform
                    uint16_t* to = p.rows_out + row_at(r, p.max_m, p.ld_out, p.gs_out) + col;
                    if (!p.w) {
                        store8(to, raw);
                        continue;
                    }
                    const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), j + q));
                    float y[8], o[8];
                    unpack8(v[q], y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot[q] += d[e] * y[e], o[e] = w * d[e];
                    store8(to, pack8(o));
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

// Routed rows larger than the 256 MB of the last cache would push each other out of it: from 100 MB of
// them on, their loads are nontemporal. Plain / nontemporal, us (dispatch; combination, whose stores
// are nontemporal in both): 2048 tokens x 8 of 2048 columns (67 MB) 12.8/13.5; 24.3/29.7, 1024 x 8 of
// 7168 (117 MB) 24.6/23.0; 52.4/49.5, 16384 x 2 of 4096 (268 MB) 74.9/71.8; 129/126, 8192 x 8 of 7168
// (940 MB) 193/180; 400/396. Plain stores: 13.0; 32.5, 25.0; 53.9, 79.3; 132, 205; 403.
bool stream_rows(const MoeGradArgs& a) { return (int64_t)a.t * a.k * a.n >= 50'000'000; }

template <int WPT>
void run_combine_backward(const MoeGradArgs& a, dim3 grid, dim3 block, hipStream_t stream) {
    if (stream_rows(a)) hipLaunchKernelGGL((combine_backward_kernel<WPT, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((combine_backward_kernel<WPT, false>), grid, block, 0, stream, a);
}

}  // namespace

void launch_dispatch_backward(const MoeGradArgs& a, hipStream_t stream) {
    if (a.t == 0) return;
    const int64_t slices = a.n > 0 ? (a.n + 511) / 512 : 1, blocks = dispatch_backward_blocks(a.t, a.n);
    DG_CHECK_GRID(blocks, 256);
    const dim3 grid((unsigned)blocks), block(256);
    if (stream_rows(a)) hipLaunchKernelGGL(dispatch_backward_kernel<true>, grid, block, 0, stream, a, (int)slices);
    else hipLaunchKernelGGL(dispatch_backward_kernel<false>, grid, block, 0, stream, a, (int)slices);
    DG_HIP_CHECK(hipGetLastError());
}

void launch_combine_backward(const MoeGradArgs& a, hipStream_t stream) {
    if (a.t == 0) return;
    const int64_t blocks = combine_backward_blocks(a.t, a.n);
    const int threads = combine_backward_threads(a.t, a.n);
    DG_CHECK_GRID(blocks, threads);
    const dim3 grid((unsigned)blocks), block(threads);
    switch (moe_grad_waves(a.t, a.n)) {
        case 1: run_combine_backward<1>(a, grid, block, stream); break;
        case 2: run_combine_backward<2>(a, grid, block, stream); break;
        case 4: run_combine_backward<4>(a, grid, block, stream); break;
        case 8: run_combine_backward<8>(a, grid, block, stream); break;
        default: run_combine_backward<16>(a, grid, block, stream); break;
    }
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
