// SwiGLU x routing weight with an 8-bit checkpoint of its input, and its backward pass
// from the checkpoint (gfx950).
//
// Forward, for a row of gate g and up u (BF16 [2I], halves of I columns) with weight w:
//   h = silu(g) u w, silu(g) = g s, s = 1 / (1 + exp(-g)), in FP32, rounded once to BF16;
//   checkpoint: e4m3 codes of g and u with one power-of-two scale per 128 columns of each
//   half (the per-token cast's arithmetic: amax clamped at 1e-4, times fl32(1/448), up to
//   a power of two), so that code x scale is exact in BF16.
// Backward, from g and u as the checkpoint holds them and the gradient dh of h:
//   h  = g s u w (recomputed for the weight gradient of the next product)
//   du = dh w g s,  dg = dh w u s (1 + g (1 - s)),  dw = sum over the row of dh g s u.
// With a clamp c, u is clamped to [-c, c] and g to at most c before all of it, and du, dg
// are zero where the clamp holds the value (|u| > c, g > c).
// Both are one pass over HBM, which bounds them: forward 8 bytes per element of h (4 in, 2 +
// 2 out), backward 10 (2 + 2 in, 4 + 2 out). A lane owns 8 columns: 16-byte accesses of the
// BF16 rows, 8 of the codes. 16384 x 2048: forward 48.6 us (5.6 TB/s; the kernel alone 43),
// backward 60.7 (5.6 TB/s), a copy of 1 GiB 5.1 TB/s; the exponentials and reciprocals hide
// under it. (Columns in whole 512s; the forward pass gives a wave 512 of them, so at 768 a
// quarter of the lanes have nothing to do, at 520 almost half.) 33 x 1024: 9 us a call, of which the kernel 4.
#include <hip/hip_runtime.h>

#include "dg_internal.hpp"
#include "dg_swiglu.hpp"

namespace dgm {
namespace {

using namespace dev;
constexpr int kSwThreads = 256;

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

// s = 1 / (1 + exp(-g)) by the hardware's exponential and reciprocal: off by (|g| + 8) 2^-23 of
// itself at most (the exponent is an FP32 product), beside BF16's half step of 2^-8 in all
// results but dw; zero below g = -87.3, NaN for NaN.
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// The power-of-two scale and the codes of one lane's 8 values, the group being the 16
// lanes of its row of lanes (every lane of the wave calls it). A NaN orders above every
// number in the bit patterns, as in the per-token cast.
__device__ __forceinline__ uint2 quantize_pow2(const uint4& raw, float& sf_out) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    u16x2 m2 = u16x2{0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(u16x2, w[e] & 0x7FFF7FFFu));
    uint32_t amax = (uint32_t)(m2.x > m2.y ? m2.x : m2.y) << 16;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, o));
    amax = max(amax, 0x38D1B717u);   // 1e-4f
    const uint32_t b = __float_as_uint(f32_mul(__uint_as_float(amax), 1.0f / 448.0f));
    const uint32_t e8 = min(((b >> 23) & 0xFFu) + ((b & 0x7FFFFFu) != 0 ? 1u : 0u), 254u);
    sf_out = __uint_as_float(e8 << 23);
    const float inv = __uint_as_float(e8 < 254u ? (254u - e8) << 23 : 0x00400000u);   // 1 / sf, exact
    float v[8];
    unpack8(raw, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f32_mul(v[e], inv);
    uint32_t lo = 0, hi = 0;
    if (__builtin_expect(__ballot(amax >= 0x7F800000u) == 0, 1)) {
        int l = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        l = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], l, true);
        int h = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
        h = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], h, true);
        lo = (uint32_t)l, hi = (uint32_t)h;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo |= e4m3_code_slow(v[e]) << (8 * e);
            hi |= e4m3_code_slow(v[4 + e]) << (8 * e);
        }
    }
    return uint2{lo, hi};
}

// One wave per (row, 512 columns of h).
__global__ void __launch_bounds__(kSwThreads) swiglu_checkpoint_kernel(const SwigluCheckpointArgs p, int slices) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rb = blockIdx.x / slices, slice = blockIdx.x - rb * slices;
    const int row = rb * (kSwThreads / 64) + wave;
    if (row >= p.m) return;   // wave-uniform
    const int col = slice * 512 + lane * 8;
    const bool in = col < p.n;   // p.n % 8 == 0 (host check)
    const bool skip = p.row_layout && p.row_layout[row] < 0;
    uint4 graw{0, 0, 0, 0}, uraw{0, 0, 0, 0};
    if (in && !skip) {
        const uint16_t* xr = p.x + (int64_t)row * p.ldx;
        graw = *reinterpret_cast<const uint4*>(xr + col);
        uraw = *reinterpret_cast<const uint4*>(xr + p.n + col);
    }
    const float w = p.row_weight ? p.row_weight[row] : 1.f;
    float g[8], u[8], h[8];
    unpack8(graw, g), unpack8(uraw, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (p.clamp > 0.f) {
            g[e] = g[e] > p.clamp ? p.clamp : g[e];   // (NaN stays)
            u[e] = u[e] > p.clamp ? p.clamp : u[e] < -p.clamp ? -p.clamp : u[e];
        }
        h[e] = skip ? 0.f : g[e] * sigmoid(g[e]) * u[e] * w;
    }
    float sg, su;
    const uint2 qg = quantize_pow2(graw, sg), qu = quantize_pow2(uraw, su);
    if (!in) return;
    *reinterpret_cast<uint4*>(p.h + (int64_t)row * p.ldh + col) = pack8(h);
    uint8_t* qr = p.q + (int64_t)row * p.ldq;
    *reinterpret_cast<uint2*>(qr + col) = qg;
    *reinterpret_cast<uint2*>(qr + p.n + col) = qu;
    if ((lane & 15) == 0) {
        float* s = p.sf + (int64_t)row * p.sf_sm;
        s[(int64_t)(col >> 7) * p.sf_sk] = sg;
        s[(int64_t)((p.n + 127) / 128 + (col >> 7)) * p.sf_sk] = su;
    }
}

__device__ __forceinline__ void decode8(const uint2& q, float sf, float (&x)[8]) {
    const uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
        x[4 * i] = lo[0] * sf, x[4 * i + 1] = lo[1] * sf, x[4 * i + 2] = hi[0] * sf, x[4 * i + 3] = hi[1] * sf;
    }
}

// WPR waves per row (1, 2 or 4, one for each 512 columns of h up to four), 4 / WPR rows per workgroup.
// dw: each lane's columns in order, then the lanes of a wave, then the waves, always in
// the same order.
template <int WPR>
__global__ void __launch_bounds__(kSwThreads) swiglu_backward_kernel(const SwigluBackwardArgs p) {
    __shared__ float s_dw[kSwThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (kSwThreads / 64 / WPR) + wave / WPR;
    const bool live = row < p.m;
    const bool skip = live && p.row_layout && p.row_layout[row] < 0;
    float dw = 0.f;
    if (live) {
        const float w = p.row_weight ? p.row_weight[row] : 1.f;
        const uint16_t* dhr = p.dh + row * p.lddh;
        const uint8_t* qr = p.q + row * p.ldq;
        const float* sr = p.sf + row * p.sf_sm;
        uint16_t* dxr = p.dx + row * p.lddx;
        uint16_t* hr = p.h + row * p.ldh;
        const int parts = (p.n + 127) / 128;
        for (int col = (wave % WPR) * 512 + lane * 8; col < p.n; col += WPR * 512) {
            float g[8], u[8], dh[8], dg[8], du[8], h[8];
            if (!skip) {
                const uint4 draw = *reinterpret_cast<const uint4*>(dhr + col);
                const uint2 qg = *reinterpret_cast<const uint2*>(qr + col);
                const uint2 qu = *reinterpret_cast<const uint2*>(qr + p.n + col);
                const float sg = sr[(int64_t)(col >> 7) * p.sf_sk], su = sr[(int64_t)(parts + (col >> 7)) * p.sf_sk];
                unpack8(draw, dh), decode8(qg, sg, g), decode8(qu, su, u);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (skip) {
                    dg[e] = du[e] = h[e] = 0.f;
                    continue;
                }
                bool free_g = true, free_u = true;
                if (p.clamp > 0.f) {
                    free_g = !(g[e] > p.clamp), free_u = !(fabsf(u[e]) > p.clamp);
                    g[e] = free_g ? g[e] : p.clamp;
                    u[e] = free_u ? u[e] : __builtin_copysignf(p.clamp, u[e]);
                }
                const float s = sigmoid(g[e]), act = g[e] * s, dy = dh[e] * w;
                dw += dh[e] * act * u[e];
                h[e] = act * u[e] * w;
                du[e] = free_u ? dy * act : 0.f;
                dg[e] = free_g ? dy * u[e] * (s + act * (1.0f - s)) : 0.f;
            }
            *reinterpret_cast<uint4*>(dxr + col) = pack8(dg);
            *reinterpret_cast<uint4*>(dxr + p.n + col) = pack8(du);
            *reinterpret_cast<uint4*>(hr + col) = pack8(h);
        }
    }
    if (p.dw == nullptr) return;   // uniform over the launch
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) dw += __shfl_xor(dw, o);
    if constexpr (WPR > 1) {
        if (lane == 0) s_dw[wave] = dw;
        __syncthreads();
        if (wave % WPR == 0)
            for (int i = 1; i < WPR; ++i) dw += s_dw[wave + i];
    }
    if (live && lane == 0 && wave % WPR == 0) p.dw[row] = dw;
}

}  // namespace

void launch_swiglu_checkpoint(const SwigluCheckpointArgs& a, hipStream_t stream) {
    if (a.m == 0 || a.n == 0) return;
    const int64_t blocks = swiglu_checkpoint_blocks(a.m, a.n);
    DG_CHECK_GRID(blocks, kSwThreads);
    hipLaunchKernelGGL(swiglu_checkpoint_kernel, dim3((unsigned)blocks), dim3(kSwThreads), 0, stream, a, (a.n + 511) / 512);
    DG_HIP_CHECK(hipGetLastError());
}

void launch_swiglu_backward(const SwigluBackwardArgs& a, hipStream_t stream) {
    if (a.m == 0) return;
    const int64_t blocks = swiglu_backward_blocks(a.m, a.n);
    DG_CHECK_GRID(blocks, kSwThreads);
    const dim3 grid((unsigned)blocks), block(kSwThreads);
    switch (swiglu_backward_waves(a.n)) {
        case 1: hipLaunchKernelGGL(swiglu_backward_kernel<1>, grid, block, 0, stream, a); break;
        case 2: hipLaunchKernelGGL(swiglu_backward_kernel<2>, grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL(swiglu_backward_kernel<4>, grid, block, 0, stream, a); break;
    }
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
