// Per-token cast of BF16 activations or weights to e2m1 codes, and back (gfx950).
//
// Cast, per group of `gran` columns of a row (the arithmetic of the torch form in
// deep_gemm/utils/math.py, to the bit):
//   amax = max |x|, at least 1e-4;  sf = amax * fl32(1 / 6), up to a power of two with UE8M0;
//   code = e2m1(x * fl32(1 / sf)), round to nearest even, at most 6, no negative zero; NaN
//   takes the code of 6.
// Columns past the last are zeros for their group, and scales past the last in a word are 1.
// Back: value = code * sf in FP32 (an UE8M0 byte e is the float of exponent bits e), rounded
// once to BF16 where that is asked for: exact there for powers of two.
//
// HBM-bound: 2 bytes in and 1/2 out an element (and the reverse), plus the scales. A lane has 8
// columns, 16 bytes of BF16 and 4 of codes; a wave converts 1024 columns of a row, both of its
// loads issued first (four: 170 us against 111); the gran / 8 lanes of a group find its largest magnitude by shuffles. BF16 and
// FP32 values pass by the caches' order (nontemporal: plain / so, us: cast of 16384 x 7168 111/98,
// 65536 x 2048 159/110, 4096 x 7168 28/28; back, 16384 x 7168, to BF16 69/41, to FP32 143/74); codes do not, which the
// next kernel reads (nontemporal as well: 117 and 137 for the casts). Alone, 16384 x 7168: cast 58 us (5.2 TB/s), back 40 us (7.4 TB/s).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "dg_internal.hpp"
#include "dg_kernel_common.hpp"

namespace dgm {
namespace {

using namespace dev;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;      // rows per workgroup, one wave each
constexpr int kChunk = 512;    // columns of a wave-wide access (64 lanes x 8)
constexpr int kChunks = 2;     // loaded before converting
constexpr int kSlice = kChunk * kChunks;

// e2m1 code of v as the torch form gives it (the boundaries' ties go to the even code).
__device__ __forceinline__ uint32_t e2m1_code_slow(float v) {
    const float a = fabsf(v);
    if (!(a <= 6.0f)) return v < 0.f ? 15u : 7u;   // (NaN: 7)
    const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
    return c | (v < 0.f && c ? 8u : 0u);
}

// 8 codes without negative zeros.
__device__ __forceinline__ uint32_t without_negative_zeros(uint32_t w) {
    const uint32_t any = (w | w >> 1 | w >> 2) & 0x11111111u;   // (bits of one code only meet at its lowest)
    return w & (0x77777777u | any << 3);
}

// Row slice and columns of a workgroup: each XCD takes a contiguous range of them.
struct Slice {
    int row, col;
    __device__ __forceinline__ Slice(int slices) {
        const int lw = xcd_remap(blockIdx.x, gridDim.x);
        const int rb = lw / slices;
        row = rb * kWaves + (int)(threadIdx.x >> 6);
        col = (lw - rb * slices) * kSlice;
    }
};

// VEC: rows begin at whole 16-byte (x) and 4-byte (codes) pieces.
template <int GRAN, int VEC>
__global__ void __launch_bounds__(kWaves * 64) cast4_kernel(const Cast4Args p, int slices) {
    constexpr int TPG = GRAN / 8;   // lanes of a group
    const Slice s(slices);
    if (s.row >= p.m) return;   // wave-uniform
    const int lane = threadIdx.x & 63;
    const uint16_t* xr = p.x + (int64_t)s.row * p.ldx;
    uint8_t* qr = p.q + (int64_t)s.row * p.ldq;
    const int groups = (p.n + GRAN - 1) / GRAN;
    uint4 raw[kChunks];
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
        const int col = s.col + u * kChunk + lane * 8;
        if (VEC && col + 8 <= p.n) {
            const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(xr + col));
            raw[u] = uint4{v.x, v.y, v.z, v.w};
        } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)   // (n is even)
                w[e] = col + 2 * e < p.n ? xr[col + 2 * e] | (uint32_t)xr[col + 2 * e + 1] << 16 : 0u;
            raw[u] = uint4{w[0], w[1], w[2], w[3]};
        }
    }
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
        const int col = s.col + u * kChunk + lane * 8;
        if (s.col + u * kChunk >= p.n) continue;   // wave-uniform
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        // Largest magnitude by the bit patterns: |bf16| orders as its 15 low bits, a NaN above all.
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        u16x2 m2 = u16x2{0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(u16x2, w[e] & 0x7FFF7FFFu));
        uint32_t amax = (uint32_t)(m2.x > m2.y ? m2.x : m2.y) << 16;
#pragma unroll
        for (int o = TPG / 2; o > 0; o >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, o));
        amax = max(amax, 0x38D1B717u);   // 1e-4f
        float sf = __fmul_rn(__uint_as_float(amax), 1.0f / 6.0f);
        if (p.ue8m0) {
            const uint32_t b = __float_as_uint(sf);
            sf = __uint_as_float(min((b >> 23) + ((b & 0x7FFFFFu) != 0 ? 1u : 0u), 254u) << 23);
        }
        const float inv = __fdiv_rn(1.0f, sf);
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __fmul_rn(__uint_as_float(w[e] << 16), inv);
            v[2 * e + 1] = __fmul_rn(__uint_as_float(w[e] & 0xFFFF0000u), inv);
        }
        uint32_t codes = 0;
        if (__builtin_expect(__ballot(amax >= 0x7F800000u) == 0, 1)) {
            // |v| is at most 6 (1 + 2^-22), which the conversion rounds and saturates as above
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], 1.0f, 0);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], 1.0f, 1);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], 1.0f, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], 1.0f, 3);
            codes = without_negative_zeros(codes);
        } else {   // an Inf or NaN in a group of the wave
#pragma unroll
            for (int e = 0; e < 8; ++e) codes |= e2m1_code_slow(v[e]) << (4 * e);
        }
        if (VEC && col + 8 <= p.n) {
            *reinterpret_cast<uint32_t*>(qr + col / 2) = codes;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + 2 * e < p.n) qr[col / 2 + e] = (uint8_t)(codes >> (8 * e));
        }
        const int group = col / GRAN;
        if (!p.packed) {
            if (lane % TPG == 0 && group < groups)
                static_cast<float*>(p.sf)[(int64_t)s.row * p.sf_sm + (int64_t)group * p.sf_sk] = sf;
        } else {
            // four groups to a word (an access begins at a word)
            const uint32_t byte = group < groups ? __float_as_uint(sf) >> 23 : 127u;
            const uint32_t b1 = __shfl_down(byte, TPG), b2 = __shfl_down(byte, 2 * TPG), b3 = __shfl_down(byte, 3 * TPG);
            if (lane % (4 * TPG) == 0 && group < groups)
                static_cast<uint32_t*>(p.sf)[(int64_t)s.row * p.sf_sm + (int64_t)(group / 4) * p.sf_sk] =
                    byte | b1 << 8 | b2 << 16 | b3 << 24;
        }
    }
}

// A lane's W values fill 16 bytes, so that a wave's store is one stretch: W is 8 for BF16, 4 for FP32.
// VEC: rows begin at whole W / 2-byte (codes) and 16-byte (values) pieces.
template <int GRAN, int VEC, int W>
__global__ void __launch_bounds__(kWaves * 64) cast_back4_kernel(const Cast4Args p, int slices) {
    constexpr int CHUNK = 64 * W, CHUNKS = kSlice / CHUNK;
    using Codes = std::conditional_t<W == 8, uint32_t, uint16_t>;
    const Slice s(slices);
    if (s.row >= p.m) return;   // wave-uniform
    const int lane = threadIdx.x & 63;
    const uint8_t* qr = p.q + (int64_t)s.row * p.ldq;
    uint32_t codes[CHUNKS];
    float sf[CHUNKS];
#pragma unroll
    for (int u = 0; u < CHUNKS; ++u) {
        const int col = s.col + u * CHUNK + lane * W;
        codes[u] = 0, sf[u] = 0.f;
        if (VEC && col + W <= p.n) {
            codes[u] = *reinterpret_cast<const Codes*>(qr + col / 2);
        } else {
#pragma unroll
            for (int e = 0; e < W / 2; ++e)
                if (col + 2 * e < p.n) codes[u] |= (uint32_t)qr[col / 2 + e] << (8 * e);
        }
        if (col < p.n) {
            const int group = col / GRAN;
            if (p.packed) {
                const uint32_t w = static_cast<const uint32_t*>(p.sf)[(int64_t)s.row * p.sf_sm + (int64_t)(group >> 2) * p.sf_sk];
                sf[u] = __uint_as_float((w >> (8 * (group & 3)) & 0xFFu) << 23);
            } else {
                sf[u] = static_cast<const float*>(p.sf)[(int64_t)s.row * p.sf_sm + (int64_t)group * p.sf_sk];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < CHUNKS; ++u) {
        const int col = s.col + u * CHUNK + lane * W;
        if (col >= p.n) continue;
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        float v[W];
        auto pair = [&](auto at) {
            constexpr int e = decltype(at)::value;
            const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[u], 1.0f, e);
            v[2 * e] = __fmul_rn(c.x, sf[u]), v[2 * e + 1] = __fmul_rn(c.y, sf[u]);
        };
        pair(std::integral_constant<int, 0>{});
        pair(std::integral_constant<int, 1>{});
        if constexpr (W == 8) {
            pair(std::integral_constant<int, 2>{});
            pair(std::integral_constant<int, 3>{});
        }
        const int64_t at = (int64_t)s.row * p.ldx + col;
        const bool whole = VEC && col + W <= p.n;
        if constexpr (W == 4) {
            float* y = static_cast<float*>(p.y) + at;
            if (whole) {
                __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(y));
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if (col + e < p.n) y[e] = v[e];
            }
        } else {
            uint16_t* y = static_cast<uint16_t*>(p.y) + at;
            if (whole) {
                __builtin_nontemporal_store(u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                                  pack_bf16x2(v[6], v[7])}, reinterpret_cast<u32x4*>(y));
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if (col + e < p.n) y[e] = bf16_bits(v[e]);
            }
        }
    }
}

bool aligned(const void* p, int64_t pitch_bytes, int64_t to) { return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)pitch_bytes) % to == 0; }

template <typename F>
void by_gran(int gran, bool vec, F&& launch) {
    auto with = [&](auto g) {
        if (vec) launch(g, std::integral_constant<int, 1>{});
        else launch(g, std::integral_constant<int, 0>{});
    };
    switch (gran) {
        case 32: with(std::integral_constant<int, 32>{}); break;
        case 64: with(std::integral_constant<int, 64>{}); break;
        case 128: with(std::integral_constant<int, 128>{}); break;
        default: DG_UNSUPPORTED("4-bit cast: gran_k must be 32, 64 or 128");
    }
}

}  // namespace

void launch_cast4(const Cast4Args& a, hipStream_t stream) {
    if (a.m == 0 || a.n == 0) return;
    const int64_t blocks = cast4_blocks(a.m, a.n);
    DG_CHECK_GRID(blocks, kWaves * 64);
    by_gran(a.gran, aligned(a.x, a.ldx * 2, 16) && aligned(a.q, a.ldq, 4), [&](auto gran, auto vec) {
        hipLaunchKernelGGL((cast4_kernel<decltype(gran)::value, decltype(vec)::value>), dim3((unsigned)blocks),
                           dim3(kWaves * 64), 0, stream, a, (a.n + kSlice - 1) / kSlice);
    });
    DG_HIP_CHECK(hipGetLastError());
}

void launch_cast_back4(const Cast4Args& a, hipStream_t stream) {
    if (a.m == 0 || a.n == 0) return;
    const int64_t blocks = cast4_blocks(a.m, a.n);
    DG_CHECK_GRID(blocks, kWaves * 64);
    by_gran(a.gran, aligned(a.y, a.ldx * (a.out_f32 ? 4 : 2), 16) && aligned(a.q, a.ldq, a.out_f32 ? 2 : 4),
            [&](auto gran, auto vec) {
        constexpr int G = decltype(gran)::value, V = decltype(vec)::value;
        const dim3 grid((unsigned)blocks), block(kWaves * 64);
        const int slices = (a.n + kSlice - 1) / kSlice;
        if (a.out_f32) hipLaunchKernelGGL((cast_back4_kernel<G, V, 4>), grid, block, 0, stream, a, slices);
        else hipLaunchKernelGGL((cast_back4_kernel<G, V, 8>), grid, block, 0, stream, a, slices);
    });
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
