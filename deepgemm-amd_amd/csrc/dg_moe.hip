// MoE plumbing around the grouped GEMMs on one GPU (gfx950): dispatch of
// token-major FP8, BF16 or 4-bit activations into the expert-grouped layouts the grouped GEMMs
// read, the fused SwiGLU x routing-weight -> FP8 cast between the two grouped
// GEMMs, and combine. The reference runs this layer as DeepEP dispatch, L1 GEMM,
// tilelang SwiGLU, L2 GEMM, DeepEP combine (tests/test_mega_moe.py:296-330); the
// layouts are those of its generators (tests/generators.py:383-478).
//
// Dispatch (all integer work, deterministic): each (token t, slot j) routed to
// expert e gets the next row of e's segment, in token-then-slot order. Few tokens: in one launch
// (moe_dispatch_few_kernel); others in three, or four (moe_starts_kernel between the last two):
//   1. count:   per chunk of 64 tokens, one wave ranks the chunk's entries
//               among equal experts with ballots (in entry order; the rank goes
//               to pos) and leaves the chunk's count per expert;
//   2. scan:    one wave per expert: exclusive prefix over chunks, the total,
//               and the masked counts;
//   3. scatter: each workgroup scans the aligned totals into the segment starts
//               (contiguous / psum) and turns its ranks into rows; a wave reads a
//               token's K bytes once and stores them to each routed row, with
//               the SF row, the weight and m_indices; beside them (contiguous /
//               psum) a block per expert fills its padding rows (zero A, SF and
//               weight, m_indices = -1), and some more set m_indices = -1 and zero weights
//               past the segments.
// Bytes: the scatter reads each token row once and writes each routed row once
// (HBM-bound copy); counts and scans touch 4 bytes per entry and per
// (chunk, expert). 8192 tokens x 8 of 7168 BF16 columns, 256 experts: 230 us, 4.7 TB/s (the scatter
// alone 188).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <mutex>
#include <type_traits>

#include "dg_internal.hpp"
#include "dg_swiglu.hpp"

namespace dgm {
namespace {

constexpr int kThreads = 256;
constexpr int kPastBlocks = 16;   // workgroups of the scatter for the rows past the segments
using dev::i32x4;

__device__ __forceinline__ int align_up(int x, int a) { return (x + a - 1) / a * a; }

// Expert id of (token t, slot j); int64 ids outside [0, E) come back as -1
// (unrouted) before the value is narrowed, so 2^32 + e is not taken for e.
__device__ __forceinline__ int topk_at(const MoeDispatchArgs& p, int t, int j) {
    const int64_t off = (int64_t)t * p.topk_st + (int64_t)j * p.topk_sk;
    if (p.topk_i64) {
        const int64_t e = static_cast<const int64_t*>(p.topk)[off];
        return (e >= 0 && e < p.num_experts) ? (int)e : -1;
    }
    return static_cast<const int32_t*>(p.topk)[off];
}

__device__ __forceinline__ bool routed(const MoeDispatchArgs& p, int e) { return e >= 0 && e < p.num_experts; }

// Workspace: counts [E][chunks] (exclusive prefixes over chunks after the
// scan), then totals [E], then, where a launch of their own finds them, the segments' first rows [E + 1].
__device__ __forceinline__ int32_t* ws_counts(const MoeDispatchArgs& p) { return p.ws; }
__device__ __forceinline__ int32_t* ws_totals(const MoeDispatchArgs& p) { return p.ws + (int64_t)p.chunks * p.num_experts; }
__device__ __forceinline__ int32_t* ws_starts(const MoeDispatchArgs& p) { return ws_totals(p) + p.num_experts; }

// Inclusive prefix sum over the 64 lanes of a wave.
__device__ __forceinline__ int wave_inclusive_sum(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// One workgroup per chunk of kMoeChunkTokens tokens. Wave 0 walks the chunk's
// entries in (token, slot) order, 64 at a time: each routed entry's rank among
// the chunk's earlier entries of its expert (ballots over the lanes holding
// that expert) goes to pos[t, j]; the per-expert counts go to counts[e][chunk].
__global__ void __launch_bounds__(kThreads) moe_count_kernel(const MoeDispatchArgs p) {
    __shared__ int run[kMoeMaxExperts];
    __shared__ int ids[kMoeChunkTokens * kMoeMaxTopk];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x;
    const int t0 = c * kMoeChunkTokens;
    const int entries = min(kMoeChunkTokens, p.t - t0) * p.k;
    for (int e = threadIdx.x; e < p.num_experts; e += kThreads) run[e] = 0;
    for (int i = threadIdx.x; i < entries; i += kThreads) ids[i] = topk_at(p, t0 + i / p.k, i % p.k);
    __syncthreads();
    if (wave == 0) {
        for (int b = 0; b < entries; b += 64) {
            const int i = b + lane;
            const int e = i < entries ? ids[i] : -1;
            const bool ok = i < entries && routed(p, e);
            // peers: the routed lanes whose expert id equals this lane's, one
            // ballot per id bit (ids < kMoeMaxExperts = 2^10)
            static_assert(kMoeMaxExperts <= 1024, "expert ids fit 10 bits");
            uint64_t peers = __ballot(ok);
#pragma unroll
            for (int bit = 0; bit < 10; ++bit) {
                const bool set = (e >> bit) & 1;
                const uint64_t m = __ballot(ok && set);
                peers &= set ? m : ~m;
            }
            const uint64_t below = lane ? (~0ull >> (64 - lane)) : 0ull;
            if (ok) {
                const int base = run[e];
                p.pos[(int64_t)t0 * p.k + i] = base + __popcll(peers & below);
                if ((peers >> lane) == 1ull) run[e] = base + __popcll(peers);   // the group's last lane
            }
            // (all lanes read run[] before any lane of this batch writes it: one
            // wave, in program order; the next batch's reads follow the writes)
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.num_experts; e += kThreads)
        ws_counts(p)[(int64_t)e * p.chunks + c] = run[e];
}

// Contiguous and psum layouts, one workgroup: the exclusive prefix of the aligned expert totals
// (E <= 4 * kThreads, 4 experts per thread) gives the segment starts. total(e): expert e's rows;
// start(e, first row, rows). Returns, in the last thread, the rows that the segments use.
template <typename Total, typename Start>
__device__ __forceinline__ int segment_starts(const MoeDispatchArgs& p, Total&& total, Start&& start) {
    static_assert(kMoeMaxExperts <= 4 * kThreads, "4 experts per thread");
    __shared__ int wsum[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int v[4], tot[4], s = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int e = threadIdx.x * 4 + q;
        tot[q] = e < p.num_experts ? total(e) : 0;
        v[q] = align_up(tot[q], p.alignment);
        s += v[q];
    }
    const int incl = wave_inclusive_sum(s, lane);
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int x = incl - s;
    for (int w = 0; w < wave; ++w) x += wsum[w];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int e = threadIdx.x * 4 + q;
        if (e < p.num_experts) start(e, x, tot[q]);
        x += v[q];
    }
    return x;
}

// Contiguous and psum layouts, in four launches: the segments' first rows, once for all, and the psum ends.
__global__ void __launch_bounds__(kThreads) moe_starts_kernel(const MoeDispatchArgs p) {
    const int used = segment_starts(p, [&](int e) { return ws_totals(p)[e]; }, [&](int e, int start, int total) {
        ws_starts(p)[e] = start;
        if (p.layout == kMoePsum) p.meta[e] = start + total;   // psum[e] = align(psum[e-1]) + count
    });
    if (threadIdx.x == kThreads - 1) ws_starts(p)[p.num_experts] = used;
}

// One wave per expert: the exclusive prefix of its chunk counts (in place, 256
// chunks per round, 4 consecutive chunks per lane), its total, and for the
// masked layout masked_m = min(total, max_m).
__global__ void __launch_bounds__(kThreads) moe_scan_kernel(const MoeDispatchArgs p) {
    const int lane = threadIdx.x & 63;
    const int e = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (e >= p.num_experts) return;   // wave-uniform
    int32_t* cnt = ws_counts(p) + (int64_t)e * p.chunks;
    int carry = 0;
    for (int c0 = 0; c0 < p.chunks; c0 += 256) {
        const int c = c0 + lane * 4;
        int v[4], s = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            v[q] = c + q < p.chunks ? cnt[c + q] : 0;
            s += v[q];
        }
        const int incl = wave_inclusive_sum(s, lane);
        int x = carry + incl - s;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (c + q < p.chunks) cnt[c + q] = x;
            x += v[q];
        }
        carry += __shfl(incl, 63);
    }
    if (lane == 0) {
        ws_totals(p)[e] = carry;
        if (p.layout == kMoeMasked) p.meta[e] = min(carry, p.max_m);
    }
}

// Row p of the output layout (flattened for masked: e * max_m + r).
__device__ __forceinline__ int64_t row_a(const MoeDispatchArgs& p, int64_t r) {
    return p.layout == kMoeMasked ? (r / p.max_m) * p.a_gs + (r % p.max_m) * p.lda : r * p.lda;
}
__device__ __forceinline__ int64_t row_sf(const MoeDispatchArgs& p, int64_t r) {
    return p.layout == kMoeMasked ? (r / p.max_m) * p.sf_gs + (r % p.max_m) * p.sf_sm : r * p.sf_sm;
}

// Contiguous and psum layouts: the padding rows [r0, r1) of a segment get zero A, SF and
// weight and m_indices = -1.
__device__ __forceinline__ void pad_rows(const MoeDispatchArgs& p, int r0, int r1) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = r0 + wave; r < r1; r += kThreads / 64) {
        uint8_t* a = p.a + row_a(p, r);
        for (int c = lane * 16; c < p.kdim; c += 64 * 16)
            __builtin_nontemporal_store(i32x4{0, 0, 0, 0}, reinterpret_cast<i32x4*>(a + c));
        for (int c = lane; c < p.sfk; c += 64) p.sf[row_sf(p, r) + (int64_t)c * p.sf_sk_o] = 0.f;
        if (lane == 0) {
            if (p.w_out) p.w_out[r] = 0.f;
            if (p.layout == kMoeContiguous) p.meta[r] = -1;
        }
    }
}
// Past the segments (from row r0 on, every `step`-th): m_indices = -1, weights zero.
__device__ __forceinline__ void pad_past(const MoeDispatchArgs& p, int64_t r0, int64_t step) {
    for (int64_t r = r0; r < p.cap_rows; r += step) {
        if (p.layout == kMoeContiguous) p.meta[r] = -1;
        if (p.w_out) p.w_out[r] = 0.f;
    }
}

// A wave has TOKENS tokens: 1, or 4 short ones. Lane i turns
// the chunk rank of the wave's entry i into its output row (segment start + the expert's prefix over
// earlier chunks + the rank; for the masked layout the slot in the group's buffer, -1 past max_m);
// then the wave stores the tokens' K bytes, read once (8 KB per round of one token, 8 x 16 B per
// lane in flight), to each routed row, then the SF row. The segment starts lie in the workspace, or
// every workgroup scans the totals into them for itself (SCAN; see launch_moe_dispatch; in the last workgroup
// of the scan, by an atomic count: 8192 x 8 rows of 7168 BF16 columns 239 us, 235 and 230 for these two).
// The first pad_blocks blocks (E + kPastBlocks for the
// contiguous and psum layouts, else 0) fill an expert's padding rows each, and what is past the
// segments, beside the copies (by one block, 8192 x 8 rows of 512 bytes, 1024 experts, alignment 128: 35.0 us, 31.3
// by sixteen); the first writes the psum ends.
template <int TOKENS, bool SCAN>
__global__ void __launch_bounds__(kThreads) moe_scatter_kernel(const MoeDispatchArgs p, int pad_blocks) {
    __shared__ int s_start[SCAN ? kMoeMaxExperts + 1 : 1];
    const auto start_of = [&](int x) { return SCAN ? s_start[x] : ws_starts(p)[x]; };
    constexpr int UNITS = TOKENS == 1 ? 8 : 1;   // 16-byte pieces of a token and lane at a time
    static_assert(TOKENS * kMoeMaxTopk <= 64, "a wave's entries");
    const bool padding = (int)blockIdx.x < pad_blocks;
    const int lane = threadIdx.x & 63;
    const int t0 = padding ? p.t : ((int)blockIdx.x - pad_blocks) * (kThreads / 64 * TOKENS) + (int)(threadIdx.x >> 6) * TOKENS;
    const int tokens = min(TOKENS, p.t - t0);   // wave-uniform; none or fewer behind the last
    // The first 8 KB are loaded before the rows are looked up (the two
    // are independent), so the lookup's load latency hides behind them.
    const int units = p.kdim / 16;
    i32x4 v[TOKENS][UNITS];
#pragma unroll
    for (int i = 0; i < TOKENS; ++i)
#pragma unroll
        for (int q = 0; q < UNITS; ++q)
            if (i < tokens && q * 64 + lane < units)
                v[i][q] = reinterpret_cast<const i32x4*>(p.x + (int64_t)(t0 + i) * p.ldx)[q * 64 + lane];
    const bool mine = lane < tokens * p.k;
    const int own = TOKENS == 1 ? 0 : lane / p.k, slot = lane - own * p.k;   // this lane's entry
    const int64_t entry = (int64_t)t0 * p.k + lane;
    int e = -1, rank = 0;
    if (mine) {
        e = topk_at(p, t0 + own, slot);
        if (routed(p, e)) {
            rank = ws_counts(p)[(int64_t)e * p.chunks + (t0 + own) / kMoeChunkTokens] + p.pos[entry];
            if (!SCAN && p.layout != kMoeMasked) rank += ws_starts(p)[e];   // (a row then)
        }
    }
    if constexpr (SCAN) {
        const int used = segment_starts(p, [&](int x) { return ws_totals(p)[x]; }, [&](int x, int start, int total) {
            s_start[x] = start;
            if (blockIdx.x == 0 && p.layout == kMoePsum) p.meta[x] = start + total;   // psum[e] = align(psum[e-1]) + count
        });
        if (threadIdx.x == kThreads - 1) s_start[p.num_experts] = used;
        __syncthreads();
    }
    if (padding) {
        const int x = blockIdx.x;
        const int past = x - p.num_experts;
        if (past >= 0) pad_past(p, (int64_t)start_of(p.num_experts) + past * kThreads + (int)threadIdx.x, kPastBlocks * kThreads);
        else pad_rows(p, start_of(x) + ws_totals(p)[x], start_of(x + 1));
        return;
    }
    if (tokens <= 0) return;   // (no barrier follows)
    int flat = -1;
    if (mine) {
        if (routed(p, e)) {
            if constexpr (SCAN) flat = s_start[e] + rank;
            else flat = p.layout == kMoeMasked ? (rank < p.max_m ? e * p.max_m + rank : -1) : rank;
            if (flat >= 0) {
                if (p.w_out) p.w_out[flat] = p.topk_w ? p.topk_w[(int64_t)(t0 + own) * p.w_st + (int64_t)slot * p.w_sk] : 1.f;
                if (p.layout == kMoeContiguous) p.meta[flat] = e;
            }
        }
        p.pos[entry] = flat;
    }
    // The rows are written once and read by the next kernel, not by this one:
    // non-temporal stores (about 1.5x the copy rate of plain ones here).
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        if (i >= tokens) break;
        for (int u0 = 0; u0 < units; u0 += 64 * UNITS) {
            if (u0 > 0) {
#pragma unroll
                for (int q = 0; q < UNITS; ++q) {
                    const int u = u0 + q * 64 + lane;
                    if (u < units) v[i][q] = reinterpret_cast<const i32x4*>(p.x + (int64_t)(t0 + i) * p.ldx)[u];
                }
            }
            for (int j = 0; j < p.k; ++j) {
                const int r = __builtin_amdgcn_readlane(flat, i * p.k + j);
                if (r < 0) continue;   // wave-uniform
                i32x4* dst = reinterpret_cast<i32x4*>(p.a + row_a(p, r));
#pragma unroll
                for (int q = 0; q < UNITS; ++q) {
                    const int u = u0 + q * 64 + lane;
                    if (u < units) __builtin_nontemporal_store(v[i][q], dst + u);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        if (i >= tokens) break;
        for (int s = lane; s < p.sfk; s += 64) {
            const float sv = p.x_sf[(int64_t)(t0 + i) * p.sf_st + (int64_t)s * p.sf_sk];
            for (int j = 0; j < p.k; ++j) {
                const int r = __builtin_amdgcn_readlane(flat, i * p.k + j);
                if (r >= 0) p.sf[row_sf(p, r) + (int64_t)s * p.sf_sk_o] = sv;
            }
        }
    }
}

// Few tokens: the whole dispatch in one launch, without a workspace. Every workgroup counts all
// entries by expert in LDS, those before its own tokens apart, and scans the totals into the segment
// starts for itself; its entries' rows are the starts, plus the earlier entries of their
// experts, plus those among its own. TOKENS 1: the four waves share a token's row, 4: a token
// each. The first 16 (8) KB of a row are loaded before the counting, whose latency they cover. The first
// pad_blocks workgroups (contiguous and psum layouts) share the experts' padding rows and what
// is past the segments, and the first one of all writes the ends.
template <int TOKENS>
__global__ void __launch_bounds__(kThreads) moe_dispatch_few_kernel(const MoeDispatchArgs p, int pad_blocks) {
    constexpr int LANES = kThreads / TOKENS, UNITS = TOKENS == 1 ? 4 : 8;   // lanes of a row, 16-byte pieces of each at a time
    __shared__ int s_total[kMoeMaxExperts], s_before[kMoeMaxExperts];
    __shared__ int s_used;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool padding = (int)blockIdx.x < pad_blocks;
    const int t0 = padding ? 0 : ((int)blockIdx.x - pad_blocks) * TOKENS;   // the first token
    const int mine = TOKENS == 1 ? 0 : wave, t = t0 + mine;
    const int at = (int)threadIdx.x % LANES, units = p.kdim / 16;
    const bool live = !padding && t < p.t;
    const i32x4* src = reinterpret_cast<const i32x4*>(p.x + (int64_t)(live ? t : 0) * p.ldx);
    i32x4 v[UNITS];
    if (live) {
#pragma unroll
        for (int q = 0; q < UNITS; ++q)
            if (q * LANES + at < units) v[q] = src[q * LANES + at];
    }
    for (int e = threadIdx.x; e < p.num_experts; e += kThreads) s_total[e] = s_before[e] = 0;
    __syncthreads();
    // entry i: slot i % k of token i / k
    const int entries = p.t * p.k, first = t0 * p.k;
    const bool flat_ids = p.topk_st == p.k && p.topk_sk == 1;
    auto id_of = [&](int i) {
        if (flat_ids) return topk_at(p, 0, i);
        const int row = i / p.k;
        return topk_at(p, row, i - row * p.k);
    };
    for (int i0 = threadIdx.x; i0 < entries; i0 += 4 * kThreads) {
        int e[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) e[q] = i0 + q * kThreads < entries ? id_of(i0 + q * kThreads) : -1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (!routed(p, e[q])) continue;
            atomicAdd(&s_total[e[q]], 1);
            if (!padding && i0 + q * kThreads < first) atomicAdd(&s_before[e[q]], 1);
        }
    }
    __syncthreads();
    if (p.layout != kMoeMasked) {
        // s_total becomes the first row; padding workgroups keep the rows in s_before
        const int x = segment_starts(p, [&](int e) { return s_total[e]; }, [&](int e, int start, int total) {
            s_total[e] = start;
            if (padding) s_before[e] = total;
            if (blockIdx.x == 0 && p.layout == kMoePsum) p.meta[e] = start + total;
        });
        if (threadIdx.x == kThreads - 1) s_used = x;
        __syncthreads();
    } else if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < p.num_experts; e += kThreads) p.meta[e] = min(s_total[e], p.max_m);
    }
    if (padding) {
        if (p.layout == kMoeMasked) return;   // (no tokens)
        if (p.alignment > 1)
            for (int e = blockIdx.x; e < p.num_experts; e += pad_blocks)
                pad_rows(p, s_total[e] + s_before[e], s_total[e] + align_up(s_before[e], p.alignment));
        pad_past(p, (int64_t)s_used + (int)blockIdx.x * kThreads + (int)threadIdx.x, (int64_t)pad_blocks * kThreads);
        return;
    }
    // Lane i of every wave: the row of the workgroup's i-th entry.
    const int own = min(TOKENS, p.t - t0) * p.k;
    const int e = lane < own ? id_of(first + lane) : -1;
    const bool ok = routed(p, e);
    static_assert(kMoeMaxExperts <= 1024 && 4 * kMoeMaxTopk <= 64, "expert ids fit 10 bits, a workgroup's entries a wave");
    uint64_t peers = __ballot(ok);   // the lanes with this lane's expert
#pragma unroll
    for (int bit = 0; bit < 10; ++bit) {
        const bool set = (e >> bit) & 1;
        const uint64_t m = __ballot(ok && set);
        peers &= set ? m : ~m;
    }
    int flat = -1;
    if (ok) {
        const int r = s_before[e] + __popcll(peers & ((1ull << lane) - 1));
        flat = p.layout == kMoeMasked ? (r < p.max_m ? e * p.max_m + r : -1) : s_total[e] + r;
    }
    if (wave == 0 && lane < own) {
        p.pos[(int64_t)first + lane] = flat;
        if (flat >= 0) {
            const int row = lane / p.k;
            if (p.w_out)
                p.w_out[flat] = p.topk_w ? p.topk_w[(int64_t)(t0 + row) * p.w_st + (int64_t)(lane - row * p.k) * p.w_sk] : 1.f;
            if (p.layout == kMoeContiguous) p.meta[flat] = e;
        }
    }
    if (!live) return;   // wave-uniform; no barrier follows
    for (int u0 = 0; u0 < units; u0 += UNITS * LANES) {
        if (u0 > 0) {
#pragma unroll
            for (int q = 0; q < UNITS; ++q)
                if (u0 + q * LANES + at < units) v[q] = src[u0 + q * LANES + at];
        }
        for (int j = 0; j < p.k; ++j) {
            const int r = __builtin_amdgcn_readlane(flat, mine * p.k + j);
            if (r < 0) continue;   // wave-uniform
            i32x4* dst = reinterpret_cast<i32x4*>(p.a + row_a(p, r));
#pragma unroll
            for (int q = 0; q < UNITS; ++q) {
                const int u = u0 + q * LANES + at;
                if (u < units) __builtin_nontemporal_store(v[q], dst + u);
            }
        }
    }
    for (int s = at; s < p.sfk; s += LANES) {
        const float sv = p.x_sf[(int64_t)t * p.sf_st + (int64_t)s * p.sf_sk];
        for (int j = 0; j < p.k; ++j) {
            const int r = __builtin_amdgcn_readlane(flat, mine * p.k + j);
            if (r >= 0) p.sf[row_sf(p, r) + (int64_t)s * p.sf_sk_o] = sv;
        }
    }
}

// ---------------------------------------------------------------- SwiGLU -> FP8

__device__ __forceinline__ float bf16_to_f32(uint32_t b) { return __uint_as_float(b << 16); }

// One wave per (row, 512 output columns): lane l owns columns 8l .. 8l + 7 of
// the slice. gate = x[row, c], up = x[row, I + c]; y = silu(gate) * up * w in
// float32; then the per-token quantizer (amax over GRAN columns, clamped at
// 1e-4, sf = amax * fl32(1/448), code = e4m3(y * (1 / sf))). The arithmetic is
// dev::swiglu_weighted and dev::quantize_group8, which the GEMMs' fused SwiGLU
// epilogue calls too.
template <int GRAN>
__global__ void __launch_bounds__(kThreads) moe_swiglu_cast_kernel(const SwigluCastArgs p, int slices) {
    constexpr int TPG = GRAN / 8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lw = blockIdx.x;
    const int rb = lw / slices, slice = lw - rb * slices;
    const int row = rb * (kThreads / 64) + wave;
    if (row >= p.m) return;   // wave-uniform
    const int col = slice * 512 + lane * 8;
    const bool in = col < p.n;   // p.n % 8 == 0 (host check)
    const bool skip = p.row_layout && p.row_layout[row] < 0;
    float y[8];
    if (in && !skip) {
        const uint16_t* xr = p.x + (int64_t)row * p.ldx;
        const uint4 g4 = *reinterpret_cast<const uint4*>(xr + col);
        const uint4 u4 = *reinterpret_cast<const uint4*>(xr + p.n + col);
        const uint32_t gw[4] = {g4.x, g4.y, g4.z, g4.w}, uw[4] = {u4.x, u4.y, u4.z, u4.w};
        const float w = p.row_weight ? p.row_weight[row] : 1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float g = bf16_to_f32(e & 1 ? gw[e >> 1] >> 16 : gw[e >> 1] & 0xFFFFu);
            const float u = bf16_to_f32(e & 1 ? uw[e >> 1] >> 16 : uw[e >> 1] & 0xFFFFu);
            y[e] = dev::swiglu_weighted(g, u, w, p.clamp);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.f;
    }
    float sf;
    const uint2 codes = dev::quantize_group8<TPG>(y, sf);
    if (in) {
        *reinterpret_cast<uint2*>(p.q + (int64_t)row * p.ldq + col) = codes;
        if (lane % TPG == 0)
            p.sf[(int64_t)row * p.sf_sm + (int64_t)(col / GRAN) * p.sf_sk] = sf;
    }
}

// ---------------------------------------------------------------- combine

// One wave per (token, 512 columns): out[t, c] = sum over slots j (in order) of
// w[t, j] * y[pos[t, j], c], each product and sum rounded to float32, then bf16.
__global__ void __launch_bounds__(kThreads) moe_combine_kernel(const CombineArgs p, int slices) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lw = blockIdx.x;
    const int tb = lw / slices, slice = lw - tb * slices;
    const int t = tb * (kThreads / 64) + wave;
    if (t >= p.t) return;
    const int col = slice * 512 + lane * 8;
    if (col >= p.n) return;
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int j = 0; j < p.k; ++j) {
        const int r = p.pos[(int64_t)t * p.k + j];
        if (r < 0 || r >= p.rows) continue;   // unrouted, or not a row of y
        const int64_t off = p.max_m ? (int64_t)(r / p.max_m) * p.y_gs + (int64_t)(r % p.max_m) * p.ldy
                                    : (int64_t)r * p.ldy;
        const uint4 v4 = *reinterpret_cast<const uint4*>(p.y + off + col);
        const uint32_t vw[4] = {v4.x, v4.y, v4.z, v4.w};
        const float w = p.topk_w ? p.topk_w[(int64_t)t * p.w_st + (int64_t)j * p.w_sk] : 1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float yv = bf16_to_f32(e & 1 ? vw[e >> 1] >> 16 : vw[e >> 1] & 0xFFFFu);
            acc[e] = dev::f32_add(acc[e], p.topk_w ? dev::f32_mul(w, yv) : yv);
        }
    }
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t lo = __builtin_bit_cast(uint16_t, static_cast<__bf16>(acc[2 * e]));
        const uint32_t hi = __builtin_bit_cast(uint16_t, static_cast<__bf16>(acc[2 * e + 1]));
        o[e] = lo | (hi << 16);
    }
    *reinterpret_cast<uint4*>(p.out + (int64_t)t * p.ldo + col) = uint4{o[0], o[1], o[2], o[3]};
}

// Scratch of the dispatch entry point that allocates nothing: the workspace of
// one call (per-chunk expert counts, starts, totals), kMoeScratchInts int32 on
// each GPU the library runs on, held until the process ends. Host code must not
// pass `scratch` itself (a host-side stand-in): it passes the device address
// that hipGetSymbolAddress returns for the current device.
static __device__ __align__(256) int32_t scratch[kMoeScratchInts];

}  // namespace

int32_t* moe_scratch_device_ptr() {
    static std::mutex mu;
    static int32_t* ptrs[kMoeMaxDevices] = {};
    int dev = -1;
    DG_HIP_CHECK(hipGetDevice(&dev));
    DG_CHECK(dev >= 0 && dev < kMoeMaxDevices);
    std::lock_guard<std::mutex> lock(mu);
    if (ptrs[dev] == nullptr) {   // once per device, with that device current
        void* p = nullptr;
        DG_HIP_CHECK(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
        DG_CHECK(p != nullptr);
        ptrs[dev] = static_cast<int32_t*>(p);
    }
    return ptrs[dev];
}

int moe_dispatch_chunks(int64_t tokens) { return (int)((tokens + kMoeChunkTokens - 1) / kMoeChunkTokens); }

int64_t moe_dispatch_workspace_ints(int64_t tokens, int num_experts) {
    return (int64_t)moe_dispatch_chunks(tokens) * num_experts + 2 * (int64_t)num_experts + 1;
}

void launch_moe_dispatch(const MoeDispatchArgs& a, hipStream_t stream) {
    DG_CHECK(a.num_experts > 0 && a.num_experts <= kMoeMaxExperts && a.k > 0 && a.k <= kMoeMaxTopk);
    DG_CHECK(a.chunks == moe_dispatch_chunks(a.t));
    // One launch or several: every workgroup of the one counts all entries for itself, work that grows
    // with the square of the tokens, against two launches and a workspace's round trip. BF16 rows, tokens
    // x slots (columns), 64 experts, one launch / three, us in a graph: 4 x 8 (7168) 6.1/12.9, 256 x 8 (7168)
    // 15.2/22.8, 1024 x 8 (2048) 13.4/17.3, 1449 x 8 (1024) 14.1/15.8, 1700 x 8 16.2/16.6, 2048 x 8 18.7/17.5, 2900 x 4
    // 14.1/14.0, 4000 x 2 13.0/12.4, 4000 x 1 9.6/11.0; masked 1700 x 8 15.3/15.4, 2900 x 4 13.1/13.1. Rows of 4 KB and more
    // hide more of it: 2048 x 8 (4096) 37.3/37.8, 2048 x 4 20.6/23.0, 4000 x 2 22.9/23.4. Padding has a workgroup for each
    // expert, which counts as well, and six workgroups fit a CU at a time: 1024 experts 1448 x 8 18.8/17.9, 2048 x 2
    // 11.4/14.4, 2900 x 2 16.5/15.0, 2900 x 1 12.1/13.4, rows of 8 KB 2048 x 8 50.9/51.9. The counts are atomics, which
    // take their turns where the entries go to few experts: FP8 rows of 1 KB, masked, to one expert 1448 x 1 8.4/8.4, 2048 x 1
    // 10.4/8.6, 4096 x 1 27/9.5; to two 2048 x 1 8.1/8.7, 2500 x 1 10.3/9.0; to four 2500 x 1 8.5/9.1, 3547 x 1 11.4/9.3,
    // 2508 x 2 12.1/10.3; to eight 2048 x 2 8.1/10.0, 2900 x 2 11.8/10.8, 4096 x 1 10.4/9.7; hence most by experts. (All
    // tokens to one of 256 experts: 1448 x 1 10.5/10.5, 2048 x 1 13.1/10.5, 4096 x 1 32/12.)
    // One token a workgroup or four, us: 64 x 8 of 7168 10.2/11.9, 512 x 8 of 2048 8.3/8.2, 777 x 6 10.8/9.9, all to
    // one expert 1000 x 1 9.8/6.5.
    if (const int tokens = moe_few_tokens(a.t, a.k, a.kdim, a.num_experts, a.layout)) {   // of a workgroup
        // (without tokens or padding rows: one workgroup for the ends, masked counts and weights)
        const int pad_blocks = a.layout != kMoeMasked ? (a.alignment > 1 ? a.num_experts : 1) : a.t == 0 ? 1 : 0;
        const dim3 grid(pad_blocks + (a.t + tokens - 1) / tokens), block(kThreads);
        if (tokens == 1) hipLaunchKernelGGL(moe_dispatch_few_kernel<1>, grid, block, 0, stream, a, pad_blocks);
        else hipLaunchKernelGGL(moe_dispatch_few_kernel<4>, grid, block, 0, stream, a, pad_blocks);
        DG_HIP_CHECK(hipGetLastError());
        return;
    }
    hipLaunchKernelGGL(moe_count_kernel, dim3(a.chunks), dim3(kThreads), 0, stream, a);
    DG_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(moe_scan_kernel, dim3((a.num_experts + kThreads / 64 - 1) / (kThreads / 64)), dim3(kThreads), 0,
                       stream, a);
    DG_HIP_CHECK(hipGetLastError());
    const int launches = moe_dispatch_launches(a.t, a.k, a.kdim, a.num_experts, a.layout);
    if (launches == 4) {
        hipLaunchKernelGGL(moe_starts_kernel, dim3(1), dim3(kThreads), 0, stream, a);
        DG_HIP_CHECK(hipGetLastError());
    }
    const int pad_blocks = a.layout == kMoeMasked ? 0 : a.num_experts + kPastBlocks;
    // Short rows four tokens a wave, where the workgroups of a token a wave no longer fit the card at a time (1792 of
    // them; 2048 without the scan) and a token has little to store: the scan of the totals weighs less. One / four, us
    // in a graph (FP8 rows, alignment 16): 64 experts, 512 bytes 5000 x 8 18.7/21.2, 7200 x 2 15.0/13.8, 8192 x 1
    // 14.5/12.6, 8192 x 4 18.1/16.4, 8192 x 16 34.6/36.7, 16384 x 2 20.8/15.6, 16384 x 16 47.3/54.3; of 256 bytes
    // 16384 x 8 30.9/26.1; masked 256 bytes 5000 x 8 20.5/25.7, 10000 x 4 19.9/20.7, 12000 x 4 21.6/21.0, 16384 x 8
    // 38.3/36.8. Of 1 KB, 16384 x 8 (BF16) 38.8/42.2.
    const bool several = moe_four_tokens(a.t, a.k, a.kdim, a.layout);
    // Every workgroup that scans the totals for itself starts some microseconds later, and there are many where
    // each has little to store: a launch of their own for the starts is then shorter. Three / four launches, us
    // in a graph (FP8 rows, alignment 16): 64 experts 16384 x 8 of 512 bytes 31.9/30.5, of 1 KB 7900 x 1 14.7/13.3, 12000 x 2
    // 17.7/16.9, 32768 x 2 36.1/32.1, of 2 KB 32768 x 2 45.2/43.9, 8192 x 8 39.5/41.0; 384 experts, 7 KB, 12000 x 2
    // 55.7/52.6, 16384 x 4 113.6/108.1 (64 experts 110.0/108.9); 1024 experts, 1 KB, 32768 x 2 45.6/37.5, 4096 x 1
    // 16.2/14.4. 256 experts, 8192 x 8 of 7168 BF16 columns 230/235; rows of 128 bytes, four tokens a wave, 16384 x 4
    // 18.5/19.9.
    const int per = kThreads / 64 * (several ? 4 : 1);   // tokens of a workgroup
    const dim3 grid((unsigned)(pad_blocks + ((int64_t)a.t + per - 1) / per)), block(kThreads);
    // (the masked layout has no starts, and without their scan 56 registers instead of 66: eight waves on a SIMD, not seven)
    const bool scan = launches == 3 && a.layout != kMoeMasked;
    auto run = [&](auto tokens) {
        constexpr int T = decltype(tokens)::value;
        if (scan) hipLaunchKernelGGL((moe_scatter_kernel<T, true>), grid, block, 0, stream, a, pad_blocks);
        else hipLaunchKernelGGL((moe_scatter_kernel<T, false>), grid, block, 0, stream, a, pad_blocks);
    };
    if (several) run(std::integral_constant<int, 4>{});
    else run(std::integral_constant<int, 1>{});
    DG_HIP_CHECK(hipGetLastError());
}

void launch_moe_swiglu_cast(const SwigluCastArgs& a, hipStream_t stream) {
    if (a.m == 0 || a.n == 0) return;
    const int64_t row_blocks = (a.m + 3) / 4, slices = (a.n + 511) / 512;
    DG_CHECK(row_blocks * slices < ((int64_t)1 << 31));
    const dim3 grid((unsigned)(row_blocks * slices)), block(kThreads);
    switch (a.gran) {
        case 32: hipLaunchKernelGGL(moe_swiglu_cast_kernel<32>, grid, block, 0, stream, a, (int)slices); break;
        case 128: hipLaunchKernelGGL(moe_swiglu_cast_kernel<128>, grid, block, 0, stream, a, (int)slices); break;
        default: DG_UNSUPPORTED("SwiGLU FP8 cast: gran_k must be 32 or 128");
    }
    DG_HIP_CHECK(hipGetLastError());
}

void launch_moe_combine(const CombineArgs& a, hipStream_t stream) {
    if (a.t == 0 || a.n == 0) return;
    const int64_t tb = (a.t + 3) / 4, slices = (a.n + 511) / 512;
    DG_CHECK(tb * slices < ((int64_t)1 << 31));
    hipLaunchKernelGGL(moe_combine_kernel, dim3((unsigned)(tb * slices)), dim3(kThreads), 0, stream, a, (int)slices);
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace dgm
