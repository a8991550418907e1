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
//
// Measured on MI355X: 8192^3 as one group NT 930-980 us (16 KB rows of both operands meet in
// few L2 channels; with 128 bytes more 905), NN 825-880, TN 805-855, with an 8-bit B
// 960-1010; torch's library product 802, 888, 996. Under matrix load the clock falls to
// 1.4-1.7 GHz: 2091 TFLOP/s of zeros become 1371 of random values in the library's NT
// product, 1814 and 1250 in NN here, so bytes moved cost time even where they are hidden.
// Matrix cores busy 74-78% of the cycles of NT 16384 x 4096 x 7168 and NN 8192 x 7168 x 4096.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dg_internal.hpp"
#include "dg_ragged.hpp"

namespace dgm {
namespace {

using namespace dev;

// Group at place q of the groups from the longest to the shortest, so that the last tiles of
// a launch are the short ones; more than 16 groups in their own order (one of them weighs
// little, and the ranking takes a workgroup 20 instructions a group). By length and in
// their own order, shortest first, us: 7 x 300 and 6000 rows to 2048 x 2304 137 and 191, 16 of
// 32 to 4096 rows to 1408 x 2048 116 and 138, of 32 to 8192 to 4096 x 2048 with C 523 and 564,
// 8 of 455 to 3640 to 4096 x 7168 with C 1036 and 1058, 3 x 100 and 8000 to 4096 x 4096 (whole
// rounds) even. It loses where the long group would have been the quarters of the last round,
// 8 of 64 to 8192 to 2048 x 1408 166 and 133, and on short equal groups by the ranking itself,
// 8 x 64 to 2048 x 2048 32.7 and 31.3, 16 x 64 to 576 x 2048 23.2 and 21.2.
__device__ __forceinline__ int group_by_length(const RaggedGemmArgs& p, int q) {
    if (p.groups > 16) return q;
    const int lane = threadIdx.x & 63;
    int start = 0, end = -1;
    if (lane < p.groups) group_rows(p.ends, lane, p.rows, p.alignment, start, end);
    const int size = end - start;
    int place = 0;
    for (int j = 0; j < p.groups; ++j) {
        const int other = __builtin_amdgcn_readlane(size, j);
        place += other > size || (other == size && j < lane);
    }
    return __ffsll((unsigned long long)__ballot(place == q && lane < p.groups)) - 1;
}

__host__ __device__ __forceinline__ bool deals_eighths(int per) { return per % 8 == 0 || per >= 64; }
__host__ __device__ __forceinline__ int eighth_start(int x, int per) { return (int)((int64_t)x * per / 8); }

// TN: every group has the same tiles. Every XCD takes an eighth of each group's, group
// after group, so that groups of different lengths weigh on all of them alike (groups
// of few tiles: tiles dealt out one by one).
template <int BM, int BN, int PART>
__device__ __forceinline__ bool locate_outputs(const RaggedGemmArgs& p, const RaggedLaunch& l, RaggedTile& t) {
    const int per = l.row_blocks * l.col_blocks;
    int lo = 0, mine = per, i = blockIdx.x, slots = l.slots;
    if (deals_eighths(per)) {
        const int x = blockIdx.x & 7;
        lo = eighth_start(x, per);
        mine = eighth_start(x + 1, per) - lo;
        i = blockIdx.x >> 3;
        slots = max(l.slots / 8, 1);
    }
    int quarter;
    const int at = list_tile<PART>(i, mine * p.groups, slots, quarter);
    if (at < 0) return false;
    const int q = at / mine;
    int mb, nb;
    raster_tile(lo + at - q * mine, l.row_blocks, l.col_blocks, kRasterBlocks, mb, nb);
    t.g = group_by_length(p, q);
    t.m0 = mb * BM + (quarter >> 1) * (BM / 2), t.n0 = nb * BN + (quarter & 1) * (BN / 2);
    t.m_end = p.m;
    group_rows(p.ends, t.g, p.rows, p.alignment, t.k0, t.k_end);
    return t.m0 < p.m && t.n0 < p.n;
}

// ---------------------------------------------------------------- tiles
//
// One workgroup per BM x BN tile of D: 256 x 256 on eight waves (128 x 64 each), one
// workgroup on a CU, or 128 x 128 on four (64 x 64), two on a CU. 64 reduced elements a step,
// three steps of A and two of B in LDS (160 or 80 KB), so that every load has most of two
// steps to arrive: with two of each, 128 x 128 tiles of few rows, which wait for HBM, took
// 35.4 us instead of 25.7 (1001 x 1413 x 2048 over 16 groups), 256 x 256 the same.
// Operands go straight to LDS by buffer loads (16 bytes a lane) whose descriptor ends at
// the last valid byte: rows past the group's, columns past N and reduced elements past the
// end arrive as zeros, in both operands, and nothing is read there. So there are no edge
// variants, and steps past the end may be issued freely (they read nothing).
//
// An operand whose reduced dimension is contiguous ("K-major": A of NT and NN, B of NT)
// holds 64 reduced elements of a row in 128 bytes, 16-byte chunk c of row r at c ^ g(r); a
// matrix instruction's fragment (row lane & 31, 8 reduced elements) is one 16-byte read.
// The others ("MN-major": B of NN, both of TN) hold one reduced row of BM or BN columns
// after another; their fragments are read by ds_read_b64_tr_b16, which hands 16 lanes a
// transposed 4 x 16 block: 4 reduced rows of 32 bytes each. The 32-byte units of a row are
// permuted (column unit 2a + b of reduced row k at b * 4 + (a & 3 ^ k & 3) + (a >> 2) * 8)
// so that the four rows of a block, and the two blocks side by side, lie in distinct banks.
//
// Two barriers a step. The hand-off (the next step's loads have arrived, and every wave has
// read A's last slice of this one: A's step after the next three goes there) comes before
// the last 32-row slice of a step's matrix instructions, with the next step's fragments read
// under them; the other one, a slice after the step's start (128 x 128: at it), when every
// wave holds its B fragments, hands B's place on.

// An 8-bit B of TN: the codes of 64 reduced rows and their scales go to LDS as they are, three
// steps ahead (each lane's 16 codes of one row, and their scale, to a place of its own, so
// that only the lane's own loads have to be waited for), and from there as BF16 into the
// MN-major layout. code x scale is rounded to BF16, which the matrix instructions take (the
// scale goes by the reduced row, so the sums cannot take it instead): exact for powers of
// two, otherwise half a step, 2^-8 of a value at most. Measured then, of the sum of the
// products' magnitudes: 3.8e-3 for a single row, 2.7e-4 for 1500; with powers of two 8e-8.
// Doing it once per value on the way to LDS takes 64 vector instructions a thread and step,
// doing it on fragments 128 (two waves hold the same fragment).
template <int BN, int NW>
struct CodeOperand {
    static constexpr int kPieces = BN * BK / (16 * 64 * NW);   // 16-code pieces of each lane
    static constexpr int kLoads = 2 * kPieces;                 // loads of a step for each wave
    static constexpr int kCodes = BN * BK, kBytes = kCodes + NW * kPieces * 256;   // LDS of a step
    static constexpr int LPR = BN / 16;                        // lanes per reduced row
    static_assert(kPieces * 16 * 64 * NW == BN * BK, "whole wave loads");

    const uint8_t* base;   // the tile's first code of the step to be loaded next
    const float* sf;       // the scales' first row of that step
    int64_t pitch, sf_row;
    int64_t sf_col;        // this lane's column of scales
    int cols, left;
    uint32_t vlane;
    int row;               // this lane's reduced row in a wave load

    __device__ __forceinline__ void init(const RaggedGemmArgs& p, int k0, int reduced, int n0, int lane) {
        pitch = p.ldb, sf_row = p.sf_sr;
        base = static_cast<const uint8_t*>(p.b) + (int64_t)k0 * pitch + n0;
        cols = min(BN, p.n - n0);
        left = reduced;
        row = lane / LPR;
        const int col = lane % LPR * 16;
        vlane = col < cols ? (uint32_t)(row * (int)pitch) + col : kPastEnd;
        sf = p.b_sf + (int64_t)k0 * sf_row;
        sf_col = (int64_t)min((n0 + col) >> 7, (p.n - 1) >> 7) * p.sf_sc;
    }
    // The next step's codes and scales to lds (codes, then scales). Rows past the end: zero
    // codes; a scale is read of the last row there is.
    __device__ __forceinline__ void issue(uint32_t lds, int wave) {
        if (left <= 0) {   // (uniform) nothing left: as many loads, of no bytes
            const i32x4 none = descriptor(base, 0);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) dma16_buffer(none, kPastEnd, lds + (uint32_t)((i % kPieces * NW + wave) * 1024));
        } else {
            const int n = min(left, BK);
            const i32x4 rsrc = descriptor(base, (n - 1) * (int)pitch + ((cols + 3) & ~3));
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int seg = i * NW + wave;
                dma16_buffer(rsrc, vlane + (uint32_t)(seg * (1024 / BN) * (int)pitch), lds + seg * 1024);
                const float* at = sf + (int64_t)min(seg * (1024 / BN) + row, n - 1) * sf_row + sf_col;
                dma4_vaddr(at, lds + kCodes + seg * 256);
            }
        }
        base += BK * pitch, sf += BK * sf_row, left -= BK;
    }
    // The codes of the step at `from` (already there) to BF16 in `to`; valid: its rows.
    __device__ __forceinline__ void convert(const uint8_t* from, uint8_t* to, int valid, int wave, int lane) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int seg = i * NW + wave, k = seg * (1024 / BN) + row;
            const uint4 c = *reinterpret_cast<const uint4*>(from + seg * 1024 + lane * 16);
            float scale = *reinterpret_cast<const float*>(from + kCodes + seg * 256 + lane * 4);
            scale = k < valid ? scale : 0.f;   // (a scale of another row may be anything)
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
            uint32_t o[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], false);
                const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], true);
                o[2 * q] = pack2(lo[0] * scale, lo[1] * scale);
                o[2 * q + 1] = pack2(hi[0] * scale, hi[1] * scale);
            }
            const int u = lane % LPR, a = u >> 1;   // 16-column unit of the row: 2a + (u & 1)
            uint8_t* at = to + k * (BN * 2) + (u & 1) * 128 + (((a & 3) ^ (k & 3)) << 5) + (a >> 2) * 256;
            reinterpret_cast<uint4*>(at)[0] = uint4{o[0], o[1], o[2], o[3]};
            reinterpret_cast<uint4*>(at)[1] = uint4{o[4], o[5], o[6], o[7]};
        }
    }
};

// PART 2: 128 x 128 tiles, quarters of 256 x 256 ones.
template <int KIND, int BM, int BN, int WGM, int WGN, int PART, int EIGHT, int AHEAD>
__global__ void __launch_bounds__(WGM * WGN * 64, WGM * WGN == 4 ? 2 : 1)
ragged_tile_kernel(const RaggedGemmArgs p, const RaggedLaunch l) {
    constexpr int NW = WGM * WGN;
    constexpr int WM = BM / WGM, WN = BN / WGN, SM = WM / 32, SN = WN / 32;
    constexpr int A_KMAJOR = KIND != kRaggedTN, B_KMAJOR = KIND == kRaggedNT;
    constexpr int KS = BK / 16;
    constexpr int A_STEP = BM * BK * 2, B_STEP = BN * BK * 2;   // bytes of a step
    // LDS: A's steps, B's (8-bit: one, beside three steps of codes, in the place of A's third)
    using Codes = CodeOperand<BN, NW>;
    constexpr int A_SLOTS = EIGHT ? 2 : 3, B_SLOTS = EIGHT ? 1 : 2;
    constexpr int B_AT = A_SLOTS * A_STEP, C_AT = B_AT + B_SLOTS * B_STEP;
    constexpr int LDS_BYTES = C_AT + (EIGHT ? 3 * Codes::kBytes : 0);
    static_assert(SM % 2 == 0, "A fragments alternate between two buffers");
    static_assert(128 * BN * 4 <= LDS_BYTES && LDS_BYTES <= 160 * 1024, "the epilogue's rows fit");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[LDS_BYTES];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WGN, wn = wave % WGN;

    constexpr int LIST_BM = PART == 2 ? 2 * BM : BM, LIST_BN = PART == 2 ? 2 * BN : BN;
    RaggedTile t{};
    if constexpr (KIND == kRaggedTN) {
        if (!locate_outputs<LIST_BM, LIST_BN, PART>(p, l, t)) return;
    } else {
        if (!locate_rows<LIST_BM, LIST_BN, PART>(p, l, t)) return;
    }
    const int g = t.g, m0 = t.m0, n0 = t.n0, m_end = t.m_end;
    // this workgroup's piece of the reduced axis, in whole steps (none: it writes zeros)
    const int piece = ((t.k_end - t.k0 + BK - 1) / BK + l.splits - 1) / l.splits * BK;
    const int k0 = min(t.k0 + (int)blockIdx.y * piece, t.k_end);
    const int reduced = min(piece, t.k_end - k0);
    const uint16_t* b = static_cast<const uint16_t*>(p.b);

    Operand<BM, A_KMAJOR, NW> oa;
    Operand<BN, B_KMAJOR, NW> ob;
    Codes oc;
    if constexpr (A_KMAJOR)
        oa.init(p.a + (int64_t)m0 * p.lda + k0, p.lda, min(BM, m_end - m0), reduced, wave, lane);
    else
        oa.init(p.a + (int64_t)k0 * p.lda + m0, p.lda, min(BM, p.m - m0), reduced, wave, lane);
    if constexpr (EIGHT)
        oc.init(p, k0, reduced, n0, lane);
    else if constexpr (KIND == kRaggedNT)
        ob.init(b + (int64_t)g * p.b_gs + (int64_t)n0 * p.ldb + k0, p.ldb, min(BN, p.n - n0), reduced, wave, lane);
    else if constexpr (KIND == kRaggedNN)
        ob.init(b + (int64_t)g * p.b_gs + (int64_t)k0 * p.ldb + n0, p.ldb, min(BN, p.n - n0), reduced, wave, lane);
    else
        ob.init(b + (int64_t)k0 * p.ldb + n0, p.ldb, min(BN, p.n - n0), reduced, wave, lane);

    f32x16 acc[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem));
    Fragments<BM, A_KMAJOR, SM> fa;
    Fragments<BN, B_KMAJOR, SN> fb;
    fa.init(wm * WM, lane);
    fb.init(wn * WN, lane);
    bf16x8 op_b[SN][KS], op_a[2][KS];
    auto read_a = [&](const uint8_t* stage, int buf, int slab) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) op_a[buf][ks] = fa.read(stage, slab, ks);
    };
    auto read_b = [&](const uint8_t* stage, int slab) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) op_b[slab][ks] = fb.read(stage, slab, ks);
    };

    const int steps = (reduced + BK - 1) / BK;
    // Loads of a wave for a step of A and of B (codes and scales). At a hand-off those of the
    // step after the next may be in flight: A's and B's, or the codes of four steps on.
    constexpr int A_LOADS = decltype(oa)::kInstr, B_LOADS = EIGHT ? Codes::kLoads : decltype(ob)::kInstr;
    constexpr int IN_FLIGHT = EIGHT ? B_LOADS : A_LOADS + B_LOADS;
    if constexpr (EIGHT) {
        oc.issue(lds0 + C_AT, wave);
        oa.issue(lds0, wave);
        oc.issue(lds0 + C_AT + Codes::kBytes, wave);
        oa.issue(lds0 + A_STEP, wave);
        oc.issue(lds0 + C_AT + 2 * Codes::kBytes, wave);
        // (waits for the first step's codes, and for A's)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * B_LOADS + A_LOADS) : "memory");
        oc.convert(smem + C_AT, smem + B_AT, reduced, wave, lane);
        oc.issue(lds0 + C_AT, wave);
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt_barrier<2 * B_LOADS + A_LOADS>();
    } else {
        oa.issue(lds0, wave);
        ob.issue(lds0 + B_AT, wave);
        oa.issue(lds0 + A_STEP, wave);
        ob.issue(lds0 + B_AT + B_STEP, wave);
        oa.issue(lds0 + 2 * A_STEP, wave);
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt_barrier<2 * A_LOADS + B_LOADS>();
    }
    __builtin_amdgcn_sched_barrier(0);
    read_a(smem, 0, 0);
#pragma unroll
    for (int j = 0; j < SN; ++j) read_b(smem + B_AT, j);

    // A's steps kb, kb + 1 (and kb + 2), and the codes of steps kb + 1, kb + 2, kb + 3
    uint32_t a_cur = 0, a_next = A_STEP, a_last = A_SLOTS > 2 ? 2 * A_STEP : 0;
    uint32_t c_next = C_AT + Codes::kBytes, c_after = C_AT + 2 * Codes::kBytes, c_last = C_AT;
    auto advance = [&] {
        const uint32_t a_freed = a_cur, c_freed = c_next;
        a_cur = a_next, a_next = A_SLOTS > 2 ? a_last : a_freed, a_last = a_freed;
        c_next = c_after, c_after = c_last, c_last = c_freed;
    };
    // B's place of this step is free: the next step's codes go there as BF16, and the codes
    // of the step three after that one to the place they leave (the lane has read its own:
    // it has stored what they became).
    auto next_codes = [&](int kb) {
        oc.convert(smem + c_next, smem + B_AT, reduced - (kb + 1) * BK, wave, lane);
        oc.issue(lds0 + c_next, wave);
    };
    // FP32 C of 256 x 256 tiles: half of it on its way to LDS under the last three steps (with
    // codes, whose places are smaller, a quarter under the last two), in the places that
    // the steps past the end would take, a 32-row slab for each: slab i of wave row e as
    // A (i = 0) or B (i = 1) of step `steps + e`. A wave load is a row of the tile, whose
    // 16-byte unit u goes to u ^ (row & 7). Otherwise every CU waits for all of its C at the
    // same time as the others: 16384 rows to 8 x 4096 x 7168 1087 -> 1028 us, 5000 to 8 x 4000
    // x 7000 664 -> 593, with codes 692 -> 618. (Kernels of their own: without C the
    // loop's conditions would cost 1 to 2%.)
    static_assert(!AHEAD || (KIND == kRaggedTN && BM == 256 && AHEAD == (EIGHT ? 1 : 2)));
    const bool ahead = AHEAD && p.c && p.out_f32 && l.vec && steps >= A_SLOTS;
    const int c_pitch = (int)p.ldc * 4;
    auto c_slab = [&](int e, int i) {
        const int row = m0 + e * WM + i * 32, rows = min(m_end - row, 32), cols = min(BN, p.n - n0);
        const float* at = static_cast<const float*>(p.c) + (int64_t)g * p.c_gs + (int64_t)row * p.ldc + n0;
        const uint32_t unit = (uint32_t)((lane ^ (wave & 7)) * 16);
        return typename decltype(oa)::Step{descriptor(at, rows > 0 ? (rows - 1) * c_pitch + cols * 4 : 0),
                                           unit < (uint32_t)cols * 4 ? unit : kPastEnd};
    };
    // The loads of A for step kb + A_SLOTS and of B for kb + 2; `apart`: bytes between wave loads.
    auto next_a = [&](int kb, int& apart) {
        auto s = oa.next();
        apart = oa.kRows * (int)oa.pitch;
        if constexpr (AHEAD != 0)
            if (ahead && kb + A_SLOTS >= steps && kb + A_SLOTS <= steps + 1) s = c_slab(kb + A_SLOTS - steps, 0), apart = c_pitch;
        return s;
    };
    auto next_b = [&](int kb, int& apart) {
        auto s = ob.next();
        apart = ob.kRows * (int)ob.pitch;
        if constexpr (AHEAD != 0)
            if (ahead && kb + 2 >= steps) s = c_slab(kb + 2 - steps, 1), apart = c_pitch;
        return s;
    };
    const bool computes = m0 + wm * WM < m_end;   // else a wave of rows past the group's: it loads and synchronises only
    if (!computes) {
        for (int kb = 0; kb < steps; ++kb) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if constexpr (EIGHT) {
                next_codes(kb);
            } else {
                int apart = 0;
                const auto s = next_b(kb, apart);
#pragma unroll
                for (int q = 0; q < B_LOADS; ++q) ob.load(s, q, lds0 + B_AT + (kb & 1) * B_STEP, wave, apart);
            }
            wait_vmcnt_barrier<IN_FLIGHT>();
            int apart = 0;
            const auto s = next_a(kb, apart);
#pragma unroll
            for (int q = 0; q < A_LOADS; ++q) oa.load(s, q, lds0 + a_cur, wave, apart);
            advance();
        }
    } else
    for (int kb = 0; kb < steps; ++kb) {
        const uint32_t b_cur = B_AT + (EIGHT ? 0 : (kb & 1) * B_STEP), b_next = B_AT + (EIGHT ? 0 : (~kb & 1) * B_STEP);
        // A slice's matrix instructions with the LDS reads and loads of the steps to come
        // set between them one by one, in this order: a burst of loads keeps a wave from
        // issuing matrix instructions for as long as the address unit takes them in.
        constexpr int N = SN * KS, TOP = SM > 2 ? 1 : 0;
#pragma unroll
        for (int i = 0; i < SM; ++i) {
            const bool last = i + 1 == SM;
            typename decltype(oa)::Step sa;
            typename decltype(ob)::Step sb;
            int a_apart = 0, b_apart = 0;
            __builtin_amdgcn_sched_barrier(0);
            if (i == TOP) {
                // every wave holds its B fragments of this step: their place is free
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if constexpr (EIGHT) next_codes(kb);
                else sb = next_b(kb, b_apart);
            }
            if (last) {
                wait_vmcnt_barrier<IN_FLIGHT>();
                sa = next_a(kb, a_apart);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                // (the last slice by columns of fragments, whose registers are then free)
                const int j = last ? n / KS : n % SN, ks = last ? n % KS : n / SN;
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op_b[j][ks], op_a[i & 1][ks], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                if (n < KS) {
                    if (last) op_a[0][n] = fa.read(smem + a_next, 0, n);
                    else op_a[(i + 1) & 1][n] = fa.read(smem + a_cur, i + 1, n);
                }
                if (last && n >= KS) op_b[n / KS - 1][n % KS] = fb.read(smem + b_next, n / KS - 1, n % KS);
                if (!EIGHT && i == TOP) {
#pragma unroll
                    for (int q = n * B_LOADS / N; q < (n + 1) * B_LOADS / N; ++q) ob.load(sb, q, lds0 + b_cur, wave, b_apart);
                }
                if (last) {
#pragma unroll
                    for (int q = n * A_LOADS / N; q < (n + 1) * A_LOADS / N; ++q) oa.load(sa, q, lds0 + a_cur, wave, a_apart);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (last) read_b(smem + b_next, SN - 1);
        }
        advance();
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt_barrier<0>();   // (loads of steps past the end wrote zeros to LDS)
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (AHEAD != 0) {
        if (ahead) {
            if (computes) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const uint8_t* slab = smem + (i == 0 ? (steps + wm) % A_SLOTS * A_STEP : B_AT + ((steps + wm) & 1) * B_STEP);
#pragma unroll
                    for (int j = 0; j < SN; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int unit = (wn * WN + j * 32 + 8 * q) / 4 + (lane >> 5);
                            const f32x4 v = *reinterpret_cast<const f32x4*>(slab + (lane & 31) * (BN * 4) +
                                                                            ((unit ^ (lane & 7)) << 4));
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += v[e];
                        }
                }
            }
            __syncthreads();
            store_tile<1, BM, BN, WGM, WGN, AHEAD>(p, acc, smem, g, m0, m_end, n0, wave, lane, true);
            return;
        }
    }
    auto store = [&](auto out) {
        store_tile<decltype(out)::value, BM, BN, WGM, WGN>(p, acc, smem, KIND == kRaggedTN ? g : 0, m0, m_end, n0, wave, lane,
                                                           l.vec);
    };
    if (p.out_f32) store(std::integral_constant<int, 1>{});
    else if (KIND == kRaggedTN && p.c) store(std::integral_constant<int, KIND == kRaggedTN ? 2 : 0>{});
    else store(std::integral_constant<int, 0>{});
}

// NT and NN with at most 32 rows a group on average (decode): 32 x 128 tiles on four waves of 32 x
// 32, two workgroups on a CU, which stream the weights from HBM. A step is 4 KB of A and 16 of B, so
// four steps fit where a 128 x 128 tile has three and two, and a workgroup keeps 60 KB in
// flight; one barrier a step (it certifies the next step's loads and frees this one's
// place, whose fragments every wave holds).
template <int KIND>
__global__ void __launch_bounds__(256, 2) ragged_few_rows_kernel(const RaggedGemmArgs p, const RaggedLaunch l) {
    static_assert(KIND == kRaggedNT || KIND == kRaggedNN, "A is K-major");
    constexpr int BM = kFewRows, BN = 128, NW = 4, KS = BK / 16, SLOTS = 4;
    constexpr int A_STEP = BM * BK * 2, STEP = A_STEP + BN * BK * 2;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[SLOTS * STEP];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    RaggedTile t{};
    if (!locate_rows<BM, BN, 0>(p, l, t)) return;
    const int piece = ((p.k + BK - 1) / BK + l.splits - 1) / l.splits * BK;   // (as in the tile kernel)
    const int k0 = min((int)blockIdx.y * piece, p.k);
    const int reduced = min(piece, p.k - k0);
    const uint16_t* b = static_cast<const uint16_t*>(p.b) + (int64_t)t.g * p.b_gs;

    Operand<BM, 1, NW> oa;
    Operand<BN, KIND == kRaggedNT, NW> ob;
    oa.init(p.a + (int64_t)t.m0 * p.lda + k0, p.lda, min(BM, t.m_end - t.m0), reduced, wave, lane);
    ob.init(KIND == kRaggedNT ? b + (int64_t)t.n0 * p.ldb + k0 : b + (int64_t)k0 * p.ldb + t.n0, p.ldb, min(BN, p.n - t.n0),
            reduced, wave, lane);
    constexpr int LOADS = decltype(oa)::kInstr + decltype(ob)::kInstr;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem));
    auto issue = [&](int slot) {
        oa.issue(lds0 + slot * STEP, wave);
        ob.issue(lds0 + slot * STEP + A_STEP, wave);
    };
    Fragments<BM, 1, 1> fa;
    Fragments<BN, KIND == kRaggedNT, 1> fb;
    fa.init(0, lane);
    fb.init(wave * 32, lane);
    bf16x8 op_a[2][KS], op_b[2][KS];
    auto read = [&](int to, int slot) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            op_a[to][ks] = fa.read(smem + slot * STEP, 0, ks);
            op_b[to][ks] = fb.read(smem + slot * STEP + A_STEP, 0, ks);
        }
    };
    f32x16 acc[1][1];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][0][e] = 0.f;

    const int steps = (reduced + BK - 1) / BK;
#pragma unroll
    for (int st = 0; st < SLOTS; ++st) issue(st);
    wait_vmcnt_barrier<(SLOTS - 1) * LOADS>();
    read(0, 0);
    for (int kb = 0; kb < steps; kb += 2) {   // (a step past an odd end: zeros)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wait_vmcnt_barrier<(SLOTS - 2) * LOADS>();
            issue((kb + h) % SLOTS);
            read(h ^ 1, (kb + h + 1) % SLOTS);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op_b[h][ks], op_a[h][ks], acc[0][0], 0, 0, 0);
        }
    }
    wait_vmcnt_barrier<0>();   // (loads of steps past the end wrote zeros to LDS)
    if (p.out_f32) store_tile<1, BM, BN, 1, NW>(p, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
    else store_tile<0, BM, BN, 1, NW>(p, acc, smem, 0, t.m0, t.m_end, t.n0, wave, lane, l.vec);
}

// Whether 256 x 256 tiles load FP32 C under their last products.
bool loads_c_ahead(RaggedKind kind, const RaggedGemmArgs& a) {
    return kind == kRaggedTN && a.c && a.out_f32 && takes_vectors(a);
}

template <int KIND>
void launch_few_rows(const RaggedGemmArgs& a, int slots, int splits, hipStream_t stream) {
    const int64_t mb = row_blocks((RaggedKind)KIND, a, kFewRows), nb = ceil_div(a.n, 128);
    const RaggedLaunch l{(int)mb, (int)nb, slots, splits, takes_vectors(a)};
    hipLaunchKernelGGL(ragged_few_rows_kernel<KIND>, dim3((unsigned)(mb * nb), (unsigned)splits), dim3(256), 0, stream, a, l);
    DG_HIP_CHECK(hipGetLastError());
}

template <int KIND, int BM, int BN, int WGM, int WGN, int PART, int EIGHT, int AHEAD = 0>
void launch_tiles(const RaggedGemmArgs& a, int slots, int splits, hipStream_t stream) {
    constexpr int LIST = PART == 2 ? 2 : 1;
    const int64_t mb = row_blocks((RaggedKind)KIND, a, LIST * BM), nb = ceil_div(a.n, LIST * BN);
    const int64_t blocks = tile_blocks((RaggedKind)KIND, a, LIST * BM, PART == 2, slots);
    const RaggedLaunch l{(int)mb, (int)nb, slots, splits, takes_vectors(a)};
    hipLaunchKernelGGL((ragged_tile_kernel<KIND, BM, BN, WGM, WGN, PART, EIGHT, AHEAD>), dim3((unsigned)blocks, (unsigned)splits),
                       dim3(WGM * WGN * 64), 0, stream, a, l);
    DG_HIP_CHECK(hipGetLastError());
}

// Whether a TN launch of 256 x 256 tiles leaves tiles to a second one.
bool has_tail(const RaggedGemmArgs& a, int slots) {
    const int64_t per = ceil_div(a.m, 256) * ceil_div(a.n, 256);
    if (!deals_eighths((int)per)) return tail_tiles((int)per * a.groups, slots) > 0;
    for (int x = 0; x < 8; ++x)
        if (tail_tiles((eighth_start(x + 1, (int)per) - eighth_start(x, (int)per)) * a.groups, std::max(slots / 8, 1)) > 0)
            return true;
    return false;
}

template <int KIND, int EIGHT>
void launch_kind(const RaggedGemmArgs& a, const RaggedPlan& plan, float* ws, int slots, hipStream_t stream) {
    if (plan.block == 256) {
        auto launch_256 = [&](auto ahead) {
            if (KIND == kRaggedTN && !has_tail(a, slots)) {   // (known here: its tiles do not depend on group_ends)
                launch_tiles<KIND, 256, 256, 2, 4, 0, EIGHT, decltype(ahead)::value>(a, slots, 1, stream);
            } else {
                launch_tiles<KIND, 256, 256, 2, 4, 1, EIGHT, decltype(ahead)::value>(a, slots, 1, stream);
                launch_tiles<KIND, 128, 128, 2, 2, 2, EIGHT>(a, slots, 1, stream);
            }
        };
        constexpr int AHEAD = KIND == kRaggedTN ? (EIGHT ? 1 : 2) : 0;
        if (loads_c_ahead((RaggedKind)KIND, a)) launch_256(std::integral_constant<int, AHEAD>{});
        else launch_256(std::integral_constant<int, 0>{});
        return;
    }
    auto launch = [&](const RaggedGemmArgs& args) {
        if constexpr (KIND != kRaggedTN) {
            if (plan.block == kFewRows) return launch_few_rows<KIND>(args, slots, plan.splits, stream);
        }
        launch_tiles<KIND, 128, 128, 2, 2, 0, EIGHT>(args, slots, plan.splits, stream);
    };
    if (plan.splits == 1) {
        launch(a);
        return;
    }
    const int64_t rows = KIND == kRaggedTN ? (int64_t)a.groups * a.m : a.rows, ld = ceil_div(a.n, 4) * 4;
    RaggedGemmArgs part = a;
    part.d = ws, part.ldd = ld, part.d_gs = KIND == kRaggedTN ? a.m * ld : 0, part.d_split = rows * ld;
    part.c = nullptr, part.out_f32 = 1;
    launch(part);
    RaggedGemmArgs whole = a;
    whole.d_split = part.d_split;
    hipLaunchKernelGGL(ragged_join_kernel<KIND>, dim3((unsigned)join_blocks((RaggedKind)KIND, a)), dim3(256), 0, stream, whole,
                       (const float*)ws, ld, plan.splits, (int)ceil_div(a.n, 1024));
    DG_HIP_CHECK(hipGetLastError());
}

}  // namespace

// The tile and the pieces of the reduced axis that take the fewest microseconds by measured
// times: of a 64-element step of a round of tiles (256 x 256: 1.7; 128 x 128: 0.42 with one
// workgroup on a CU, 1.05 with two; more with an 8-bit B; 32 x 128, for at most 32 rows a
// group on average: 0.25 and 0.5), of a round's stores in TN, and of the pieces' sums on their way
// through the workspace. 256 x 256 tiles have to fill 150 CUs, and in NT and NN win where
// they are within 15%: with K long the 128 x 128 ones' operands, read twice as often, slow
// their steps (8 groups, 17648 x 517 x 7272 231 and 289 us). What it decides between, in us:
// 256 x 256 against 128 x 128: NT, 4096 columns, K = 2048, 8 groups of 256 rows 38.1 and 35.5,
//   of 512 61.9 and 67.2, 32 of 512 252 and 311; TN without C, 8 groups of 512 rows to 4096 x
//   2048 133 and 114, of 1024 to 4096 x 4096 312 and 408; with FP32 C, 32 of 47 to 2048 x 2048
//   271 and 196 (two small workgroups on a CU read C for one under the other's products; two
//   steps leave no time to load it ahead), 8 of 256 to 4096 x 2048 119 and 128, of 512 152 and
//   164, to 2048 x 2048 76 and 68, of 2048 to 4096 x 7168 1028 and 1207.
// 128 x 128 against 32 x 128: NT, 64 x 2048 x 2048 over 8 groups 17.8 and 13.3, 14 x 512 x
//   8192 over 2, in pieces, 14.0 and 9.6; even where HBM bounds both.
// It knows the buffer's rows, not which of them are in groups (the ends are on the device), and
// no group's own: 32 experts of 32 rows to 4096 x 2048 with FP32 C 367 in a buffer of their
// 1024 rows, 522 in one of 8672, which a dispatch of 8192 ids takes (371 on 128 x 128); NT, 32
// of 4096 x 7168, 2 rows each 303 and, in 4224 rows, 312; 1024 rows 109 all in one group (32 x
// 128 tiles, each of which reads its weights; 65 on 128 x 128), 309 spread over them.
// Whole and in 4, 8 and 16 pieces: 32 x 128, 8 x 4096 x 7168 30.4, 15.4, 15.4, 16.8; 128 x
//   128, 256 x 2112 x 7168 50.9, 22.5, 24.2, 31.0, 512 x 4096 x 2048 19.5, 28.4, 41.9, 66.3,
//   TN of 20000 rows to 104 x 504 124, 39.2, 24.8, 19.5.
RaggedPlan plan_ragged_gemm(RaggedKind kind, const RaggedGemmArgs& a, int slots, int block, int splits) {
    const bool tn = kind == kRaggedTN, eight = a.b_sf != nullptr;
    const int64_t used = std::max<int64_t>(1, std::min<int64_t>(a.groups, a.rows));   // groups with rows, at most
    const int64_t length = tn ? ceil_div(a.rows, used) : a.k;
    auto tiles = [&](int b) {   // expected
        const double mb = tn ? (double)ceil_div(a.m, b) * a.groups
                          : a.rows <= used * b ? (double)used
                                               : (double)a.rows / b + 0.5 * used;
        return mb * ceil_div(a.n, b);
    };
    // (the longest of several groups counts in TN: half as long again as the others, say)
    const double steps = (double)ceil_div(length, BK) * (tn && used > 1 ? 1.5 : 1.0), t256 = tiles(256), t128 = tiles(128);
    const bool few = !tn && (block == kFewRows || (block == 0 && a.rows <= kFewRows * used));
    const double alone = few ? 0.25 : eight ? 1.1 : 0.42, both = few ? 0.5 : eight ? 1.3 : 1.05;   // a step of 32 or 128 rows
    const bool ahead = loads_c_ahead(kind, a) && length > 2 * BK;   // (shorter groups have no steps to load C under)
    const double store256 = !tn ? 0 : ahead ? 24 : a.c ? 30 : a.out_f32 ? 15 : 9, store128 = !tn ? 0 : a.c ? 11.5 : a.out_f32 ? 7.7 : 5;
    auto us128 = [&](double t, double n) {   // t tiles of n steps: whole rounds, and what is left for a CU
        const double per_cu = t / slots, whole = std::floor(per_cu / 2), rest = per_cu - 2 * whole;
        return whole * (n * both + store128) +
               (rest > 0 ? n * (alone + (both - alone) * std::max(0.0, rest - 1)) + store128 * rest / 2 : 0.0);
    };
    RaggedPlan plan{few ? kFewRows : 128, 1, 0};
    if (block == 0 && !few && t256 * 128 >= slots * 75 &&
        std::max(1.0, t256 / slots) * (steps * (eight ? 1.95 : 1.7) + store256) < (tn ? 1.0 : 1.15) * us128(t128, steps))
        block = 256;
    if (block == 256) {
        plan.block = 256;
        return plan;
    }
    const int64_t out_rows = tn ? (int64_t)a.groups * a.m : a.rows;
    const double sums = (double)out_rows * a.n * 4;   // bytes of a piece's
    double best = 1e300;
    for (int s = 1; s <= 32; ++s) {
        if (splits > 0 ? s != splits : (s > 1 && steps < 4 * s)) continue;
        const double us = us128(t128 * s, std::ceil(steps / s)) + (s > 1 ? 5.0 + 2 * sums * s / 3e6 : 0.0);
        if (us < best) best = us, plan.splits = s;
    }
    if (plan.splits > 1) plan.workspace_bytes = out_rows * ceil_div(a.n, 4) * 16 * plan.splits;
    return plan;
}

// (Every launch of a call is within these before the first of them is queued; they keep the
// kernels' tile numbers within 32 bits too.)
void check_ragged_launches(RaggedKind kind, const RaggedGemmArgs& a, const RaggedPlan& plan, int slots) {
    if (plan.block == kFewRows) {
        DG_CHECK_GRID(row_blocks(kind, a, kFewRows) * ceil_div(a.n, 128), 256);
    } else {
        DG_CHECK_GRID(tile_blocks(kind, a, plan.block, false, slots), plan.block * 2);
        if (plan.block == 256) DG_CHECK_GRID(tile_blocks(kind, a, 256, true, slots), 256);
    }
    if (plan.splits > 1) DG_CHECK_GRID(join_blocks(kind, a), 256);
}

void launch_ragged_gemm(RaggedKind kind, const RaggedGemmArgs& a, const RaggedPlan& plan, float* ws, int slots,
                        hipStream_t stream) {
    DG_CHECK(plan.splits == 1 || ws != nullptr);
    switch (kind) {
        case kRaggedNT: launch_kind<kRaggedNT, 0>(a, plan, ws, slots, stream); break;
        case kRaggedNN: launch_kind<kRaggedNN, 0>(a, plan, ws, slots, stream); break;
        case kRaggedTN:
            if (a.b_sf) launch_kind<kRaggedTN, 1>(a, plan, ws, slots, stream);
            else launch_kind<kRaggedTN, 0>(a, plan, ws, slots, stream);
            break;
    }
}

}  // namespace dgm
