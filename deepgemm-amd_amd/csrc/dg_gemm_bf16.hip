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
#include "dg_kernel_common.hpp"
#include "dg_lds_dma.hpp"

namespace dgm {
namespace {

using namespace dev;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Two values rounded to BF16 by one v_cvt_pk_bf16_f32.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

// Tiles of a launch: row and column blocks (NT, NN: row blocks at most; of 256 for quarters),
// CUs, pieces of the reduced axis (blockIdx.y), and whether D and C take 16-byte accesses.
struct RaggedLaunch {
    int row_blocks, col_blocks, slots, splits;
    bool vec;
};
constexpr int kRasterBlocks = 8;   // row blocks of a raster band
constexpr int kFewRows = 32;       // rows of the tile for decode

// Rows [start, end) of group g, inside the `rows` that exist whatever group_ends holds.
__device__ __forceinline__ void group_rows(const int32_t* ends, int g, int rows, int alignment, int& start, int& end) {
    const int prev = g > 0 ? min(max(ends[g - 1], 0), rows) : 0;
    start = min(align_up(prev, alignment), rows);
    end = max(start, min(ends[g], rows));
}

// A launch of 256 x 256 tiles whose last round (a tile per CU) would be at most 58% full
// leaves that round's tiles to a second launch, as four 128 x 128 quarters each: two
// workgroups of those fit a CU, so 150 tiles' quarters take 1.2 rounds of 512, about 0.65
// of a 256 x 256 round (PART 1 and 2; 0 is a launch by itself). Both launches work it
// out alike, from the tiles that there are; in NT and NN the host does not know them, and
// the second one is made also where it has nothing to do (4 to 5 us). 8 experts, 16384 x 4096 x 7168 (NT, 1088
// tiles, 4.25 rounds): 889 -> 861 us; 8192 x 7168 x 4096 (NN, 3.94 rounds, no tail) 437 and 439.
__host__ __device__ __forceinline__ int tail_tiles(int tiles, int slots) {
    const int rest = tiles % slots;
    return rest * 128 <= slots * 75 ? rest : 0;
}

// What a workgroup computes: rows [m0, m_end) of D and columns from n0, for group g,
// reduced over [k0, k_end).
struct RaggedTile {
    int g, m0, m_end, n0, k0, k_end;
};

// Item `i` of the `tiles` items of a list (PART 2: a quarter of one of its last tiles):
// the tile, or -1.
template <int PART>
__device__ __forceinline__ int list_tile(int i, int tiles, int slots, int& quarter) {
    const int full = PART == 0 ? tiles : tiles - tail_tiles(tiles, slots);
    quarter = 0;
    if constexpr (PART == 2) {
        quarter = i & 3;
        i = full + (i >> 2);
        return i < tiles ? i : -1;
    }
    return i < full ? i : -1;
}

// NT, NN: row blocks of BM rows, groups in order; a wave looks at 64 groups at a time, every
// lane counting one group's blocks, a prefix sum over the lanes placing them. Each XCD
// gets a contiguous part of the tiles that there are (the grid is an upper bound:
// group_ends is on the device).
template <int BM, int BN, int PART>
__device__ __forceinline__ bool locate_rows(const RaggedGemmArgs& p, const RaggedLaunch& l, RaggedTile& t) {
    const int lane = threadIdx.x & 63;
    int start = 0, end = 0, mine = 0, incl = 0;
    auto count = [&](int g0) {   // blocks of groups [g0, g0 + 64): this lane's, and up to it
        start = end = 0;
        if (g0 + lane < p.groups) group_rows(p.ends, g0 + lane, p.rows, p.alignment, start, end);
        mine = (end - start + BM - 1) / BM;
        incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            incl += lane >= o ? v : 0;
        }
        return __builtin_amdgcn_readlane(incl, 63);
    };
    int total = 0;   // (decreasing ends could count more than the launch holds)
    for (int g0 = 0; g0 < p.groups; g0 += 64) total = min(total + count(g0), l.row_blocks);
    const int tiles = total * l.col_blocks;
    const int full = PART == 0 ? tiles : tiles - tail_tiles(tiles, l.slots);
    const int items = PART == 2 ? (tiles - full) * 4 : full;
    if ((int)blockIdx.x >= items) return false;
    int quarter;
    const int lt = list_tile<PART>(xcd_remap(blockIdx.x, items), tiles, l.slots, quarter);
    const int block = lt / l.col_blocks;
    int base = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
        const int here = p.groups <= 64 ? total : count(g0);
        if (block < base + here) {
            const int at = __ffsll((unsigned long long)__ballot(base + incl > block)) - 1;
            const int blocks = __builtin_amdgcn_readlane(mine, at);
            const int first = base + __builtin_amdgcn_readlane(incl, at) - blocks;
            int mb, nb;
            raster_tile(lt - first * l.col_blocks, blocks, l.col_blocks, kRasterBlocks, mb, nb);
            t.g = g0 + at;
            t.m0 = __builtin_amdgcn_readlane(start, at) + mb * BM + (quarter >> 1) * (BM / 2);
            t.m_end = __builtin_amdgcn_readlane(end, at);
            t.n0 = nb * BN + (quarter & 1) * (BN / 2);
            t.k0 = 0, t.k_end = p.k;
            return t.m0 < t.m_end && t.n0 < p.n;
        }
        base += here;
    }
    return false;
}

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

__device__ __forceinline__ int swz_g(int r) { return ((r >> 1) ^ ((r & 1) << 2)) & 7; }

// 16 bytes a lane from `rsrc` at byte voff (zeros past its end) to lds + 16 * lane. Inline
// asm: the compiler would wait for every load in flight before each LDS read.
__device__ __forceinline__ void dma16_buffer(const i32x4& rsrc, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc)
                 : "memory", "m0");
}

// Buffer descriptor of `bytes` bytes (a multiple of 4 is read, dword by dword) from `base`.
__device__ __forceinline__ i32x4 descriptor(const void* base, int bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xFFFFu)),
                 __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}

// No offset of a valid byte: past the end of every descriptor here.
constexpr uint32_t kPastEnd = 0x80000000u;

constexpr int BK = 64;

// One operand of a tile: where its steps come from. ROWS: BM or BN; KMAJOR as above.
template <int ROWS, int KMAJOR, int NW>
struct Operand {
    static constexpr int kInstr = ROWS * BK / (512 * NW);   // wave loads (1 KB) of a step for each wave
    static_assert(kInstr * 512 * NW == ROWS * BK && (KMAJOR || ROWS == 128 || ROWS == 256), "whole wave loads");

    const uint8_t* base;   // the tile's first element of the step to be issued next
    int64_t pitch;         // bytes
    int rows;              // valid rows (KMAJOR) or columns of the tile
    int left;              // reduced elements from there on
    uint32_t vlane;        // this lane's offset in a wave load
    int chunk;             // KMAJOR: first reduced element of this lane's chunk

    __device__ __forceinline__ void init(const uint16_t* at, int64_t ld, int valid, int reduced, int wave, int lane) {
        base = reinterpret_cast<const uint8_t*>(at);
        pitch = ld * 2;
        rows = valid;
        left = reduced;
        if constexpr (KMAJOR) {
            const int rs = lane / (BK / 8);
            // (NW is even, so a wave's 8-row pieces share a parity)
            chunk = ((lane & 7) ^ swz_g((wave & 1) * 8 + rs)) * 8;
            vlane = (uint32_t)(rs * (int)pitch) + chunk * 2;
        } else {
            constexpr int LPR = ROWS / 8;   // lanes per reduced row
            const int k = lane / LPR + (ROWS == 256 ? (wave & 1) * 2 : 0);   // its two low bits
            const int slot = lane % LPR, pu = slot >> 1;
            const int a = ((pu & 3) ^ (k & 3)) | (pu >> 3) << 2, b = (pu >> 2) & 1;
            const int col = (2 * a + b) * 16 + (slot & 1) * 8;
            vlane = col < valid ? (uint32_t)(lane / LPR * (int)pitch) + col * 2 : kPastEnd;
        }
    }
    // Loads of the next step: its descriptor and lane offset, then wave load i to lds (this
    // operand's part of LDS), and on to the step after it.
    static constexpr int kRows = 512 / (KMAJOR ? BK : ROWS);   // rows of a wave load
    struct Step {
        i32x4 rsrc;
        uint32_t v;
    };
    __device__ __forceinline__ Step next() {
        // (without branches, which would split the loop's instruction sequence; nothing
        // left: every lane past the end, or no bytes, as a row is no longer than the pitch)
        const int n = min(max(left, 0), BK);
        const int bytes = KMAJOR ? (rows - 1) * (int)pitch + n * 2 : max((n - 1) * (int)pitch + ((rows * 2 + 3) & ~3), 0);
        const Step s{descriptor(base, bytes), !KMAJOR || chunk < left ? vlane : kPastEnd};
        base += KMAJOR ? (int64_t)BK * 2 : BK * pitch;
        left -= BK;
        return s;
    }
    __device__ __forceinline__ void load(const Step& s, int i, uint32_t lds, int wave) const {
        load(s, i, lds, wave, kRows * (int)pitch);
    }
    __device__ __forceinline__ void load(const Step& s, int i, uint32_t lds, int wave, int apart) const {
        const int seg = i * NW + wave;
        dma16_buffer(s.rsrc, s.v + (uint32_t)(seg * apart), lds + seg * 1024);
    }
    __device__ __forceinline__ void issue(uint32_t lds, int wave) {
        const Step s = next();
#pragma unroll
        for (int i = 0; i < kInstr; ++i) load(s, i, lds, wave);
    }
};

// Fragment reads of a 32-row slab: off[] for slab 0 of the wave, see above.
template <int ROWS, int KMAJOR, int SLABS>
struct Fragments {
    uint32_t off[KMAJOR ? BK / 16 : SLABS];
    __device__ __forceinline__ void init(int first_row, int lane) {
        if constexpr (KMAJOR) {
            const int r = lane & 31;
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks)
                off[ks] = (first_row + r) * (BK * 2) + (((2 * ks + (lane >> 5)) ^ swz_g(r)) << 4);
        } else {
            const int i = lane & 15, a = first_row >> 5;
#pragma unroll
            for (int s = 0; s < SLABS; ++s)
                off[s] = ((lane >> 5) * 8 + (i >> 2)) * (ROWS * 2) + ((lane >> 4) & 1) * 128 +
                         ((((a + s) & 3) ^ (i >> 2)) << 5) + ((a + s) >> 2) * 256 + (i & 3) * 8;
        }
    }
    __device__ __forceinline__ bf16x8 read(const uint8_t* tile, int slab, int ks) const {
        if constexpr (KMAJOR) {
            return *reinterpret_cast<const bf16x8*>(tile + off[ks] + slab * 32 * (BK * 2));
        } else {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const uint8_t* at = tile + off[slab] + ks * 16 * (ROWS * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * (ROWS * 2)));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

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

// The tile's sums to D (+ C) through LDS, so that each access of a wave covers whole rows of
// the tile (256 to 1024 bytes in one piece; every lane 16 of them). OUT: 0 BF16 without C
// (staged as BF16), 1 FP32, 2 BF16 with C (staged as FP32: the sum is rounded once).
// Staged as FP32, 256 rows take two passes of 128 (64 of each wave row). C's values of a
// pass are loaded before its sums are in LDS: their latency would otherwise come with
// every access. AHEAD: four passes of 64 rows, the first AHEAD of which have C in the sums
// already; C of the next two is loaded at once, of a fourth when the registers of the
// second's are free.
template <int OUT, int BM, int BN, int WGM, int WGN, int AHEAD = 0, int SM, int SN>
__device__ __forceinline__ void store_tile(const RaggedGemmArgs& p, const f32x16 (&acc)[SM][SN], uint8_t* lds, int g, int m0,
                                           int m_end, int n0, int wave, int lane, bool vec) {
    constexpr int NW = WGM * WGN, SIZE = OUT == 1 ? 4 : 2, CPL = 16 / SIZE;   // columns of a lane
    constexpr int PASSES = AHEAD ? 4 : OUT && BM == 256 ? 2 : 1, PS = SM / PASSES;        // slabs of a pass
    constexpr int STAGED = OUT ? 4 : 2, ROW_BYTES = BN * STAGED;
    constexpr int LPR = BN / CPL, RPT = 64 / LPR, T = BM / PASSES / (NW * RPT);   // lanes of a row, rows of an access
    static_assert(T * NW * RPT * PASSES == BM, "whole accesses");
    const int lrow = lane & 31, lhalf = lane >> 5, wm = wave / WGN, wn = wave % WGN;
    const int c = n0 + lane % LPR * CPL;
    const bool whole = vec && c + CPL <= p.n;
    const int64_t d_tile = (int64_t)blockIdx.y * p.d_split + (int64_t)g * p.d_gs + n0, c_tile = (int64_t)g * p.c_gs + n0;
    const int64_t d_off = d_tile + (c - n0), c_off = c_tile + (c - n0);
    uint4 c_values[AHEAD ? PASSES : 1][T];
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        const bool add = OUT && p.c && pass >= AHEAD;
        // row of D of the row r of a pass (which has PS slabs of each wave row)
        auto row_in = [&](int r, int of) { return m0 + (r / (PS * 32)) * (SM * 32) + of * (PS * 32) + r % (PS * 32); };
        auto row_of = [&](int r) { return row_in(r, pass); };
        uint4 (&cv)[T] = c_values[AHEAD ? pass : 0];
#pragma unroll
        for (int of = pass; of < PASSES; ++of) {
            const int when = !AHEAD ? of : of < AHEAD + 2 ? 0 : of - 1;
            if (of < AHEAD || pass != when || (!AHEAD && !add)) continue;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int r = row_in((t * NW + wave) * RPT + lane / LPR, of);
                if (r < m_end && whole)
                    c_values[AHEAD ? of : 0][t] =
                        *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.c) + (c_off + (int64_t)r * p.ldc) * SIZE);
            }
        }
        if (pass > 0) __syncthreads();
        // 16-byte unit u of row r at u ^ (r & 7): 8 rows on distinct banks
#pragma unroll
        for (int i = 0; i < PS; ++i)
#pragma unroll
            for (int j = 0; j < SN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x16& v = acc[pass * PS + i][j];
                    const int r = wm * (PS * 32) + i * 32 + lrow, col = wn * (SN * 32) + j * 32 + 8 * q + 4 * lhalf;
                    uint8_t* at = lds + r * ROW_BYTES + ((col * STAGED >> 4 ^ (r & 7)) << 4) + (OUT ? 0 : lhalf * 8);
                    if constexpr (OUT)
                        *reinterpret_cast<f32x4*>(at) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                    else
                        *reinterpret_cast<uint2*>(at) = uint2{pack2(v[4 * q], v[4 * q + 1]), pack2(v[4 * q + 2], v[4 * q + 3])};
                }
        __syncthreads();
        if (!vec) {   // rows that begin anywhere: 64 elements of a row an access, one a lane
            for (int t = 0; t < T * RPT; ++t) {
                const int lr = t * NW + wave, r = row_of(lr);
                if (r >= m_end) continue;
#pragma unroll
                for (int q = 0; q < BN / 64; ++q) {
                    const int col = q * 64 + lane, at = col * STAGED;
                    if (n0 + col >= p.n) continue;
                    const uint8_t* src = lds + lr * ROW_BYTES + (((at >> 4) ^ (lr & 7)) << 4) + (at & 15);
                    const int64_t to = d_tile + (int64_t)r * p.ldd + col, from = c_tile + (int64_t)r * p.ldc + col;
                    if constexpr (OUT == 0) {
                        static_cast<uint16_t*>(p.d)[to] = *reinterpret_cast<const uint16_t*>(src);
                    } else {
                        float v = *reinterpret_cast<const float*>(src);
                        if constexpr (OUT == 1) {
                            if (add) v += static_cast<const float*>(p.c)[from];
                            static_cast<float*>(p.d)[to] = v;
                        } else {
                            v += bf16_to_f32(static_cast<const uint16_t*>(p.c)[from]);
                            static_cast<uint16_t*>(p.d)[to] = bf16_bits(v);
                        }
                    }
                }
            }
            continue;
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int lr = (t * NW + wave) * RPT + lane / LPR, r = row_of(lr);
            auto unit = [&](int u) { return *reinterpret_cast<const uint4*>(lds + lr * ROW_BYTES + ((u ^ (lr & 7)) << 4)); };
            const uint4 x = unit(lane % LPR * (OUT == 2 ? 2 : 1));
            uint32_t w[4] = {x.x, x.y, x.z, x.w};   // D's 16 bytes
            float f[OUT ? CPL : 1];
            if constexpr (OUT) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(w[e]);
                if constexpr (OUT == 2) {
                    const uint4 y = unit(lane % LPR * 2 + 1);
                    f[4] = __uint_as_float(y.x), f[5] = __uint_as_float(y.y), f[6] = __uint_as_float(y.z), f[7] = __uint_as_float(y.w);
                }
            }
            if (r >= m_end || c >= p.n) continue;
            const int64_t to = d_off + (int64_t)r * p.ldd, from = c_off + (int64_t)r * p.ldc;
            if (whole) {
                if constexpr (OUT) {
                    if (add) {
                        const uint32_t y[4] = {cv[t].x, cv[t].y, cv[t].z, cv[t].w};
#pragma unroll
                        for (int e = 0; e < CPL; ++e)
                            f[e] += OUT == 1 ? __uint_as_float(y[e & 3])
                                             : __uint_as_float(e & 1 ? y[e >> 1] & 0xFFFF0000u : y[e >> 1] << 16);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = OUT == 1 ? __float_as_uint(f[e]) : pack2(f[(2 * e) % CPL], f[(2 * e + 1) % CPL]);
                }
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.d) + to * SIZE) = uint4{w[0], w[1], w[2], w[3]};
            } else {
#pragma unroll
                for (int e = 0; e < CPL; ++e) {
                    if (c + e >= p.n) break;
                    if constexpr (OUT == 1)
                        static_cast<float*>(p.d)[to + e] = add ? f[e] + static_cast<const float*>(p.c)[from + e] : f[e];
                    else if constexpr (OUT == 2)
                        static_cast<uint16_t*>(p.d)[to + e] =
                            bf16_bits(f[e] + bf16_to_f32(static_cast<const uint16_t*>(p.c)[from + e]));
                    else
                        static_cast<uint16_t*>(p.d)[to + e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                }
            }
        }
    }
}

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

// D (+ C) from the pieces' sums in the workspace, added in the order of the pieces: four
// columns a thread, 1024 of a row a workgroup. rows: of D, in all groups (TN).
template <int KIND>
__global__ void __launch_bounds__(256) ragged_join_kernel(const RaggedGemmArgs p, const float* __restrict__ ws,
                                                          const int64_t ws_ld, const int splits, const int chunks) {
    const int64_t row = blockIdx.x / chunks;
    const int c = ((int)(blockIdx.x - row * chunks) * 256 + (int)threadIdx.x) * 4;
    int64_t to, from = 0;
    if constexpr (KIND == kRaggedTN) {
        const int64_t g = row / p.m, m = row - g * p.m;
        to = g * p.d_gs + m * p.ldd, from = g * p.c_gs + m * p.ldc;
    } else {
        // the first group whose end is past the row has it, or none
        int lo = 0, hi = p.groups;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.ends[mid] > row) hi = mid;
            else lo = mid + 1;
        }
        if (lo == p.groups) return;
        int start, end;
        group_rows(p.ends, lo, p.rows, p.alignment, start, end);
        if (row < start) return;
        to = row * p.ldd;
    }
    if (c >= p.n) return;
    const float* src = ws + row * ws_ld + c;   // (ws_ld: n up to a multiple of 4)
    f32x4 v = *reinterpret_cast<const f32x4*>(src);
    for (int s = 1; s < splits; s += 8) {   // eight loads at a time
        f32x4 x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (s + q < splits) x[q] = *reinterpret_cast<const f32x4*>(src + (s + q) * p.d_split);
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (s + q < splits) v[e] += x[q][e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (c + e >= p.n) break;
        if (p.out_f32) {
            if (p.c) v[e] += static_cast<const float*>(p.c)[from + c + e];
            static_cast<float*>(p.d)[to + c + e] = v[e];
        } else {
            if (p.c) v[e] += bf16_to_f32(static_cast<const uint16_t*>(p.c)[from + c + e]);
            static_cast<uint16_t*>(p.d)[to + c + e] = bf16_bits(v[e]);
        }
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Row blocks of `bm` rows at most: whole ones, and a partial one for each group that has rows.
int64_t row_blocks(RaggedKind kind, const RaggedGemmArgs& a, int bm) {
    return kind == kRaggedTN ? ceil_div(a.m, bm) : a.rows / bm + std::min<int64_t>(a.groups, a.rows);
}

// Whether D's rows, and C's, begin at multiples of 16 bytes.
bool takes_vectors(const RaggedGemmArgs& a) {
    const int64_t size = a.out_f32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(a.d) % 16 == 0 && a.ldd * size % 16 == 0 && a.d_gs * size % 16 == 0 &&
           (!a.c || (reinterpret_cast<uintptr_t>(a.c) % 16 == 0 && a.ldc * size % 16 == 0 && a.c_gs * size % 16 == 0));
}

// Whether 256 x 256 tiles load FP32 C under their last products.
bool loads_c_ahead(RaggedKind kind, const RaggedGemmArgs& a) {
    return kind == kRaggedTN && a.c && a.out_f32 && takes_vectors(a);
}

// Workgroups of a launch of `tile` x `tile` tiles (quarters: of its tail).
int64_t tile_blocks(RaggedKind kind, const RaggedGemmArgs& a, int tile, bool quarters, int slots) {
    const int64_t tiles = row_blocks(kind, a, tile) * ceil_div(a.n, tile);
    const int64_t blocks = kind == kRaggedTN ? ceil_div(tiles, 8) * 8 * a.groups : tiles;
    // (a tail has at most 58% of a round's tiles, for each XCD by itself in TN)
    return quarters ? std::min<int64_t>(blocks, kind == kRaggedTN ? std::max(slots / 8, 1) * 8 : slots) * 4 : blocks;
}

// Workgroups of the join of a call's pieces: 1024 columns of a row each.
int64_t join_blocks(RaggedKind kind, const RaggedGemmArgs& a) {
    return (kind == kRaggedTN ? (int64_t)a.groups * a.m : a.rows) * ceil_div(a.n, 1024);
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
