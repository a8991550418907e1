// Building blocks of the products over ragged row segments (gfx950): which rows and columns a
// workgroup has, an operand's way to LDS and its fragments, and the way of the sums to D.
//
// Group g owns rows [s_g, e_g), e_g = group_ends[g] and s_g = align(e_{g-1}, alignment). Operands
// are counted in 16-bit units: one BF16 value, or four 4-bit ones. 64 units of the reduced axis
// are a step; a "K-major" operand (its reduced axis is contiguous) holds a row's step in 128
// bytes of LDS, 16-byte chunk c of row r at c ^ g(r), an "MN-major" one a reduced row of the
// tile's columns after another, in the permutation that ds_read_b64_tr_b16 reads without
// bank conflicts. Loads past an operand's end bring zeros.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

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
        load_rows(s, i * NW + wave, lds, apart);
    }
    // the wave load of rows (KMAJOR) 8 seg to 8 seg + 7; seg of the wave's parity
    __device__ __forceinline__ void load_rows(const Step& s, int seg, uint32_t lds, int apart) const {
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
            // Four rows read from LDS at a time. One after the other / four, 4-bit products of 1001 rows over 16
            // groups, n 1413, k 2080: BF16 14.6/13.5 us, FP32 15.6/14.1 us.
            constexpr int ROWS = 4;
            static_assert(T * RPT % ROWS == 0, "whole batches");
            for (int t = 0; t < T * RPT; t += ROWS) {
                uint32_t v[ROWS][BN / 64];
                auto each = [&](auto&& body) {
#pragma unroll
                    for (int u = 0; u < ROWS; ++u) {
                        const int r = row_of((t + u) * NW + wave);
                        if (r >= m_end) continue;
#pragma unroll
                        for (int q = 0; q < BN / 64; ++q)
                            if (n0 + q * 64 + lane < p.n) body(v[u][q], r, q * 64 + lane);
                    }
                };
#pragma unroll
                for (int u = 0; u < ROWS; ++u)
#pragma unroll
                    for (int q = 0; q < BN / 64; ++q) {
                        const int lr = (t + u) * NW + wave, at = (q * 64 + lane) * STAGED;
                        const uint8_t* src = lds + lr * ROW_BYTES + (((at >> 4) ^ (lr & 7)) << 4) + (at & 15);
                        if constexpr (OUT == 0) v[u][q] = *reinterpret_cast<const uint16_t*>(src);
                        else v[u][q] = *reinterpret_cast<const uint32_t*>(src);
                    }
                if (add)   // uniform over the launch
                    each([&](uint32_t& x, int r, int col) {
                        const int64_t from = c_tile + (int64_t)r * p.ldc + col;
                        if constexpr (OUT == 1) x = __float_as_uint(__uint_as_float(x) + static_cast<const float*>(p.c)[from]);
                        if constexpr (OUT == 2) x = __float_as_uint(__uint_as_float(x) + bf16_to_f32(static_cast<const uint16_t*>(p.c)[from]));
                    });
                each([&](uint32_t x, int r, int col) {
                    const int64_t to = d_tile + (int64_t)r * p.ldd + col;
                    if constexpr (OUT == 0) static_cast<uint16_t*>(p.d)[to] = (uint16_t)x;
                    if constexpr (OUT == 1) static_cast<float*>(p.d)[to] = __uint_as_float(x);
                    if constexpr (OUT == 2) static_cast<uint16_t*>(p.d)[to] = bf16_bits(__uint_as_float(x));
                });
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
                // Past the caches' order, in whole lines: it leaves them to the operands. Plain / so, us (4-bit NT, groups x
                // rows, n, k): 8 x 16384, 7168, 2048 177/163 (FP32 226/196), 4096, 7168 284/282, 32 x 4096, 2048, 2048
                // 28.0/25.4; BF16 TN 16384 rows to 8 x 4096 x 7168, FP32 + C, 1070/1034, NT 8 x 1000, 4096, 2048 38.4/37.1.
                // What reads D next finds less of it in the caches, so that a whole forward layer (NT, SwiGLU, NT, combination;
                // rows in groups, hidden, inner columns) gains little from it, and loses where D is small: BF16 16384 in 8, 7168,
                // 2048 1305/1295, 2048 in 8, 4096, 2048 152.8/152.0, 4096 in 8, 7168, 2048 353/354, 1001 in 16, 2048, 704 38.6/39.2;
                // in 4 bits (and a cast) 567/558, 63.6/62.6, 160/162, 30.1/30.8. TN of 4096 rows with a pass over D after it 391/377.
                // The sums of pieces, which the join reads: even (64 rows, 2112, 7168 17.0/17.0).
                typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
                __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]},
                                            reinterpret_cast<u32x4*>(static_cast<uint8_t*>(p.d) + to * SIZE));
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

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Row blocks of `bm` rows at most: whole ones, and a partial one for each group that has rows.
inline int64_t row_blocks(RaggedKind kind, const RaggedGemmArgs& a, int bm) {
    return kind == kRaggedTN ? ceil_div(a.m, bm) : a.rows / bm + std::min<int64_t>(a.groups, a.rows);
}

// Whether D's rows, and C's, begin at multiples of 16 bytes.
inline bool takes_vectors(const RaggedGemmArgs& a) {
    const int64_t size = a.out_f32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(a.d) % 16 == 0 && a.ldd * size % 16 == 0 && a.d_gs * size % 16 == 0 &&
           (!a.c || (reinterpret_cast<uintptr_t>(a.c) % 16 == 0 && a.ldc * size % 16 == 0 && a.c_gs * size % 16 == 0));
}

// Workgroups of a launch of `tile` x `tile` tiles (quarters: of its tail).
inline int64_t tile_blocks(RaggedKind kind, const RaggedGemmArgs& a, int tile, bool quarters, int slots) {
    const int64_t tiles = row_blocks(kind, a, tile) * ceil_div(a.n, tile);
    const int64_t blocks = kind == kRaggedTN ? ceil_div(tiles, 8) * 8 * a.groups : tiles;
    // (a tail has at most 58% of a round's tiles, for each XCD by itself in TN)
    return quarters ? std::min<int64_t>(blocks, kind == kRaggedTN ? std::max(slots / 8, 1) * 8 : slots) * 4 : blocks;
}

// Workgroups of the join of a call's pieces: 1024 columns of a row each.
inline int64_t join_blocks(RaggedKind kind, const RaggedGemmArgs& a) {
    return (kind == kRaggedTN ? (int64_t)a.groups * a.m : a.rows) * ceil_div(a.n, 1024);
}

}  // namespace
}  // namespace dgm
