// Attention of single tokens over the 8-bit paged key/value cache.
//
// Work. A unit is one row and four or eight query heads of one KV head; its tokens are cut into tiles of 128 (of 64 with head sizes above
// 128). The tiles of all units form one line (rows in order, then heads, then tokens), of which every CTA of a grid that fits the GPU takes an equal piece. The
// lengths are on the device, so each CTA works the line out for itself from the rows' positions. A unit that lies within a piece is
// finished there; the parts of one that is cut are left in the workspace, and the CTA that arrives last at the unit's counter joins
// them in order, so results do not hang on who arrives when.
//
// Mathematics. s = scale * ks_j * (q . kc_j), weights p_j = 2^(s_j log2 e - m) with a running reference m, and
// out = sum p_j vs_j vc_j / sum p_j. Both products are of integers: a query is rounded to 31 bits of its head's largest element and
// cut into four signed bytes (a balanced radix of 256), and the weight w_j = 2^(s_j log2 e - E) vs_j is cut into eight of them, in units of
// 2^-32, with a power of two E that moves on when a weight would pass 2^30. Two bytes of four heads are the columns of an mma.m16n8k32
// (int8, sums in int32), whose rows are tokens (keys) or elements (values): the codes go in as they are, without a conversion
// (values after a transpose of four by four bytes), and a step's sums are exact. E follows the weights with the scale, so scales of
// values may differ by any factor between tokens; m and E are whole numbers, so that moving them on rounds nothing.
//
// What small weights keep. A token far above the others says nothing about an element where its code is 0; that is made up of the
// others, whose weights must not drown in the digits of the large one. A warp's largest weight times scale is above 2^26, so one within
// 2^-41 of it (28 nats) is off by 2^-18 of itself at most. What the smaller ones lose is added up, and where it could be more than 2^-13 of an
// output, the warp goes over its tokens again for the digits behind those (exponentials end at 2^-126, 120 octaves below or more). Four bytes alone, which lose a weight of 2^-28 of the
// largest, took (us) 191 for 16 rows at 32000, 11.3 for one row at 3901, 12.9 for 32 rows at 512, 18.9 for 64 rows with a window of 1000; these take
// 207, 11.5, 13.6 and 21.6. A second pass doubles a warp's time; with scores of 3 nats some warp of a large grid has one in one call of three or so.
//
// What bounds it (back to back on three sets of inputs in turn; copy rate 6.46 TB/s). 16 rows at 32000 tokens of 8 KV heads of 128, 1.08 GB: 207 us, 5.2
// TB/s, after a second at the power limit of the card (1000 W, 1.5 GHz), 192 us in front of it: the bytes, and the energy of what is computed.
// 64 rows with a window of 1000 of 8 KV heads of 64, 70 MB: 21.6 us, 3.2 TB/s: instructions, issued in 0.58 of the cycles by 13 warps of an SM. 32
// rows at 512 of 8 of 128, 31 MB: 13.6 us; one row at 3901, 8 MB: 11.5 us; one at 57: 5.0 us. These are chains: lengths, blocks, keys, one to five steps
// of about 1 us, 0.6 us to fold the warps, 2 us to publish a part and hear who is last, 1.5 us to join. Dealing the last quarter of a long
// line out in chunks was slower (a change of units costs more than what the SMs differ by), and so were warps of their own for units,
// next segments entered ahead, and a smaller kernel made of loops.
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kv8.cuh"

namespace jl {
namespace {

constexpr int kStep = 32;                // tokens that a warp takes at a time
constexpr uint32_t kLongQuota = 8;       // tiles for each CTA from which on lines are cut without regard to units. 4 / 8 / 16: 64 rows with a
                                         // window of 1000 27.5 / 21.6 / 21.6 us, 8 rows at 2000 of 8 groups of 8 heads 22.6 / 20.6 / 20.6
constexpr int kRowsPerLane = 4;          // of up to 128 rows, short lines of which are cut by units
constexpr int kMostSms = 160, kMostCtas = 4 * kMostSms;
constexpr uint32_t kGroup = 32;          // parts that are joined at once
constexpr int kSlots = 4;                // for parts, of a CTA
static_assert(kMostCtas <= int(kGroup * kGroup));
constexpr int kFlush = 2048;             // steps after which sums of 2^14 a token could pass 2^30
constexpr float kNothing = -3e38f;       // m and E before there is a token
constexpr float kHeadroom = 26.f;        // E moves on so that weights are below 2^27, and again when one passes 1.5e9 or could pass 2^30
constexpr float kDeep = 0x1p1f, kLow = 0x1p-15f;  // weights that are off by 2^-18 of themselves at most with six bytes, and with eight
constexpr float kLoss = 0x1p-13f;        // of an output, that weights below the second may lose
constexpr float kMagic = 12582912.f;     // 1.5 * 2^23: a sum's low bits are those of the whole number, to the nearest
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// ---- layout of a stage in shared memory: 32 rows of keys, 32 rows of values, their scales, the mask of tokens that count -----------
// Rows are read in pieces of 4 to 16 bytes, eight rows (keys) or four (values) at once. With 64, 128 and 256 bytes a row, 16-byte pieces
// are exchanged within a 128-byte line so that neither read meets in a bank; rows of 96 bytes need nothing, rows of 192 are 208 apart.
template <int HD>
struct Layout {
    static constexpr int kPitch = HD == 192 ? 208 : HD;
    static constexpr int kValues = kStep * kPitch, kScales = 2 * kValues, kMask = kScales + 2 * kStep * 4;
    static constexpr int kStage = kMask + 16;
    static constexpr int kQuads = HD / 32;               // words of four elements that a lane has of a head's values
    static constexpr int kLoad = HD == 96 ? 1 : 2;       // words of values that one load brings

    // where 16-byte piece c of row r is
    __device__ static int piece(int r, int c) {
        if constexpr (HD == 64) return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (r & 2)) << 4);
        else if constexpr (HD == 128 || HD == 256) return r * HD + ((c ^ ((r & 1) << 2 | (r & 2))) << 4);
        else return r * kPitch + (c << 4);
    }
    // byte (= element) of a row that lane t's word w of keys starts at
    __device__ static constexpr int key_element(int t, int w) { return (w >> 1) * 32 + t * 8 + (w & 1) * 4; }
    // byte of a row that lane g's word j of values starts at
    __device__ static int value_element(int g, int j) {
        if constexpr (HD == 64) return g * 8 + j * 4;
        else if constexpr (HD == 96) return j * 32 + g * 4;
        else if constexpr (HD == 192) return (j >> 1) * 64 + g * 8 + (j & 1) * 4;
        else return (j >> 2) * 128 + g * 16 + (j & 3) * 4;
    }
};

// NT groups of four query heads have 3 / 8 * HD * NT accumulators. What these and the stages leave room for, with both sides measured (us): head
// size 128, 2 CTAs of 3 stages and 3 CTAs of 2: 13.6 / 15.8 (32 rows at 512 of 8 KV heads), 18.1 / 20.8 (1 row at 20000), 192 / 192 (16 rows at 32000), but
// 24.8 / 20.1 (128 rows at 100); 64 with one group, 4 CTAs of 3 and 3 of 4: 21.6 / 25.0 (64 rows, a window of 1000), but 124 / 117 (16 rows at 32000), with
// two groups, 2 of 6 and 3 of 4: 13.3 / 15.2 (8 rows at 2000 of 4 KV heads); 96, 3 of 2 and 2 of 4: 17.9 / 18.6 (16 rows at 2000); 192, 3 of 2 and 2 of
// 3: 33.3 / 36.8 (16 rows at 2000), 84 / 89 (at 8000), but 20.5 / 18.0 (1 row at 5000); 256, 2 of 3 and 2 of 2: 49.3 / 52.7 (16 rows at 2000).
template <int HD, int NT>
struct Shape {
    static constexpr int kWarps = HD <= 128 ? 4 : 2, kThreads = 32 * kWarps;
    static constexpr int kTile = kStep * kWarps;  // tokens of a tile
    static constexpr int kStages = HD == 64 ? (NT == 1 ? 3 : 6) : HD == 96 || HD == 192 ? 2 : 3;
    static constexpr int kRing = kStages * Layout<HD>::kStage, kBytes = kWarps * kRing;
    static constexpr int kHeads = 4 * NT, kPartFloats = kHeads * (HD + 3);
    static constexpr int kShare = HD / 16 / kWarps + (HD / 16 % kWarps != 0);  // words of the queries that a warp prepares
    static constexpr int kResident = NT == 1 && HD == 64 ? 4 : HD == 96 || HD == 192 ? 3 : 2;  // CTAs per SM
    static_assert(kResident * kMostSms <= kMostCtas);
    static_assert(Layout<HD>::kStage >= kHeads * HD * 4);  // a stage also holds a warp's outputs
    static_assert(kResident * (kBytes + NT * HD * 16 + kWarps * kShare * (NT * 256 + 64) + 128 * kHeads + 1024) <= 228 * 1024);
};

struct Params {
    jl_kv8_attention_args a;
    uint64_t divide;   // j / block_tokens = j * divide >> shift for j < 2^31
    int shift;
    int group, head_tiles;         // query heads per KV head, units that these are
    unsigned *arrivals;            // [3][CTAs], zero between launches
    float *parts;                  // [kSlots * CTAs][part floats]
};

__device__ __forceinline__ void mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x = b3 2^24 + b2 2^16 + b1 2^8 + b0 with signed bytes, for |x| below 2^31 - 2^24
__device__ __forceinline__ uint32_t signed_bytes(int x) { return (uint32_t(x) + 0x00808080u) ^ 0x00808080u; }
// Words of bytes x[i].b to words y[b].i.
__device__ __forceinline__ void transpose_bytes(const uint32_t (&x)[4], uint32_t (&y)[4]) {
    const uint32_t low01 = __byte_perm(x[0], x[1], 0x5140), high01 = __byte_perm(x[0], x[1], 0x7362);
    const uint32_t low23 = __byte_perm(x[2], x[3], 0x5140), high23 = __byte_perm(x[2], x[3], 0x7362);
    y[0] = __byte_perm(low01, low23, 0x5410), y[1] = __byte_perm(low01, low23, 0x7632);
    y[2] = __byte_perm(high01, high23, 0x5410), y[3] = __byte_perm(high01, high23, 0x7632);
}
__device__ __forceinline__ uint32_t pack(__half lo, __half hi) {
    const __half2 x = __halves2half2(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&x);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(from - to) of whole numbers from <= to, exactly (below 2^-126, and from kNothing: 0)
__device__ __forceinline__ float step_down(float from, float to) {
    return from == to ? 1.f : __int_as_float((__float_as_int(fmaxf(from - to, -127.f) + kMagic) - __float_as_int(kMagic) + 127) << 23);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t policy_normal() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
// SIZE bytes, or as many zeros
template <int SIZE>
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void *src, bool copy) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(SIZE), "r"(copy ? SIZE : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// A row's tokens [first, end) in its sequence's line of the table.
struct Row {
    uint32_t first, end;
    int slot;
};
__device__ __forceinline__ Row row_at(const jl_kv8_attention_args &a, int r) {
    const int slot = a.kv_slots ? a.kv_slots[r] : r, pos = a.positions[r];
    const int64_t seen = int64_t(pos) + 1, length = min(seen, int64_t(a.blocks_per_slot) * a.pages.block_tokens);
    const int64_t first = a.window > 0 ? max(seen - a.window, int64_t(0)) : 0;
    Row row = {0, 0, slot};
    if (slot >= 0 && slot < a.slots && first < length) row.first = uint32_t(first), row.end = uint32_t(length);
    return row;
}
// Tiles of a row's unit; the first begins at a multiple of 16 tokens. One at least, so that a row without tokens gets its zeros.
__device__ __forceinline__ uint32_t tiles_of(const Row &row, int tile) { return max(1u, (row.end - (row.first & ~15u) + tile - 1) / tile); }

// Sum of v over the CTA's threads; `before`: over those in front of this one.
template <int kWarps>
__device__ __forceinline__ uint32_t block_sum(uint32_t v, uint32_t *before, uint32_t *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(~0u, s, d);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    uint32_t base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) base += warp_sums[w];
        all += warp_sums[w];
    }
    *before = base + s - v;
    return all;
}

// PAGED16: blocks are multiples of 16 tokens, so sixteen rows from a multiple of sixteen on lie behind one another.
template <int HD, int NT, bool PAGED16>
__global__ void __launch_bounds__((Shape<HD, NT>::kThreads), (Shape<HD, NT>::kResident)) attention_kernel(const Params p) {
    using L = Layout<HD>;
    using S = Shape<HD, NT>;
    constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kTile = S::kTile, kHeads = S::kHeads;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t warp_sums[kWarps], start_row, start_tile;
    __shared__ float s_m[kWarps][kHeads], s_e[kWarps][kHeads], s_l[kWarps][kHeads];
    __shared__ int s_last;
    __shared__ uint32_t s_largest[kWarps][8 * NT];
    __shared__ float s_scale[kHeads];
    __shared__ uint4 s_query[NT][HD / 32][32];
    constexpr int kShare = S::kShare;
    __shared__ float4 s_raw[kWarps][kShare][NT][16], s_turn[kWarps][kShare][4];
    const jl_kv8_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    const int rows = a.token_count ? min(a.token_count[0], a.rows) : a.rows;

    // ---- what this CTA takes. Short lines: a piece of one unit, every unit cut into equal pieces of `quota` tiles at most, as
    // many as there are CTAs. Long ones, and more rows than four for each lane: [at, end) of the line, cut without regard to units.
    // Where a KV head has more query heads than a unit, neighbouring CTAs take the same tokens for their own heads at the same time,
    // and all but the first read them from L2.
    const uint32_t head_tile = blockIdx.x % p.head_tiles, cta = blockIdx.x / p.head_tiles;
    const int head0 = head_tile * kHeads, units = a.pages.kv_heads;
    uint32_t at = 0, end = 0, piece = 0, pieces = 0, in_row = 0, ctas = gridDim.x / p.head_tiles, quota = 0, more_than = 0, total = 0;
    int r = 0;
    Row row = {};
    if (rows <= 32 * kRowsPerLane) {
        Row mine[kRowsPerLane];  // rows lane + 32 k
        uint32_t tiles[kRowsPerLane] = {}, sum = 0;
#pragma unroll
        for (int k = 0; k < kRowsPerLane; ++k)
            if (32 * k < rows && lane + 32 * k < rows) {
                mine[k] = row_at(a, lane + 32 * k);
                sum += tiles[k] = tiles_of(mine[k], kTile);
            }
        total = __reduce_add_sync(~0u, sum) * units;
        const uint32_t whole_units = uint32_t(rows) * units;
        if (whole_units <= ctas && total < ctas * kLongQuota) {
            // a unit has half a piece more than its share on average
            quota = total / max(1u, ctas - whole_units / 2);
            uint32_t n[kRowsPerLane] = {}, all;
            do {
                quota += max(1u, quota / 8);
                sum = 0;
                const float inverse = __fdividef(1.f, float(quota));
#pragma unroll
                for (int k = 0; k < kRowsPerLane; ++k)
                    // the quotient's fraction is at least half a quota's part away from a whole number, and tiles are below 2^16
                    if (32 * k < rows) sum += n[k] = tiles[k] ? uint32_t((float(tiles[k] - 1) + 0.5f) * inverse) + 1 : 0;
                all = __reduce_add_sync(~0u, sum);
            } while (all * units > ctas);
            if (cta >= all * units) return;
            uint32_t front = 0;  // pieces of the rows before 32 k
#pragma unroll
            for (int k = 0; k < kRowsPerLane; ++k)
                if (32 * k < rows && pieces == 0) {
                    uint32_t before = n[k];
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const uint32_t o = __shfl_up_sync(~0u, before, d);
                        if (lane >= d) before += o;
                    }
                    const uint32_t in_chunk = __shfl_sync(~0u, before, 31);
                    const unsigned here = __ballot_sync(~0u, cta < (front + before) * units);  // the first of these lanes has it
                    if (here) {
                        const int from = __ffs(here) - 1;
                        r = from + 32 * k;
                        pieces = __shfl_sync(~0u, n[k], from);
                        piece = cta - (front + __shfl_sync(~0u, before, from) - pieces) * units;
                        row = {__shfl_sync(~0u, mine[k].first, from), __shfl_sync(~0u, mine[k].end, from), __shfl_sync(~0u, mine[k].slot, from)};
                    }
                    front += in_chunk;
                }
            in_row = piece / pieces;  // the unit
            piece -= in_row * pieces;
        }
    }
    if (pieces == 0) {
        if (rows > 32 * kRowsPerLane) {
            uint32_t mine = 0, before;
            for (int i = tid; i < rows; i += kThreads) mine += tiles_of(row_at(a, i), kTile);
            total = block_sum<kWarps>(mine, &before, warp_sums) * units;
        }
        if (total == 0) return;
        ctas = min(ctas, total);
        if (cta >= ctas) return;
        quota = total / ctas;
        more_than = total % ctas;  // so many CTAs take one more
        at = cta * quota + min(cta, more_than);
        end = at + quota + (cta < more_than);
        uint32_t front = 0;  // tiles in front of the rows from `base` on
        for (int base = 0; base < rows && front <= at; base += kThreads) {
            uint32_t before;
            const uint32_t mine = base + tid < rows ? tiles_of(row_at(a, base + tid), kTile) * units : 0, all = block_sum<kWarps>(mine, &before, warp_sums);
            if (at >= front + before && at < front + before + mine) {
                start_row = base + tid;
                start_tile = at - front - before;
            }
            front += all;
        }
        __syncthreads();
        r = start_row;
        in_row = start_tile;
    }
    auto owner = [&](uint32_t tile) {
        const uint32_t longer = more_than * (quota + 1);
        return tile < longer ? tile / (quota + 1) : more_than + (tile - longer) / quota;
    };

    unsigned char *ring = smem + warp * S::kRing;
    const uint32_t ring_at = smem_u32(ring);
    const int bt = a.pages.block_tokens;

    // The segment under way: tiles [tile, tile + take) of a unit, tokens [from, to); `mine` steps of them are this warp's, step i at
    // token from + (warp + warps i) 32.
    struct Segment {
        uint32_t first, from, to, tiles, tile, take;
        int kv, mine, pos;
        const int32_t *line;
    } seg;
    auto enter = [&]() {
        if (!pieces) row = row_at(a, r);
        seg.tiles = tiles_of(row, kTile);
        uint32_t unit = in_row;
        if (pieces) {
            seg.take = seg.tiles / pieces;
            const uint32_t longer = seg.tiles - seg.take * pieces;
            seg.tile = piece * seg.take + min(piece, longer);
            seg.take += piece < longer;
        } else {
            unit = in_row / seg.tiles;
            seg.tile = in_row % seg.tiles;
            seg.take = min(seg.tiles - seg.tile, end - at);
        }
        seg.kv = unit;
        seg.first = row.first;
        seg.from = (row.first & ~15u) + seg.tile * kTile;
        seg.to = min(row.end, seg.from + seg.take * kTile);
        const int steps = seg.to > seg.from ? int((seg.to - seg.from + kStep - 1) / kStep) : 0;
        seg.mine = steps > warp ? (steps - warp + kWarps - 1) / kWarps : 0;
        seg.pos = a.positions[r];
        seg.line = a.block_table + int64_t(row.slot) * a.blocks_per_slot;
    };
    auto step_at = [&](int i) { return seg.from + uint32_t(warp + i * kWarps) * kStep; };
    auto block_of = [&](uint32_t j) { return uint32_t((j * p.divide) >> p.shift); };

    // PAGED16: lane i looks up the sixteen tokens i & 1 of step 16 k + i / 2 of this warp, 16 steps ahead: where their codes and scales
    // begin, or -1. Otherwise it looks up token i of a step, one step ahead.
    int64_t code_at = -1, scale_at = -1;
    int ahead;
    auto my_token = [&](int i) { return PAGED16 ? step_at(i + (lane >> 1)) + 16 * (lane & 1) : step_at(i) + lane; };
    auto look_up = [&](int i) {
        const uint32_t j = my_token(i);
        return i + (PAGED16 ? lane >> 1 : 0) < seg.mine && j < seg.to ? seg.line[block_of(j)] : -1;
    };
    auto place = [&](int block, uint32_t j) {
        const bool good = block >= 0 && block < a.pages.blocks;
        const int64_t in_block = int64_t(seg.kv) * bt + (j - block_of(j) * bt);
        code_at = good ? block * a.pages.block_stride + in_block * HD : -1;
        scale_at = good ? block * a.pages.scale_stride + in_block : -1;
    };
    // Codes that no CTA reads for other heads of its unit's are the first to leave L2: with and without, 16 rows at 32000 192 / 197 us, 64 rows with a
    // window of 1000 21.6 / 22.8, 16 rows at 8000 of head size 192 84 / 89. Rows that read the same blocks find most of them there all the same: 32 rows of
    // one sequence of 4000 tokens 50.5 / 50.4, of 16000 168 / 157, 128 rows of 4000 166 / 166, a third of the blocks in common 50.5 / 51.0.
    const uint64_t policy = p.head_tiles == 1 ? policy_evict_first() : policy_normal();
    // Keys, scales and mask of step i, and its values, as groups of copies of their own.
    auto copy_rows = [&](int i, const int8_t *pages, uint32_t stage) {
        if constexpr (PAGED16) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int64_t code = __shfl_sync(~0u, code_at, 2 * (i & 15) + half);
                if (code >= 0) {
                    const int8_t *src = pages + code + lane * 16;
#pragma unroll
                    for (int n = 0; n < HD / 32; ++n) {
                        const int piece16 = n * 32 + lane;
                        copy16(stage + L::piece(16 * half + piece16 / (HD / 16), piece16 % (HD / 16)), src + n * 512, policy);
                    }
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                const int piece16 = n * 32 + lane, row32 = piece16 / (HD / 16), c = piece16 % (HD / 16);
                const int64_t src = __shfl_sync(~0u, code_at, row32);
                if (src >= 0) copy16(stage + L::piece(row32, c), pages + src + c * 16, policy);
            }
        }
    };
    auto issue_keys = [&](int i) {
        if (i < seg.mine) {
            const uint32_t stage = ring_at + uint32_t(i % S::kStages) * L::kStage, j0 = step_at(i);
            unsigned mask = (j0 < seg.first ? ~0u << (seg.first - j0) : ~0u) & (seg.to - j0 < 32 ? (1u << (seg.to - j0)) - 1 : ~0u);
            int64_t scale;
            if constexpr (PAGED16) {
                if (i % 16 == 0) {
                    place(ahead, my_token(i));
                    ahead = look_up(i + 16);
                }
                scale = __shfl_sync(~0u, scale_at, 2 * (i & 15) + (lane >> 4));
                if (scale >= 0) scale += lane & 15;
            } else {
                place(ahead, j0 + lane);
                ahead = look_up(i + 1);
                scale = scale_at;
            }
            copy_rows(i, a.pages.k, stage);
            if (scale >= 0) {
                copy4(stage + L::kScales + 4 * lane, a.pages.k_scale + scale);
                copy4(stage + L::kScales + 4 * kStep + 4 * lane, a.pages.v_scale + scale);
            }
            mask &= __ballot_sync(~0u, scale >= 0);
            if (lane == 0) *reinterpret_cast<unsigned *>(ring + (i % S::kStages) * L::kStage + L::kMask) = mask;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto issue_values = [&](int i) {
        if (i < seg.mine) copy_rows(i, a.pages.v, ring_at + uint32_t(i % S::kStages) * L::kStage + L::kValues);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Queries of a segment, as they are, and their places in the rotation tables: the words that this warp prepares. On the way before the keys.
    auto load_queries = [&]() {
#pragma unroll
        for (int i = 0; i < kShare; ++i) {
            const int word = warp * kShare + i, el = L::key_element(t, word);
            if (word >= HD / 16) continue;
            if ((g & 1) == 0)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int head = head0 + 4 * n + (g >> 1);
                    const bool here = head < p.group;
                    const int64_t at_q = here ? int64_t(r) * a.q_stride + int64_t(seg.kv * p.group + head) * HD + el : 0;
                    const uint32_t dst = smem_u32(&s_raw[warp][i][n][(g >> 1) * 4 + t]);
                    if (a.ggml_type == JL_F16) copy_or_zero<8>(dst, static_cast<const __half *>(a.q) + at_q, here);
                    else copy_or_zero<16>(dst, static_cast<const float *>(a.q) + at_q, here);
                }
            else if (g == 1 && a.rope_cos && seg.pos >= 0 && seg.pos < a.rope_rows) {
                const int64_t angle = int64_t(seg.pos) * (HD / 2) + el / 2;
                const uint32_t dst = smem_u32(&s_turn[warp][i][t]);
                copy_or_zero<8>(dst, a.rope_cos + angle, true);
                copy_or_zero<8>(dst + 8, a.rope_sin + angle, true);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto begin = [&]() {
        enter();
        ahead = look_up(0);
        load_queries();
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) {
            issue_keys(i);
            issue_values(i);
        }
    };

    // Units of this CTA that others have a part of: two at most, its first and its last. Whether it was the last to arrive at one
    // is asked for at once, and looked at when nothing else is left to do.
    struct Shared {
        int r, kv;
        uint32_t first, parts;
    } shared[2];
    int n_shared = 0;
    bool arrived_last[2] = {false, false};  // thread 0
    // A CTA's slots: the part of its first segment, of its last, and joined parts of a group that begins behind or with a unit's first CTA.
    auto slot_of = [&](uint32_t owner, int slot) { return p.parts + ((size_t(owner) * p.head_tiles + head_tile) * kSlots + slot) * S::kPartFloats; };
    // Thread 0: whether this CTA is the last of its unit, or, of a unit of more than kGroup parts, of its group. The last one to come sets
    // the counter back to zero. Counters: by a unit's first CTA, by a later group's first CTA, and of the groups by the unit's first CTA.
    auto count_in = [&](int which, uint32_t owner, uint32_t all) {
        __threadfence();
        const bool is_last = atomicInc(p.arrivals + which * kMostCtas + owner * p.head_tiles + head_tile, all - 1) == all - 1;
        __threadfence();
        return is_last;
    };
    auto arrive = [&](const Shared &unit) {
        const uint32_t group = (cta - unit.first) / kGroup, in_front = group * kGroup;
        return count_in(group > 0, unit.first + in_front, unit.parts > kGroup ? min(kGroup, unit.parts - in_front) : unit.parts);
    };

    // quad f = n kQuads + j of lane (g, t): four elements of head 4 n + t
    auto finish = [&](int f, int row, int kv, float4 x, float top, float etop, float sum) {
        const int head = 4 * (f / L::kQuads) + t;
        if (head0 + head >= p.group) return;
        // 2^(etop - top) / sum, in two factors: either may be beyond binary32 where the output is not. The two are less than 200 apart:
        // a scale's exponent is between -126 and 128, E within 30 of the largest weight's, m within 20 of the largest score.
        const float inverse = sum == 0.f ? 0.f : 1.f / sum;
        const int power = sum == 0.f || !(fabsf(etop - top) < 200.f) ? 0 : int(etop - top), h1 = power / 2;
        const float f1 = inverse * __int_as_float((127 + h1) << 23), f2 = __int_as_float((127 + power - h1) << 23);
        x = make_float4(x.x * f1 * f2, x.y * f1 * f2, x.z * f1 * f2, x.w * f1 * f2);
        const int64_t out_at = int64_t(row) * a.out_stride + int64_t(kv * p.group + head0 + head) * HD + L::value_element(g, f % L::kQuads);
        if (a.ggml_type == JL_F16) {
            const uint2 h = make_uint2(pack(__float2half_rn(x.x), __float2half_rn(x.y)), pack(__float2half_rn(x.z), __float2half_rn(x.w)));
            *reinterpret_cast<uint2 *>(static_cast<__half *>(a.out) + out_at) = h;
        } else {
            *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + out_at) = x;
        }
        if (a.lse && f % L::kQuads == 0 && g == 0)
            a.lse[int64_t(row) * a.heads + kv * p.group + head0 + head] = sum == 0.f ? -CUDART_INF_F : fmaf(top, kLn2, logf(sum));
    };

    begin();
    for (;;) {
        const int mine = seg.mine, kv = seg.kv;

        // ---- queries: of group n, column g of the first product is byte 3 (g even) or 2 of head 4 n + g / 2, of the second byte 1 or 0.
        // Rotated, as whole numbers below 2^30. A warp does its share of the words, and takes the others' from shared memory.
        {
            const bool outside = a.rope_cos && seg.pos >= a.rope_rows, turn = a.rope_cos && seg.pos >= 0 && !outside;
            const uint32_t select_high = g & 1 ? 0x0062 : 0x0073, select_low = g & 1 ? 0x0040 : 0x0051;
            float x[NT][kShare][4];
            asm volatile("cp.async.wait_group %0;" ::"n"(2 * S::kStages - 2) : "memory");
            __syncwarp();
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t largest = outside ? 0x7f800000u : 0u;  // of the elements' magnitudes, as bits
#pragma unroll
                for (int i = 0; i < kShare; ++i) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (warp * kShare + i < HD / 16) {
                        v = s_raw[warp][i][n][(g >> 1) * 4 + t];
                        if (a.ggml_type == JL_F16) {
                            const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)), hi = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
                            v = make_float4(lo.x, lo.y, hi.x, hi.y);
                        }
                        if (turn) {
                            const float4 c = s_turn[warp][i][t];  // two cosines, two sines
                            v = make_float4(v.x * c.x - v.y * c.z, v.x * c.z + v.y * c.x, v.z * c.y - v.w * c.w, v.z * c.w + v.w * c.y);
                        }
                    }
                    x[n][i][0] = v.x, x[n][i][1] = v.y, x[n][i][2] = v.z, x[n][i][3] = v.w;
#pragma unroll
                    for (int k = 0; k < 4; ++k) largest = max(largest, __float_as_uint(x[n][i][k]) & 0x7fffffffu);
                }
                largest = max(largest, __shfl_xor_sync(~0u, largest, 1));
                largest = max(largest, __shfl_xor_sync(~0u, largest, 2));
                if (t == 0) s_largest[warp][n * 8 + g] = largest;
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t largest = 0;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) largest = max(largest, s_largest[w][n * 8 + g]);
                const bool finite = largest < 0x7f800000u;
                // 2^(29 - exponent of the largest), which may be 2^156, in two factors
                const int shift = finite ? 29 - (int(largest >> 23) - 127) : 0, rest = max(shift - 126, 0);
                const float up = __uint_as_float(uint32_t(127 + shift - rest) << 23), up_rest = __uint_as_float(uint32_t(127 + rest) << 23);
#pragma unroll
                for (int i = 0; i < kShare; ++i) {
                    const int word = warp * kShare + i;
                    uint32_t b[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) b[k] = signed_bytes(finite ? __float2int_rn(x[n][i][k] * up * up_rest) : 0);
                    if (word < HD / 16) {
                        uint32_t *to = reinterpret_cast<uint32_t *>(&s_query[n][word / 2][lane]) + (word & 1);
                        to[0] = __byte_perm(__byte_perm(b[0], b[1], select_high), __byte_perm(b[2], b[3], select_high), 0x5410);
                        to[2] = __byte_perm(__byte_perm(b[0], b[1], select_low), __byte_perm(b[2], b[3], select_low), 0x5410);
                    }
                }
                if (warp == 0 && t == 0 && (g & 1) == 0)
                    s_scale[4 * n + g / 2] = finite ? a.scale * kLog2e * __uint_as_float(uint32_t(127 - shift + rest) << 23) * __uint_as_float(uint32_t(127 - rest) << 23) : CUDART_NAN_F;
            }
            __syncthreads();
        }
        float factor[NT];  // of head 4 n + t
#pragma unroll
        for (int n = 0; n < NT; ++n) factor[n] = s_scale[4 * n + t];

        // ---- one pass over this warp's tokens, or more where small weights want it: lane (g, t) has tokens g, g + 8, g + 16, g + 24 of a
        // step, heads 4 n + t, elements of column g. The four tokens of g are bytes of one word of weights, and so are those of t and of t + 4 in a word of values.
        float m[NT], e[NT], l[NT], o[NT][L::kQuads][4];
        int acc[NT][2 * L::kQuads][4];  // elements 2 i and 2 i + 1 of a word; bytes 7 and 6 of the weights
        float loss[NT];                 // of weights below kLow
        bool bad = false;               // a value's scale was no number
        int since, pass = 0;            // steps in `acc`; passes over the tokens in front of this one
        float unit = 1.f;               // of this pass's weights, next to 2^E
        volatile float sums[NT * L::kQuads * 4];  // of the passes in front
        // o = (o + acc) keep, acc = 0; the other bytes' products are in `o` already
        auto flush = [&](int n, float keep) {
#pragma unroll
            for (int j = 0; j < 2 * L::kQuads; ++j)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    int(&c)[4] = acc[n][j];
                    float &y = o[n][j / 2][2 * (j & 1) + k];
                    // below 2^22 each: two fit one number
                    const float x = since <= 8 ? float(c[2 * k] * 256 + c[2 * k + 1]) : fmaf(float(c[2 * k]), 256.f, float(c[2 * k + 1]));
                    y = fmaf(x, unit * 0x1p16f, y) * keep;
                    c[2 * k] = c[2 * k + 1] = 0;
                }
        };
    again:
        since = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n] = e[n] = kNothing;
            l[n] = loss[n] = 0.f;
#pragma unroll
            for (int j = 0; j < L::kQuads; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
#pragma unroll
            for (int j = 0; j < 2 * L::kQuads; ++j) acc[n][j][0] = acc[n][j][1] = acc[n][j][2] = acc[n][j][3] = 0;
        }
        // A step's keys are free when its scores are done, its values when they are added: both are refilled then, kStages steps ahead.
        issue_keys(S::kStages - 1);
        issue_values(S::kStages - 1);
        for (int i = 0; i < mine; ++i) {
            const unsigned char *stage = ring + (i % S::kStages) * L::kStage;
            asm volatile("cp.async.wait_group %0;" ::"n"(2 * S::kStages - 1) : "memory");
            __syncwarp();

            int s[NT][2][2][4] = {};  // tokens g and g + 8, g + 16 and g + 24; bytes 3 and 2, 1 and 0
#pragma unroll
            for (int w = 0; w < HD / 16; w += 2) {
                uint4 q[NT];  // the first product's words w and w + 1, the second's
#pragma unroll
                for (int n = 0; n < NT; ++n) q[n] = s_query[n][w / 2][lane];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int rk = g + 16 * half, el = L::key_element(t, w);
                    const uint2 x = *reinterpret_cast<const uint2 *>(stage + L::piece(rk, el >> 4) + (el & 15)), y = *reinterpret_cast<const uint2 *>(stage + L::piece(rk + 8, el >> 4) + (el & 15));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma(s[n][half][0], x.x, y.x, x.y, y.y, q[n].x, q[n].y);
                        mma(s[n][half][1], x.x, y.x, x.y, y.y, q[n].z, q[n].w);
                    }
                }
            }

            // scores in units of ln 2 and weights
            const unsigned mask = *reinterpret_cast<const unsigned *>(stage + L::kMask) >> g;
            const float *ks = reinterpret_cast<const float *>(stage + L::kScales) + g, *vs = ks + kStep;
            float v[4];
            bool odd_scale = false;  // beyond 2^-60 .. 2^4: exponents are taken apart below, so that no exponential is lost in front of a large scale
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = mask >> (8 * k) & 1 ? vs[8 * k] : 1.f;
                odd_scale = odd_scale || (__float_as_uint(v[k]) & 0x7fffffffu) - 0x21800000u > 0x41800000u - 0x21800000u;
            }
            float y[NT][4], keep[NT];
            float least = kDeep;  // of the weights
            bool moved = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4];
                keep[n] = 1.f;
                bool beyond = odd_scale;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int(&c)[2][4] = s[n][k >> 1];
                    const int at2 = 2 * (k & 1);
                    const float dot = fmaf(float(c[0][at2] * 256 + c[0][at2 + 1]), 65536.f, float(c[1][at2] * 256 + c[1][at2 + 1]));
                    x[k] = mask >> (8 * k) & 1 ? dot * factor[n] * ks[8 * k] : -CUDART_INF_F;
                    // from the largest's place, not from the unit's, which is 26 octaves away: the difference would be rounded 2^5 times as coarsely
                    y[n][k] = exp2_approx(x[k] - (e[n] + kHeadroom)) * (v[k] * 0x1p26f);
                    beyond = beyond || x[k] - m[n] > 20.f || fabsf(y[n][k]) > 1.5e9f;
                }
                if (__any_sync(~0u, beyond)) {
                    float mantissa[4], exponent[4], top = kNothing, etop = kNothing;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t bits = __float_as_uint(v[k]), ex = bits >> 23 & 255;
                        bad = bad || ex == 255;
                        mantissa[k] = ex ? __uint_as_float((bits & 0x807fffffu) | 0x3f800000u) : v[k] * 0x1p126f;
                        exponent[k] = __uint_as_float(0x4b000000u | max(ex, 1u)) - 8388735.f;  // 2^23 + 127
                        top = fmaxf(top, x[k]), etop = fmaxf(etop, x[k] + exponent[k]);
                    }
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                        etop = fmaxf(etop, __shfl_xor_sync(~0u, etop, d));
                    }
                    const float m_new = top - m[n] > 20.f ? ceilf(top) : m[n], e_new = etop - e[n] > 29.f ? ceilf(etop) - kHeadroom : e[n];
                    l[n] *= step_down(m[n], m_new);
                    keep[n] = step_down(e[n], e_new);
                    moved = moved || __any_sync(~0u, keep[n] != 1.f);
                    m[n] = m_new;
                    e[n] = e_new;
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[n][k] = exp2_approx(x[k] - (e[n] + kHeadroom) + exponent[k]) * (mantissa[k] * 0x1p26f);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) l[n] += exp2_approx(x[k] - m[n]);
                for (int times = 0; times < pass; ++times)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float z = y[n][k] * 0x1p32f;
                        y[n][k] = (z - __ll2float_rn(__float2ll_rn(z))) * 0x1p26f;  // exact
                    }
#pragma unroll
                for (int k = 0; k < 4; ++k) least = fminf(least, fabsf(y[n][k]));
            }
            // The last two bytes only where a weight is below 2: 16 rows at 32000 207 us, 214 with them always; 32 rows at 512 13.6 / 13.9; 64 rows
            // with a window of 1000 21.6 / 22.3.
            const bool deep = __any_sync(~0u, least < kDeep);
            if (moved || since == kFlush) {
#pragma unroll
                for (int n = 0; n < NT; ++n) flush(n, keep[n]);
                since = 0;
            }
            ++since;
            // Weights as eight signed bytes, in units of 2^-32; pairs of them are columns, as of the queries. Lane (g, t) has the bytes of head t and
            // tokens g; column g is of head g / 2; groups of tokens t and t + 4.
            uint32_t w[NT][4][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t low[4], high[4], digit[4];
                auto columns = [&](int pair, int upper) {
#pragma unroll
                    for (int far = 0; far < 2; ++far) {
                        const int from = (t + 4 * far) * 4 + (g >> 1);
                        const uint32_t even = __shfl_sync(~0u, digit[upper], from), odd = __shfl_sync(~0u, digit[upper - 1], from);
                        w[n][pair][far] = g & 1 ? odd : even;
                    }
                };
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t bytes = (uint64_t(__float2ll_rn(y[n][k] * 0x1p32f)) + 0x0080808080808080u) ^ 0x0080808080808080u;
                    low[k] = uint32_t(bytes), high[k] = uint32_t(bytes >> 32);
                }
                transpose_bytes(high, digit);
                columns(0, 3);
                columns(1, 1);
                transpose_bytes(low, digit);
                columns(2, 3);
                if (deep) columns(3, 1);
            }
            if (deep && __any_sync(~0u, least < kLow)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) loss[n] += fabsf(y[n][k]) < kLow ? fminf(fabsf(y[n][k]), 0x1p-33f) : 0.f;
            }

            __syncwarp();  // every lane has read keys and scales
            issue_keys(i + S::kStages);
            asm volatile("cp.async.wait_group %0;" ::"n"(2 * S::kStages - 1) : "memory");
            __syncwarp();
            // values: of a word of column g, elements 0 and 1 are rows g and g + 8 of one product, 2 and 3 of the next
            auto multiply = [&](auto pairs) {
#pragma unroll
                for (int j0 = 0; j0 < L::kQuads; j0 += L::kLoad) {
                    uint32_t near[L::kLoad][4], far[L::kLoad][4];  // tokens t + 8 k, t + 4 + 8 k
                    const int el = L::value_element(g, j0);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const unsigned char *at_near = stage + L::kValues + L::piece(t + 8 * k, el >> 4) + (el & 15), *at_far = stage + L::kValues + L::piece(t + 4 + 8 * k, el >> 4) + (el & 15);
                        if constexpr (L::kLoad == 2) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(at_near), z = *reinterpret_cast<const uint2 *>(at_far);
                            near[0][k] = x.x, near[1][k] = x.y, far[0][k] = z.x, far[1][k] = z.y;
                        } else {
                            near[0][k] = *reinterpret_cast<const uint32_t *>(at_near), far[0][k] = *reinterpret_cast<const uint32_t *>(at_far);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < L::kLoad; ++j) {
                        uint32_t x[4], z[4];
                        transpose_bytes(near[j], x);
                        transpose_bytes(far[j], z);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                float(&to)[4] = o[n][j0 + j];
#pragma unroll
                                for (int b = decltype(pairs)::value - 1; b > 0; --b) {
                                    int c[4] = {0, 0, 0, 0};
                                    mma(c, x[2 * half], x[2 * half + 1], z[2 * half], z[2 * half + 1], w[n][b][0], w[n][b][1]);
                                    const float of = unit * (b == 3 ? 0x1p-32f : b == 2 ? 0x1p-16f : 1.f);
                                    to[2 * half] = fmaf(float(c[0] * 256 + c[1]), of, to[2 * half]);
                                    to[2 * half + 1] = fmaf(float(c[2] * 256 + c[3]), of, to[2 * half + 1]);
                                }
                                mma(acc[n][2 * (j0 + j) + half], x[2 * half], x[2 * half + 1], z[2 * half], z[2 * half + 1], w[n][0][0], w[n][0][1]);
                            }
                    }
                }
            };
            if (deep) multiply(std::integral_constant<int, 4>());
            else multiply(std::integral_constant<int, 3>());
            __syncwarp();  // every lane has read the values
            issue_values(i + S::kStages);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        bool some = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            flush(n, 1.f);
            some = some || loss[n] != 0.f;
        }
        bad = __any_sync(~0u, bad);
        some = __any_sync(~0u, some);
        // Another pass, for the digits behind those of this one, where weights below kLow may have lost too much; E takes the same way. 58 binary
        // digits a pass; what is below 2^-148 is left out.
        if (pass || some) {
            bool lost = some && pass < 2 && !bad;
            if (pass == 0) {
                bool small = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) loss[n] += __shfl_xor_sync(~0u, loss[n], d);
#pragma unroll
                    for (int j = 0; j < L::kQuads; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) small = small || fabsf(o[n][j][k]) * kLoss < 128.f * loss[n];
                }
                lost = __any_sync(~0u, small) && lost;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < L::kQuads; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (pass) o[n][j][k] += sums[(n * L::kQuads + j) * 4 + k];
                        if (lost) sums[(n * L::kQuads + j) * 4 + k] = o[n][j][k];
                    }
            if (lost) {
                ++pass;
                unit *= 0x1p-58f;
                ahead = look_up(0);
                for (int i = 0; i < S::kStages - 1; ++i) {
                    issue_keys(i);
                    issue_values(i);
                }
                goto again;
            }
        }
        if (bad)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < L::kQuads; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = CUDART_NAN_F;

        // ---- the next segment's first stages are on their way while this one's warps are folded, in the stage that they leave free.
        // Outputs lie there as [group][quad][lane], four elements of head t each.
        const int row = r;
        // the CTAs that have a part of this unit
        const uint32_t first_cta = pieces ? cta - piece : owner(at - seg.tile), last_cta = pieces ? first_cta + pieces - 1 : owner(at - seg.tile + seg.tiles - 1);
        at += seg.take;
        in_row += seg.take;
        if (in_row == seg.tiles * uint32_t(units)) ++r, in_row = 0;
        const bool more = !pieces && at < end;
        if (!more) pdl_launch_dependents();  // not before: early CTAs of the next launch would take the places that spread this one's out
        if (more) begin();
        float4 *out_w = reinterpret_cast<float4 *>(ring + (S::kStages - 1) * L::kStage);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[n] += __shfl_xor_sync(~0u, l[n], d);
            if (g == 0) s_m[warp][4 * n + t] = m[n], s_e[warp][4 * n + t] = e[n], s_l[warp][4 * n + t] = l[n];
#pragma unroll
            for (int j = 0; j < L::kQuads; ++j) out_w[(n * L::kQuads + j) * 32 + lane] = make_float4(o[n][j][0], o[n][j][1], o[n][j][2], o[n][j][3]);
        }
        __syncthreads();
        const bool whole = first_cta == last_cta;
        float *part = slot_of(cta, cta == first_cta);
        for (int f = warp; f < NT * L::kQuads; f += kWarps) {
            const int head = 4 * (f / L::kQuads) + t;
            float top = -CUDART_INF_F, etop = -CUDART_INF_F, sum = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][head]), etop = fmaxf(etop, s_e[w][head]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float keep = step_down(s_e[w][head], etop);
                const float4 y = reinterpret_cast<const float4 *>(smem + w * S::kRing + (S::kStages - 1) * L::kStage)[f * 32 + lane];
                sum += s_l[w][head] * step_down(s_m[w][head], top);
                x.x += y.x * keep, x.y += y.y * keep, x.z += y.z * keep, x.w += y.w * keep;
            }
            if (whole) {
                finish(f, row, kv, x, top, etop, sum);
            } else {
                reinterpret_cast<float4 *>(part)[f * 32 + lane] = x;
                if (f % L::kQuads == 0 && g == 0) {
                    float *stats = part + kHeads * HD + head;
                    stats[0] = top, stats[kHeads] = etop, stats[2 * kHeads] = sum;
                }
            }
        }
        __syncthreads();  // the part is written, the fold's stage is free
        if (!whole) {
            const Shared unit = {row, kv, first_cta, last_cta - first_cta + 1};
            if (tid == 0) {
                const bool is_last = arrive(unit);
                if (n_shared == 0) arrived_last[0] = is_last;
                else arrived_last[1] = is_last;
            }
            if (n_shared == 0) shared[0] = unit;
            else shared[1] = unit;
            ++n_shared;
        }
        if (!more) break;
    }

    // ---- join the units that this CTA came last to: a group's parts, 32 at most, then the groups. Every warp works out the parts' weights for
    // itself (lane (g, t) those of parts g, g + 8, ... of heads 4 n + t) and has its own quads of the outputs, so nothing is waited for in between.
    for (int u = 0; u < n_shared; ++u) {
        const Shared unit = u ? shared[1] : shared[0];
        if (tid == 0) s_last = u ? arrived_last[1] : arrived_last[0];
        __syncthreads();
        bool here = s_last;
        const uint32_t group = (cta - unit.first) / kGroup, in_front = group * kGroup;
        for (int level = unit.parts > kGroup ? 0 : 1; here; ++level) {
            const bool groups = unit.parts > kGroup && level == 1;
            const int n = level == 0 ? min(kGroup, unit.parts - in_front) : groups ? (unit.parts + kGroup - 1) / kGroup : unit.parts;
            // part k, and its slot: that of the unit's first part is another one
            const float *base = slot_of(unit.first + (level == 0 ? in_front : 0), groups ? 2 : 0);
            const size_t stride = size_t(p.head_tiles) * kSlots * S::kPartFloats * (groups ? kGroup : 1);
            const int first_slot = groups ? S::kPartFloats : level == 0 && group ? 0 : S::kPartFloats;
            auto part_of = [&](int k) { return base + k * stride + (k ? 0 : first_slot); };
            // sixteen parts' quads at once
            float4 y[16];
            auto load = [&](int f, int k0) {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (k0 + k < n) y[k] = __ldcg(reinterpret_cast<const float4 *>(part_of(k0 + k)) + f * 32 + lane);
            };
            if (warp < L::kQuads) load(warp, 0);
            float top[NT], etop[NT], sum[NT], keep[NT][kGroup / 8];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float m[kGroup / 8], e[kGroup / 8], l[kGroup / 8];
                top[i] = etop[i] = -CUDART_INF_F;
                sum[i] = 0.f;
#pragma unroll
                for (int k = 0; k < int(kGroup / 8); ++k) {
                    m[k] = e[k] = -CUDART_INF_F;
                    l[k] = 0.f;
                    if (g + 8 * k < n) {
                        const float *stats = part_of(g + 8 * k) + kHeads * HD + 4 * i + t;
                        m[k] = __ldcg(stats), e[k] = __ldcg(stats + kHeads), l[k] = __ldcg(stats + 2 * kHeads);
                    }
                    top[i] = fmaxf(top[i], m[k]), etop[i] = fmaxf(etop[i], e[k]);
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], d));
                    etop[i] = fmaxf(etop[i], __shfl_xor_sync(~0u, etop[i], d));
                }
#pragma unroll
                for (int k = 0; k < int(kGroup / 8); ++k) {
                    sum[i] += l[k] * step_down(m[k], top[i]);
                    keep[i][k] = step_down(e[k], etop[i]);
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum[i] += __shfl_xor_sync(~0u, sum[i], d);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
                for (int j = warp; j < L::kQuads; j += kWarps) {
                    const int f = i * L::kQuads + j;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int half = 0; half < int(kGroup / 16); ++half) {
                        if (16 * half >= n) break;
                        if (f != warp || half) load(f, 16 * half);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float w = __shfl_sync(~0u, keep[i][2 * half + k / 8], 4 * (k & 7) + t);
                            if (16 * half + k < n) x.x += y[k].x * w, x.y += y[k].y * w, x.z += y[k].z * w, x.w += y[k].w * w;
                        }
                    }
                    if (level == 1) {
                        finish(f, unit.r, unit.kv, x, top[i], etop[i], sum[i]);
                    } else {
                        float *to = slot_of(unit.first + in_front, group ? 2 : 3);
                        reinterpret_cast<float4 *>(to)[f * 32 + lane] = x;
                        if (j == 0 && g == 0) {
                            float *stats = to + kHeads * HD + 4 * i + t;
                            stats[0] = top[i], stats[kHeads] = etop[i], stats[2 * kHeads] = sum[i];
                        }
                    }
                }
            if (level == 1) break;
            __syncthreads();
            if (tid == 0) s_last = count_in(2, unit.first, (unit.parts + kGroup - 1) / kGroup);
            __syncthreads();
            here = s_last;
        }
        __syncthreads();  // s_last has been read
    }
}

template <int HD, int NT, bool PAGED16>
cudaError_t launch(Params &p, const Kv8Scratch &s, const Kv8Launch &l) {
    using S = Shape<HD, NT>;
    static std::atomic<uint64_t> configured{0};  // a bit for each device
    const cudaError_t e = kv8_allow_shared(reinterpret_cast<const void *>(attention_kernel<HD, NT, PAGED16>), S::kBytes, configured);
    if (e != cudaSuccess) return e;
    // never more CTAs than tiles if every row were as long as the table is (a window may begin inside sixteen tokens)
    const jl_kv8_attention_args &a = p.a;
    int64_t most = int64_t(a.blocks_per_slot) * a.pages.block_tokens;
    if (a.window > 0) most = std::min(most, int64_t(a.window) + 15);
    p.head_tiles = (p.group + S::kHeads - 1) / S::kHeads;
    const int64_t tiles = (most + S::kTile - 1) / S::kTile * a.pages.kv_heads * a.rows, resident = std::max(1, l.sm_count * S::kResident / p.head_tiles);
    p.arrivals = static_cast<unsigned *>(s.memory);
    p.parts = reinterpret_cast<float *>(static_cast<char *>(s.memory) + kKv8CounterBytes);
    return kv8_launch(attention_kernel<HD, NT, PAGED16>, unsigned(std::min(tiles, resident)) * p.head_tiles, S::kThreads, S::kBytes, l.stream, l.programmatic, p);
}

template <int HD>
cudaError_t launch_head(Params &p, const Kv8Scratch &s, const Kv8Launch &l) {
    // Blocks of multiples of 16 tokens: one lookup for sixteen rows instead of one for each. One row at 3901 11.5 / 12.0 us, 32 rows at 512
    // 13.6 / 15.5, 16 rows at 32000 192 / 227.
    const bool paged16 = p.a.pages.block_tokens % 16 == 0;
    // More than four query heads of a KV head: eight to a unit, or four, whose CTAs then read a token's keys and values twice (from L2 the
    // second time). Eight heads, four and eight to a unit (us): head size 128, 8 rows at 2000 of 8 KV heads 20.6 / 21.6, 1 row at 100000 of one
    // 21.8 / 25.5, at 16000 92 / 80; where units are many, 32 rows at 300 22.4 / 16.7, 24 rows at 800 27.8 / 25.4, 64 rows at 1500 82 / 92. Head size 64: 16
    // rows at 16000 of 4 KV heads 64 / 56. Head size 96: 24 rows at 300 11.2 / 14.0, 64 rows at 1000 48 / 64, 32 rows at 2000 43 / 49, but 32 rows at 300 18.1 / 14.4.
    if constexpr (HD == 64 || HD == 128)
        if (p.group > 4 && (HD == 64 || int64_t(p.a.rows) * p.a.pages.kv_heads >= l.sm_count)) return paged16 ? launch<HD, 2, true>(p, s, l) : launch<HD, 2, false>(p, s, l);
    return paged16 ? launch<HD, 1, true>(p, s, l) : launch<HD, 1, false>(p, s, l);
}

static_assert(3 * kMostCtas * 4 <= kKv8MapCounter);

template <int HD, int NT>
constexpr size_t kPartsPerSm = size_t(kSlots) * Shape<HD, NT>::kResident *Shape<HD, NT>::kPartFloats * sizeof(float);

}  // namespace

cudaError_t kv8_scratch_create(Kv8Scratch *s, int sm_count) {
    if (sm_count > kMostSms) return cudaErrorInvalidValue;  // more CTAs than there are counters, or than a join has room for
    // for the CTAs of the largest grid, of the largest kind
    const size_t parts = std::max({kPartsPerSm<64, 1>, kPartsPerSm<64, 2>, kPartsPerSm<96, 1>, kPartsPerSm<128, 1>, kPartsPerSm<128, 2>, kPartsPerSm<192, 1>,
                                   kPartsPerSm<256, 1>});
    cudaError_t e = cudaMalloc(&s->memory, kKv8CounterBytes + size_t(sm_count) * parts);
    if (e == cudaSuccess) e = cudaMemset(s->memory, 0, kKv8CounterBytes);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // the memset is over before a launch on any stream
    return e;
}

void kv8_scratch_free(Kv8Scratch *s) {
    if (s->memory) cudaFree(s->memory);
    s->memory = nullptr;
}

cudaError_t kv8_attention_launch(const jl_kv8_attention_args &a, const Kv8Scratch &s, const Kv8Launch &l) {
    Params p = {};
    p.a = a;
    kv8_division(a.pages.block_tokens, &p.divide, &p.shift);
    p.group = a.heads / a.pages.kv_heads;
    switch (a.pages.head_dim) {
        case 64: return launch_head<64>(p, s, l);
        case 96: return launch_head<96>(p, s, l);
        case 128: return launch_head<128>(p, s, l);
        case 192: return launch_head<192>(p, s, l);
        default: return launch_head<256>(p, s, l);
    }
}

}  // namespace jl
