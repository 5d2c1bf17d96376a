// Attention of single tokens over the 8-bit paged key/value cache.
//
// Work. A unit is one row and four or eight query heads of one KV head; its tokens are cut into tiles of 64. The tiles of all units
// form one line (rows in order, then heads, then tokens), of which every CTA of a grid that fits the GPU takes an equal piece. The
// lengths are on the device, so each CTA works the line out for itself from the rows' positions. A unit that lies within a piece is
// finished there; the parts of one that is cut are left in the workspace, and the CTA that arrives last at the unit's counter joins
// them in order, so results do not hang on who arrives when.
//
// Mathematics. s = scale * ks_j * (q . kc_j), weights p_j = 2^(s_j log2 e - m) with a running maximum m, and
// out = sum p_j vs_j vc_j / sum p_j. Codes are exact in binary16; a query is split into two binary16 parts of eleven bits each
// (scaled by the power of two that takes its largest element to [2^14, 2^15)), and so is p_j vs_j. The two parts of four heads are
// the eight columns of an mma.m16n8k16 whose sixteen rows are tokens (keys) or elements (values), so products are exact to 22 bits;
// the instructions' sums of sixteen tokens are added in binary32. w_j = 2^(s_j log2 e - E) vs_j has a running power of two E of its
// own that keeps it below 2^15: scales of values may differ by any factor between tokens. m and E are whole numbers, so that
// moving them on rounds nothing.
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kv8.cuh"

namespace jl {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 16;                // tokens that a warp takes at a time
constexpr int kTile = kStep * kWarps;    // tokens of a tile
constexpr uint32_t kMinTiles = 2;        // that a piece of a unit has at least
constexpr uint32_t kLongQuota = 16;      // tiles for each CTA from which on lines are cut without regard to units
constexpr int kRowsPerLane = 4;
constexpr int kMostResident = 4;         // CTAs per SM
constexpr int kMostSms = 160;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// ---- layout of a stage in shared memory: 16 rows of keys, 16 rows of values, their scales, the mask of tokens that count -----------
// Rows are read as 16-byte pieces across eight rows (keys) or every second row (values). With 64, 128 and 256 bytes a row, pieces are
// exchanged within a 128-byte line so that both reads are free of bank conflicts; rows of 96 and 192 bytes are 16 bytes apart instead.
template <int HD>
struct Layout {
    static constexpr int kPitch = HD == 96 || HD == 192 ? HD + 16 : HD;
    static constexpr int kValues = kStep * kPitch, kScales = 2 * kValues, kMask = kScales + 2 * kStep * 4;
    static constexpr int kStage = kMask + 16;
    static constexpr int kStages = HD <= 96 ? 4 : 3;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kQuads = HD / 32;               // groups of four elements that a lane has of a head's output
    static constexpr int kLoad = HD == 96 ? 1 : HD == 64 || HD == 192 ? 2 : 4;  // quads that one load of values brings
    static constexpr int kBytes = kWarps * kRing;
    static_assert(kStage >= 8 * HD * 4);                 // a stage also holds a warp's outputs of eight heads

    // where 16-byte piece c of row r is
    __device__ static int piece(int r, int c) {
        if constexpr (HD == 64) return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ ((r >> 1 & 3) << 1)) << 4);
        else if constexpr (HD == 128 || HD == 256) return r * HD + ((c ^ (r & 7)) << 4);
        else return r * kPitch + (c << 4);
    }
    // byte (= element) of a row that lane t's word w of keys starts at
    __device__ static int key_element(int t, int w) {
        if constexpr (HD == 64) return t * 16 + w * 4;
        else if constexpr (HD == 96) return (w >> 1) * 32 + t * 8 + (w & 1) * 4;
        else if constexpr (HD == 192) return (w >> 2) * 64 + t * 16 + (w & 3) * 4;
        else return (w >> 3) * 128 + t * 32 + (w & 7) * 4;
    }
    // byte of a row that lane g's word j of values starts at
    __device__ static int value_element(int g, int j) {
        if constexpr (HD == 64) return g * 8 + j * 4;
        else if constexpr (HD == 96) return j * 32 + g * 4;
        else if constexpr (HD == 192) return (j >> 1) * 64 + g * 8 + (j & 1) * 4;
        else return (j >> 2) * 128 + g * 16 + (j & 3) * 4;
    }
};

// CTAs per SM: registers are the limit (accumulators and queries of NT groups of heads)
template <int HD, int NT>
constexpr int kResident = HD <= 96 || (HD == 128 && NT == 1) ? 4 : HD == 128 ? 3 : 2;

struct Params {
    jl_kv8_attention_args a;
    uint64_t divide;   // j / block_tokens = j * divide >> shift for j < 2^31
    int shift;
    int group, head_tiles, units;  // query heads per KV head, units per KV head and per row
    unsigned *arrivals;            // [CTAs], zero between launches
    float *parts;                  // [2 * CTAs][part floats]
};
template <int HD, int NT>
constexpr int kPartFloats = 4 * NT * (HD + 3);

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two bytes (signed codes with their top bit flipped) as binary16: 0x64uu is 1024 + u, and u is code + 128.
template <int SELECT>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t flipped) {
    const uint32_t biased = __byte_perm(flipped, 0x64646464u, SELECT);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&x);
}
__device__ __forceinline__ uint32_t pack(__half lo, __half hi) {
    const __half2 x = __halves2half2(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&x);
}
// x and y as two binary16 parts each: `big` rounded to eleven bits, `rest` what that leaves.
__device__ __forceinline__ void split(float x, float y, uint32_t &big, uint32_t &rest) {
    const __half bx = __float2half_rn(x), by = __float2half_rn(y);
    big = pack(bx, by);
    rest = pack(__float2half_rn(x - __half2float(bx)), __float2half_rn(y - __half2float(by)));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(from - to) of whole numbers from <= to, exactly (from -inf: nothing is there, 0; below 2^-126: 0)
__device__ __forceinline__ float step_down(float from, float to) {
    const float magic = 12582912.f;  // 1.5 * 2^23: the sum's low bits are the whole number
    return from == to ? 1.f : __int_as_float((__float_as_int(fmaxf(from - to, -127.f) + magic) - __float_as_int(magic) + 127) << 23);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// The transpose of an 8 x 8 matrix of binary16 whose row g is held by lanes 4g .. 4g + 3, two columns each.
__device__ __forceinline__ uint32_t transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
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
__device__ __forceinline__ uint32_t tiles_of(const Row &row) { return max(1u, (row.end - (row.first & ~15u) + kTile - 1) / kTile); }

// Sum of v over the CTA's threads; `before`: over those in front of this one.
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

// NT: groups of four query heads. PAGED16: blocks are multiples of 16 tokens, so a step's sixteen rows lie behind one another.
template <int HD, int NT, bool PAGED16>
__global__ void __launch_bounds__(kThreads, (kResident<HD, NT>)) attention_kernel(const Params p) {
    using L = Layout<HD>;
    constexpr int kHeads = 4 * NT;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t warp_sums[kWarps], start_row, start_tile;
    __shared__ float s_m[kWarps][kHeads], s_e[kWarps][kHeads], s_l[kWarps][kHeads];
    __shared__ int s_last[2];
    const jl_kv8_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int rows = a.token_count ? min(a.token_count[0], a.rows) : a.rows;

    // ---- what this CTA takes. Short lines: a piece of one unit, every unit cut into equal pieces of `quota` tiles at most, as
    // many as there are CTAs. Long ones, and more rows than a warp holds: [at, end) of the line, cut without regard to units.
    uint32_t at = 0, end = 0, piece = 0, pieces = 0, in_row = 0, ctas = gridDim.x, quota = 0, more_than = 0, total = 0;
    int r = 0;
    if (rows <= 32 * kRowsPerLane) {
        uint32_t tiles[kRowsPerLane], mine = 0;
#pragma unroll
        for (int k = 0; k < kRowsPerLane; ++k) {
            const int i = lane * kRowsPerLane + k;
            tiles[k] = i < rows ? tiles_of(row_at(a, i)) : 0;
            mine += tiles[k];
        }
        total = __reduce_add_sync(~0u, mine) * p.units;
        if (uint32_t(rows) * p.units <= ctas && total < ctas * kLongQuota) {
            quota = max(kMinTiles, (total + ctas - 1) / ctas);
            uint32_t n[kRowsPerLane], sum;
            for (;;) {
                sum = 0;
#pragma unroll
                for (int k = 0; k < kRowsPerLane; ++k) sum += n[k] = (tiles[k] + quota - 1) / quota;
                if (__reduce_add_sync(~0u, sum) * p.units <= ctas) break;
                quota += max(1u, quota / 8);
            }
            uint32_t before = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t o = __shfl_up_sync(~0u, before, d);
                if (lane >= d) before += o;
            }
            if (blockIdx.x >= __shfl_sync(~0u, before, 31) * p.units) return;
            before = (before - sum) * p.units;
            uint32_t found = 0, found_in = 0, found_n = 0;
#pragma unroll
            for (int k = 0; k < kRowsPerLane; ++k) {
                if (blockIdx.x >= before && blockIdx.x < before + n[k] * p.units) {
                    found = lane * kRowsPerLane + k + 1;
                    found_in = blockIdx.x - before;
                    found_n = n[k];
                }
                before += n[k] * p.units;
            }
            const int from_lane = __ffs(__ballot_sync(~0u, found != 0)) - 1;
            r = __shfl_sync(~0u, found, from_lane) - 1;
            found_in = __shfl_sync(~0u, found_in, from_lane);
            pieces = __shfl_sync(~0u, found_n, from_lane);
            piece = found_in % pieces;
            in_row = found_in / pieces;  // the unit, until enter() knows the row's tiles
        }
    }
    if (pieces == 0) {
        if (rows > 32 * kRowsPerLane) {
            uint32_t mine = 0, before;
            for (int i = tid; i < rows; i += kThreads) mine += tiles_of(row_at(a, i));
            total = block_sum(mine, &before, warp_sums) * p.units;
        }
        if (total == 0) return;
        ctas = min(ctas, total);
        if (blockIdx.x >= ctas) return;
        quota = total / ctas;
        more_than = total % ctas;  // so many CTAs take one more
        at = blockIdx.x * quota + min(blockIdx.x, more_than);
        end = at + quota + (blockIdx.x < more_than);
        uint32_t front = 0;  // tiles in front of the rows from `base` on
        for (int base = 0; base < rows && front <= at; base += kThreads) {
            uint32_t before;
            const uint32_t mine = base + tid < rows ? tiles_of(row_at(a, base + tid)) * p.units : 0, all = block_sum(mine, &before, warp_sums);
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

    unsigned char *ring = smem + warp * L::kRing;
    const uint32_t ring_at = smem_u32(ring);
    const int bt = a.pages.block_tokens;

    // The segment under way: tiles [tile, tile + take) of a unit, tokens [from, to); `mine` steps of them are this warp's, step i at
    // token from + (warp + 4 i) 16.
    struct Segment {
        uint32_t first, from, to, tiles, tile, take;
        int kv, head0, mine;  // head0: within the group
        const int32_t *line;
    } seg;
    auto enter = [&]() {
        const Row row = row_at(a, r);
        seg.tiles = tiles_of(row);
        uint32_t unit = in_row;
        if (pieces) {
            seg.tile = seg.tiles * piece / pieces;
            seg.take = seg.tiles * (piece + 1) / pieces - seg.tile;
        } else {
            unit = in_row / seg.tiles;
            seg.tile = in_row % seg.tiles;
            seg.take = min(seg.tiles - seg.tile, end - at);
        }
        seg.kv = unit / p.head_tiles;
        seg.head0 = (unit % p.head_tiles) * kHeads;
        seg.first = row.first;
        seg.from = (row.first & ~15u) + seg.tile * kTile;
        seg.to = min(row.end, seg.from + seg.take * kTile);
        const int steps = seg.to > seg.from ? int((seg.to - seg.from + kStep - 1) / kStep) : 0;
        seg.mine = steps > warp ? (steps - warp + kWarps - 1) / kWarps : 0;
        seg.line = a.block_table + int64_t(row.slot) * a.blocks_per_slot;
    };
    auto step_at = [&](int i) { return seg.from + uint32_t(warp + i * kWarps) * kStep; };
    auto block_of = [&](uint32_t j) { return uint32_t((j * p.divide) >> p.shift); };

    // PAGED16: lane i looks up step 32 k + i of this warp, 32 steps ahead; where its codes and scales begin, or -1.
    // Otherwise lanes i and i + 16 look up token i of a step, one step ahead.
    int64_t code_at = -1, scale_at = -1;
    int ahead;
    auto look_up = [&](int i) {
        if constexpr (PAGED16) return i + lane < seg.mine ? seg.line[block_of(step_at(i + lane))] : -1;
        const uint32_t j = step_at(i) + (lane & 15);
        return i < seg.mine && j < seg.to ? seg.line[block_of(j)] : -1;
    };
    auto place = [&](int block, uint32_t j) {
        const bool good = block >= 0 && block < a.pages.blocks;
        const int64_t in_block = int64_t(seg.kv) * bt + (j - block_of(j) * bt);
        code_at = good ? block * a.pages.block_stride + in_block * HD : -1;
        scale_at = block * a.pages.scale_stride + in_block;
    };
    auto issue = [&](int i) {
        if (i < seg.mine) {
            const uint32_t stage = ring_at + uint32_t(i % L::kStages) * L::kStage, j0 = step_at(i);
            unsigned mask = (j0 < seg.first ? 0xffffu << (seg.first - j0) : 0xffffu) & (seg.to - j0 < 16 ? (1u << (seg.to - j0)) - 1 : 0xffffu);
            if constexpr (PAGED16) {
                if (i % 32 == 0) {
                    place(ahead, step_at(i + lane));
                    ahead = look_up(i + 32);
                }
                const int64_t code = __shfl_sync(~0u, code_at, i & 31), scale = __shfl_sync(~0u, scale_at, i & 31);
                if (code < 0) mask = 0;
                if (code >= 0) {
                    const int8_t *k = a.pages.k + code + lane * 16, *v = a.pages.v + code + lane * 16;
                    copy4(stage + L::kScales + 4 * lane, (lane < 16 ? a.pages.k_scale : a.pages.v_scale) + scale + (lane & 15));
#pragma unroll
                    for (int n = 0; n < HD / 32; ++n) {
                        const int piece = n * 32 + lane;
                        const uint32_t dst = stage + L::piece(piece / (HD / 16), piece % (HD / 16));
                        copy16(dst, k + n * 512);
                        copy16(dst + L::kValues, v + n * 512);
                    }
                }
            } else {
                place(ahead, j0 + (lane & 15));
                ahead = look_up(i + 1);
                mask &= __ballot_sync(~0u, code_at >= 0);
                if (code_at >= 0) copy4(stage + L::kScales + 4 * lane, (lane < 16 ? a.pages.k_scale : a.pages.v_scale) + scale_at);
#pragma unroll
                for (int n = 0; n < HD / 32; ++n) {
                    const int piece = n * 32 + lane, row16 = piece / (HD / 16), c = piece % (HD / 16);
                    const int64_t src = __shfl_sync(~0u, code_at, row16);
                    const uint32_t dst = stage + L::piece(row16, c);
                    if (src >= 0) {
                        copy16(dst, a.pages.k + src + c * 16);
                        copy16(dst + L::kValues, a.pages.v + src + c * 16);
                    }
                }
            }
            if (lane == 0) *reinterpret_cast<unsigned *>(ring + (i % L::kStages) * L::kStage + L::kMask) = mask;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto begin = [&]() {
        enter();
        ahead = look_up(0);
#pragma unroll
        for (int i = 0; i < L::kStages - 1; ++i) issue(i);
    };

    // Units of this CTA that others have a part of: two at most, its first and its last. Whether it was the last to arrive at one
    // is asked for at once, and looked at when nothing else is left to do.
    struct Shared {
        int r, kv, head0;
        uint32_t first, parts;
    } shared[2];
    int n_shared = 0;
    bool arrived_last[2] = {false, false};  // thread 0

    // quad f = n kQuads + j of lane (g, t): four elements of head 4 n + t
    auto finish = [&](int f, int row, int kv, int head0, float4 x, float top, float etop, float sum) {
        const int head = 4 * (f / L::kQuads) + t;
        if (head0 + head >= p.group) return;
        // 2^(etop - top) / sum, in two factors: either may be beyond binary32 where the output is not. etop is above top - 130 and
        // below top + 116, since a weight's exponent is between -113 and 128.
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
            a.lse[int64_t(row) * a.heads + kv * p.group + head0 + head] = sum == 0.f ? -CUDART_INF_F : (top + __log2f(sum)) * kLn2;
    };

    begin();
    for (;;) {
        const int mine = seg.mine, kv = seg.kv, head0 = seg.head0;

        // ---- queries: column g of group n is part g & 1 of head 4 n + g / 2. Rotated, scaled, split.
        uint32_t q[NT][HD / 16][2];
        float factor[NT];  // of head 4 n + t
        if (mine > 0) {
            const int pos = a.positions[r];
            const bool outside = a.rope_cos && pos >= a.rope_rows;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int head = head0 + 4 * n + (g >> 1);
                float x[HD / 16][4];
                uint32_t largest = outside ? 0x7f800000u : 0u;  // of the elements' magnitudes, as bits
                const int64_t q_at = int64_t(r) * a.q_stride + int64_t(kv * p.group + head) * HD;
#pragma unroll
                for (int w = 0; w < HD / 16; ++w) {
                    const int e = L::key_element(t, w);
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (head < p.group) {
                        if (a.ggml_type == JL_F16) {
                            const uint2 h = *reinterpret_cast<const uint2 *>(static_cast<const __half *>(a.q) + q_at + e);
                            const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&h.x)), hi = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
                            v = make_float4(lo.x, lo.y, hi.x, hi.y);
                        } else {
                            v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + q_at + e);
                        }
                    }
                    if (a.rope_cos && !outside) {
                        const int64_t angle = int64_t(pos) * (HD / 2) + e / 2;
                        const float2 c = *reinterpret_cast<const float2 *>(a.rope_cos + angle), s = *reinterpret_cast<const float2 *>(a.rope_sin + angle);
                        v = make_float4(v.x * c.x - v.y * s.x, v.x * s.x + v.y * c.x, v.z * c.y - v.w * s.y, v.z * s.y + v.w * c.y);
                    }
                    x[w][0] = v.x, x[w][1] = v.y, x[w][2] = v.z, x[w][3] = v.w;
#pragma unroll
                    for (int k = 0; k < 4; ++k) largest = max(largest, __float_as_uint(x[w][k]) & 0x7fffffffu);
                }
                largest = max(largest, __shfl_xor_sync(~0u, largest, 1));
                largest = max(largest, __shfl_xor_sync(~0u, largest, 2));
                const bool finite = largest < 0x7f800000u;
                // 2^(14 - exponent of the largest), at most 2^126
                const int shift = finite ? min(14 - (int(largest >> 23) - 127), 126) : 0;
                const float up = __uint_as_float(uint32_t(127 + shift) << 23);
#pragma unroll
                for (int w = 0; w < HD / 16; ++w)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t big, rest;
                        split(finite ? x[w][2 * k] * up : 0.f, finite ? x[w][2 * k + 1] * up : 0.f, big, rest);
                        q[n][w][k] = g & 1 ? rest : big;
                    }
                // head 4 n + t is that of lanes with g = 2 t
                factor[n] = __shfl_sync(~0u, finite ? a.scale * kLog2e * __uint_as_float(uint32_t(127 - shift) << 23) : CUDART_NAN_F, t * 8);
            }
        }

        // ---- one pass over this warp's tokens: lane (g, t) has tokens g and g + 8 of a step, heads 4 n + t, elements of column g
        float m[NT], e[NT], l[NT], o[NT][L::kQuads][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n] = e[n] = -CUDART_INF_F;
            l[n] = 0.f;
#pragma unroll
            for (int j = 0; j < L::kQuads; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
        }
        for (int i = 0; i < mine; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
            __syncwarp();
            issue(i + L::kStages - 1);
            const unsigned char *stage = ring + (i % L::kStages) * L::kStage;
            const uint32_t stage_at = ring_at + (i % L::kStages) * L::kStage;

            float s[NT][4] = {};
            {
                uint32_t kw[2][HD / 16];  // tokens g and g + 8
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int rk = g + 8 * half;
                    if constexpr (HD == 96) {
#pragma unroll
                        for (int w = 0; w < HD / 16; w += 2) {
                            const uint2 x = lds64(stage_at + rk * L::kPitch + L::key_element(t, w));
                            kw[half][w] = x.x, kw[half][w + 1] = x.y;
                        }
                    } else {
#pragma unroll
                        for (int w = 0; w < HD / 16; w += 4) {
                            const uint4 x = lds128(stage_at + L::piece(rk, L::key_element(t, w) >> 4));
                            kw[half][w] = x.x, kw[half][w + 1] = x.y, kw[half][w + 2] = x.z, kw[half][w + 3] = x.w;
                        }
                    }
                }
#pragma unroll
                for (int w = 0; w < HD / 16; ++w) {
                    const uint32_t u0 = kw[0][w] ^ 0x80808080u, u1 = kw[1][w] ^ 0x80808080u;
                    const uint32_t a0 = codes_to_half2<0x4140>(u0), a1 = codes_to_half2<0x4140>(u1), a2 = codes_to_half2<0x4342>(u0), a3 = codes_to_half2<0x4342>(u1);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma(s[n], a0, a1, a2, a3, q[n][w][0], q[n][w][1]);
                }
            }

            // scores in units of ln 2 and weights; maxima are moved on where a score or a weight is beyond them
            const unsigned mask = *reinterpret_cast<const unsigned *>(stage + L::kMask);
            const float *ks = reinterpret_cast<const float *>(stage + L::kScales), *vs = ks + kStep;
            const bool counts[2] = {bool(mask >> g & 1), bool(mask >> (g + 8) & 1)};
            const float key_scale[2] = {ks[g], ks[g + 8]}, v[2] = {counts[0] ? vs[g] : 0.f, counts[1] ? vs[g + 8] : 0.f};
            uint32_t b[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[2], w[2];
                bool beyond = false;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    x[k] = counts[k] ? (s[n][2 * k] + s[n][2 * k + 1]) * factor[n] * key_scale[k] : -CUDART_INF_F;
                    w[k] = exp2_approx(x[k] - e[n]) * v[k];
                    beyond = beyond || x[k] > m[n] || fabsf(w[k]) > 32768.f;
                }
                if (__any_sync(~0u, beyond)) {
                    float top = fmaxf(x[0], x[1]), etop = -CUDART_INF_F;
#pragma unroll
                    for (int k = 0; k < 2; ++k) etop = fmaxf(etop, x[k] + fmaxf(float(int(__float_as_uint(v[k]) >> 23 & 255) - 127), -113.f));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                        etop = fmaxf(etop, __shfl_xor_sync(~0u, etop, d));
                    }
                    const float m_new = fmaxf(m[n], ceilf(top)), e_new = fmaxf(e[n], ceilf(etop) - 14.f), keep = step_down(e[n], e_new);
                    l[n] *= step_down(m[n], m_new);
#pragma unroll
                    for (int j = 0; j < L::kQuads; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[n][j][k] *= keep;
                    m[n] = m_new;
                    e[n] = e_new;
#pragma unroll
                    for (int k = 0; k < 2; ++k) w[k] = exp2_approx(x[k] - e[n]) * v[k];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    // nothing has been seen yet (m = E = -inf, which -inf may not be taken from), or a token does not count
                    const bool none = x[k] == -CUDART_INF_F;
                    l[n] += none ? 0.f : exp2_approx(x[k] - m[n]);
                    const float y = none ? 0.f * v[k] : w[k];
                    const __half big = __float2half_rn(y);
                    b[n][k] = transpose(pack(big, __float2half_rn(y - __half2float(big))));
                }
            }

            // values: of word j of column g, elements 0 and 1 are rows g and g + 8 of one product, 2 and 3 of the next
#pragma unroll
            for (int j0 = 0; j0 < L::kQuads; j0 += L::kLoad) {
                uint32_t vw[4][L::kLoad];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int rv = 2 * t + (k & 1) + 8 * (k >> 1), el = L::value_element(g, j0);
                    const uint32_t addr = stage_at + L::kValues + L::piece(rv, el >> 4) + (el & 15);
                    if constexpr (L::kLoad == 4) {
                        const uint4 y = lds128(addr);
                        vw[k][0] = y.x, vw[k][1] = y.y, vw[k][2] = y.z, vw[k][3] = y.w;
                    } else if constexpr (L::kLoad == 2) {
                        const uint2 y = lds64(addr);
                        vw[k][0] = y.x, vw[k][1] = y.y;
                    } else {
                        vw[k][0] = lds32(addr);
                    }
                }
#pragma unroll
                for (int j = 0; j < L::kLoad; ++j) {
                    const uint32_t u0 = vw[0][j] ^ 0x80808080u, u1 = vw[1][j] ^ 0x80808080u, u2 = vw[2][j] ^ 0x80808080u, u3 = vw[3][j] ^ 0x80808080u;
                    const uint32_t near01 = __byte_perm(u0, u1, 0x5140), near23 = __byte_perm(u0, u1, 0x7362);
                    const uint32_t far01 = __byte_perm(u2, u3, 0x5140), far23 = __byte_perm(u2, u3, 0x7362);
                    const uint32_t x0 = codes_to_half2<0x4140>(near01), x1 = codes_to_half2<0x4342>(near01), x2 = codes_to_half2<0x4140>(far01), x3 = codes_to_half2<0x4342>(far01);
                    const uint32_t y0 = codes_to_half2<0x4140>(near23), y1 = codes_to_half2<0x4342>(near23), y2 = codes_to_half2<0x4140>(far23), y3 = codes_to_half2<0x4342>(far23);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float c[4] = {}, d[4] = {};
                        mma(c, x0, x1, x2, x3, b[n][0], b[n][1]);
                        mma(d, y0, y1, y2, y3, b[n][0], b[n][1]);
                        float(&out)[4] = o[n][j0 + j];
                        out[0] += c[0] + c[1], out[1] += c[2] + c[3], out[2] += d[0] + d[1], out[3] += d[2] + d[3];
                    }
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();

        // ---- the next segment's first stages are on their way while this one's warps are folded, in the stage that they leave free.
        // Outputs lie there as [group][quad][lane], four elements of head t each.
        const int row = r;
        // the CTAs that have a part of this unit
        const uint32_t first_cta = pieces ? blockIdx.x - piece : owner(at - seg.tile), last_cta = pieces ? first_cta + pieces - 1 : owner(at - seg.tile + seg.tiles - 1);
        at += seg.take;
        in_row += seg.take;
        if (in_row == seg.tiles * uint32_t(p.units)) ++r, in_row = 0;
        const bool more = !pieces && at < end;
        if (more) begin();
        float4 *out_w = reinterpret_cast<float4 *>(ring + (L::kStages - 1) * L::kStage);
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
        float *part = p.parts + (size_t(blockIdx.x) * 2 + (blockIdx.x == first_cta)) * kPartFloats<HD, NT>;
        for (int f = warp; f < NT * L::kQuads; f += kWarps) {
            const int head = 4 * (f / L::kQuads) + t;
            float top = -CUDART_INF_F, etop = -CUDART_INF_F, sum = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][head]), etop = fmaxf(etop, s_e[w][head]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float keep = step_down(s_e[w][head], etop);
                const float4 y = reinterpret_cast<const float4 *>(smem + w * L::kRing + (L::kStages - 1) * L::kStage)[f * 32 + lane];
                sum += s_l[w][head] * step_down(s_m[w][head], top);
                x.x += y.x * keep, x.y += y.y * keep, x.z += y.z * keep, x.w += y.w * keep;
            }
            if (whole) {
                finish(f, row, kv, head0, x, top, etop, sum);
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
            const unsigned others = last_cta - first_cta;
            if (tid == 0) {
                __threadfence();
                const bool is_last = atomicInc(p.arrivals + first_cta, others) == others;  // the last one to come sets it back to zero
                if (n_shared == 0) arrived_last[0] = is_last;
                else arrived_last[1] = is_last;
            }
            const Shared unit = {row, kv, head0, first_cta, others + 1};
            if (n_shared == 0) shared[0] = unit;
            else shared[1] = unit;
            ++n_shared;
        }
        if (!more) break;
    }

    // ---- join the units that this CTA came last to
    if (n_shared == 0) return;
    if (tid == 0) {
        s_last[0] = arrived_last[0];
        s_last[1] = arrived_last[1];
        __threadfence();
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (u >= n_shared || !s_last[u]) continue;
        const Shared &unit = shared[u];
        const int n = int(unit.parts);
        auto part_of = [&](int k) { return p.parts + (size_t(unit.first + k) * 2 + (k == 0)) * kPartFloats<HD, NT>; };
        // maxima and sums: thread i has head i mod heads of every (threads / heads)-th part
        const int my_head = tid % kHeads;
        float top = -CUDART_INF_F, etop = -CUDART_INF_F, sum = 0.f;
#pragma unroll 4
        for (int k = tid / kHeads; k < n; k += kThreads / kHeads) {
            const float *stats = part_of(k) + kHeads * HD + my_head;
            top = fmaxf(top, __ldcg(stats));
            etop = fmaxf(etop, __ldcg(stats + kHeads));
        }
#pragma unroll
        for (int d = kHeads; d < 32; d <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            etop = fmaxf(etop, __shfl_xor_sync(~0u, etop, d));
        }
        __syncthreads();  // what was kept here before has been read
        if (lane < kHeads) s_m[warp][lane] = top, s_e[warp][lane] = etop;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][my_head]), etop = fmaxf(etop, s_e[w][my_head]);
        float *keep = reinterpret_cast<float *>(smem);  // [part][head]
#pragma unroll 4
        for (int k = tid / kHeads; k < n; k += kThreads / kHeads) {
            const float *stats = part_of(k) + kHeads * HD + my_head;
            sum += __ldcg(stats + 2 * kHeads) * step_down(__ldcg(stats), top);
            keep[k * kHeads + my_head] = step_down(__ldcg(stats + kHeads), etop);
        }
#pragma unroll
        for (int d = kHeads; d < 32; d <<= 1) sum += __shfl_xor_sync(~0u, sum, d);
        if (lane < kHeads) s_l[warp][lane] = sum;
        __syncthreads();
        // outputs: a warp has every fourth part
        constexpr int kUnroll = NT * L::kQuads <= 4 ? 4 : NT * L::kQuads <= 8 ? 2 : 1;
        float4 x[NT * L::kQuads];
#pragma unroll
        for (int f = 0; f < NT * L::kQuads; ++f) x[f] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll kUnroll
        for (int k = warp; k < n; k += kWarps) {
            const float4 *src = reinterpret_cast<const float4 *>(part_of(k)) + lane;
#pragma unroll
            for (int f = 0; f < NT * L::kQuads; ++f) {
                const float4 y = __ldcg(src + f * 32);
                const float w = keep[k * kHeads + 4 * (f / L::kQuads) + t];
                x[f].x += y.x * w, x[f].y += y.y * w, x[f].z += y.z * w, x[f].w += y.w * w;
            }
        }
        float4 *warp_out = reinterpret_cast<float4 *>(smem + kMostResident * kMostSms * kHeads * 4);  // behind `keep`
        static_assert(kMostResident * kMostSms * kHeads * 4 + kWarps * NT * HD * 16 <= L::kBytes);
#pragma unroll
        for (int f = 0; f < NT * L::kQuads; ++f) warp_out[(warp * NT * L::kQuads + f) * 32 + lane] = x[f];
        __syncthreads();
        for (int f = warp; f < NT * L::kQuads; f += kWarps) {
            const int head = 4 * (f / L::kQuads) + t;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            float all = 0.f, head_top = -CUDART_INF_F, head_etop = -CUDART_INF_F;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 z = warp_out[(w * NT * L::kQuads + f) * 32 + lane];
                y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
                all += s_l[w][head];
                head_top = fmaxf(head_top, s_m[w][head]), head_etop = fmaxf(head_etop, s_e[w][head]);
            }
            finish(f, unit.r, unit.kv, unit.head0, y, head_top, head_etop, all);
        }
        __syncthreads();
    }
}

template <int HD, int NT, bool PAGED16>
cudaError_t launch(Params &p, const Kv8Scratch &s, int sm_count, cudaStream_t stream) {
    using L = Layout<HD>;
    static std::atomic<uint64_t> configured{0};  // a bit for each device
    const cudaError_t e = kv8_allow_shared(reinterpret_cast<const void *>(attention_kernel<HD, NT, PAGED16>), L::kBytes, configured);
    if (e != cudaSuccess) return e;
    // never more CTAs than tiles if every row were as long as the table is (a window may begin inside sixteen tokens)
    const jl_kv8_attention_args &a = p.a;
    int64_t most = int64_t(a.blocks_per_slot) * a.pages.block_tokens;
    if (a.window > 0) most = most < int64_t(a.window) + 15 ? most : int64_t(a.window) + 15;
    p.head_tiles = (p.group + 4 * NT - 1) / (4 * NT);
    p.units = p.head_tiles * a.pages.kv_heads;
    const int64_t tiles = (most + kTile - 1) / kTile * p.units * a.rows;
    const int grid = int(tiles < int64_t(sm_count) * kResident<HD, NT> ? tiles : int64_t(sm_count) * kResident<HD, NT>);
    p.arrivals = static_cast<unsigned *>(s.memory);
    p.parts = reinterpret_cast<float *>(static_cast<char *>(s.memory) + kKv8CounterBytes);
    attention_kernel<HD, NT, PAGED16><<<grid, kThreads, L::kBytes, stream>>>(p);
    return cudaGetLastError();
}

template <int HD>
cudaError_t launch_variant(Params &p, const Kv8Scratch &s, int sm_count, cudaStream_t stream) {
    const bool paged16 = p.a.pages.block_tokens % 16 == 0;
    if (p.group <= 4) return paged16 ? launch<HD, 1, true>(p, s, sm_count, stream) : launch<HD, 1, false>(p, s, sm_count, stream);
    return paged16 ? launch<HD, 2, true>(p, s, sm_count, stream) : launch<HD, 2, false>(p, s, sm_count, stream);
}

static_assert(kMostSms * kMostResident * 4 <= kKv8MapCounter);
}  // namespace

cudaError_t kv8_scratch_create(Kv8Scratch *s, int sm_count) {
    // two parts for each CTA of the largest grid, of the largest kind
    const int part = std::max({kResident<64, 2> * kPartFloats<64, 2>, kResident<96, 2> * kPartFloats<96, 2>, kResident<128, 1> * kPartFloats<128, 1>,
                               kResident<128, 2> * kPartFloats<128, 2>, kResident<192, 2> * kPartFloats<192, 2>, kResident<256, 2> * kPartFloats<256, 2>});
    if (sm_count > kMostSms) return cudaErrorInvalidValue;  // more CTAs than there are counters, or than a join has room for
    cudaError_t e = cudaMalloc(&s->memory, kKv8CounterBytes + size_t(sm_count) * 2 * part * sizeof(float));
    if (e == cudaSuccess) e = cudaMemset(s->memory, 0, kKv8CounterBytes);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // the memset is over before a launch on any stream
    return e;
}

void kv8_scratch_free(Kv8Scratch *s) {
    if (s->memory) cudaFree(s->memory);
    s->memory = nullptr;
}

cudaError_t kv8_attention_launch(const jl_kv8_attention_args &a, const Kv8Scratch &s, int sm_count, cudaStream_t stream) {
    Params p = {};
    p.a = a;
    kv8_division(a.pages.block_tokens, &p.divide, &p.shift);
    p.group = a.heads / a.pages.kv_heads;
    switch (a.pages.head_dim) {
        case 64: return launch_variant<64>(p, s, sm_count, stream);
        case 96: return launch_variant<96>(p, s, sm_count, stream);
        case 128: return launch_variant<128>(p, s, sm_count, stream);
        case 192: return launch_variant<192>(p, s, sm_count, stream);
        default: return launch_variant<256>(p, s, sm_count, stream);
    }
}

}  // namespace jl
