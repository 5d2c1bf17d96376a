// Block tables, slot maps and the append of the 8-bit paged key/value cache.
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kv8.cuh"

namespace jl {
namespace {

// ---- block tables and slot maps -----------------------------------------------------------------
//
// With t_r = max(added_r, 0) and its running sum, need_r = ceil((held_r + added_r) / B) - ceil(held_r / B) blocks and their running
// sum, everything a token or a new block needs is known: token i belongs to the last sequence whose sum begins at or below i, block
// number b to the last sequence whose blocks begin at or below b. Every CTA works both sums out for itself (at most 8192
// sequences, 64 KB from L2) and keeps them in shared memory; then tokens and blocks are dealt out evenly, whatever the
// sequences' lengths. So there is one launch and nothing to wait for between CTAs. What may be an input and an output at once
// (lengths, cursor) is written by the CTA that is through last.
// Bound by the chain of loads, sums and searches, not by bytes: 8 sequences 3.3 us, 201 sequences with 3 800 tokens 4.2 us, 4096 sequences
// with 10^6 tokens (16.3 MB) 14.1 us. One token for each thread, and four in a row with wide stores: 3.3 / 4.6, 4.2 / 6.7, 15.0 / 14.1 us.

constexpr int kMapThreads = 512;
constexpr int kMapWarps = kMapThreads / 32;

struct MapParams {
    jl_kv8_map_args a;
    uint64_t divide;  // j / block_tokens = j * divide >> shift for j < 2^31
    int shift;
    bool in_place;
    bool wide;        // the token arrays are 16-byte aligned
    unsigned *arrivals;
};

__device__ __forceinline__ uint32_t add_saturated(uint32_t a, uint32_t b) { return a + b < a ? ~0u : a + b; }

// Saturated sums of v over the threads in front of this one; that of all threads in *all.
__device__ uint32_t exclusive_sum(uint32_t v, uint32_t *warp_sums, uint32_t *all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(~0u, s, d);
        if (lane >= d) s = add_saturated(s, o);
    }
    const uint32_t in_front = __shfl_up_sync(~0u, s, 1);
    __syncthreads();
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    uint32_t w = lane < kMapWarps ? warp_sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < kMapWarps; d <<= 1) {
        const uint32_t o = __shfl_up_sync(~0u, w, d);
        if (lane >= d) w = add_saturated(w, o);
    }
    const uint32_t before = __shfl_sync(~0u, w, max(warp - 1, 0));
    *all = __shfl_sync(~0u, w, kMapWarps - 1);
    return add_saturated(warp ? before : 0, lane ? in_front : 0);
}

// The last r in [low, high] with starts[r] <= x; starts ascend and starts[low] <= x.
__device__ __forceinline__ int last_at_most(const uint32_t *starts, int low, int high, uint32_t x) {
    while (low < high) {
        const int middle = (low + high + 1) >> 1;
        if (starts[middle] <= x) low = middle;
        else high = middle - 1;
    }
    return low;
}

// EACH: tokens in a row that a thread has. One where there are few, four (a wide store for each array) where there are many.
template <int EACH>
__global__ void __launch_bounds__(kMapThreads) map_kernel(const MapParams p) {
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t warp_sums[32], s_taken, s_refused;
    __shared__ bool s_last;
    const jl_kv8_map_args &a = p.a;
    const int n = a.sequences, tid = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    uint32_t *token_start = smem, *block_start = smem + n;
    int32_t *kept = reinterpret_cast<int32_t *>(smem + 2 * n);  // held; below 0: the sequence is refused
    auto block_of = [&](uint32_t position) { return uint32_t((uint64_t(position) * p.divide) >> p.shift); };
    auto blocks_for = [&](uint32_t tokens) { return tokens ? block_of(tokens - 1) + 1 : 0; };

    if (tid == 0) s_taken = s_refused = 0;
    const int cursor = a.cursor[0];
    const uint32_t free_blocks = cursor < 0 || cursor > a.free_count ? 0 : a.free_count - cursor;
    const int64_t room = min(int64_t(a.blocks_per_slot) * a.block_tokens, int64_t(INT32_MAX));
    // each thread has sequences [from, to), an odd number of them, so that a warp's threads meet in no bank
    const int each = (n + kMapThreads - 1) / kMapThreads | 1, from = min(n, tid * each), to = min(n, from + each);
    for (int r = tid; r < n; r += kMapThreads) block_start[r] = a.added[r], kept[r] = a.held[r];
    __syncthreads();
    uint32_t sum = 0, tokens, asked;
    for (int r = from; r < to; ++r) sum = add_saturated(sum, uint32_t(max(int32_t(block_start[r]), 0)));
    uint32_t at = exclusive_sum(sum, warp_sums, &tokens);
    sum = 0;
    for (int r = from; r < to; ++r) {
        const int held = kept[r], added = int32_t(block_start[r]);
        token_start[r] = at;
        at = add_saturated(at, uint32_t(max(added, 0)));
        const bool bad = held < 0 || added < 0 || int64_t(held) + added > room || at > uint32_t(a.capacity);
        const uint32_t need = bad ? 0 : blocks_for(held + added) - blocks_for(held);
        kept[r] = bad ? -1 : held;
        block_start[r] = need;
        sum = add_saturated(sum, need);
    }
    at = exclusive_sum(sum, warp_sums, &asked);
    uint32_t taken = 0, refused = 0;
    for (int r = from; r < to; ++r) {
        const uint32_t need = block_start[r], block_end = add_saturated(at, need);
        block_start[r] = at;
        at = block_end;
        if (kept[r] >= 0 && need != 0) {
            if (block_end <= free_blocks) taken = block_end;
            else kept[r] = -1;
        }
        refused += kept[r] < 0;
    }
    taken = __reduce_max_sync(~0u, taken);
    refused = __reduce_add_sync(~0u, refused);
    if ((tid & 31) == 0 && taken) atomicMax(&s_taken, taken);
    if ((tid & 31) == 0 && refused) atomicAdd(&s_refused, refused);
    __syncthreads();
    taken = s_taken;

    // ---- new blocks: numbers 0 .. taken - 1, all of sequences that are served
    const int step = gridDim.x * kMapThreads;
    for (uint32_t b = blockIdx.x * kMapThreads + tid; b < taken; b += step) {
        const int r = last_at_most(block_start, 0, n - 1, b);
        a.block_table[int64_t(r) * a.blocks_per_slot + blocks_for(kept[r]) + (b - block_start[r])] = a.free_blocks[cursor + b];
    }
    // ---- new tokens
    const uint32_t written = min(tokens, uint32_t(a.capacity));
    int low = 0;
    for (uint32_t i0 = EACH * (blockIdx.x * kMapThreads + tid); i0 < written; i0 += EACH * step) {
        int r = low = last_at_most(token_start, low, n - 1, i0);
        int slot[EACH], position[EACH];
        int64_t place[EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const uint32_t i = i0 + k;
            if (k && i < written && r < n - 1 && token_start[r + 1] <= i) r = last_at_most(token_start, r + 1, n - 1, i);
            slot[k] = r;
            position[k] = -1;
            place[k] = -1;
            if (i < written && kept[r] >= 0) {
                position[k] = int32_t(uint32_t(kept[r]) + (i - token_start[r]));
                const uint32_t index = block_of(position[k]), have = blocks_for(kept[r]);
                // an entry below `have` is one that was there and that nobody writes
                const int block = index < have ? a.block_table[int64_t(r) * a.blocks_per_slot + index] : a.free_blocks[cursor + block_start[r] + (index - have)];
                if (block >= 0) place[k] = int64_t(block) * a.block_tokens + (uint32_t(position[k]) - index * a.block_tokens);
            }
        }
        if (EACH == 4 && p.wide && i0 + 4 <= written) {
            reinterpret_cast<longlong2 *>(a.slot_map + i0)[0] = make_longlong2(place[0], place[EACH / 4]);
            reinterpret_cast<longlong2 *>(a.slot_map + i0)[1] = make_longlong2(place[EACH / 2], place[EACH - 1]);
            if (a.positions) *reinterpret_cast<int4 *>(a.positions + i0) = make_int4(position[0], position[EACH / 4], position[EACH / 2], position[EACH - 1]);
            if (a.token_slots) *reinterpret_cast<int4 *>(a.token_slots + i0) = make_int4(slot[0], slot[EACH / 4], slot[EACH / 2], slot[EACH - 1]);
        } else {
#pragma unroll
            for (int k = 0; k < EACH; ++k)
                if (i0 + k < written) {
                    a.slot_map[i0 + k] = place[k];
                    if (a.positions) a.positions[i0 + k] = position[k];
                    if (a.token_slots) a.token_slots[i0 + k] = slot[k];
                }
        }
    }
    // ---- what goes by sequences
    if (a.offsets)
        for (int r = blockIdx.x * kMapThreads + tid; r <= n; r += step) a.offsets[r] = int32_t(min(r < n ? token_start[r] : tokens, 0x7fffffffu));
    auto length = [&](int r) { return kept[r] < 0 ? a.held[r] : kept[r] + a.added[r]; };
    if (!p.in_place)
        for (int r = blockIdx.x * kMapThreads + tid; r < n; r += step) a.lengths[r] = length(r);
    bool last = blockIdx.x == 0;
    if (p.in_place && gridDim.x > 1) {
        __syncthreads();  // this CTA has read all it reads of held and cursor
        if (tid == 0) {
            __threadfence();
            s_last = atomicInc(p.arrivals, gridDim.x - 1) == gridDim.x - 1;
            __threadfence();
        }
        __syncthreads();
        last = s_last;
    } else if (p.in_place) {
        __syncthreads();
    }
    if (!last) return;
    if (p.in_place)
        for (int r = tid; r < n; r += kMapThreads) a.lengths[r] = length(r);
    if (tid == 0) {
        a.cursor_out[0] = cursor + int32_t(taken);
        a.result[0] = int32_t(written);
        a.result[1] = int32_t(taken);
        a.result[2] = int32_t(s_refused);
        a.result[3] = int32_t(min(asked, 0x7fffffffu));
    }
}

template <int EACH>
cudaError_t map_launch(const MapParams &p, int64_t most, int ctas, const Kv8Launch &l) {
    const size_t bytes = size_t(p.a.sequences) * 12;
    if (bytes > 40 * 1024) {  // 48 KB with what the kernel has besides
        static std::atomic<uint64_t> configured{0};  // a bit for each device
        const cudaError_t e = kv8_allow_shared(reinterpret_cast<const void *>(map_kernel<EACH>), 8192 * 12, configured);
        if (e != cudaSuccess) return e;
    }
    const int64_t grid = (most + EACH * kMapThreads - 1) / (EACH * kMapThreads);
    return kv8_launch(map_kernel<EACH>, unsigned(std::max(int64_t(1), std::min(int64_t(ctas), grid))), kMapThreads, bytes, l.stream, l.programmatic, p);
}

// ---- append -------------------------------------------------------------------------------------
//
// A row (a token's keys or values of one head) is held by D / 8 lanes, eight elements each, so a warp has one to four rows and reads
// them in 16-byte pieces; the lanes take the keys and the values of their token and head, whose places are the same. Codes are
// those of the unrounded values, so that they are a function of the row alone: 127 x / max |x| in binary32 is off by less than 1.6e-5
// (the quotient 2 of 127 * 2^-24), rotated by less than 5.3e-5 (the rotation 2.5, the maximum as much), and a row that has an
// element nearer than 2^-16 (rotated 2^-14) to the border of two codes is done again in 64 bits; so are rows whose largest element is
// infinite, NaN, above 2^125 or close to 2^-100. That is a row in 250, rotated one in 60.
// Bound by what it reads, and by its instructions (23 for an element, issued in 0.66 of the cycles): 8191 tokens of 8 heads of 128 in
// binary32, 84.5 MB, take 18.3 us = 4.6 TB/s, 0.72 of the measured copy rate; a row for each side by lanes of its own took 28.6 us. A
// single token takes 2.2 us.

// Nine CTAs of 128 threads per SM, 56 registers each: those 8191 tokens took 18.8 us with 62 to 64 registers (eight CTAs), 18.5 with 48 and
// spills outside the second look, 19.5 as four CTAs of 256 threads.
constexpr int kAppendThreads = 128;

template <typename T>
struct Eight;
template <>
struct Eight<float> {
    float4 lo, hi;
    __device__ void load(const float *p) {
        lo = __ldcs(reinterpret_cast<const float4 *>(p));
        hi = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    }
    __device__ void get(float (&x)[8]) const { x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w; }
};
template <>
struct Eight<__half> {
    uint4 v;
    __device__ void load(const __half *p) { v = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
};

struct AppendParams {
    jl_kv8_append_args a;
    uint64_t divide, divide_rows;  // j / block_tokens = j * divide >> shift for j < 2^31; the same for the heads of a token
    int shift, shift_rows;
};

template <int HD, typename T>
__global__ void __launch_bounds__(kAppendThreads, 9) append_kernel(const AppendParams p) {
    constexpr int kLanes = HD <= 64 ? 8 : HD <= 128 ? 16 : 32;  // HD / 8 of them have elements
    const jl_kv8_append_args &a = p.a;
    const int sub = threadIdx.x % kLanes;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t heads = a.pages.kv_heads, row = blockIdx.x * uint32_t(kAppendThreads / kLanes) + threadIdx.x / kLanes;  // rows: token, head
    const uint32_t t = uint32_t((uint64_t(row) * p.divide_rows) >> p.shift_rows), head = row - t * heads;
    const int count = a.token_count ? min(a.token_count[0], a.tokens) : a.tokens;
    const bool here = int64_t(t) < count, mine = here && sub < HD / 8;
    Eight<T> raw[2] = {};  // keys, values
    if (mine) {
        raw[0].load(static_cast<const T *>(a.k) + t * a.k_stride + (head * HD + sub * 8));
        raw[1].load(static_cast<const T *>(a.v) + t * a.v_stride + (head * HD + sub * 8));
    }
    const int64_t place = here ? a.slot_map[t] : -1;
    const bool turn = a.rope_cos != nullptr;
    const int pos = turn && here ? a.positions[t] : 0;
    const bool outside = turn && (pos < 0 || pos >= a.rope_rows);
    float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (turn && !outside && mine) {
        c = *reinterpret_cast<const float4 *>(a.rope_cos + int64_t(pos) * (HD / 2) + sub * 4);
        s = *reinterpret_cast<const float4 *>(a.rope_sin + int64_t(pos) * (HD / 2) + sub * 4);
    }
    // a place may be beyond 31 bits
    const int64_t block = place < 0x7fffffff ? int64_t((uint64_t(place) * p.divide) >> p.shift) : place / a.pages.block_tokens;
    const int64_t at = int64_t(head) * a.pages.block_tokens + (place - block * a.pages.block_tokens);
    const int64_t code_at = block * a.pages.block_stride + at * HD + sub * 8, scale_at = block * a.pages.scale_stride + at;
    const bool stored = mine && place >= 0 && place < int64_t(a.pages.blocks) * a.pages.block_tokens;

    // side 0: keys, 1: values
    auto store = [&](const int side) {
        const bool turned = side == 0 && turn, lost = side == 0 && outside;
        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
        float in[8], x[8];
        raw[side].get(in);
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = turned ? in[2 * i] * cs[i] - in[2 * i + 1] * sn[i] : in[2 * i];
            x[2 * i + 1] = turned ? in[2 * i] * sn[i] + in[2 * i + 1] * cs[i] : in[2 * i + 1];
            bits = max(bits, max(__float_as_uint(x[2 * i]) & 0x7fffffffu, __float_as_uint(x[2 * i + 1]) & 0x7fffffffu));
        }
#pragma unroll
        for (int d = kLanes / 2; d; d >>= 1) bits = max(bits, __shfl_xor_sync(~0u, bits, d));
        const float most = __uint_as_float(bits), up = 127.f * __frcp_rn(most), magic = 12582912.f;  // 1.5 * 2^23: a sum's low byte is the code
        float border = 0.f;
        uint32_t code[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = fmaf(x[i], up, magic);
            border = fmaxf(border, fabsf(fmaf(x[i], up, magic - y)));
            code[i] = __float_as_uint(y);
        }
        const bool again = lost || !(most >= 0x1p-99f && most < 0x1p125f) || border > 0.5f - (turned ? 0x1p-14f : 0x1p-16f);
        // most / 127 with one rounding: the quotient by the rounded reciprocal, and its remainder, which is exact (Markstein 1990). The largest element
        // of a rotated row is off by 2.5 of 2^-24 itself; that of the exact rotation took 23.1 us in place of 19.8 for 8191 rotated tokens.
        float scale = most * (1.f / 127.f);
        scale = fmaf(fmaf(-127.f, scale, most), 1.f / 127.f, scale);
        // whether any lane of the row says so
        const unsigned says = __ballot_sync(~0u, again && here);
        if (says) {
            const unsigned row_lanes = kLanes == 32 ? ~0u : ((1u << (kLanes & 31)) - 1) << (threadIdx.x & 31 & ~(kLanes - 1));
            double exact[8], largest = 0;
            bool good = !lost;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double u = in[2 * i], w = in[2 * i + 1];
                exact[2 * i] = turned ? u * double(cs[i]) - w * double(sn[i]) : u;
                exact[2 * i + 1] = turned ? u * double(sn[i]) + w * double(cs[i]) : w;
                good = good && isfinite(exact[2 * i]) && isfinite(exact[2 * i + 1]);
                largest = fmax(largest, fmax(fabs(exact[2 * i]), fabs(exact[2 * i + 1])));
            }
            good = (__ballot_sync(~0u, good) & row_lanes) == row_lanes;
#pragma unroll
            for (int d = kLanes / 2; d; d >>= 1) largest = fmax(largest, __shfl_xor_sync(~0u, largest, d));
            if (says & row_lanes) {
                const bool some = good && largest >= 0x1p-100;
#pragma unroll
                for (int i = 0; i < 8; ++i) code[i] = some ? uint32_t(int(rint(exact[i] * 127.0 / largest))) : 0;
                scale = good ? (some ? float(largest / 127.0) : 0.f) : CUDART_NAN_F;
            }
        }
        if (!stored) return;
        uint2 packed;
        packed.x = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
        packed.y = __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2 *>((side ? a.pages.v : a.pages.k) + code_at) = packed;
        if (sub == 0) (side ? a.pages.v_scale : a.pages.k_scale)[scale_at] = scale;
    };
    store(0);
    store(1);
}

template <int HD>
cudaError_t append_launch(const AppendParams &p, const Kv8Launch &l) {
    constexpr int kLanes = HD <= 64 ? 8 : HD <= 128 ? 16 : 32;
    const int64_t rows = int64_t(p.a.tokens) * p.a.pages.kv_heads;
    const unsigned grid = unsigned((rows * kLanes + kAppendThreads - 1) / kAppendThreads);
    return kv8_launch(p.a.ggml_type == JL_F16 ? append_kernel<HD, __half> : append_kernel<HD, float>, grid, kAppendThreads, 0, l.stream, l.programmatic, p);
}

}  // namespace

void kv8_division(int divisor, uint64_t *divide, int *shift) {
    int bits = 0;
    while ((int64_t(1) << bits) < divisor) ++bits;
    // floor(2^(31 + bits) / n) + 1 gives exact quotients of 31-bit numbers by n <= 2^bits (Granlund and Montgomery 1994)
    *shift = 31 + bits;
    *divide = (uint64_t(1) << *shift) / uint64_t(divisor) + 1;
}

cudaError_t kv8_map_launch(const jl_kv8_map_args &a, const Kv8Scratch &s, const Kv8Launch &l) {
    MapParams p = {};
    p.a = a;
    kv8_division(a.block_tokens, &p.divide, &p.shift);
    auto aligned = [](const void *x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
    p.wide = aligned(a.slot_map) && aligned(a.positions) && aligned(a.token_slots);
    p.in_place = a.lengths == a.held || a.cursor_out == a.cursor;
    p.arrivals = reinterpret_cast<unsigned *>(static_cast<char *>(s.memory) + kKv8MapCounter);
    const int64_t most = std::max(a.capacity, a.sequences);
    return most <= int64_t(l.sm_count) * kMapThreads ? map_launch<1>(p, most, l.sm_count, l) : map_launch<4>(p, most, 2 * l.sm_count, l);
}

cudaError_t kv8_append_launch(const jl_kv8_append_args &a, const Kv8Launch &l) {
    AppendParams p = {};
    p.a = a;
    kv8_division(a.pages.block_tokens, &p.divide, &p.shift);
    kv8_division(a.pages.kv_heads, &p.divide_rows, &p.shift_rows);
    switch (a.pages.head_dim) {
        case 64: return append_launch<64>(p, l);
        case 96: return append_launch<96>(p, l);
        case 128: return append_launch<128>(p, l);
        case 192: return append_launch<192>(p, l);
        default: return append_launch<256>(p, l);
    }
}

cudaError_t kv8_allow_shared(const void *kernel, int bytes, std::atomic<uint64_t> &configured) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device <= 63 && (configured.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device <= 63) configured.fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace jl
