// Block tables, slot maps and the append of the 8-bit paged key/value cache.
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"
#include "kv8.cuh"

namespace jl {
namespace {

constexpr int kMapThreads = 1024;

// Sum over the block's threads up to and including this one; the whole sum goes to every thread.
__device__ long long block_inclusive(long long v, long long *warp_sums, long long *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < int(blockDim.x) / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    *total = all;
    return before + v;
}

// One CTA walks the sequences, a thread each, and writes a sequence's blocks and tokens one after the other.
__global__ void __launch_bounds__(kMapThreads) map_kernel(jl_kv8_map_args a) {
    __shared__ long long warp_sums[kMapThreads / 32];
    const int tid = threadIdx.x;
    const int cursor = a.cursor[0];
    const long long free_blocks = cursor < 0 || cursor > a.free_count ? 0 : a.free_count - cursor;
    const long long room = (long long)a.blocks_per_slot * a.block_tokens;
    long long tokens = 0, asked = 0, taken = 0, refused = 0;
    for (int base = 0; base < a.sequences; base += kMapThreads) {
        const int r = base + tid;
        const bool here = r < a.sequences;
        const long long held = here ? a.held[r] : 0, added = here ? a.added[r] : 0;
        const long long count = added > 0 ? added : 0;
        long long all;
        const long long end = tokens + block_inclusive(count, warp_sums, &all);
        tokens += all;
        const bool bad = held < 0 || added < 0 || held + added > room || end > a.capacity;
        const long long have = bad ? 0 : (held + a.block_tokens - 1) / a.block_tokens;
        const long long need = bad ? 0 : (held + added + a.block_tokens - 1) / a.block_tokens - have;
        const long long block_end = asked + block_inclusive(need, warp_sums, &all);
        asked += all;
        const bool served = !bad && (need == 0 || block_end <= free_blocks);
        block_inclusive(here && !served, warp_sums, &all);
        refused += all;
        block_inclusive(served ? need : 0, warp_sums, &all);
        taken += all;
        if (!here) continue;
        int32_t *row = a.block_table + (size_t)r * a.blocks_per_slot;
        if (served)
            for (long long j = 0; j < need; ++j) row[have + j] = a.free_blocks[cursor + block_end - need + j];
        a.lengths[r] = int32_t(served ? held + added : held);
        const long long start = end - count;
        if (a.offsets) {
            a.offsets[r] = int32_t(min(start, (long long)INT32_MAX));
            if (r == a.sequences - 1) a.offsets[r + 1] = int32_t(min(end, (long long)INT32_MAX));
        }
        for (long long i = 0; i < count && start + i < a.capacity; ++i) {
            const long long t = start + i, pos = served ? held + i : -1;
            const int block = pos < 0 ? -1 : row[pos / a.block_tokens];
            a.slot_map[t] = block < 0 ? -1 : (long long)block * a.block_tokens + pos % a.block_tokens;
            if (a.positions) a.positions[t] = int32_t(pos);
            if (a.token_slots) a.token_slots[t] = r;
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.cursor_out[0] = cursor + int32_t(taken);
        a.result[0] = int32_t(min(tokens, (long long)a.capacity));
        a.result[1] = int32_t(taken);
        a.result[2] = int32_t(refused);
        a.result[3] = int32_t(min(asked, (long long)INT32_MAX));
    }
}

__device__ __forceinline__ double load_as_double(const void *p, bool f16, int64_t i) {
    return f16 ? double(__half2float(static_cast<const __half *>(p)[i])) : double(static_cast<const float *>(p)[i]);
}

// A warp per token, head and side, in 64 bits throughout.
__global__ void __launch_bounds__(256) append_kernel(jl_kv8_append_args a) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int heads = a.pages.kv_heads, d = a.pages.head_dim;
    const int64_t t = unit / (2 * heads);
    const int side = int(unit % 2), head = int(unit % (2 * heads)) / 2;
    const int count = a.token_count ? min(a.token_count[0], a.tokens) : a.tokens;
    if (t >= count) return;
    const int64_t place = a.slot_map[t];
    if (place < 0 || place >= int64_t(a.pages.blocks) * a.pages.block_tokens) return;
    const void *src = side ? a.v : a.k;
    const int64_t at = t * (side ? a.v_stride : a.k_stride) + int64_t(head) * d;
    const bool f16 = a.ggml_type == JL_F16, turn = side == 0 && a.rope_cos;
    const int pos = turn ? a.positions[t] : 0;
    const bool outside = turn && (pos < 0 || pos >= a.rope_rows);
    double x[4][2], most = 0;
    bool good = !outside;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = 2 * (lane + 32 * i);
        x[i][0] = x[i][1] = 0;
        if (e >= d) continue;
        double p = load_as_double(src, f16, at + e), q = load_as_double(src, f16, at + e + 1);
        if (turn && !outside) {
            const int64_t angle = int64_t(pos) * (d / 2) + e / 2;
            const double c = a.rope_cos[angle], s = a.rope_sin[angle], rotated = p * c - q * s;
            q = p * s + q * c;
            p = rotated;
        }
        x[i][0] = p;
        x[i][1] = q;
        good = good && isfinite(p) && isfinite(q);
        most = fmax(most, fmax(fabs(p), fabs(q)));
    }
    good = __all_sync(~0u, good);
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmax(most, __shfl_xor_sync(~0u, most, o));
    const bool some = good && most >= 0x1p-100;
    const int64_t block = place / a.pages.block_tokens, row = int64_t(head) * a.pages.block_tokens + place % a.pages.block_tokens;
    int8_t *codes = (side ? a.pages.v : a.pages.k) + block * a.pages.block_stride + row * d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = 2 * (lane + 32 * i);
        if (e >= d) continue;
        const int lo = some ? int(rint(x[i][0] * 127.0 / most)) : 0, hi = some ? int(rint(x[i][1] * 127.0 / most)) : 0;
        *reinterpret_cast<char2 *>(codes + e) = make_char2(char(lo), char(hi));
    }
    if (lane == 0)
        (side ? a.pages.v_scale : a.pages.k_scale)[block * a.pages.scale_stride + row] = good ? (some ? float(most / 127.0) : 0.f) : CUDART_NAN_F;
}

}  // namespace

cudaError_t kv8_map_launch(const jl_kv8_map_args &a, const Kv8Scratch &, int, cudaStream_t stream) {
    map_kernel<<<1, kMapThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t kv8_append_launch(const jl_kv8_append_args &a, int, cudaStream_t stream) {
    const int64_t warps = int64_t(a.tokens) * a.pages.kv_heads * 2;
    append_kernel<<<unsigned((warps + 7) / 8), 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace jl
