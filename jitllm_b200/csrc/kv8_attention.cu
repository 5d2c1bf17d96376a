// Attention of single tokens over the 8-bit paged key/value cache.
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"
#include "kv8.cuh"

namespace jl {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxPairs = 4;  // pairs of elements that a lane has of a head of 256

// A CTA per row and query head: its warps take tokens in turn, one at a time, with a running maximum and sum (a rescaled
// softmax, so one pass over the cache), and are folded at the end.
__global__ void __launch_bounds__(32 * kWarps) attention_kernel(jl_kv8_attention_args a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x, h = blockIdx.y, d = a.pages.head_dim;
    if (a.token_count && r >= a.token_count[0]) return;
    const int kv = h / (a.heads / a.pages.kv_heads), bt = a.pages.block_tokens;
    const int slot = a.kv_slots ? a.kv_slots[r] : r, pos = a.positions[r];
    const bool there = slot >= 0 && slot < a.slots;
    const int64_t length = there ? min(int64_t(pos) + 1, int64_t(a.blocks_per_slot) * bt) : 0;
    const int64_t first = a.window > 0 ? max(int64_t(pos) + 1 - a.window, int64_t(0)) : 0;
    const bool f16 = a.ggml_type == JL_F16, outside = a.rope_cos && pos >= a.rope_rows;

    float q[kMaxPairs][2], o[kMaxPairs][2];
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        const int e = 2 * (lane + 32 * i);
        q[i][0] = q[i][1] = o[i][0] = o[i][1] = 0.f;
        if (e >= d || pos < 0) continue;
        const int64_t at = int64_t(r) * a.q_stride + int64_t(h) * d + e;
        q[i][0] = f16 ? __half2float(static_cast<const __half *>(a.q)[at]) : static_cast<const float *>(a.q)[at];
        q[i][1] = f16 ? __half2float(static_cast<const __half *>(a.q)[at + 1]) : static_cast<const float *>(a.q)[at + 1];
        if (a.rope_cos) {
            const int64_t angle = int64_t(outside ? 0 : pos) * (d / 2) + e / 2;
            const float c = outside ? CUDART_NAN_F : a.rope_cos[angle], s = outside ? CUDART_NAN_F : a.rope_sin[angle];
            const float rotated = q[i][0] * c - q[i][1] * s;
            q[i][1] = q[i][0] * s + q[i][1] * c;
            q[i][0] = rotated;
        }
    }
    float most = -CUDART_INF_F, sum = 0.f;
    for (int64_t j = first + warp; j < length; j += kWarps) {
        const int block = a.block_table[int64_t(slot) * a.blocks_per_slot + j / bt];
        if (block < 0 || block >= a.pages.blocks) continue;
        const int64_t row = int64_t(kv) * bt + j % bt;
        const int8_t *k = a.pages.k + block * a.pages.block_stride + row * d, *v = a.pages.v + block * a.pages.block_stride + row * d;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxPairs; ++i) {
            const int e = 2 * (lane + 32 * i);
            if (e >= d) continue;
            const char2 c = *reinterpret_cast<const char2 *>(k + e);
            s += q[i][0] * float((signed char)c.x) + q[i][1] * float((signed char)c.y);
        }
#pragma unroll
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(~0u, s, w);
        s *= a.scale * a.pages.k_scale[block * a.pages.scale_stride + row];
        const float now = fmaxf(most, s), base = now == -CUDART_INF_F ? 0.f : now, keep = expf(most - base), p = expf(s - base);
        // o is the mean of the values so far, which is never larger than they are; their sum could be beyond binary32
        const float before = sum * keep, vs = a.pages.v_scale[block * a.pages.scale_stride + row];
        most = now;
        sum = before + p;
        const float old = sum == 0.f ? 0.f : before / sum, fresh = sum == 0.f ? 0.f : p / sum;
#pragma unroll
        for (int i = 0; i < kMaxPairs; ++i) {
            const int e = 2 * (lane + 32 * i);
            if (e >= d) continue;
            const char2 c = *reinterpret_cast<const char2 *>(v + e);
            o[i][0] = o[i][0] * old + fresh * (vs * float((signed char)c.x));
            o[i][1] = o[i][1] * old + fresh * (vs * float((signed char)c.y));
        }
    }
    __shared__ float warp_most[kWarps], warp_sum[kWarps], warp_out[kWarps][64 * kMaxPairs];
    if (lane == 0) {
        warp_most[warp] = most;
        warp_sum[warp] = sum;
    }
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        warp_out[warp][2 * (lane + 32 * i)] = o[i][0];
        warp_out[warp][2 * (lane + 32 * i) + 1] = o[i][1];
    }
    __syncthreads();
    float all = -CUDART_INF_F, total = 0.f;
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, warp_most[w]);
    const float base = all == -CUDART_INF_F ? 0.f : all;
    float part[kWarps];
    for (int w = 0; w < kWarps; ++w) {
        part[w] = expf(warp_most[w] - base);
        total += warp_sum[w] * part[w];
    }
    for (int e = threadIdx.x; e < d; e += 32 * kWarps) {
        float x = 0.f;
        for (int w = 0; w < kWarps; ++w) x += total == 0.f ? 0.f : warp_out[w][e] * (warp_sum[w] * part[w] / total);
        const int64_t at = int64_t(r) * a.out_stride + int64_t(h) * d + e;
        if (f16)
            static_cast<__half *>(a.out)[at] = __float2half_rn(x);
        else
            static_cast<float *>(a.out)[at] = x;
    }
    if (a.lse && threadIdx.x == 0) a.lse[int64_t(r) * a.heads + h] = total == 0.f ? -CUDART_INF_F : base + logf(total);
}

}  // namespace

cudaError_t kv8_attention_launch(const jl_kv8_attention_args &a, const Kv8Scratch &, int, cudaStream_t stream) {
    attention_kernel<<<dim3(a.rows, a.heads), 32 * kWarps, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace jl
