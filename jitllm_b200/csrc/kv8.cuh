// The 8-bit paged key/value cache (jl_kv8_* of include/jitllm_b200.h): launches of kv8.cu and kv8_attention.cu.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "../../include/jitllm_b200.h"

namespace jl {

// What is wrong with the arguments: a status and, unless it is JL_OK, a message of at most n - 1 characters.
int kv8_check_map(const jl_kv8_map_args *a, char *message, size_t n);
int kv8_check_append(const jl_kv8_append_args *a, char *message, size_t n);
int kv8_check_attention(const jl_kv8_attention_args *a, char *message, size_t n);

// The device half of a jl_kv8_workspace: counters that are zero between launches, then the attention's parts.
constexpr size_t kKv8CounterBytes = 16384, kKv8MapCounter = kKv8CounterBytes - 128;
struct Kv8Scratch {
    void *memory = nullptr;
};
cudaError_t kv8_scratch_create(Kv8Scratch *s, int sm_count);
void kv8_scratch_free(Kv8Scratch *s);

// Constants with which j / divisor = j * divide >> shift for j < 2^31; divisor at most 2^31.
void kv8_division(int divisor, uint64_t *divide, int *shift);
// Lets a kernel have so many bytes of dynamic shared memory on the current device; `configured` has a bit for each device.
cudaError_t kv8_allow_shared(const void *kernel, int bytes, std::atomic<uint64_t> &configured);

// One launch; programmatic: the grid may be set up while the kernel ahead of it in the stream still runs. Map and append let their
// successor do so as soon as they start, the attention when its CTAs are through their last loops; each touches no memory before
// everything ahead of it is over (pdl_wait).
template <typename P>
cudaError_t kv8_launch(void (*kernel)(const P), unsigned grid, unsigned threads, size_t shared, cudaStream_t stream, bool programmatic, const P &params) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = programmatic ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, params);
}

// Arguments that have passed the checks, on the current device.
struct Kv8Launch {
    int sm_count;
    bool programmatic;
    cudaStream_t stream;
};
cudaError_t kv8_map_launch(const jl_kv8_map_args &a, const Kv8Scratch &s, const Kv8Launch &l);
cudaError_t kv8_append_launch(const jl_kv8_append_args &a, const Kv8Launch &l);
cudaError_t kv8_attention_launch(const jl_kv8_attention_args &a, const Kv8Scratch &s, const Kv8Launch &l);

}  // namespace jl
