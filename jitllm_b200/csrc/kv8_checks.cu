// Checks of the arguments of the jl_kv8_* calls. They touch no device: what a kernel would read or write out of bounds, or with
// addresses that it cannot use, is refused here before any launch.
#include <cmath>
#include <cstdio>

#include "kv8.cuh"

namespace jl {
namespace {

#define KV8_REQUIRE(cond, code, ...)              \
    do {                                          \
        if (!(cond)) {                            \
            snprintf(message, n, __VA_ARGS__);    \
            return code;                          \
        }                                         \
    } while (0)

bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_pages(const jl_kv8_pages &p, char *message, size_t n) {
    KV8_REQUIRE(p.k && p.v && p.k_scale && p.v_scale, JL_ERR_INVALID, "k, v, k_scale and v_scale of the pages must not be NULL");
    KV8_REQUIRE(p.head_dim == 64 || p.head_dim == 96 || p.head_dim == 128 || p.head_dim == 192 || p.head_dim == 256, JL_ERR_UNSUPPORTED,
                "head size %d (supported: 64, 96, 128, 192, 256)", p.head_dim);
    KV8_REQUIRE(p.blocks > 0 && p.block_tokens > 0 && p.block_tokens <= 65536 && p.kv_heads > 0 && p.kv_heads <= 1024, JL_ERR_INVALID,
                "blocks must be positive, block_tokens in 1..65536 and kv_heads in 1..1024, got %d, %d and %d", p.blocks, p.block_tokens, p.kv_heads);
    const int64_t rows = int64_t(p.kv_heads) * p.block_tokens;
    KV8_REQUIRE(p.block_stride >= rows * p.head_dim && p.block_stride % 16 == 0 && p.scale_stride >= rows, JL_ERR_INVALID,
                "block_stride %lld and scale_stride %lld: blocks of %lld rows of %d need at least that, block_stride a multiple of 16",
                (long long)p.block_stride, (long long)p.scale_stride, (long long)rows, p.head_dim);
    KV8_REQUIRE(p.block_stride <= INT64_MAX / p.blocks && p.scale_stride <= INT64_MAX / 4 / p.blocks, JL_ERR_INVALID,
                "%d blocks at these strides are beyond 64-bit addresses", p.blocks);
    KV8_REQUIRE(aligned(p.k, 16) && aligned(p.v, 16) && aligned(p.k_scale, 4) && aligned(p.v_scale, 4), JL_ERR_INVALID,
                "k and v of the pages must be 16-byte aligned, their scales 4-byte aligned");
    return JL_OK;
}

int check_rope(const float *cos_table, const float *sin_table, const int32_t *positions, int32_t rows, char *message, size_t n) {
    KV8_REQUIRE((cos_table == nullptr) == (sin_table == nullptr), JL_ERR_INVALID, "rope_cos and rope_sin: both or neither");
    if (!cos_table) return JL_OK;
    KV8_REQUIRE(positions && rows > 0, JL_ERR_INVALID, "rotation tables need positions and a positive rope_rows, got %d", rows);
    KV8_REQUIRE(aligned(cos_table, 16) && aligned(sin_table, 16), JL_ERR_INVALID, "rope_cos and rope_sin must be 16-byte aligned");
    return JL_OK;
}

int check_rows(const char *what, const void *p, int64_t stride, int64_t least, int32_t type, char *message, size_t n) {
    KV8_REQUIRE(type == JL_F32 || type == JL_F16, JL_ERR_UNSUPPORTED, "GGML type %d (supported: F32=0, F16=1)", type);
    KV8_REQUIRE(p, JL_ERR_INVALID, "%s must not be NULL", what);
    const int64_t bytes = type == JL_F32 ? 4 : 2;
    KV8_REQUIRE(stride >= least && stride <= (int64_t(1) << 40) && stride * bytes % 16 == 0 && aligned(p, 16), JL_ERR_INVALID,
                "%s must be 16-byte aligned, its row stride (%lld elements) a multiple of 16 bytes of at least %lld and at most 2^40 elements", what, (long long)stride, (long long)least);
    return JL_OK;
}

}  // namespace

int kv8_check_map(const jl_kv8_map_args *a, char *message, size_t n) {
    KV8_REQUIRE(a, JL_ERR_INVALID, "args must not be NULL");
    KV8_REQUIRE(a->sequences >= 1 && a->sequences <= 8192, JL_ERR_UNSUPPORTED, "%d sequences (1..8192)", a->sequences);
    KV8_REQUIRE(a->blocks_per_slot > 0 && a->block_tokens > 0 && a->block_tokens <= 65536 && a->free_count >= 0 && a->capacity >= 0, JL_ERR_INVALID,
                "blocks_per_slot must be positive, block_tokens in 1..65536, free_count and capacity not negative, got %d, %d, %d and %d",
                a->blocks_per_slot, a->block_tokens, a->free_count, a->capacity);
    KV8_REQUIRE(a->held && a->added && a->cursor && a->cursor_out && a->block_table && a->lengths && a->result, JL_ERR_INVALID,
                "held, added, cursor, cursor_out, block_table, lengths and result must not be NULL");
    KV8_REQUIRE(a->free_blocks || a->free_count == 0, JL_ERR_INVALID, "free_blocks must not be NULL with a free_count of %d", a->free_count);
    KV8_REQUIRE(a->slot_map || a->capacity == 0, JL_ERR_INVALID, "slot_map must not be NULL with a capacity of %d", a->capacity);
    for (const void *p : {(const void *)a->held, (const void *)a->added, (const void *)a->free_blocks, (const void *)a->cursor,
                          (const void *)a->cursor_out, (const void *)a->block_table, (const void *)a->lengths, (const void *)a->offsets,
                          (const void *)a->token_slots, (const void *)a->positions, (const void *)a->result})
        KV8_REQUIRE(aligned(p, 4), JL_ERR_INVALID, "int32 arrays must be 4-byte aligned");
    KV8_REQUIRE(aligned(a->slot_map, 8), JL_ERR_INVALID, "slot_map must be 8-byte aligned");
    return JL_OK;
}

int kv8_check_append(const jl_kv8_append_args *a, char *message, size_t n) {
    KV8_REQUIRE(a, JL_ERR_INVALID, "args must not be NULL");
    int rc = check_pages(a->pages, message, n);
    if (rc) return rc;
    const int64_t row = int64_t(a->pages.kv_heads) * a->pages.head_dim;
    KV8_REQUIRE(a->tokens >= 0 && int64_t(a->tokens) * a->pages.kv_heads <= 1 << 29, JL_ERR_INVALID,
                "tokens must not be negative, and tokens times heads at most 2^29, got %d tokens of %d heads", a->tokens, a->pages.kv_heads);
    if ((rc = check_rows("k", a->k, a->k_stride, row, a->ggml_type, message, n))) return rc;
    if ((rc = check_rows("v", a->v, a->v_stride, row, a->ggml_type, message, n))) return rc;
    if ((rc = check_rope(a->rope_cos, a->rope_sin, a->positions, a->rope_rows, message, n))) return rc;
    KV8_REQUIRE(a->slot_map, JL_ERR_INVALID, "slot_map must not be NULL");
    KV8_REQUIRE(aligned(a->slot_map, 8) && aligned(a->positions, 4) && aligned(a->token_count, 4), JL_ERR_INVALID,
                "slot_map must be 8-byte aligned, positions and token_count 4-byte aligned");
    return JL_OK;
}

int kv8_check_attention(const jl_kv8_attention_args *a, char *message, size_t n) {
    KV8_REQUIRE(a, JL_ERR_INVALID, "args must not be NULL");
    int rc = check_pages(a->pages, message, n);
    if (rc) return rc;
    KV8_REQUIRE(a->rows >= 0 && a->rows <= 1 << 16 && a->slots > 0 && a->blocks_per_slot > 0 && a->window >= 0, JL_ERR_INVALID,
                "rows must be in 0..2^16, slots and blocks_per_slot positive, window not negative, got %d, %d, %d and %d", a->rows, a->slots,
                a->blocks_per_slot, a->window);
    KV8_REQUIRE(a->heads > 0 && a->heads % a->pages.kv_heads == 0 && a->heads <= 16384, JL_ERR_INVALID,
                "heads must be a multiple of kv_heads and at most 16384, got %d and %d", a->heads, a->pages.kv_heads);
    const int64_t tiles = (int64_t(a->blocks_per_slot) * a->pages.block_tokens + 63) / 64 * a->heads;
    KV8_REQUIRE(a->rows == 0 || tiles <= INT32_MAX / a->rows, JL_ERR_UNSUPPORTED,
                "rows times heads times the tokens of a table row must be below 2^37, got %d rows, %d heads, %d blocks of %d", a->rows, a->heads,
                a->blocks_per_slot, a->pages.block_tokens);
    KV8_REQUIRE(std::isfinite(a->scale), JL_ERR_INVALID, "scale must be finite");
    const int64_t row = int64_t(a->heads) * a->pages.head_dim;
    if ((rc = check_rows("q", a->q, a->q_stride, row, a->ggml_type, message, n))) return rc;
    if ((rc = check_rows("out", a->out, a->out_stride, row, a->ggml_type, message, n))) return rc;
    if ((rc = check_rope(a->rope_cos, a->rope_sin, a->positions, a->rope_rows, message, n))) return rc;
    KV8_REQUIRE(a->block_table && a->positions, JL_ERR_INVALID, "block_table and positions must not be NULL");
    for (const void *p : {(const void *)a->lse, (const void *)a->block_table, (const void *)a->kv_slots, (const void *)a->positions, (const void *)a->token_count})
        KV8_REQUIRE(aligned(p, 4), JL_ERR_INVALID, "int32 and float arrays must be 4-byte aligned");
    return JL_OK;
}

}  // namespace jl
