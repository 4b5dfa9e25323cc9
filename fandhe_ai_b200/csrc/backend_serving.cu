// C-ABI implementation, part 3: the serving step of a ragged batch - rotating cache append, attention of ragged chunks over the
// paged cache, token sampling.  Everything a call needs lives on the device, so a step needs no host data.  Arguments are
// checked before the first driver call; what only the device knows (lengths, block ids, per-row sampling parameters) is checked
// by the kernels.
#include <cmath>

#include "backend.h"
#include "kernels.cuh"

using namespace b200;

namespace {

constexpr uint64_t kI32Max = 0x7FFFFFFFull;

int32_t bad(const char* op, const std::string& msg) { return fail(B200_INVALID_ARGUMENT, std::string(op) + ": " + msg); }

bool cmul(uint64_t a, uint64_t b, uint64_t* out) { return !__builtin_mul_overflow(a, b, out); }

size_t item_bytes(int32_t dtype) { return dtype == B200_BF16 ? 2 : 4; }

// A buffer range that starts on a 16-byte boundary (imported memory may start anywhere)
int32_t check_aligned(const b200_ctx* ctx, const char* op, const b200_buf* buf, size_t off, uint64_t need, const char* name, size_t align,
                      bool optional = false) {
    const std::string label = std::string(op) + " " + name;
    if (int32_t st = check_buf(ctx, buf, off, need, label.c_str(), optional)) return st;
    if (buf && ((reinterpret_cast<uintptr_t>(buf->ptr) + off) & (align - 1)) != 0)
        return bad(op, std::string(name) + " must start on a " + std::to_string(align) + "-byte boundary");
    return B200_OK;
}

// Do two ranges of the caller's memory share a byte?  (Handles of imported memory may name the same one.)
bool overlap(const b200_buf* a, size_t a_off, uint64_t a_bytes, const b200_buf* b, size_t b_off, uint64_t b_bytes) {
    if (!a || !b || a_bytes == 0 || b_bytes == 0) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a->ptr) + a_off, y = reinterpret_cast<uintptr_t>(b->ptr) + b_off;
    return x < y + b_bytes && y < x + a_bytes;
}

// The part of the arguments that append and attention share
struct Ragged {
    RaggedShape sh;
    uint64_t head_dim, pool_bytes, table_bytes;
};

int32_t check_ragged(const char* op, const b200_paged_kv_layout* l, uint64_t batch, uint64_t rows, uint64_t row_stride, uint64_t row_width,
                     uint64_t num_heads, uint64_t num_kv_heads, uint64_t max_blocks_per_seq, int32_t io_dtype, Ragged* out) {
    // the layout's own rules, by the validator that every paged entry uses
    const b200_paged_attention_args probe = {*l, 0, 0, num_heads, num_kv_heads, 0, 1.0f};
    if (int32_t st = b200_validate_paged_attention(0, l->num_blocks * l->block_size * l->embed_dim, l->num_blocks * l->block_size * l->embed_dim,
                                                   nullptr, 0, nullptr, 0, &probe, nullptr))
        return st;
    if (io_dtype != B200_F32 && io_dtype != B200_BF16) return bad(op, "io_dtype must be F32 or BF16");
    if (batch > kI32Max || rows > kI32Max || max_blocks_per_seq > kI32Max) return bad(op, "batch, rows and max_blocks_per_seq must not exceed i32::MAX");
    if (l->num_blocks > kI32Max) return fail(B200_UNSUPPORTED, std::string(op) + ": num_blocks above i32::MAX is not supported");
    const uint64_t dh = l->embed_dim / num_kv_heads;
    if (dh > 256) return fail(B200_UNSUPPORTED, std::string(op) + ": head_dim above 256 is not supported");
    if (num_heads > 65535) return fail(B200_UNSUPPORTED, std::string(op) + ": more than 65535 query heads are not supported");
    if (row_stride != 0 && row_stride < row_width) return bad(op, "row stride is smaller than a row");
    const uint64_t stride = row_stride ? row_stride : row_width;
    uint64_t span;
    if (!cmul(rows, stride, &span) || span > (1ull << 60)) return bad(op, "rows * row stride overflows");
    uint64_t tables;
    if (!cmul(batch, max_blocks_per_seq, &tables) || tables > (1ull << 60)) return bad(op, "batch * max_blocks_per_seq overflows");
    uint64_t cap;
    if (!cmul(max_blocks_per_seq, l->block_size, &cap) || cap > kI32Max) return bad(op, "max_blocks_per_seq * block_size exceeds i32::MAX");
    out->head_dim = dh;
    out->pool_bytes = l->num_blocks * l->block_size * l->embed_dim * item_bytes(l->dtype);
    out->table_bytes = tables * 4;
    RaggedShape& s = out->sh;
    s = RaggedShape{};
    s.rows = int64_t(rows);
    s.row_stride = int64_t(stride);
    s.batch = int(batch);
    s.num_q_heads = int(num_heads);
    s.num_kv_heads = int(num_kv_heads);
    s.head_dim = int(dh);
    s.block_size = int(l->block_size);
    s.num_blocks = int(l->num_blocks);
    s.max_blocks_per_seq = int(max_blocks_per_seq);
    return B200_OK;
}

// Bytes from the first element of a strided array of rows to its last
uint64_t span_bytes(uint64_t rows, uint64_t stride, uint64_t width, size_t item) { return rows == 0 ? 0 : ((rows - 1) * stride + width) * item; }

int32_t check_index_buffers(const b200_ctx* ctx, const char* op, const Ragged& r, uint64_t batch, const b200_buf* tables,
                            const b200_buf* q_starts, const b200_buf* seq_lens) {
    if (int32_t st = check_aligned(ctx, op, tables, 0, r.table_bytes, "block_tables", 4)) return st;
    if (int32_t st = check_aligned(ctx, op, q_starts, 0, (batch + 1) * 4, "q_starts", 4)) return st;
    return check_aligned(ctx, op, seq_lens, 0, batch * 4, "seq_lens", 4);
}

int32_t chunk_args(const b200_paged_chunk_args* a, Ragged* r) {
    const char* op = "paged_chunk_attention";
    if (!a) return bad(op, "args is null");
    if (a->num_kv_heads == 0 || a->layout.embed_dim % a->num_kv_heads != 0) return bad(op, "num_kv_heads must be >= 1 and divide embed_dim");
    const uint64_t dh = a->layout.embed_dim / a->num_kv_heads;
    uint64_t width;
    if (!cmul(a->num_heads, dh, &width) || width > kI32Max) return bad(op, "num_heads * head_dim exceeds i32::MAX");
    if (int32_t st = check_ragged(op, &a->layout, a->batch, a->rows, a->q_stride, width, a->num_heads, a->num_kv_heads, a->max_blocks_per_seq, a->io_dtype, r))
        return st;
    if (!std::isfinite(a->scale)) return bad(op, "scale must be finite");
    const uint64_t cap = a->max_blocks_per_seq * a->layout.block_size;
    if (a->max_seq_len > cap) return bad(op, "max_seq_len exceeds max_blocks_per_seq * block_size");
    if (a->max_q_len > a->max_seq_len) return bad(op, "max_q_len exceeds max_seq_len");
    r->sh.scale = a->scale;
    r->sh.max_q_len = int(a->max_q_len);
    r->sh.max_seq_len = int(a->max_seq_len);
    return B200_OK;
}

int32_t append_args(const b200_rope_append_args* a, Ragged* r, uint64_t* row_width) {
    const char* op = "rope_paged_kv_append";
    if (!a) return bad(op, "args is null");
    if (a->num_kv_heads == 0 || a->layout.embed_dim % a->num_kv_heads != 0) return bad(op, "num_kv_heads must be >= 1 and divide embed_dim");
    const uint64_t dh = a->layout.embed_dim / a->num_kv_heads;
    if (a->num_heads > kI32Max || !cmul(a->num_heads + 2 * a->num_kv_heads, dh, row_width) || *row_width > kI32Max)
        return bad(op, "a row of q, k and v exceeds i32::MAX elements");
    if (int32_t st = check_ragged(op, &a->layout, a->batch, a->rows, a->qkv_stride, *row_width, a->num_heads, a->num_kv_heads, a->max_blocks_per_seq, a->io_dtype, r))
        return st;
    r->sh.max_q_len = r->sh.max_seq_len = r->sh.max_blocks_per_seq * r->sh.block_size;
    if (a->rotary_dim % 2 != 0 || a->rotary_dim > dh) return bad(op, "rotary_dim must be even and at most head_dim");
    if (a->adjacent_pairs && (dh % 2 != 0 || r->sh.row_stride % 2 != 0)) return bad(op, "adjacent pairs need an even head_dim and an even row stride");
    if (a->n_positions > kI32Max) return bad(op, "n_positions exceeds i32::MAX");
    return B200_OK;
}

int32_t sample_args(const b200_sample_args* a, uint64_t* stride) {
    const char* op = "sample_tokens";
    if (!a) return bad(op, "args is null");
    if (a->dtype != B200_F32 && a->dtype != B200_BF16) return bad(op, "dtype must be F32 or BF16");
    if (a->rows > (1ull << 27)) return bad(op, "rows must not exceed 2^27");
    if (a->vocab == 0) return bad(op, "vocab must be at least 1");
    if (a->vocab > uint64_t(sample_tokens_max_vocab()))
        return fail(B200_UNSUPPORTED, std::string(op) + ": a vocabulary above " + std::to_string(sample_tokens_max_vocab()) + " tokens is not supported");
    if (a->row_stride != 0 && a->row_stride < a->vocab) return bad(op, "row stride is smaller than a row");
    *stride = a->row_stride ? a->row_stride : a->vocab;
    uint64_t span;
    if (!cmul(a->rows, *stride, &span) || span > (1ull << 60)) return bad(op, "rows * row stride overflows");
    return B200_OK;
}

}  // namespace

extern "C" {

int32_t b200_validate_ragged_batch(const uint32_t* block_tables, const uint32_t* q_starts, const uint32_t* seq_lens,
                                   const b200_paged_chunk_args* a) {
    const char* op = "ragged_batch";
    Ragged r;
    if (int32_t st = chunk_args(a, &r)) return st;
    if (a->batch == 0) return B200_OK;
    if (!q_starts || !seq_lens || (a->max_blocks_per_seq > 0 && !block_tables)) return bad(op, "null array");
    if (q_starts[0] != 0) return bad(op, "q_starts[0] must be 0");
    for (uint64_t b = 0; b < a->batch; ++b) {
        const std::string who = "sequence " + std::to_string(b) + ": ";
        if (q_starts[b + 1] < q_starts[b]) return bad(op, who + "q_starts decreases");
        const uint64_t n = q_starts[b + 1] - q_starts[b], len = seq_lens[b];
        if (n > len) return bad(op, who + std::to_string(n) + " new tokens, but only " + std::to_string(len) + " cached ones");
        if (n > a->max_q_len) return bad(op, who + std::to_string(n) + " new tokens exceed max_q_len");
        if (len > a->max_seq_len) return bad(op, who + "length " + std::to_string(len) + " exceeds max_seq_len");
        const uint64_t used = (len + a->layout.block_size - 1) / a->layout.block_size;
        for (uint64_t i = 0; i < used; ++i)
            if (block_tables[b * a->max_blocks_per_seq + i] >= a->layout.num_blocks)
                return bad(op, who + "block id " + std::to_string(block_tables[b * a->max_blocks_per_seq + i]) + " in slot " + std::to_string(i) + " is >= num_blocks");
    }
    if (q_starts[a->batch] > a->rows) return bad(op, "q_starts ends behind the last row");
    return B200_OK;
}

int32_t b200_validate_rope_append(const b200_rope_append_args* a) {
    Ragged r;
    uint64_t width;
    return append_args(a, &r, &width);
}

int32_t b200_validate_sample(const b200_sample_args* a) {
    uint64_t stride;
    return sample_args(a, &stride);
}

int32_t b200_rope_table(double theta, uint64_t rotary_dim, uint64_t n_positions, float* cos_out, float* sin_out) {
    const char* op = "rope_table";
    if (!(theta > 0.0) || !std::isfinite(theta)) return bad(op, "theta must be finite and positive");
    if (rotary_dim == 0 || rotary_dim % 2 != 0 || rotary_dim > 65536) return bad(op, "rotary_dim must be even and in 2..65536");
    if (n_positions > kI32Max) return bad(op, "n_positions exceeds i32::MAX");
    if (n_positions > 0 && (!cos_out || !sin_out)) return bad(op, "null output");
    const uint64_t half = rotary_dim / 2;
    for (uint64_t i = 0; i < half; ++i) {
        const double inv = std::pow(theta, -2.0 * double(i) / double(rotary_dim));
        for (uint64_t p = 0; p < n_positions; ++p) {
            const double angle = double(p) * inv;       // in f64: far positions turn many times
            cos_out[p * half + i] = float(std::cos(angle));
            sin_out[p * half + i] = float(std::sin(angle));
        }
    }
    return B200_OK;
}

int32_t b200_rope_paged_kv_append(b200_ctx* ctx, const b200_buf* qkv, size_t qkv_off, const b200_buf* cos_table, const b200_buf* sin_table,
                                  const b200_buf* positions, const b200_buf* block_tables, const b200_buf* q_starts,
                                  const b200_buf* seq_lens, b200_buf* k_pool, b200_buf* v_pool, const b200_rope_append_args* a,
                                  b200_buf* q_out, size_t q_out_off) {
    const char* op = "rope_paged_kv_append";
    if (int32_t st = check_ctx(ctx)) return st;
    Ragged r;
    uint64_t width;
    if (int32_t st = append_args(a, &r, &width)) return st;
    const uint64_t heads = a->num_heads * r.head_dim;
    const size_t item = item_bytes(a->io_dtype);
    const uint64_t table = a->n_positions * (a->rotary_dim / 2) * 4;
    if (int32_t st = check_aligned(ctx, op, qkv, qkv_off, span_bytes(a->rows, r.sh.row_stride, width, item), "qkv", 16)) return st;
    if (int32_t st = check_aligned(ctx, op, q_out, q_out_off, a->rows * heads * item, "q_out", 16)) return st;
    if (int32_t st = check_aligned(ctx, op, cos_table, 0, table, "cos_table", 16, table == 0)) return st;
    if (int32_t st = check_aligned(ctx, op, sin_table, 0, table, "sin_table", 16, table == 0)) return st;
    if (int32_t st = check_aligned(ctx, op, positions, 0, a->rows * 4, "positions", 4, true)) return st;
    if (int32_t st = check_index_buffers(ctx, op, r, a->batch, block_tables, q_starts, seq_lens)) return st;
    if (int32_t st = check_aligned(ctx, op, k_pool, 0, r.pool_bytes, "k_pool", 16)) return st;
    if (int32_t st = check_aligned(ctx, op, v_pool, 0, r.pool_bytes, "v_pool", 16)) return st;
    if (a->rows == 0 || a->batch == 0) return B200_OK;
    const uint64_t in_bytes = span_bytes(a->rows, r.sh.row_stride, width, item), out_bytes = a->rows * heads * item;
    if (overlap(qkv, qkv_off, in_bytes, q_out, q_out_off, out_bytes)) return bad(op, "q_out overlaps qkv");
    for (const b200_buf* pool : {k_pool, v_pool}) {
        if (overlap(pool, 0, r.pool_bytes, qkv, qkv_off, in_bytes) || overlap(pool, 0, r.pool_bytes, q_out, q_out_off, out_bytes))
            return bad(op, "a pool overlaps qkv or q_out");
    }
    if (overlap(k_pool, 0, r.pool_bytes, v_pool, 0, r.pool_bytes)) return bad(op, "k_pool overlaps v_pool");
    if (int32_t st = set_device(ctx)) return st;
    const RopeShape rope = {int(a->rotary_dim), a->adjacent_pairs != 0, int64_t(a->n_positions)};
    const cudaError_t e = rope_paged_kv_append(
        r.sh, rope, buf_ptr<const uint8_t>(qkv, qkv_off), a->io_dtype == B200_BF16, buf_ptr<const float>(cos_table, 0),
        buf_ptr<const float>(sin_table, 0), buf_ptr<const uint32_t>(positions, 0), buf_ptr<const uint32_t>(block_tables, 0),
        buf_ptr<const uint32_t>(q_starts, 0), buf_ptr<const uint32_t>(seq_lens, 0), buf_ptr<uint8_t>(q_out, q_out_off), k_pool->ptr,
        v_pool->ptr, a->layout.dtype == B200_BF16, ctx->sm_count, ctx->err_dev, ctx->stream);
    if (e != cudaSuccess) return fail_runtime(ctx, B200_KERNEL_LAUNCH_FAILED, std::string(op) + ": " + cudaGetErrorString(e));
    return B200_OK;
}

int32_t b200_paged_chunk_workspace(b200_ctx* ctx, const b200_paged_chunk_args* a, size_t* bytes) {
    if (int32_t st = check_ctx(ctx)) return st;
    if (!bytes) return bad("paged_chunk_workspace", "bytes is null");
    Ragged r;
    if (int32_t st = chunk_args(a, &r)) return st;
    *bytes = paged_chunk_workspace_bytes(r.sh, a->io_dtype == B200_BF16, a->layout.dtype == B200_BF16, ctx->sm_count);
    return B200_OK;
}

int32_t b200_paged_chunk_attention(b200_ctx* ctx, const b200_buf* q, size_t q_off, const b200_buf* k_pool, const b200_buf* v_pool,
                                   const b200_buf* block_tables, const b200_buf* q_starts, const b200_buf* seq_lens,
                                   const b200_paged_chunk_args* a, b200_buf* workspace, b200_buf* out, size_t out_off) {
    const char* op = "paged_chunk_attention";
    if (int32_t st = check_ctx(ctx)) return st;
    Ragged r;
    if (int32_t st = chunk_args(a, &r)) return st;
    const size_t item = item_bytes(a->io_dtype);
    const uint64_t width = a->num_heads * r.head_dim;
    if (int32_t st = check_aligned(ctx, op, q, q_off, span_bytes(a->rows, r.sh.row_stride, width, item), "q", 16)) return st;
    if (int32_t st = check_aligned(ctx, op, out, out_off, a->rows * width * item, "out", 16)) return st;
    if (int32_t st = check_aligned(ctx, op, k_pool, 0, r.pool_bytes, "k_pool", 16)) return st;
    if (int32_t st = check_aligned(ctx, op, v_pool, 0, r.pool_bytes, "v_pool", 16)) return st;
    if (int32_t st = check_index_buffers(ctx, op, r, a->batch, block_tables, q_starts, seq_lens)) return st;
    const size_t need = paged_chunk_workspace_bytes(r.sh, a->io_dtype == B200_BF16, a->layout.dtype == B200_BF16, ctx->sm_count);
    if (int32_t st = check_aligned(ctx, op, workspace, 0, need, "workspace", 16, need == 0)) return st;
    if (a->rows == 0 || a->batch == 0 || a->max_q_len == 0) return B200_OK;
    // Results in the queries' own places are fine: a row and head is read by the blocks that write it, or before the join does.
    const uint64_t in_bytes = span_bytes(a->rows, r.sh.row_stride, width, item), out_bytes = a->rows * width * item;
    const bool in_place = static_cast<uint8_t*>(q->ptr) + q_off == static_cast<uint8_t*>(out->ptr) + out_off && uint64_t(r.sh.row_stride) == width;
    if (!in_place && overlap(q, q_off, in_bytes, out, out_off, out_bytes)) return bad(op, "out overlaps q (it may only be q itself, with dense rows)");
    for (const b200_buf* pool : {k_pool, v_pool})
        if (overlap(pool, 0, r.pool_bytes, out, out_off, out_bytes) || overlap(pool, 0, r.pool_bytes, workspace, 0, need))
            return bad(op, "a pool overlaps out or the workspace");
    if (overlap(workspace, 0, need, q, q_off, in_bytes) || overlap(workspace, 0, need, out, out_off, out_bytes))
        return bad(op, "the workspace overlaps q or out");
    if (int32_t st = set_device(ctx)) return st;
    const cudaError_t e = paged_chunk_attention(
        r.sh, buf_ptr<const uint8_t>(q, q_off), a->io_dtype == B200_BF16, k_pool->ptr, v_pool->ptr, a->layout.dtype == B200_BF16,
        buf_ptr<const uint32_t>(block_tables, 0), buf_ptr<const uint32_t>(q_starts, 0), buf_ptr<const uint32_t>(seq_lens, 0),
        buf_ptr<uint8_t>(workspace, 0), buf_ptr<uint8_t>(out, out_off), ctx->sm_count, ctx->err_dev, ctx->stream);
    if (e != cudaSuccess) return fail_runtime(ctx, B200_KERNEL_LAUNCH_FAILED, std::string(op) + ": " + cudaGetErrorString(e));
    return B200_OK;
}

int32_t b200_sample_tokens(b200_ctx* ctx, const b200_buf* logits, size_t logits_off, const b200_sample_args* a, const b200_buf* temperature,
                           const b200_buf* top_k, const b200_buf* top_p, const b200_buf* min_p, const b200_buf* uniform, b200_buf* ids,
                           b200_buf* prob, b200_buf* kept) {
    const char* op = "sample_tokens";
    if (int32_t st = check_ctx(ctx)) return st;
    uint64_t stride;
    if (int32_t st = sample_args(a, &stride)) return st;
    const size_t item = item_bytes(a->dtype);
    if (int32_t st = check_aligned(ctx, op, logits, logits_off, span_bytes(a->rows, stride, a->vocab, item), "logits", item)) return st;
    if (int32_t st = check_aligned(ctx, op, temperature, 0, a->rows * 4, "temperature", 4, true)) return st;
    if (int32_t st = check_aligned(ctx, op, top_k, 0, a->rows * 4, "top_k", 4, true)) return st;
    if (int32_t st = check_aligned(ctx, op, top_p, 0, a->rows * 4, "top_p", 4, true)) return st;
    if (int32_t st = check_aligned(ctx, op, min_p, 0, a->rows * 4, "min_p", 4, true)) return st;
    if (int32_t st = check_aligned(ctx, op, uniform, 0, a->rows * 4, "uniform", 4)) return st;
    if (int32_t st = check_aligned(ctx, op, ids, 0, a->rows * 4, "ids", 4)) return st;
    if (int32_t st = check_aligned(ctx, op, prob, 0, a->rows * 4, "prob", 4, true)) return st;
    if (int32_t st = check_aligned(ctx, op, kept, 0, a->rows * 4, "kept", 4, true)) return st;
    if (a->rows == 0) return B200_OK;
    if (int32_t st = set_device(ctx)) return st;
    SampleShape sh = {};
    sh.rows = int64_t(a->rows);
    sh.row_stride = int64_t(stride);
    sh.vocab = int(a->vocab);
    const cudaError_t e = sample_tokens(sh, buf_ptr<const uint8_t>(logits, logits_off), a->dtype == B200_BF16, buf_ptr<const float>(temperature, 0),
                                        buf_ptr<const int>(top_k, 0), buf_ptr<const float>(top_p, 0), buf_ptr<const float>(min_p, 0),
                                        buf_ptr<const float>(uniform, 0), buf_ptr<int>(ids, 0), buf_ptr<float>(prob, 0),
                                        buf_ptr<int>(kept, 0), ctx->sm_count, ctx->stream);
    if (e != cudaSuccess) return fail_runtime(ctx, B200_KERNEL_LAUNCH_FAILED, std::string(op) + ": " + cudaGetErrorString(e));
    return B200_OK;
}

}  // extern "C"
