// Dispatchers of the KV cache in blocks: its tables, its writes and read-back, and the attention
// over it.  Nothing of the reference corresponds: its decoder keeps one contiguous cache per layer
// for one sequence (src/models/qwen2/attention.hpp:108-123) and attends it one sequence per call.
#include "op_common.hpp"

namespace llaisys::ops {

namespace {

constexpr size_t kLimit = size_t(1) << 31;

void requireContiguous(std::initializer_list<const tensor_t *> all, const char *op) {
    for (const tensor_t *t : all) ASSERT((*t)->isContiguous(), op << ": tensors must be contiguous");
}

void requireType(std::initializer_list<const tensor_t *> all, llaisysDataType_t dt, const char *what) {
    for (const tensor_t *t : all) ASSERT((*t)->dtype() == dt, what);
}

void requireBlock(size_t block, const char *op) {
    ASSERT(block >= 16 && block <= 256 && (block & (block - 1)) == 0,
           op << ": block must be a power of two in [16, 256]");
}

void requireAligned(const tensor_t &t, const char *op) {
    ASSERT(reinterpret_cast<uintptr_t>(t->data()) % 16 == 0, op << ": tensors must start on 16 bytes");
}

kernels::PagedCache checkCache(const tensor_t &k_cache, const tensor_t &k_scale, const tensor_t &v_cache,
                               const tensor_t &v_scale, const char *op) {
    CHECK_SAME_DEVICE(k_cache, k_scale, v_cache, v_scale);
    requireContiguous({&k_cache, &k_scale, &v_cache, &v_scale}, op);
    ASSERT(k_cache->dtype() == LLAISYS_DTYPE_I8 && v_cache->dtype() == LLAISYS_DTYPE_I8,
           op << ": cache codes must be INT8");
    ASSERT(k_scale->dtype() == LLAISYS_DTYPE_F32 && v_scale->dtype() == LLAISYS_DTYPE_F32,
           op << ": cache scales must be F32");
    ASSERT(k_cache->ndim() == 4 && k_scale->ndim() == 2,
           op << ": cache [n_blocks, n_kvh, block, d], scales [n_blocks, n_kvh]");
    CHECK_SAME_SHAPE(k_cache->shape(), v_cache->shape());
    CHECK_SAME_SHAPE(k_scale->shape(), v_scale->shape());
    const auto &s = k_cache->shape();
    ASSERT(k_scale->shape()[0] == s[0] && k_scale->shape()[1] == s[1], op << ": scale cache shape mismatch");
    requireBlock(s[2], op);
    ASSERT(s[3] > 0 && s[3] % 16 == 0 && s[3] <= 256, op << ": head_dim must be a multiple of 16, at most 256");
    ASSERT(s[0] < kLimit && s[1] <= 65535, op << ": fewer than 2^31 blocks and at most 65535 heads");
    requireAligned(k_cache, op);
    requireAligned(v_cache, op);
    return {reinterpret_cast<int8_t *>(k_cache->data()), reinterpret_cast<int8_t *>(v_cache->data()),
            reinterpret_cast<float *>(k_scale->data()), reinterpret_cast<float *>(v_scale->data()), s[0], s[1], s[2], s[3]};
}

// k and v rows [rows, n_kvh, d] of one float type, and their slots; returns the row count.
size_t checkRows(const tensor_t &k, const tensor_t &v, const tensor_t &slots, const kernels::PagedCache &c,
                 const char *op) {
    CHECK_SAME_DEVICE(k, v, slots);
    requireContiguous({&k, &v, &slots}, op);
    CHECK_SAME_DTYPE(k->dtype(), v->dtype());
    requireFloat(k->dtype());
    ASSERT(slots->dtype() == LLAISYS_DTYPE_I64, op << ": slots must be INT64");
    ASSERT(k->ndim() == 3, op << ": k and v [rows, n_kvh, d]");
    CHECK_SAME_SHAPE(k->shape(), v->shape());
    ASSERT(k->shape()[1] == c.heads && k->shape()[2] == c.dim, op << ": kv head shape mismatch");
    const size_t rows = k->shape()[0];
    ASSERT(slots->numel() == rows, op << ": one slot per row");
    ASSERT(rows < kLimit && rows * c.heads / 8 < size_t(1) << 24, op << ": too many rows and heads for one call");
    requireAligned(k, op);
    requireAligned(v, op);
    return rows;
}

// Bytes of a contiguous tensor.
struct Range {
    const std::byte *begin, *end;
    Range(const tensor_t &t) : begin(t->data()), end(begin + t->numel() * t->elementSize()) {}
    bool meets(const Range &o) const { return begin < o.end && o.begin < end; }
};

template <typename P>
P *ptr(const tensor_t &t) {
    return reinterpret_cast<P *>(t->data());
}

} // namespace

void pagedTables(tensor_t block_table, tensor_t slots, tensor_t pos_ids, tensor_t row_starts, tensor_t free_out,
                 tensor_t old_lens, tensor_t new_lens, tensor_t free_blocks, tensor_t free_in, size_t block) {
    const char *op = "PagedTables";
    CHECK_SAME_DEVICE(block_table, slots, pos_ids, row_starts, free_out, old_lens, new_lens, free_blocks, free_in);
    requireContiguous({&block_table, &slots, &pos_ids, &row_starts, &free_out, &old_lens, &new_lens, &free_blocks, &free_in}, op);
    requireType({&block_table, &row_starts, &old_lens, &new_lens, &free_blocks}, LLAISYS_DTYPE_I32,
                "PagedTables: block_table, row_starts, lengths and free_blocks must be INT32");
    requireType({&slots, &pos_ids, &free_in, &free_out}, LLAISYS_DTYPE_I64,
                "PagedTables: slots, pos_ids and the ring's state must be INT64");
    ASSERT(block_table->ndim() == 2, "PagedTables: block_table [requests, width]");
    const size_t requests = block_table->shape()[0], width = block_table->shape()[1];
    ASSERT(old_lens->numel() == requests && new_lens->numel() == requests, "PagedTables: one old and one new length per request");
    ASSERT(row_starts->numel() == requests + 1, "PagedTables: row_starts must hold requests + 1 elements");
    ASSERT(slots->numel() == pos_ids->numel(), "PagedTables: slots and pos_ids must have the same length");
    ASSERT(free_in->numel() == 2 && free_out->numel() == 2, "PagedTables: the ring's state is (head, tail)");
    requireBlock(block, op);
    ASSERT(requests <= kernels::kPagedTablesRequests, "PagedTables: at most " << kernels::kPagedTablesRequests << " requests");
    ASSERT(width < kLimit && slots->numel() < kLimit / 2 && free_blocks->numel() < kLimit / 2,
           "PagedTables: rows and free_blocks must be below 2^30");
    // each row of what is written is written once, and nothing that is read changes under its readers
    const Range written[] = {block_table, slots, pos_ids, row_starts, free_blocks, free_out}, read[] = {old_lens, new_lens, free_in};
    for (const Range *w = written; w != written + 6; ++w) {
        for (const Range *o = w + 1; o != written + 6; ++o) ASSERT(!w->meets(*o), "PagedTables: outputs must not overlap");
        for (const Range &r : read)
            ASSERT(!w->meets(r) || (w == written + 5 && &r == read + 2 && r.begin == w->begin),
                   "PagedTables: outputs must not overlap inputs (free_out may be free_in)");
    }
    auto s = streamFor(block_table);
    const kernels::PagedTablesCall c{ptr<int32_t>(block_table), ptr<int64_t>(slots), ptr<int64_t>(pos_ids), ptr<int32_t>(row_starts),
                               ptr<int64_t>(free_out), ptr<const int32_t>(old_lens), ptr<const int32_t>(new_lens),
                               ptr<int32_t>(free_blocks), ptr<const int64_t>(free_in), requests, width, slots->numel(),
                               free_blocks->numel(), block, device::amd::errorWord(block_table->deviceId())};
    kernels::pagedTables(c, device::amd::workspace(block_table->deviceId(), kernels::kScratchReserved), s);
    launched("pagedTables");
}

void pagedKvAppendInt8(tensor_t k_cache, tensor_t k_scale, tensor_t v_cache, tensor_t v_scale, tensor_t k, tensor_t v,
                       tensor_t slots) {
    const char *op = "PagedKVAppendInt8";
    CHECK_SAME_DEVICE(k_cache, k);
    const kernels::PagedCache c = checkCache(k_cache, k_scale, v_cache, v_scale, op);
    const size_t rows = checkRows(k, v, slots, c, op);
    ASSERT(!overlaps(k_cache, v_cache) && !overlaps(k_scale, v_scale), "PagedKVAppendInt8: the k and v caches must not overlap");
    auto s = streamFor(k);
    kernels::pagedKvAppendInt8(c, k->data(), v->data(), ptr<const int64_t>(slots), rows, k->dtype(),
                               device::amd::errorWord(k->deviceId()), s);
    launched("pagedKvAppendInt8");
}

void pagedKvReadInt8(tensor_t k, tensor_t v, tensor_t k_cache, tensor_t k_scale, tensor_t v_cache, tensor_t v_scale,
                     tensor_t slots) {
    const char *op = "PagedKVReadInt8";
    CHECK_SAME_DEVICE(k_cache, k);
    const kernels::PagedCache c = checkCache(k_cache, k_scale, v_cache, v_scale, op);
    const size_t rows = checkRows(k, v, slots, c, op);
    ASSERT(!overlaps(k, v), "PagedKVReadInt8: k and v must not overlap");
    auto s = streamFor(k);
    kernels::pagedKvReadInt8(k->data(), v->data(), c, ptr<const int64_t>(slots), rows, k->dtype(),
                             device::amd::errorWord(k->deviceId()), s);
    launched("pagedKvReadInt8");
}

void pagedAttentionInt8KV(tensor_t attn_val, tensor_t q, tensor_t k_cache, tensor_t k_scale, tensor_t v_cache,
                          tensor_t v_scale, tensor_t block_table, tensor_t row_starts, tensor_t kv_lens, float scale) {
    const char *op = "PagedAttentionInt8KV";
    CHECK_SAME_DEVICE(attn_val, q, k_cache, block_table, row_starts, kv_lens);
    const kernels::PagedCache c = checkCache(k_cache, k_scale, v_cache, v_scale, op);
    requireContiguous({&attn_val, &q, &block_table, &row_starts, &kv_lens}, op);
    CHECK_SAME_DTYPE(attn_val->dtype(), q->dtype());
    requireFloat(q->dtype());
    requireType({&block_table, &row_starts, &kv_lens}, LLAISYS_DTYPE_I32,
                "PagedAttentionInt8KV: block_table, row_starts and kv_lens must be INT32");
    ASSERT(q->ndim() == 3, "PagedAttentionInt8KV: q [rows, nh, d]");
    CHECK_SAME_SHAPE(attn_val->shape(), q->shape());
    const size_t rows = q->shape()[0], nh = q->shape()[1];
    ASSERT(q->shape()[2] == c.dim, "PagedAttentionInt8KV: head_dim mismatch");
    ASSERT(c.n_blocks > 0, "PagedAttentionInt8KV: the cache has no blocks"); // (a bad id is read as block 0)
    ASSERT(c.heads > 0 && nh > 0 && nh % c.heads == 0, "nhead must be divisible by kv_head (GQA)");
    ASSERT(block_table->ndim() == 2, "PagedAttentionInt8KV: block_table [requests, width]");
    const size_t requests = block_table->shape()[0], width = block_table->shape()[1];
    ASSERT(kv_lens->numel() == requests && row_starts->numel() == requests + 1,
           "PagedAttentionInt8KV: kv_lens must hold a length per request and row_starts requests + 1 elements");
    ASSERT(rows < kLimit && requests < kLimit && nh <= 65535, "PagedAttentionInt8KV: sizes must be below 2^31, heads at most 65535");
    // one launch: fewer than 2^24 blocks of 256 threads, 16 rows of a kv head each at the least
    ASSERT(rows * nh / 16 + requests * c.heads < (size_t(1) << 24) - (size_t(1) << 17),
           "PagedAttentionInt8KV: too many rows and heads for one call");
    ASSERT(width < kLimit && width * c.block <= kLimit - 4096, "PagedAttentionInt8KV: a request's blocks must hold fewer than 2^31 tokens");
    ASSERT(!overlaps(attn_val, q), "PagedAttentionInt8KV: attn_val must not overlap q");
    requireAligned(q, op);
    requireAligned(attn_val, op);
    auto s = streamFor(q);
    const kernels::PagedAttentionCall call{attn_val->data(), q->data(), c, ptr<const int32_t>(block_table),
                                           ptr<const int32_t>(row_starts), ptr<const int32_t>(kv_lens), rows, requests, width,
                                           nh, scale, q->dtype(), device::amd::errorWord(q->deviceId())};
    const size_t want = kernels::pagedAttentionWorkspaceBytes(call);
    void *ws = want ? device::amd::tryWorkspace(q->deviceId(), kernels::kScratchReserved + want, s) : nullptr;
    kernels::pagedAttentionInt8KV(call, ws, want, s);
    launched("pagedAttentionInt8KV");
}

} // namespace llaisys::ops
