// Causal GQA attention of many requests over the INT8 KV cache in blocks: plan and launch.
//
// Row i of request r's n rows sees its cached tokens t <= lens[r] - n + i:
//   s_t = scale * k_scale[block(t)] * (q . k_codes[t]),  p_t = exp(s_t - m),  m = max s,
//   out = sum_t p_t * v_scale[block(t)] * v_codes[t] / sum_t p_t,
// the maximum and the sums running along the keys in f32; a row that sees no key gives 0.
#include "paged_attention.hpp"

#include <algorithm>
#include <climits>

namespace llaisys::kernels {

namespace {

constexpr unsigned kTarget = 512; // chunks over all heads: two blocks on each of 256 compute units

// What the sizes known to the host allow: the requests' lengths are on the device.
struct Plan {
    size_t items;  // of each head, at most
    size_t splits; // partials
    unsigned target;
};
Plan planOf(const PagedAttentionCall &c, size_t tile, size_t most_tiles) {
    const size_t h = c.cache.heads, rows = c.rows * (c.nh / h), requests = std::min(c.rows, c.requests);
    const size_t tiles = std::min(rows / tile + requests, most_tiles);
    const size_t steps = (c.width * c.cache.block + kStep - 1) / kStep;
    Plan p{tiles, 0, 0};
    const size_t per_head = (kTarget + kTarget / 32 + h - 1) / h + 1;
    if (2 * per_head * h <= kPagedCounters && steps > kLeast) {
        // the chunks of all tiles are at most the tiles and all steps over a chunk's, which are kTarget over the heads (3%
        // more, as the sum is rounded); those of split tiles at most twice the latter
        p.target = kTarget;
        p.items = std::min(tiles + per_head, tiles * ((steps + kLeast - 1) / kLeast));
        p.splits = 2 * per_head * h;
    }
    return p;
}

// Tiles of 16 rows for all requests where they have 32 rows or fewer on average (one launch; a longer request
// among them is 16 rows a tile, which is slower for its own rows alone), else two launches, each request by its rows.
bool allFew(const PagedAttentionCall &c) { return c.rows * (c.nh / c.cache.heads) <= kFewMost * c.requests; }
Plan fewPlan(const PagedAttentionCall &c) { return planOf(c, kFewTile, allFew(c) ? SIZE_MAX : kFewMost / kFewTile * c.requests); }
Plan manyPlan(const PagedAttentionCall &c) { return planOf(c, kManyTile, SIZE_MAX); }

size_t bytesOf(const PagedAttentionCall &c, const Plan &p, size_t tile) { return p.splits * tile * (c.cache.dim + 4) * sizeof(float); }

template <typename T>
void launch(PagedAttnArgs a, const PagedAttentionCall &c, bool split, hipStream_t s) {
    const auto with = [&](const Plan &p, int least, int most) {
        a.target = split ? p.target : 0;
        a.per_target = 1.0f / float(kTarget);
        a.few_most = most;
        a.many_least = least;
        return a;
    };
    const Plan few = fewPlan(c);
    if (allFew(c)) return launchPagedFew<T>(with(few, 0, INT_MAX), unsigned(few.items), s);
    const Plan many = manyPlan(c);
    launchPagedMany<T>(with(many, c.requests > 1 ? kFewMost + 1 : 0, INT_MAX), unsigned(many.items), s);
    if (c.requests > 1) launchPagedFew<T>(with(few, 0, kFewMost), unsigned(few.items), s);
}

} // namespace

size_t pagedAttentionWorkspaceBytes(const PagedAttentionCall &c) {
    if (c.rows == 0 || c.requests == 0) return 0;
    const size_t few = bytesOf(c, fewPlan(c), kFewTile);
    return allFew(c) ? few : std::max(few, bytesOf(c, manyPlan(c), kManyTile));
}

void pagedAttentionInt8KV(const PagedAttentionCall &c, void *ws, size_t ws_bytes, hipStream_t s) {
    if (c.rows == 0 || c.requests == 0) return;
    const bool split = ws && ws_bytes >= pagedAttentionWorkspaceBytes(c);
    char *head = static_cast<char *>(ws);
    const PagedAttnArgs a{c.out, c.q, c.cache.k_codes, c.cache.v_codes, c.cache.k_scale, c.cache.v_scale, c.table, c.starts, c.lens,
                          reinterpret_cast<float *>(head + kScratchReserved), reinterpret_cast<unsigned *>(head + kPagedCountersOffset),
                          0, 0.0f, 0, INT_MAX, int64_t(c.rows), int64_t(c.requests), int64_t(c.width),
                          int64_t(c.cache.n_blocks), int(c.nh), int(c.cache.heads), int(c.nh / c.cache.heads), int(c.cache.dim),
                          __builtin_ctzll(c.cache.block), SmallDiv(uint32_t(c.cache.heads)), SmallDiv(uint32_t(c.nh / c.cache.heads)), c.scale, c.err};
    switch (c.dt) {
    case LLAISYS_DTYPE_F32: return launch<F32>(a, c, split, s);
    case LLAISYS_DTYPE_BF16: return launch<BF16>(a, c, split, s);
    case LLAISYS_DTYPE_F16: return launch<F16>(a, c, split, s);
    default: return;
    }
}

} // namespace llaisys::kernels
