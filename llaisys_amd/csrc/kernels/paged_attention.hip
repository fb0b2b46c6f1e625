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

// Chunks over all heads (us of 64 ragged tokens and of one over 131072 keys, tiles of 16: 512 60.3 and 29.3, 768 60.2 and 32.2,
// 1024 57.8 and 40.9, when chunks had no other bound; a chunk of 512 tokens beside 24 of one: 512 56, 1024 60).
constexpr unsigned kTarget = 512;

// What the sizes known to the host allow: the requests' lengths are on the device.
struct Plan {
    size_t items;  // of each head, at most
    size_t splits; // partials
    unsigned target;
};
size_t stepsOf(const PagedAttentionCall &c) { return (c.width * c.cache.block + kStep - 1) / kStep; }
Plan planOf(const PagedAttentionCall &c, size_t tile, size_t least, size_t most_tiles) {
    const size_t h = c.cache.heads, rows = c.rows * (c.nh / h), requests = std::min(c.rows, c.requests);
    const size_t tiles = std::min(rows / tile + requests, most_tiles), steps = stepsOf(c);
    Plan p{tiles, 0, 0};
    const size_t per_head = (kTarget + kTarget / 32 + h - 1) / h + 1;
    if (2 * per_head * h <= kPagedCounters && steps > least) {
        // the chunks of all tiles are at most the tiles and all steps over a chunk's, which are kTarget over the heads (3%
        // more, as the sum is rounded); those of split tiles at most twice the latter
        p.target = kTarget;
        p.items = std::min(tiles + per_head, tiles * ((steps + least - 1) / least));
        p.splits = 2 * per_head * h;
    }
    return p;
}

// Steps up to which a request of any number of rows goes by 16 of them, or -1.
int fewSteps(const PagedAttentionCall &c) {
    const size_t work = c.dt == LLAISYS_DTYPE_F32 ? kFewWork<float> : kFewWork<BF16>, steps = work / std::max(c.rows * c.nh, size_t(1));
    return steps < size_t(kFewSteps) ? -1 : int(std::min(steps, size_t(INT_MAX / kStep)));
}
// One launch, 16 rows a tile, where the requests have 32 rows or fewer on average (a longer one among them is then
// attended so too, which is slower for its own rows alone) or the table holds no more steps than go so.  Else
// two launches, each request by its rows and steps.
bool allFew(const PagedAttentionCall &c) {
    return c.rows * (c.nh / c.cache.heads) <= kFewRows * c.requests || (fewSteps(c) > 0 && stepsOf(c) <= size_t(fewSteps(c)));
}
Plan fewPlan(const PagedAttentionCall &c) {
    return planOf(c, kFewTile, kFewLeast, allFew(c) || fewSteps(c) > 0 ? SIZE_MAX : kFewRows / kFewTile * c.requests);
}
Plan manyPlan(const PagedAttentionCall &c) { return planOf(c, kManyTile, kManyLeast, SIZE_MAX); }

size_t bytesOf(const PagedAttentionCall &c, const Plan &p, size_t tile) { return p.splits * tile * (c.cache.dim + 4) * sizeof(float); }

template <typename T>
void launch(PagedAttnArgs a, const PagedAttentionCall &c, bool split, hipStream_t s) {
    a.per_target = 1.0f / float(kTarget);
    const bool all = allFew(c);
    a.few_rows = all ? INT_MAX : kFewRows;
    a.few_steps = fewSteps(c);
    const bool one = c.requests == 1 && a.few_steps < 0; // (of any number of rows: others may stand behind them)
    if (!all && one) a.few_rows = 0;
    if (!all) {
        const Plan many = manyPlan(c);
        a.target = split ? many.target : 0;
        launchPagedMany<T>(a, unsigned(many.items), s);
        if (one) return;
    }
    const Plan few = fewPlan(c);
    a.target = split ? few.target : 0;
    launchPagedFew<T>(a, unsigned(few.items), s);
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
                          0, 0.0f, 0, 0, int64_t(c.rows), int64_t(c.requests), int64_t(c.width),
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
