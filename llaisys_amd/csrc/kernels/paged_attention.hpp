// Shared by the kernels of the attention over the KV cache in blocks (paged_attention*.hip).
//
// The rows of a request and a kv head are its n tokens times the group = nh / heads q heads that share the
// kv head: row m is token m / group, head m % group of the group.  Requests of few rows are attended in
// tiles of 16 rows (paged_attention_few.hpp), others in tiles of 128 (paged_attention_many.hpp).  A tile attends its
// keys in steps of 64; where the tiles of all requests would leave compute units idle, the keys
// are split into chunks of a whole number of steps, and whoever finishes a tile's last chunk merges them.
//
// Codes meet the matrix instructions as f16: a code is a whole number of magnitude <= 127, exact in f16, for
// every element type of q.  f16 rows of q enter as they are; others are multiplied by a power of two that brings their
// largest element to [2^14, 2^15): bf16 rows then are exact f16 (but for elements below 2^-38 of the row's largest), f32
// rows enter as two f16 parts (22 bits).  Weights p = 2^(t - m) lie in [0, 1], enter times 2^15 (f16's normal range
// then goes down to 2^-29), and in two parts where the rows are f16 or f32; bf16 rows round the result to 8 bits, 11 for
// a weight are enough.  A block's scale of v multiplies the weights as its ratio to the largest seen so
// far, so that nothing leaves f16's range.
#pragma once

#include "common.hpp"
#include "launch.hpp"
#include "quantize.hpp"
#include "rowplan.hpp"

#include <type_traits>

namespace llaisys::kernels {

constexpr int kStep = 64;          // keys of a step
constexpr int kFan = 16;           // chunks, and groups of them, merged at once
constexpr int kPagedThreads = 256; // of a block
constexpr int kFewTile = 16, kManyTile = 128;
// A request goes by 16 rows where it has 32 or fewer, or where rows * q heads of the call times the request's steps are at most
// kFewWork, and the steps allowed so are kFewSteps or more: 128-row tiles then leave most compute units idle.  In us by 16 and
// by 128 rows, 32 / 8 heads of 128, bf16: 1 request of 96 rows over 500 keys before them 14 and 23, of 200 over 500 25 and 24,
// of 512 over 500 33 and 37, over 1500 59 and 48; 4 of 96 over 1500 41 and 47, over 4000 90 and 82.  f32, whose products
// are two or three in either: 1 of 512 over 1500 66 and 82, over 4000 135 and 129; 4 of 512 over 500 119 and 96.
constexpr int kFewRows = 32, kFewSteps = 8;
template <typename T>
constexpr size_t kFewWork = std::is_same_v<T, float> ? 1 << 19 : 1 << 18;
// Steps of a chunk, at least: a 128-row tile's partial is 8 times as large (us of 512 rows after some 1000 keys beside 24 single
// ones: 4 58, 8 52).
constexpr int kFewLeast = 4, kManyLeast = 8;
constexpr int kMostChunks = 256; // of a tile, merged on two levels (131072 keys: 256 22.7 us, 128 25.4)
static_assert(kMostChunks <= kFan * kFan, "two levels");
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kCodeUnit = 0x1p-9f; // a code's f16 value is code * kCodeUnit
constexpr float kWeightBits = 15.0f; // weights are 2^(t - m + kWeightBits)

struct PagedAttnArgs {
    void *out;
    const void *q;
    const int8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    const int32_t *table, *starts, *lens;
    float *part;        // partials of chunks of split tiles
    unsigned *arrived;  // [2][kPagedCounters], 0 between launches
    unsigned target;    // chunks wanted over all requests and heads; 0: no tile is split
    float per_target;   // 1 / target
    int few_rows, few_steps; // a request goes by 16 rows up to so many rows, or steps
    int64_t rows, requests, width, n_blocks;
    int nh, heads, group, dim, shift;
    SmallDiv by_heads, by_group;
    float scale;
    int *err;
};

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// Two codes, given as code + 128 in bytes 0 and 2 of a word, as f16: the bytes are f16 subnormals of 2^-24,
// and one packed fma brings them to code * 2^-9, exactly.
__device__ __forceinline__ v2h codePair(uint32_t bytes) {
    const v2h up{_Float16(0x1p15f), _Float16(0x1p15f)}, bias{_Float16(-0.25f), _Float16(-0.25f)};
    return __builtin_elementwise_fma(__builtin_bit_cast(v2h, bytes), up, bias);
}

struct Pairs {
    v2h p[4];
};
__device__ __forceinline__ v8h join(const Pairs &x) { return __builtin_bit_cast(v8h, x); }

// Eight codes in a row (two words) as f16.
__device__ __forceinline__ v8h codes8(uint32_t lo, uint32_t hi) {
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    return join(Pairs{{codePair(__builtin_amdgcn_perm(lo, lo, 0x0c010c00u)), codePair(__builtin_amdgcn_perm(lo, lo, 0x0c030c02u)),
                       codePair(__builtin_amdgcn_perm(hi, hi, 0x0c010c00u)), codePair(__builtin_amdgcn_perm(hi, hi, 0x0c030c02u))}});
}

// Scales are finite and not negative; another makes NaN of what it scales, and of nothing else.
__device__ __forceinline__ float checkedScale(float s) { return s >= 0.0f && s < INFINITY ? s : __builtin_nanf(""); }

// f32 -> f16, to nearest.
__device__ __forceinline__ v8h narrow8(const float *f) {
    v8h h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = _Float16(f[e]);
    return h;
}
// f in two f16 parts.  The first is made once: where the compiler sees both uses, it rounds a product straight to f16
// for one (v_fma_mixlo) and over f32 for the other, which differ on ties, and the parts then do not add up.
__device__ __forceinline__ void split8(const float *f, v8h &hi, v8h &lo) {
    v4u bits = __builtin_bit_cast(v4u, narrow8(f));
    asm("" : "+v"(bits));
    hi = __builtin_bit_cast(v8h, bits);
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = _Float16(f[e] - float(hi[e]));
}

// Eight elements of a row as loaded, as values, and the largest finite magnitude over some of them.
template <typename T>
struct Raw8 {
    static constexpr int kN = 8 / Fmt<T>::kVec;
    v4u r[kN];
    __device__ __forceinline__ void load(const void *base, size_t elem) {
#pragma unroll
        for (int i = 0; i < kN; ++i) r[i] = load16<T>(base, elem + i * Fmt<T>::kVec);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kN; ++i) r[i] = v4u{0, 0, 0, 0};
    }
    __device__ __forceinline__ void unpack(float *f) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) Fmt<T>::unpack(r[i], f + i * Fmt<T>::kVec);
    }
};
template <typename T, int N>
__device__ __forceinline__ float largest(const Raw8<T> (&x)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
        for (int i = 0; i < Raw8<T>::kN; ++i) m = AbsBits<T>::fold(m, x[s].r[i]);
    m = AbsBits<T>::finish(m);
    if (__builtin_expect(m < AbsBits<T>::kInf, 1)) return AbsBits<T>::value(m);
    float top = 0.0f;
    for (int s = 0; s < N; ++s) {
        float f[8];
        x[s].unpack(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fabsf(f[e]) < INFINITY && fabsf(f[e]) > top ? fabsf(f[e]) : top;
    }
    return top;
}

// Eight outputs, rounded once, to nearest (f16 by the conversion instruction).
template <typename T>
__device__ __forceinline__ void store8(void *base, size_t elem, const float *f) {
    if constexpr (Fmt<T>::kVec == 4) {
        store16<T>(base, elem, Fmt<T>::pack(f));
        store16<T>(base, elem + 4, Fmt<T>::pack(f + 4));
    } else if constexpr (std::is_same_v<T, F16>) {
        store16<T>(base, elem, __builtin_bit_cast(v4u, narrow8(f)));
    } else {
        store16<T>(base, elem, Fmt<T>::packQ(f));
    }
}

template <typename T>
__device__ __forceinline__ void store4(void *base, size_t elem, const float *f) {
    if constexpr (Fmt<T>::kVec == 4) {
        store16<T>(base, elem, Fmt<T>::pack(f));
    } else {
        const float g[8] = {f[0], f[1], f[2], f[3]};
        v4u u;
        if constexpr (std::is_same_v<T, F16>) u = __builtin_bit_cast(v4u, narrow8(g));
        else u = Fmt<T>::packQ(g);
        reinterpret_cast<v2u *>(base)[elem / 4] = v2u{u.x, u.y};
    }
}

// Exponent that brings `top` to [2^14, 2^15).
__device__ __forceinline__ int rowExponent(float top) { return top > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0; }

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// What a block of threads works at: a tile of one request's rows and a chunk of its keys.
struct Item {
    bool any;
    int start;         // first row of the request in q
    int request;
    int n, len;        // rows and cached tokens of the request
    int tile;
    int step0, step1;  // steps of the chunk (not cut to what the tile sees)
    int chunk, chunks; // of the tile
    unsigned split;    // number of the tile's first chunk among those of split tiles, where chunks > 1
};

// A launch's blocks are its items, of each its heads: blocks that run at the same time then read all heads' codes, which
// lie in different channels of the memory, where those of one head lie in some (8 kB in each 64, for 8 heads of 128 in blocks of
// 64), and where the heads are as many as the XCDs each L2 holds one head's.  8419 prompt rows took 304 us the other
// way round and 273 us so when this was chosen.
//
// The item of index `index`: requests in order, of each its tiles, of each its chunks.  Every wave finds it by
// itself: sums over the requests 64 at a time, so that no table of items has to be made before.
template <int kTile>
__device__ __forceinline__ Item findItem(const PagedAttnArgs &a, int index, bool report) {
    const int lane = threadIdx.x % kWave;
    struct Request {
        int start, n, len;
    };
    const auto request = [&](int64_t r, Request &q) { // false: out of range, skipped
        q = Request{0, 0, 0};
        if (r >= a.requests) return true;
        const int s0 = a.starts[r], s1 = a.starts[r + 1], k = a.lens[r];
        if (s0 < 0 || s1 < s0 || s1 > a.rows || k < 0 || k > (a.width << a.shift)) return false;
        const bool few = (s1 - s0) * a.group <= a.few_rows || k <= a.few_steps * kStep;
        if (few == (kTile == kFewTile)) q = Request{s0, s1 - s0, k}; // (else the other launch's)
        return true;
    };
    const auto tilesOf = [&](const Request &q) { return (unsigned(q.n * a.group) + kTile - 1) / kTile; };
    const auto stepsOf = [&](const Request &q) { return (unsigned(q.len) + kStep - 1) / kStep; };
    constexpr unsigned kAll = 0x7FFFFFFFu;
    unsigned per = kAll; // steps of a chunk
    Request q, first;
    bool fine = request(lane, first);
    if (a.target || report) {
        // (in f32: off by less than the 3% that the launch has room for)
        float total = float(tilesOf(first)) * float(stepsOf(first)), most = tilesOf(first) ? float(stepsOf(first)) : 0.0f;
        for (int64_t r0 = kWave; r0 < a.requests; r0 += kWave) {
            fine = request(r0 + lane, q) && fine;
            total += float(tilesOf(q)) * float(stepsOf(q));
            most = fmaxf(most, tilesOf(q) ? float(stepsOf(q)) : 0.0f);
        }
        total = waveGroupReduce<kWave, SumOp>(total);
        most = waveGroupReduce<kWave, MaxOp>(most);
        fine = !__any(!fine);
        if (report && !fine && lane == 0) atomicOr(a.err, kErrPagedIndex);
        // row starts that go back may make more items than the grid has: a tile whose chunks did not all run
        // would leave its counter behind, so nothing is split then
        if (a.target && fine) {
            const float want = ceilf(fmaxf(total * float(a.heads) * a.per_target, most * (1.0f / kMostChunks)));
            per = want < 0x1p30f ? max(unsigned(want), unsigned(kTile == kFewTile ? kFewLeast : kManyLeast)) : kAll;
        }
    }
    per = unsigned(uniform(int(per)));
    int items = 0, splits = 0; // before this group of requests
    for (int64_t r0 = 0; r0 < a.requests; r0 += kWave) {
        if (r0) request(r0 + lane, q);
        else q = first;
        const unsigned tiles = tilesOf(q), steps = stepsOf(q);
        // Chunks of a request have one length.  128-row tiles fill the compute units' places with few blocks, and one too many
        // is a round more: as many as come next to `per` steps.  us: 64 ragged tokens, 16 rows a tile, rounded up 57.3 (with a
        // shorter last chunk 61.5), to the nearest 63.9; 2 chunks of 700 rows after 200, 128 a tile, 53.9 and 37.3.
        unsigned chunks = 1;
        if (__any(steps > per)) chunks = steps > per ? (steps + (kTile == kFewTile ? per - 1 : per / 2)) / per : 1;
        const unsigned part = chunks > 1 ? (steps + chunks - 1) / chunks : kAll;
        const unsigned mine = tiles * chunks, split = chunks > 1 ? mine : 0;
        const unsigned to = waveScan(mine), sto = __any(chunks > 1) ? waveScan(split) : 0;
        const unsigned at = unsigned(index - items); // before the group where it wraps
        const uint64_t hit = __ballot(at >= to - mine && at < to);
        if (hit) {
            const int l = uniform(__ffsll(static_cast<unsigned long long>(hit)) - 1);
            const auto of = [&](unsigned v) { return __builtin_amdgcn_readlane(int(v), l); };
            // one value for the wave in every field: scalar registers, and branches that are no masks
            const int in = uniform(index - items) - of(to - mine), c = of(chunks), t = c == 1 ? in : in / c;
            Item it;
            it.any = true;
            it.request = uniform(int(r0)) + l;
            it.start = of(unsigned(q.start));
            it.n = of(unsigned(q.n));
            it.len = of(unsigned(q.len));
            it.tile = of(tiles) - 1 - t; // the last sees most keys: first
            it.chunk = in - t * c;
            it.chunks = c;
            it.step0 = it.chunk == 0 ? 0 : it.chunk * of(part);
            it.step1 = it.step0 + of(part);
            it.split = unsigned(uniform(splits) + of(sto - split) + t * c);
            return it;
        }
        items += __builtin_amdgcn_readlane(int(to), kWave - 1);
        splits += __builtin_amdgcn_readlane(int(sto), kWave - 1);
    }
    Item none{};
    return none;
}

// Cuts the item to the `steps` its tile sees; false where its chunk has none of them (the tile's first chunk always runs).
__device__ __forceinline__ bool cutItem(Item &it, int steps) {
    if (it.chunks == 1) return true;
    const int per = it.step1 - it.step0;
    it.chunks = steps > per ? (steps + per - 1) / per : 1;
    return it.chunk < it.chunks;
}

// ---- partials: [rows of a tile][dim + 4] f32 ---------------------------------------------------
// 4 or 8 channels at a time; behind them a row's maximum and sum, those of the chunk and those of the group of chunks whose
// merge lies where its first chunk was (each thread overwrites the channels that it alone read).
// They pass between compute units of different L2s, so they are written and read past them (device scope, the
// sc1 bit), 16 bytes a lane, which needs no write-back or invalidation of an L2; a counter of arrivals orders them.

typedef __amdgpu_buffer_rsrc_t Partials;
constexpr int kPastL2 = 16; // cache policy: sc1

__device__ __forceinline__ Partials partialsAt(float *p, size_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(p, 0, int(bytes), 0x00020000); // raw, 32-bit elements, bounds in bytes
}
__device__ __forceinline__ void put4(Partials p, int at, const v4f &v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v), p, at * 4, 0, kPastL2);
}
__device__ __forceinline__ void put2(Partials p, int at, float a, float b) {
    __builtin_amdgcn_raw_buffer_store_b64(v2u{__float_as_uint(a), __float_as_uint(b)}, p, at * 4, 0, kPastL2);
}
__device__ __forceinline__ v2f get2(Partials p, int at) {
    return __builtin_bit_cast(v2f, __builtin_amdgcn_raw_buffer_load_b64(p, at * 4, 0, kPastL2));
}
__device__ __forceinline__ v4f get4(Partials p, int at) {
    return __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(p, at * 4, 0, kPastL2));
}

// After the whole block's partial stores: true for the block that is the last of `count` to come to the counter.
__device__ __forceinline__ bool arriveLast(unsigned *counter, unsigned count, unsigned *shared) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // this wave's partials are where every compute unit sees them
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == count - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *shared = before;
    }
    __syncthreads();
    const bool last = *shared == count - 1;
    __syncthreads();
    return last;
}

// Weight of a state of maximum m in a merge of maximum top (a state without keys has -inf).
__device__ __forceinline__ float mergeWeight(float m, float top) { return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top); }

// Merge of `count` partials (p's, `stride` floats apart), in order: calls done(row, c, o, m, l, W) with W channels from c
// on of each valid row, o not yet divided by l.  `level`: of chunks (0), of groups (1).  Bound by latency: all loads of
// kMany partials are asked for at once.
template <int W, int kMany, typename Done>
__device__ __forceinline__ void mergeBy(Partials p, int stride, int count, int level, int dim, int rows, Done &&done) {
    const int slots = dim / W;
    for (int j = threadIdx.x; j < rows * slots; j += kPagedThreads) {
        const int row = j / slots, c = (j - row * slots) * W, at = row * (dim + 4);
        float m = -INFINITY, l = 0.0f, o[W] = {};
        for (int k0 = 0; k0 < count; k0 += kMany) {
            v2f ml[kMany];
            v4f x[kMany][W / 4];
#pragma unroll
            for (int k = 0; k < kMany; ++k) {
                if (k0 + k >= count) continue;
                const int pk = at + (k0 + k) * stride;
                ml[k] = get2(p, pk + dim + 2 * level);
#pragma unroll
                for (int e = 0; e < W; e += 4) x[k][e / 4] = get4(p, pk + c + e);
            }
#pragma unroll
            for (int k = 0; k < kMany; ++k) {
                if (k0 + k >= count) continue;
                const float mk = ml[k].x, lk = ml[k].y, top = fmaxf(m, mk);
                const float wa = mergeWeight(m, top), wb = mergeWeight(mk, top);
                l = l * wa + lk * wb;
#pragma unroll
                for (int e = 0; e < W; ++e) o[e] = o[e] * wa + x[k][e / 4][e % 4] * wb;
                m = top;
            }
        }
        done(row, c, o, m, l, std::integral_constant<int, W>());
    }
}

// Tiles of 16 rows merge more than 8 partials by 16, of 4 channels a thread: of 8 the registers do not hold 16 at three blocks a
// compute unit (92 bytes a thread spilled: a row over 131072 keys takes 2 us more).  Tiles of 128 are seldom cut into many.
template <int kTile, typename Done>
__device__ __forceinline__ void mergePartials(Partials p, int stride, int count, int level, int dim, int rows, Done &&done) {
    if constexpr (kTile == kFewTile) {
        if (count > 8) return mergeBy<4, 16>(p, stride, count, level, dim, rows, done);
    }
    mergeBy<8, 8>(p, stride, count, level, dim, rows, done);
}

// Ends an item: `state(row, c, o, m, l)` gives 8 channels of the block's own result, `place(row)` the row's first element in the output.  One chunk: the outputs.  Several: the
// partial, and for the last of kFan chunks, and of those the last, the merge.
template <typename T, int kTile, typename Place, typename State>
__device__ __forceinline__ void finishItem(const PagedAttnArgs &a, const Item &it, int head, int rows, int dim, unsigned *shared,
                                           Place &&place, State &&state) {
    const int slots = dim / 8;
    const auto put = [&](int row, int c, const float *o, float, float l, auto w) {
        constexpr int W = decltype(w)::value;
        const size_t at = place(row) + c;
        const float d = l == 0.0f ? 0.0f : 1.0f / l; // no key: 0
        float f[W];
#pragma unroll
        for (int e = 0; e < W; ++e) f[e] = o[e] * d;
        if constexpr (W == 8) store8<T>(a.out, at, f);
        else store4<T>(a.out, at, f);
    };
    const auto all = [&](auto &&done) {
        for (int j = threadIdx.x; j < rows * slots; j += kPagedThreads) {
            const int row = j / slots, c = (j - row * slots) * 8;
            float o[8], m, l;
            state(row, c, o, m, l);
            done(row, c, o, m, l, std::integral_constant<int, 8>());
        }
    };
    if (it.chunks == 1) {
        all(put);
        return;
    }
    const int size = kTile * (dim + 4), stride = size * a.heads;
    // of the tile's chunks from one of them on, of a group's at the least
    const auto partials = [&](int chunk, int count) {
        return partialsAt(a.part + (size_t(it.split + unsigned(chunk)) * a.heads + head) * size, (size_t(count - 1) * stride + size) * sizeof(float));
    };
    const auto keep = [&](Partials p, int level) {
        return [&, p, level](int row, int c, const float *o, float m, float l, auto w) {
            const int at = row * (dim + 4);
#pragma unroll
            for (int e = 0; e < decltype(w)::value; e += 4) put4(p, at + c + e, v4f{o[e], o[e + 1], o[e + 2], o[e + 3]});
            if (c == 0) put2(p, at + dim + 2 * level, m, l);
        };
    };
    all(keep(partials(it.chunk, 1), 0));
    const auto counter = [&](int level, int chunk) {
        return a.arrived + size_t(level) * kPagedCounters + size_t(it.split + unsigned(chunk)) * a.heads + head;
    };
    const int group0 = it.chunk / kFan * kFan, in_group = min(kFan, it.chunks - group0);
    if (!arriveLast(counter(0, group0), unsigned(in_group), shared)) return;
    if (it.chunks <= kFan) {
        mergePartials<kTile>(partials(group0, in_group), stride, in_group, 0, dim, rows, put);
        return;
    }
    const int groups = (it.chunks + kFan - 1) / kFan;
    mergePartials<kTile>(partials(group0, in_group), stride, in_group, 0, dim, rows, keep(partials(group0, 1), 1));
    if (!arriveLast(counter(1, 0), unsigned(groups), shared)) return;
    mergePartials<kTile>(partials(0, (groups - 1) * kFan + 1), stride * kFan, groups, 1, dim, rows, put);
}

template <typename T>
void launchPagedFew(const PagedAttnArgs &a, unsigned items, hipStream_t s);
template <typename T>
void launchPagedMany(const PagedAttnArgs &a, unsigned items, hipStream_t s);

} // namespace llaisys::kernels
