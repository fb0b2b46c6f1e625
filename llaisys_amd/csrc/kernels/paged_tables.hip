// Block tables, slots, positions and row starts of a step, from the requests' lengths.
//
// With nb(x) = ceil(x / block), request r going from old to new tokens takes blocks nb(old) ..
// nb(new) - 1 of its table row from a ring of free block ids when it grows, and gives blocks nb(new) ..
// nb(old) - 1 back when it shrinks.  Both are exclusive sums over the requests: the i-th block taken is
// ring[(head + i) % F], the i-th given back goes to ring[(tail + i) % F].  Row t of the step (request r,
// starts[r] <= t < starts[r + 1]) is token pos = old[r] + t - starts[r], in slot
// table[r][pos / block] * block + pos % block.
//
// One block scans the requests (pagedPlan); it refuses the whole step before it writes anything.  A row
// at offset 0 of a table block is the first of a block just taken, so the rows' threads write the table.
#include "common.hpp"
#include "launch.hpp"
#include "rowplan.hpp"

namespace llaisys::kernels {

namespace {

constexpr int kPlanThreads = 1024;

struct TablesArgs {
    int32_t *table;
    int64_t *slots, *pos;
    int32_t *starts;
    int64_t *free_out;
    const int32_t *old_lens, *new_lens;
    int32_t *ring;
    const int64_t *free_in;
    int64_t requests, width, rows, ring_size;
    int shift; // log2(block)
    int64_t *taken; // scratch: [requests] sums of blocks taken, then the head before the step
    int *err;
};

struct Sums {
    int64_t rows, more, back;
};

__device__ __forceinline__ int64_t blocksOf(int64_t n, int shift) { return (n + (int64_t(1) << shift) - 1) >> shift; }

__device__ __forceinline__ Sums sumsOf(const TablesArgs &a, int64_t r, bool &ok) {
    Sums s{0, 0, 0};
    if (r >= a.requests) return s;
    const int64_t o = a.old_lens[r], n = a.new_lens[r], most = a.width << a.shift;
    ok = ok && o >= 0 && n >= 0 && o <= most && n <= most;
    const int64_t bo = blocksOf(o, a.shift), bn = blocksOf(n, a.shift);
    s.rows = n > o ? n - o : 0;
    s.more = bn > bo ? bn - bo : 0;
    s.back = bo > bn ? bo - bn : 0;
    return s;
}

__device__ __forceinline__ int64_t shflUp(int64_t v, int d) {
    const int lo = __shfl_up(int(uint32_t(uint64_t(v))), d, kWave), hi = __shfl_up(int(v >> 32), d, kWave);
    return int64_t((uint64_t(uint32_t(hi)) << 32) | uint32_t(lo));
}

// Exclusive sums over the block's threads; `total` the sums of all.
__device__ Sums blockScan(Sums v, Sums &total, Sums *red) {
    Sums in = v;
    for (int d = 1; d < kWave; d <<= 1) {
        const Sums up{shflUp(in.rows, d), shflUp(in.more, d), shflUp(in.back, d)};
        if (int(threadIdx.x % kWave) >= d) in = Sums{in.rows + up.rows, in.more + up.more, in.back + up.back};
    }
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == kWave - 1) red[wave] = in;
    __syncthreads();
    Sums before{0, 0, 0};
    total = Sums{0, 0, 0};
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
        if (w == wave) before = total;
        total = Sums{total.rows + red[w].rows, total.more + red[w].more, total.back + red[w].back};
    }
    return Sums{before.rows + in.rows - v.rows, before.more + in.more - v.more, before.back + in.back - v.back};
}

__global__ __launch_bounds__(kPlanThreads) void pagedPlan(TablesArgs a) {
    __shared__ Sums red[kPlanThreads / kWave];
    const int64_t head = a.free_in[0], tail = a.free_in[1], f = a.ring_size;
    // the totals first: a step that cannot be done changes nothing
    bool ok = head >= 0 && tail >= head && tail - head <= f && tail <= INT64_MAX / 2;
    Sums all{0, 0, 0};
    for (int64_t r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
        Sums total;
        blockScan(sumsOf(a, r0 + threadIdx.x, ok), total, red);
        all = Sums{all.rows + total.rows, all.more + total.more, all.back + total.back};
    }
    ok = ok && all.rows <= a.rows && tail + all.back - head <= f && all.more <= tail - head + all.back;
    ok = __syncthreads_and(ok);
    if (!ok) {
        for (int64_t r = threadIdx.x; r <= a.requests; r += kPlanThreads) a.starts[r] = 0;
        if (threadIdx.x == 0) {
            a.free_out[0] = head;
            a.free_out[1] = tail;
            atomicOr(a.err, kErrPagedTables);
        }
        return;
    }
    Sums carry{0, 0, 0};
    for (int64_t r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
        const int64_t r = r0 + threadIdx.x;
        Sums total;
        const Sums mine = sumsOf(a, r, ok);
        Sums at = blockScan(mine, total, red);
        at = Sums{carry.rows + at.rows, carry.more + at.more, carry.back + at.back};
        if (r < a.requests) {
            a.starts[r] = int32_t(at.rows);
            a.taken[r] = at.more;
        }
        // blocks given back: a wave copies one request's at a time
        for (uint64_t left = __ballot(mine.back > 0); left; left &= left - 1) {
            const int l = __ffsll(static_cast<unsigned long long>(left)) - 1;
            const int64_t n = __shfl(int(mine.back), l, kWave);
            const int64_t to = (int64_t(__shfl(int(at.back >> 32), l, kWave)) << 32) |
                               uint32_t(__shfl(int(uint32_t(at.back)), l, kWave));
            const int64_t q = r - int64_t(threadIdx.x % kWave) + l;
            const int64_t first = blocksOf(a.new_lens[q], a.shift);
            for (int64_t i = threadIdx.x % kWave; i < n; i += kWave)
                a.ring[(tail + to + i) % f] = a.table[q * a.width + first + i];
        }
        carry = Sums{carry.rows + total.rows, carry.more + total.more, carry.back + total.back};
    }
    if (threadIdx.x == 0) {
        a.starts[a.requests] = int32_t(carry.rows);
        a.taken[a.requests] = head;
        a.free_out[0] = head + carry.more;
        a.free_out[1] = tail + carry.back;
    }
}

__global__ __launch_bounds__(256) void pagedRows(TablesArgs a) {
    const int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (t >= a.rows) return;
    if (t >= a.starts[a.requests]) {
        a.slots[t] = -1;
        a.pos[t] = 0;
        return;
    }
    int64_t lo = 0, hi = a.requests; // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        (a.starts[mid] <= t ? lo : hi) = mid;
    }
    const int64_t o = a.old_lens[lo], p = o + t - a.starts[lo], b = p >> a.shift, off = p & ((int64_t(1) << a.shift) - 1);
    const int64_t bo = blocksOf(o, a.shift);
    int32_t id;
    if (b < bo) {
        id = a.table[lo * a.width + b];
    } else {
        id = a.ring[(a.taken[a.requests] + a.taken[lo] + b - bo) % a.ring_size];
        if (off == 0) a.table[lo * a.width + b] = id;
    }
    if (id < 0) atomicOr(a.err, kErrPagedIndex); // no block: the row is skipped, and said
    a.slots[t] = id < 0 ? -1 : (int64_t(id) << a.shift) + off;
    a.pos[t] = p;
}

} // namespace

size_t pagedTablesWorkspaceBytes(const PagedTablesCall &c) { return (c.requests + 1) * sizeof(int64_t); }

void pagedTables(const PagedTablesCall &c, void *ws, hipStream_t s) {
    const TablesArgs a{c.table, c.slots, c.pos, c.starts, c.free_out, c.old_lens, c.new_lens, c.ring, c.free_in,
                       int64_t(c.requests), int64_t(c.width), int64_t(c.rows), int64_t(c.ring_size),
                       __builtin_ctzll(c.block), static_cast<int64_t *>(ws), c.err};
    pagedPlan<<<1, kPlanThreads, 0, s>>>(a);
    if (c.rows) pagedRows<<<unsigned((c.rows + 255) / 256), 256, 0, s>>>(a);
}

} // namespace llaisys::kernels
