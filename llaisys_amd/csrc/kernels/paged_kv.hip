// Writes and read-back of the KV cache in blocks: codes [n_blocks, heads, block, dim] I8 with one F32
// scale for each (block, head).
//
// Append.  The rows of a step that go to one block are consecutive rows of consecutive slots.  With A the
// largest |x| of those rows for a head, s0 the head's scale (0 where the rows begin at offset 0: the block
// is new) and s = max(s0, A / 127), a new code is the whole number next to x / s, and where s grew the
// codes before the rows become the whole numbers next to code * s0 / s.  A block's scale so only grows
// while it fills; each growth rounds its older codes once more, by at most s / 2.
//
// Quotients are rounded as the exact quotient rounds (ties to even), so that one definition holds for any
// way of computing it: with n the whole number next to x * (1 / s), off by at most one, e = fma(-n, s, x) is
// exact (x and n * s agree in all but the last bits), and n is right wherever |e| < s / 2; else (1 in 10^5) it moves by
// one, or is a tie.  Scales below 2^-96, where 1 / s or e may leave the normal range, divide in f64, which tells any
// quotient from a half.
//
// A group of 256 threads takes `chunk` rows of one head of k or v.  Its slots come in one load of 64, in which every
// wave finds the rows where cache blocks begin and how far they go; rows stay in registers between the maximum and
// the codes.  The heads of a chunk, k and v, are next to each other in the grid: they read whole rows of the memory then
// (one head's pieces, a row's length apart, lie in few of its channels).  [7598 x 8 heads x 128] bf16, k and v (47 MB): 18 us
// (2.6 TB/s; the loads, the block's maximum and the codes of a group follow one another), the read-back 9.4 us (5 TB/s).  One row of
// each of 64 requests: 3.8 and 3.0 us, latency.
#include "common.hpp"
#include "launch.hpp"
#include "quantize.hpp"
#include "rowplan.hpp"

#include <algorithm>

namespace llaisys::kernels {

namespace {

constexpr int kThreads = 256;
constexpr size_t kChunksY = 32768;

struct AppendArgs {
    int8_t *codes[2];
    float *scale[2];
    const void *in[2];
    const int64_t *slots;
    int64_t rows, slot_end;
    int heads, dim, shift, chunk;
    SmallDiv by_vectors; // of a row
    int *err;
};

__device__ __forceinline__ uint32_t codeExact(double x, double s) {
    double n = rint(x / s);
    if (n != n) return 0; // NaN quotient
    n = n > 127.0 ? 127.0 : (n < -127.0 ? -127.0 : n);
    return uint32_t(int32_t(n)) & 0xFFu;
}

// Codes of one 16-byte vector; s is the block's scale, recip 1 / s.
template <typename T>
__device__ __forceinline__ void storeVec(int8_t *to, const v4u &r, float s, float recip) {
    constexpr int N = Fmt<T>::kVec;
    constexpr float kWhole = 12582912.0f; // 1.5 * 2^23: a sum with it rounds to a whole number, in its low bits
    float f[N];
    Fmt<T>::unpack(r, f);
    uint32_t c[N], w[N / 4];
    const float half = 0.5f * s;
    bool near = true;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float m = __builtin_fmaf(f[e], recip, kWhole), rest = __builtin_fmaf(kWhole - m, s, f[e]);
        near = near && fabsf(rest) < half;
        c[e] = __float_as_uint(m);
    }
    if (__builtin_expect(!near, 0)) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float m = __builtin_fmaf(f[e], recip, kWhole), rest = __builtin_fmaf(kWhole - m, s, f[e]);
            const bool odd = (c[e] & 1u) != 0;
            c[e] += rest > half || (rest == half && odd) ? 1u : 0u;
            c[e] -= rest < -half || (rest == -half && odd) ? 1u : 0u;
            c[e] = f[e] == f[e] ? c[e] : 0u; // NaN
        }
    }
#pragma unroll
    for (int e = 0; e < N / 4; ++e) w[e] = packCodes4(c + 4 * e);
    __builtin_memcpy(__builtin_assume_aligned(to, N), w, N);
}

// Sixteen older codes at s0 as codes at s (in the range of the f32 rule).  c * (s0 / s) in f32 is off by less than 2^-15: only
// next to a half is it not enough, and c * s0, as a product and its rest, tells there: differences of values that are nearly
// equal are exact.
__device__ __forceinline__ void rescale16(int8_t *codes, float s0, float s, float ratio) {
    const v4u r = *reinterpret_cast<const v4u *>(codes);
    const uint32_t old[4] = {r.x, r.y, r.z, r.w};
    uint32_t w[4];
    const float half = 0.5f * s;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t c[4];
        bool near = true;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float t = float(int32_t(old[e] << (24 - 8 * b)) >> 24) * ratio, n = rintf(t);
            near = near && fabsf(t - n) < 0.49996f;
            c[b] = uint32_t(int32_t(n));
        }
        if (__builtin_expect(!near, 0)) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float x = float(int32_t(old[e] << (24 - 8 * b)) >> 24), p = x * s0, more = __builtin_fmaf(x, s0, -p);
                const float rest = __builtin_fmaf(-float(int32_t(c[b])), s, p);
                const float up = (rest - half) + more, down = (rest + half) + more;
                const bool odd = (c[b] & 1u) != 0;
                c[b] += up > 0.0f || (up == 0.0f && odd) ? 1u : 0u;
                c[b] -= down < 0.0f || (down == 0.0f && odd) ? 1u : 0u;
            }
        }
        w[e] = packCodes4(c);
    }
    *reinterpret_cast<v4u *>(codes) = v4u{w[0], w[1], w[2], w[3]};
}

template <typename T>
__global__ __launch_bounds__(kThreads, 4) void pagedAppend(AppendArgs a) {
    constexpr int N = Fmt<T>::kVec;
    constexpr int kKeep = 4; // vectors a thread keeps between the maximum and the codes
    __shared__ float red[kThreads / kWave];
    const int head = blockIdx.x / 2, kv = blockIdx.x % 2, lane = threadIdx.x % kWave;
    const int nv = a.dim / N, block = 1 << a.shift;
    // slots t0 - 1 .. t0 + 62; the rows of lanes 1 .. chunk are this group's
    const int64_t t0 = (int64_t(blockIdx.z) * kChunksY + blockIdx.y) * a.chunk;
    const auto slotAt = [&](int64_t t) { return t >= 0 && t < a.rows ? a.slots[t] : int64_t(-1); };
    const int64_t mine = slotAt(t0 - 1 + lane);
    const bool ours = lane >= 1 && lane <= a.chunk;
    if (ours && mine >= a.slot_end) atomicOr(a.err, kErrPagedIndex);
    const int64_t my_block = mine < 0 ? -1 : mine >> a.shift;
    const auto pick = [](int64_t v, int l) {
        return int64_t((uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), l))) << 32) | uint32_t(__builtin_amdgcn_readlane(int(v), l)));
    };
    const int64_t before = (int64_t(__shfl_up(int(my_block >> 32), 1, kWave)) << 32) | uint32_t(__shfl_up(int(my_block), 1, kWave));
    for (uint64_t firsts = __ballot(ours && mine >= 0 && mine < a.slot_end && my_block != before); firsts; firsts &= firsts - 1) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(firsts)) - 1);
        const int64_t t = t0 - 1 + l, slot = pick(mine, l), id = slot >> a.shift;
        const int first = int(slot & (block - 1));
        // the run of rows of this block; rows that do not follow each other are refused
        int run = 0;
        bool refuse = false;
        int64_t window = mine;
        for (int at = l;; at -= kWave) { // `at`: lane of row t in the window
            const int i = lane - at;     // rows behind t
            const bool ends = i >= 1 && (first + i >= block || window != slot + i);
            const uint64_t m = __ballot(ends);
            if (m) {
                const int stop = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(m)) - 1);
                const int64_t other = pick(window, stop);
                run = stop - at;
                refuse = other >= 0 && (other >> a.shift) == id;
                break;
            }
            window = slotAt(t + (kWave - at) + lane);
        }
        if (refuse) {
            if (threadIdx.x == 0) atomicOr(a.err, kErrPagedIndex);
            continue;
        }
        const int n = run * nv;
        const size_t from = (size_t(t) * a.heads + head) * a.dim;
        const char *in = static_cast<const char *>(a.in[kv]) + from * Fmt<T>::kBytes;
        const unsigned row_elems = unsigned(a.heads) * unsigned(a.dim);
        const auto at = [&](int j) {
            const int row = a.by_vectors.div(j);
            return size_t(unsigned(row)) * row_elems + unsigned(j - row * nv) * N;
        };
        const size_t tile = size_t(id) * a.heads + head;
        const float s0 = first ? a.scale[kv][tile] : 0.0f;
        v4u keep[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const int j = threadIdx.x + i * kThreads;
            keep[i] = j < n ? load16Stream<T>(in, at(j)) : v4u{0, 0, 0, 0};
        }
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < kKeep; ++i) bits = AbsBits<T>::fold(bits, keep[i]);
        for (int j = threadIdx.x + kKeep * kThreads; j < n; j += kThreads) bits = AbsBits<T>::fold(bits, load16<T>(in, at(j)));
        bits = AbsBits<T>::finish(bits);
        float amax = AbsBits<T>::value(bits);
        if (__builtin_expect(bits > AbsBits<T>::kInf, 0)) { // a NaN, which never raises the maximum
            amax = 0.0f;
            for (int j = threadIdx.x; j < n; j += kThreads) {
                float f[N];
                Fmt<T>::unpack(load16<T>(in, at(j)), f);
#pragma unroll
                for (int e = 0; e < N; ++e) amax = MaxOp::apply(amax, fabsf(f[e]));
            }
        }
        amax = groupReduce<kThreads, MaxOp>(amax, red);
        const float grown = amax / 127.0f, s = grown > s0 ? grown : s0;
        int8_t *codes = a.codes[kv] + (tile << a.shift) * a.dim;
        if (threadIdx.x == 0 && (s != s0 || first == 0)) a.scale[kv][tile] = s;
        const bool in_f32 = s >= 0x1p-96f && s <= 0x1p120f;
        if (first && s != s0) {
            if (__builtin_expect(in_f32, 1)) {
                const float ratio = s0 / s;
                for (int j = threadIdx.x; j < first * (a.dim / 16); j += kThreads) rescale16(codes + j * 16, s0, s, ratio);
            } else {
#pragma unroll 1
                for (int j = threadIdx.x; j < first * a.dim; j += kThreads)
                    codes[j] = int8_t(codeExact(double(codes[j]) * double(s0), double(s)));
            }
        }
        int8_t *const to = codes + first * a.dim;
        if (__builtin_expect(in_f32, 1)) {
            const float recip = 1.0f / s;
#pragma unroll
            for (int i = 0; i < kKeep; ++i) {
                const int j = threadIdx.x + i * kThreads;
                if (j < n) storeVec<T>(to + j * N, keep[i], s, recip);
                __builtin_amdgcn_sched_barrier(0); // one vector's values in registers at a time
            }
            for (int j = threadIdx.x + kKeep * kThreads; j < n; j += kThreads)
                storeVec<T>(to + j * N, load16<T>(in, at(j)), s, recip);
        } else {
            for (int j = threadIdx.x; j < n; j += kThreads) {
                const size_t first_elem = at(j);
#pragma unroll 1
                for (int e = 0; e < N; ++e) to[j * N + e] = int8_t(codeExact(double(Fmt<T>::get(in, first_elem + e)), double(s)));
            }
        }
    }
}

struct ReadArgs {
    void *out[2];
    const int8_t *codes[2];
    const float *scale[2];
    const int64_t *slots;
    int64_t n, slot_end; // 8-code vectors of k or v
    DivU64 per_row, per_head;
    int heads, dim, shift;
    int *err;
};

// f16 rounds to nearest even (the conversion instruction), bf16 likewise, f32 is the product.
template <typename T>
__device__ __forceinline__ void storeRounded(void *out, size_t elem, const float *f) {
    if constexpr (Fmt<T>::kVec == 4) {
        store16Stream<T>(out, elem, Fmt<T>::pack(f));
        store16Stream<T>(out, elem + 4, Fmt<T>::pack(f + 4));
    } else if constexpr (std::is_same_v<T, F16>) {
        typedef _Float16 v8h __attribute__((ext_vector_type(8)));
        v8h h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = _Float16(f[e]);
        store16Stream<T>(out, elem, __builtin_bit_cast(v4u, h));
    } else {
        store16Stream<T>(out, elem, Fmt<T>::packQ(f));
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pagedRead(ReadArgs a) {
    const int kv = blockIdx.y;
    for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < a.n; i += int64_t(gridDim.x) * kThreads) {
        const int64_t t = int64_t(a.per_row.div(uint64_t(i)));
        const int in_row = int(i - t * (int64_t(a.heads) * (a.dim / 8)));
        const int64_t slot = a.slots[t];
        if (slot < 0) continue;
        if (slot >= a.slot_end) {
            atomicOr(a.err, kErrPagedIndex);
            continue;
        }
        const int head = int(a.per_head.div(uint64_t(in_row))), c = (in_row - head * (a.dim / 8)) * 8;
        const int64_t tile = (slot >> a.shift) * a.heads + head;
        const int8_t *from = a.codes[kv] + ((tile << a.shift) + (slot & ((1 << a.shift) - 1))) * a.dim + c;
        uint32_t w[2];
        __builtin_memcpy(w, __builtin_assume_aligned(from, 8), 8);
        const float s = a.scale[kv][tile];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = float(int32_t(w[e / 4] << (24 - 8 * (e % 4))) >> 24) * s;
        storeRounded<T>(a.out[kv], size_t(i) * 8, f);
    }
}

} // namespace

void pagedKvAppendInt8(const PagedCache &c, const void *k, const void *v, const int64_t *slots, size_t rows,
                       llaisysDataType_t dt, int *err, hipStream_t s) {
    if (rows == 0 || c.heads == 0 || c.dim == 0) return;
    // Few rows: a group of threads each, so that a step of one token per request runs in one round.  Many: up to 32 rows
    // a group (of a prompt, one or two cache blocks begin there).
    const int chunk = rows * c.heads * 2 <= 16384 ? 1 : int(c.block < 32 ? c.block : 32);
    const AppendArgs a{{c.k_codes, c.v_codes}, {c.k_scale, c.v_scale}, {k, v}, slots, int64_t(rows),
                       int64_t(c.n_blocks * c.block), int(c.heads), int(c.dim), __builtin_ctzll(c.block), chunk, SmallDiv(uint32_t(c.dim / (dt == LLAISYS_DTYPE_F32 ? 4 : 8))), err};
    const size_t chunks = (rows + chunk - 1) / chunk;
    const dim3 grid(unsigned(2 * c.heads), unsigned(std::min(chunks, kChunksY)), unsigned((chunks + kChunksY - 1) / kChunksY));
    switch (dt) {
    case LLAISYS_DTYPE_F32: pagedAppend<F32><<<grid, kThreads, 0, s>>>(a); return;
    case LLAISYS_DTYPE_BF16: pagedAppend<BF16><<<grid, kThreads, 0, s>>>(a); return;
    case LLAISYS_DTYPE_F16: pagedAppend<F16><<<grid, kThreads, 0, s>>>(a); return;
    default: return;
    }
}

void pagedKvReadInt8(void *k, void *v, const PagedCache &c, const int64_t *slots, size_t rows, llaisysDataType_t dt,
                     int *err, hipStream_t s) {
    const size_t per_row = c.heads * (c.dim / 8), n = rows * per_row;
    if (n == 0) return;
    const ReadArgs a{{k, v}, {c.k_codes, c.v_codes}, {c.k_scale, c.v_scale}, slots, int64_t(n),
                     int64_t(c.n_blocks * c.block), DivU64(per_row), DivU64(c.dim / 8), int(c.heads), int(c.dim),
                     __builtin_ctzll(c.block), err};
    const size_t blocks = (n + kThreads - 1) / kThreads;
    const dim3 grid(unsigned(std::min(blocks, size_t(1) << 22)), 2);
    switch (dt) {
    case LLAISYS_DTYPE_F32: pagedRead<F32><<<grid, kThreads, 0, s>>>(a); return;
    case LLAISYS_DTYPE_BF16: pagedRead<BF16><<<grid, kThreads, 0, s>>>(a); return;
    case LLAISYS_DTYPE_F16: pagedRead<F16><<<grid, kThreads, 0, s>>>(a); return;
    default: return;
    }
}

} // namespace llaisys::kernels
