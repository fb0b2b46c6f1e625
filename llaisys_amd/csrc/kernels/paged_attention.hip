// Causal GQA attention of many requests over the INT8 KV cache in blocks.
//
// Row i of request r's n rows sees its cached tokens t <= lens[r] - n + i:
//   s_t = scale * k_scale[block(t)] * (q . k_codes[t]),  p_t = exp(s_t - m),  m = max s,
//   out = sum_t p_t * v_scale[block(t)] * v_codes[t] / sum_t p_t,
// the maximum and the sums running along the keys in f32; a row that sees no key gives 0.
#include "common.hpp"
#include "launch.hpp"

namespace llaisys::kernels {

namespace {

struct AttnArgs {
    void *out;
    const void *q;
    const int8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    const int32_t *table, *starts, *lens;
    int64_t rows, requests, width, n_blocks;
    int nh, heads, dim, shift;
    float scale;
    int *err;
};

// One wave: one row of one q head, 64 keys a step, a key per lane for the scores and channels per lane for
// the values.
template <typename T>
__global__ __launch_bounds__(kWave) void pagedAttnRow(AttnArgs a) {
    __shared__ float q[256];
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, lane = threadIdx.x, kvh = h / (a.nh / a.heads);
    int64_t lo = 0, hi = a.requests;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        (a.starts[mid] <= t ? lo : hi) = mid;
    }
    const int64_t s0 = a.starts[lo], s1 = a.starts[lo + 1], len = a.lens[lo];
    if (t < s0 || t >= s1) return;
    if (s0 < 0 || s1 > a.rows || len < 0 || len > (a.width << a.shift)) {
        if (lane == 0) atomicOr(a.err, kErrPagedIndex);
        return;
    }
    const size_t row = (size_t(t) * a.nh + h) * a.dim;
    for (int c = lane; c < a.dim; c += kWave) q[c] = Fmt<T>::get(a.q, row + c) * a.scale;
    __syncthreads();
    const int64_t keys = len - (s1 - t) + 1; // visible
    float m = -INFINITY, l = 0.0f, acc[4] = {};
    for (int64_t k0 = 0; k0 < keys; k0 += kWave) {
        const int64_t k = k0 + lane;
        int64_t id = k < keys ? a.table[lo * a.width + (k >> a.shift)] : -1;
        if (k < keys && (id < 0 || id >= a.n_blocks)) {
            atomicOr(a.err, kErrPagedIndex);
            id = -1;
        }
        float s = -INFINITY, vs = 0.0f;
        int64_t at = 0;
        if (id >= 0) {
            const int64_t tile = id * a.heads + kvh;
            at = ((tile << a.shift) + (k & ((1 << a.shift) - 1))) * a.dim;
            float dot = 0.0f;
            for (int c = 0; c < a.dim; c += 16) {
                const v4u r = *reinterpret_cast<const v4u *>(a.k_codes + at + c);
                const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    dot = __builtin_fmaf(float(int32_t(w[e / 4] << (24 - 8 * (e % 4))) >> 24), q[c + e], dot);
            }
            s = dot * a.k_scale[tile];
            vs = a.v_scale[tile];
        }
        const float top = fmaxf(m, waveGroupReduce<kWave, MaxOp>(s));
        const float p = id >= 0 ? (s == s ? __expf(s - top) : s) : 0.0f;
        const float keep = m == -INFINITY ? 0.0f : __expf(m - top);
        m = top;
        l = l * keep + waveGroupReduce<kWave, SumOp>(p);
        const float w = id >= 0 ? p * vs : 0.0f;
        for (int c = 0; c < 4; ++c) acc[c] *= keep;
        for (int j = 0; j < kWave; ++j) {
            const float wj = __shfl(w, j, kWave);
            if (__shfl(int(id >= 0), j, kWave) == 0) continue;
            const int64_t aj = (int64_t(__shfl(int(at >> 32), j, kWave)) << 32) | uint32_t(__shfl(int(uint32_t(at)), j, kWave));
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (lane + c * kWave < a.dim)
                    acc[c] = __builtin_fmaf(float(a.v_codes[aj + lane + c * kWave]), wj, acc[c]);
        }
    }
    for (int c = 0; c < 4; ++c)
        if (lane + c * kWave < a.dim) {
            const float o = l == 0.0f ? 0.0f : acc[c] / l;
            if constexpr (std::is_same_v<T, F16>)
                static_cast<_Float16 *>(a.out)[row + lane + c * kWave] = _Float16(o);
            else
                Fmt<T>::put(a.out, row + lane + c * kWave, o);
        }
}

} // namespace

void pagedAttentionInt8KV(const PagedAttentionCall &c, hipStream_t s) {
    if (c.rows == 0 || c.nh == 0 || c.requests == 0) return;
    const AttnArgs a{c.out, c.q, c.cache.k_codes, c.cache.v_codes, c.cache.k_scale, c.cache.v_scale, c.table, c.starts,
                     c.lens, int64_t(c.rows), int64_t(c.requests), int64_t(c.width), int64_t(c.cache.n_blocks),
                     int(c.nh), int(c.cache.heads), int(c.cache.dim), __builtin_ctzll(c.cache.block), c.scale, c.err};
    const dim3 grid(unsigned(c.rows), unsigned(c.nh));
    switch (c.dt) {
    case LLAISYS_DTYPE_F32: pagedAttnRow<F32><<<grid, kWave, 0, s>>>(a); return;
    case LLAISYS_DTYPE_BF16: pagedAttnRow<BF16><<<grid, kWave, 0, s>>>(a); return;
    case LLAISYS_DTYPE_F16: pagedAttnRow<F16><<<grid, kWave, 0, s>>>(a); return;
    default: return;
    }
}

} // namespace llaisys::kernels
