// Attention over the KV cache in blocks, tiles of 16 rows: tokens one or a few at a time.
//
// Bound by the cache's bytes, so every wave reads keys of its own, 64 a step, straight into the operands' registers:
// Sᵀ = K Qᵀ and Oᵀ = Vᵀ Pᵀ on v_mfma_f32_16x16x32_f16, with the keys assigned to the operand's rows so that
// the scores a lane gets are those of the 16 keys whose values it loads: no exchange between lanes, no LDS
// until the waves' states merge.  V's codes are transposed by the byte permutes that widen them.
// Three blocks a compute unit hide each other's loads; a step ahead in registers leaves room for two.  us, bf16,
// heads of 128: 64 tokens over 100 to 8192 keys each, 32 / 8 heads, 56.9 (4.1 TB/s; before the chunks had one length 61.6, two blocks and a step ahead 67.6), one over
// 131072, 12 / 2 heads, 22.7 (3.0 TB/s, the two merges among them; 25.6), one over 200 7.0: latency of the search, of
// ids, codes and the waves' merge, one behind the other.
#pragma once

#include "paged_attention.hpp"

namespace llaisys::kernels {

constexpr int kFewWaves = kPagedThreads / kWave;

// One row vector of Q for the 16x16x32 operand: channels of step (t, half) of this lane.
template <typename T, int NT>
struct QueryRows {
    static constexpr bool kTwo = std::is_same_v<T, F32>;
    v8h hi[NT][2], lo[kTwo ? NT : 1][2];
    int exponent;
    __device__ __forceinline__ void set(const Raw8<T> (&raw)[NT][2]) {
        exponent = 0;
        if constexpr (std::is_same_v<T, F16>) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) hi[t][h] = __builtin_bit_cast(v8h, raw[t][h].r[0]);
            return;
        }
        float top = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t) top = fmaxf(top, largest(raw[t]));
        top = butterflyStep<16, MaxOp>(top);
        top = butterflyStep<32, MaxOp>(top);
        exponent = rowExponent(top);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float f[8];
                raw[t][h].unpack(f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = __builtin_amdgcn_ldexpf(f[e], exponent);
                if constexpr (kTwo) split8(f, hi[t][h], lo[t][h]);
                else hi[t][h] = narrow8(f);
            }
    }
};

// A step's codes and scales: 64 keys.
template <int NT>
struct StepData {
    v4u k[4][NT];       // [key tile][64 channels]: key 16 (m / 4) + 4 tile + m % 4, channels 64 t + 16 quarter + 0..15
    uint32_t v[16][NT]; // key 16 quarter + i, channels 4 NT m + 0 .. 4 NT - 1
    float ks, vs;       // of keys 16 quarter + 0..15
    bool bad;           // their block id is none
};

// NT: 64s of channels, rounded up; D: the head size where it is 64 NT, else 0.
template <typename T, int NT, int D>
__global__ __launch_bounds__(kPagedThreads, NT <= 2 ? 3 : 1) void pagedFew(PagedAttnArgs a) {
    constexpr bool kTwoP = !std::is_same_v<T, BF16>;
    constexpr int kRows = kFewTile, CH = 4 * NT, NW = kFewWaves;
    __shared__ struct {
        float m[NW][kRows], l[NW][kRows];
        int at[kRows]; // a row's place in the output, from the tile's first token, in rows of dim
        float o[NW][kRows][64 * NT + 4];
    } sh;
    __shared__ unsigned arrived;
    const int dim = D ? D : a.dim;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
    const int m16 = lane % 16, quarter = lane / 16, index = a.by_heads.div(int(blockIdx.x)), head = int(blockIdx.x) - index * a.heads;
    Item it = findItem<kRows>(a, index, blockIdx.x == 0 && wave == 0);
    if (!it.any) return;

    const int first_row = it.tile * kRows, rows = min(kRows, it.n * a.group - first_row);
    const int row = first_row + m16, token = a.by_group.div(row);
    const int before = it.len - it.n; // tokens cached before the rows; a row sees before + token + 1
    const int seen_last = before + a.by_group.div(first_row + rows - 1) + 1, seen_first = before + a.by_group.div(first_row) + 1;
    const int steps = seen_last > 0 ? (seen_last + kStep - 1) / kStep : 0;
    if (!cutItem(it, steps)) return;
    const int end = min(it.step1, steps);
    const int limit = before + token + 1;
    const int token0 = a.by_group.div(first_row), out_row = (token - token0) * a.nh + head * a.group + (row - token * a.group);
    const size_t out0 = size_t(it.start + token0) * a.nh;

    const int32_t *table = a.table + int64_t(it.request) * a.width;
    const int in_block = (1 << a.shift) - 1;
    const size_t tile_bytes = size_t(dim) << a.shift;

    const auto blockOf = [&](int step, int group) { // id of the block of 16 keys
        const int key = min(step * kStep + 16 * group, seen_last - 1);
        return table[key >> a.shift];
    };
    struct Ids {
        int k, v;
    };
    const auto ids = [&](int step) { return Ids{blockOf(step, m16 / 4), blockOf(step, quarter)}; };
    const auto fetch = [&](int step, const Ids &id, StepData<NT> &d) {
        const bool kbad = uint32_t(id.k) >= uint32_t(a.n_blocks);
        d.bad = uint32_t(id.v) >= uint32_t(a.n_blocks);
        const int64_t kt = (kbad ? 0 : int64_t(id.k)) * a.heads + head, vt = (d.bad ? 0 : int64_t(id.v)) * a.heads + head;
        const int kkey = (step * kStep + 16 * (m16 / 4)) & in_block, vkey = (step * kStep + 16 * quarter) & in_block;
        const int8_t *kp = a.k_codes + kt * tile_bytes + (kkey + m16 % 4) * dim;
        const int8_t *vp = a.v_codes + vt * tile_bytes + vkey * dim;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            int c = 64 * t + 16 * quarter;
            if (D != 64 * NT) c = c < dim ? c : 0; // behind the row: q is 0 there
#pragma unroll
            for (int j = 0; j < 4; ++j) d.k[j][t] = *reinterpret_cast<const v4u *>(kp + 4 * j * dim + c);
        }
        int c = CH * m16;
        if (D != 64 * NT) c = c < dim ? c : 0; // not stored
#pragma unroll
        for (int i = 0; i < 16; ++i) __builtin_memcpy(d.v[i], __builtin_assume_aligned(vp + i * dim + c, CH), CH);
        d.ks = a.k_scale[vt];
        d.vs = a.v_scale[vt];
        if (d.bad && step * kStep + 16 * quarter < seen_last) atomicOr(a.err, kErrPagedIndex);
    };

    QueryRows<T, NT> q;
    float row_scale = 0.0f;
    float mx = -INFINITY, l = 0.0f, vref = 0.0f;
    v4f acc[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) acc[c] = v4f{0, 0, 0, 0};

    const auto compute = [&](int step, const StepData<NT> &d) {
        v4f s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const v8h k0 = codes8(d.k[j][t].x, d.k[j][t].y), k1 = codes8(d.k[j][t].z, d.k[j][t].w);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q.hi[t][0], s[j], 0, 0, 0);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q.hi[t][1], s[j], 0, 0, 0);
                if constexpr (q.kTwo) {
                    s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q.lo[t][0], s[j], 0, 0, 0);
                    s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q.lo[t][1], s[j], 0, 0, 0);
                }
            }
        }
        const float c = row_scale * checkedScale(d.ks);
        const int key0 = step * kStep + 16 * quarter;
        const bool some_hidden = __any(d.bad) || (step + 1) * kStep > seen_first;
        float top = mx;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[j][i] *= c;
                if (some_hidden && (d.bad || key0 + 4 * j + i >= limit)) s[j][i] = -INFINITY;
                top = fmaxf(top, s[j][i]);
            }
        top = butterflyStep<16, MaxOp>(top);
        top = butterflyStep<32, MaxOp>(top);
        const float vs = checkedScale(d.vs);
        float vtop = d.bad || key0 >= limit ? vref : fmaxf(vref, vs);
        vtop = butterflyStep<16, MaxOp>(vtop);
        vtop = butterflyStep<32, MaxOp>(vtop);
        if (__any(top > mx || vtop > vref)) {
            const float keep = mergeWeight(mx, top), f = vtop > vref ? keep * (vref / vtop) : keep;
            l *= keep;
#pragma unroll
            for (int k = 0; k < CH; ++k) acc[k] *= f;
            mx = top;
            vref = vtop;
        }
        const float base = mx == -INFINITY ? 0.0f : mx - kWeightBits;
        const float w = vref > 0.0f ? vs / vref : vs; // 0, or NaN, where no scale was above 0
        v8h p[2], r[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = s[2 * u + e / 4][e % 4], x = __builtin_amdgcn_exp2f(t - base);
                l += x;
                f[e] = some_hidden && t == -INFINITY ? 0.0f : x * w;
            }
            if constexpr (kTwoP) split8(f, p[u], r[u]);
            else p[u] = narrow8(f);
        }
        uint32_t v[16][NT];
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) v[i][n] = d.v[i][n] ^ 0x80808080u;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            constexpr uint32_t kSel[4] = {0x0c040c00u, 0x0c050c01u, 0x0c060c02u, 0x0c070c03u};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                Pairs x;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x.p[e] = codePair(__builtin_amdgcn_perm(v[8 * u + 2 * e + 1][k / 4], v[8 * u + 2 * e][k / 4], kSel[k % 4]));
                acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(join(x), p[u], acc[k], 0, 0, 0);
                if constexpr (kTwoP) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(join(x), r[u], acc[k], 0, 0, 0);
            }
        }
    };

    // the rows, loaded while the first keys' ids are on their way, and made operands while their codes are
    int step = it.step0 + wave;
    Ids now{0, 0};
    if (step < end) now = ids(step);
    Raw8<T> raw[NT][2];
    const size_t row_at = (out0 + unsigned(out_row)) * dim;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = 64 * t + 16 * quarter + 8 * h;
            if (m16 < rows && c < dim) raw[t][h].load(a.q, row_at + c);
            else raw[t][h].zero();
        }
    q.set(raw);
    row_scale = __builtin_amdgcn_ldexpf(a.scale * kLog2e, 9 - q.exponent);
    for (; step < end; step += NW) {
        StepData<NT> d;
        fetch(step, now, d);
        if (step + NW < end) now = ids(step + NW);
        compute(step, d);
    }

    // the waves' states: [row][channel], channel CH (4 quarter + i) + k of lane (row, quarter)
    l = butterflyStep<16, SumOp>(l);
    l = butterflyStep<32, SumOp>(l);
    if (quarter == 0) {
        if (wave == 0) sh.at[m16] = out_row;
        sh.m[wave][m16] = mx;
        sh.l[wave][m16] = l;
    }
    const float unit = vref * (1.0f / kCodeUnit);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < CH; k += 4)
            *reinterpret_cast<v4f *>(&sh.o[wave][m16][CH * (4 * quarter + i) + k]) =
                v4f{acc[k][i] * unit, acc[k + 1][i] * unit, acc[k + 2][i] * unit, acc[k + 3][i] * unit};
    __syncthreads();
    const auto place = [&](int r) { return (out0 + unsigned(sh.at[r])) * dim; };
    finishItem<T, kFewTile>(a, it, head, rows, dim, &arrived, place, [&](int r, int c, float *o, float &m, float &sum) {
        m = -INFINITY;
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, sh.m[w][r]);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = mergeWeight(sh.m[w][r], m);
            sum += sh.l[w][r] * f;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += sh.o[w][r][c + e] * f;
        }
    });
}

template <typename T>
void launchPagedFew(const PagedAttnArgs &a, unsigned items, hipStream_t s) {
    const unsigned grid = items * unsigned(a.heads);
    if (a.dim == 128) pagedFew<T, 2, 128><<<grid, kPagedThreads, 0, s>>>(a);
    else if (a.dim == 64) pagedFew<T, 1, 64><<<grid, kPagedThreads, 0, s>>>(a);
    else if (a.dim < 64) pagedFew<T, 1, 0><<<grid, kPagedThreads, 0, s>>>(a);
    else if (a.dim < 128) pagedFew<T, 2, 0><<<grid, kPagedThreads, 0, s>>>(a);
    else pagedFew<T, 4, 0><<<grid, kPagedThreads, 0, s>>>(a);
}

} // namespace llaisys::kernels
