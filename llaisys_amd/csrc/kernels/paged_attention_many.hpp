// Attention over the KV cache in blocks, tiles of 128 rows: prompts and chunks of prompts.
//
// Four waves of 32 rows share tiles of 64 keys.  Each wave reads 16 of the keys (one block id) a tile ahead,
// widens their codes to f16 and writes them to LDS once for all: K as it is, V transposed by the byte permutes that widen
// it.  Sᵀ = K Qᵀ and Oᵀ = Vᵀ Pᵀ run on v_mfma_f32_32x32x16_f16; K's rows enter in the order that makes a
// lane's 16 scores those of 16 keys in a row, so that its weights are the second product's operand as they are.
// Both LDS images are read 16 bytes a lane, their 16-byte columns xor-ed with bits of the row so that neither the
// reads nor the writes meet in a bank.
//
// Bound by each wave's chain of LDS reads, products, maximum and weights, of which the registers let two blocks of waves run
// on a compute unit: 3 prompts, 8419 rows, 32 / 8 heads of 128, bf16, take 253 us (766 TFLOP/s; a large product reaches
// 1157), and leaving out the exponentials did not change that.
#pragma once

#include "paged_attention.hpp"

namespace llaisys::kernels {

typedef float v16f __attribute__((ext_vector_type(16)));

static_assert(kManyTile == 32 * (kPagedThreads / kWave), "32 rows a wave");
// Weights are 2^(t - m + 11): m stays while no score passes it by more than 2^4, so that few tiles rescale the sums.
constexpr float kManyBits = 11.0f, kLazy = 4.0f;

// Column of a 16-byte piece of a K row (key) and of a V row (channel) in LDS.  xor distributes: the pieces 2 x + half of a key
// lie at the place of piece `half`, xor 2 x.
template <int DP>
__device__ __forceinline__ int kColumn(int key, int piece) {
    // lanes of a read differ in bits 0, 1, 4, 2 of the key first
    if constexpr (DP == 64)
        return piece ^ (((key >> 1) & 1) | ((key >> 3) & 2) | (key & 4));
    else
        return piece ^ ((key & 3) | ((key >> 2) & 4) | ((key << 1) & 8));
}
__device__ __forceinline__ int vColumn(int channel, int piece) { return piece ^ (((channel >> 2) & 7) ^ ((channel << 1) & 4)); }

// Two buffers of each kind, a power of two apart: [key][channel] and [channel][key] f16, and for each 16 keys (scale of k,
// of v, log2 of v's, whether their block id is none).  The outputs take their place.
template <int DP>
struct ManyShared {
    static constexpr int kBuffer = kStep * DP * 2, kV = 2 * kBuffer, kScales = 4 * kBuffer;
    union {
        alignas(16) unsigned char in[4 * kBuffer + 128 + kWave * 16]; // the last: where lanes without a scale write theirs
        float out[kManyTile][DP + 4];
    };
    float m[kManyTile], l[kManyTile];
    int at[kManyTile]; // a row's place in the output, from the tile's first token, in rows of dim
};

// Two blocks a compute unit where 256 registers hold a wave's rows.
template <typename T, int DP>
constexpr int kManyBlocks = DP <= 128 && !std::is_same_v<T, F32> ? 2 : 1;

// DP: the head size, rounded up to a size the tiles are made for; D: the head size where it is that size, else 0.
template <typename T, int DP, int D>
__global__ __launch_bounds__(kPagedThreads, (kManyBlocks<T, DP>)) void pagedMany(PagedAttnArgs a) {
    constexpr bool kTwoQ = std::is_same_v<T, F32>, kTwoP = !std::is_same_v<T, BF16>;
    constexpr int kSteps = DP / 16, kTiles = DP / 32;
    constexpr int kK = DP / 64;                 // 16-byte pieces of K a lane brings per tile
    constexpr int kV = DP <= 128 ? 1 : 2;       // units of 8 keys x 4 channels of V
    using Sh = ManyShared<DP>;
    __shared__ Sh sh;
    __shared__ unsigned arrived;
    const int dim = D ? D : a.dim;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
    const int col = lane % 32, half = lane / 32, index = a.by_heads.div(int(blockIdx.x)), head = int(blockIdx.x) - index * a.heads;
    Item it = findItem<kManyTile>(a, index, blockIdx.x == 0 && wave == 0);
    if (!it.any) return;

    const int total_rows = it.n * a.group;
    const int first_row = it.tile * kManyTile, rows = min(kManyTile, total_rows - first_row);
    const int before = it.len - it.n;
    const auto seenBy = [&](int row) { return before + a.by_group.div(row) + 1; };
    const int seen_last = seenBy(first_row + rows - 1);
    const int steps = seen_last > 0 ? (seen_last + kStep - 1) / kStep : 0;
    if (!cutItem(it, steps)) return;
    const int end = min(it.step1, steps);

    // this wave's rows
    const int wrow = first_row + 32 * wave, row = wrow + col, token = a.by_group.div(row);
    const bool valid = row < total_rows;
    const int limit = before + token + 1;
    const int wave_last = wrow < total_rows ? seenBy(min(wrow + 31, total_rows - 1)) : 0, wave_first = seenBy(wrow);
    const int token0 = a.by_group.div(first_row), out_row = (token - token0) * a.nh + head * a.group + (row - token * a.group);
    const size_t out0 = size_t(it.start + token0) * a.nh;
    // ---- the wave's 16 keys of a tile: HBM -> registers -> LDS
    const int32_t *table = a.table + int64_t(it.request) * a.width;
    const size_t tile_bytes = size_t(dim) << a.shift;
    const int in_block = (1 << a.shift) - 1;
    const int k_key = (lane * 16) / DP, k_piece = lane % (DP / 16); // i-th piece: key k_key + i * 1024 / DP
    const int v_quad = (lane % (DP / 4 < kWave ? DP / 4 : kWave)), v_chunk = DP <= 128 ? lane / (DP / 4) : 0;
    v4u kr[kK];
    uint32_t vr[kV][8];
    float ks = 0.0f, vs = 0.0f;
    bool bad = false, any_bad = false;
    int id_next = 0;
    // past the item's keys these read keys of its last block again
    const auto idOf = [&](int step) { return table[min(step * kStep + 16 * wave, seen_last - 1) >> a.shift]; };
    struct Place {
        const int8_t *k, *v;
        const float *ks, *vs;
        bool bad;
    };
    const auto placeOf = [&](int step) { // of the step whose id is id_next
        const int id = uniform(id_next);
        Place p;
        p.bad = uint32_t(id) >= uint32_t(a.n_blocks);
        any_bad = any_bad || (p.bad && step * kStep + 16 * wave < seen_last);
        const int64_t tile = (p.bad ? 0 : int64_t(id)) * a.heads + head;
        const size_t at = tile * tile_bytes + size_t((step * kStep + 16 * wave) & in_block) * dim;
        p.k = a.k_codes + at;
        p.v = a.v_codes + at;
        p.ks = a.k_scale + tile;
        p.vs = a.v_scale + tile;
        return p;
    };
    const auto fetch = [&](int step, const Place &p) {
        id_next = idOf(step + 1); // first, as it is needed first
        int c = 16 * k_piece;
        if (D != DP) c = c < dim ? c : 0; // behind the row: q is 0 there
#pragma unroll
        for (int i = 0; i < kK; ++i) kr[i] = *reinterpret_cast<const v4u *>(p.k + unsigned((k_key + i * (1024 / DP)) * dim + c));
        if (DP >= 128 || lane < 32) {
#pragma unroll
            for (int u = 0; u < kV; ++u) {
                int ch = 4 * v_quad;
                if (D != DP) ch = ch < dim ? ch : 0; // not stored
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    vr[u][i] = *reinterpret_cast<const uint32_t *>(p.v + unsigned((8 * (v_chunk + u) + i) * dim + ch));
            }
        }
        ks = *p.ks;
        vs = *p.vs;
        bad = p.bad;
    };
    // The rows, loaded while the first keys' ids are on their way, and made operands while their codes are.
    if (it.step0 < end) id_next = idOf(it.step0);
    v8h q[kSteps], ql[kTwoQ ? kSteps : 1];
    float row_scale;
    {
        Raw8<T> raw[kSteps];
        const size_t at = (out0 + unsigned(out_row)) * dim + 8 * half;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (valid && (D || 16 * s < dim)) raw[s].load(a.q, at + 16 * s);
            else raw[s].zero();
        }
        if (it.step0 < end) fetch(it.step0, placeOf(it.step0));
        // the scale of a score is not negative below: its sign goes to the rows
        int e = 0;
        if constexpr (std::is_same_v<T, F16>) {
            const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) q[s] = __builtin_bit_cast(v8h, raw[s].r[0] ^ flip);
        } else {
            const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
            e = rowExponent(butterflyStep<32, MaxOp>(largest(raw)));
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                float f[8];
                raw[s].unpack(f);
#pragma unroll
                for (int x = 0; x < 8; ++x) f[x] = __builtin_amdgcn_ldexpf(sign * f[x], e);
                if constexpr (kTwoQ) split8(f, q[s], ql[s]);
                else q[s] = narrow8(f);
            }
        }
        row_scale = __builtin_amdgcn_ldexpf(fabsf(a.scale) * kLog2e, 9 - e);
    }
    const auto put16 = [&](int at, const v8h &x) { *reinterpret_cast<v8h *>(sh.in + at) = x; };
    const auto get16 = [&](int at) { return *reinterpret_cast<const v8h *>(sh.in + at); };
    // places in the buffers, of the next step to write and the next to read
    int k_to = (16 * wave + k_key) * DP * 2 + kColumn<DP>(16 * wave + k_key, 2 * k_piece) * 16;
    int v_to = Sh::kV + 4 * v_quad * kStep * 2 + vColumn(4 * v_quad, 2 * wave + v_chunk) * 16;
    int s_to = Sh::kScales + (lane == 0 ? wave * 16 : 128 + lane * 16);
    const int s_flip = lane == 0 ? 64 : 0;
    // The staging in halves of 16-byte pieces, to be put between products: 2 kK pieces of K, 4 kV of V.
    constexpr int kHalves = 2 * (2 * kK + 4 * kV);
    uint32_t vx[kV][8];
    Pairs piece;
    const auto stageHalf = [&](int n) {
        const int j = n / 2, h = n % 2;
        if (j < 2 * kK) {
            // keys 1024 / DP apart: bit 2 of the key, where it changes, moves the column
            const int i = j / 2, at = k_to ^ (DP == 256 ? (i & 1) * 128 : 0) ^ (j % 2 * 16);
            const uint32_t w = (j % 2 ? (h ? kr[i].w : kr[i].z) : (h ? kr[i].y : kr[i].x)) ^ 0x80808080u;
            piece.p[2 * h] = codePair(__builtin_amdgcn_perm(w, w, 0x0c010c00u));
            piece.p[2 * h + 1] = codePair(__builtin_amdgcn_perm(w, w, 0x0c030c02u));
            if (h) put16(at + i * 2048, join(piece));
            return;
        }
        const int u = (j - 2 * kK) / 4, x = (j - 2 * kK) % 4;
        constexpr uint32_t kSel[4] = {0x0c040c00u, 0x0c050c01u, 0x0c060c02u, 0x0c070c03u};
        if (x == 0) {
#pragma unroll
            for (int i = 4 * h; i < 4 * h + 4; ++i) vx[u][i] = vr[u][i] ^ 0x80808080u;
        }
#pragma unroll
        for (int e = 2 * h; e < 2 * h + 2; ++e) piece.p[e] = codePair(__builtin_amdgcn_perm(vx[u][2 * e + 1], vx[u][2 * e], kSel[x]));
        // (of 64 channels half the lanes have none: theirs go behind the scales)
        const int at = (v_to ^ (u * 16) ^ (x / 2 * 64)) + x * kStep * 2;
        if (h) put16(DP >= 128 || lane < 32 ? at : Sh::kScales + 128 + lane * 16, join(piece));
    };
    const auto stageScales = [&] {
        const float v = checkedScale(vs);
        *reinterpret_cast<v4u *>(sh.in + s_to) = v4u{__float_as_uint(checkedScale(ks)), __float_as_uint(v),
                                                     __float_as_uint(__builtin_amdgcn_logf(v)), bad ? 1u : 0u};
        k_to ^= Sh::kBuffer;
        v_to ^= Sh::kBuffer;
        s_to ^= s_flip;
    };
    const auto stage = [&] {
#pragma unroll
        for (int j = 0; j < kHalves; ++j) stageHalf(j);
        stageScales();
    };

    // ---- one step's products
    float mx = -INFINITY, l = 0.0f, vref = 0.0f, lref = 0.0f;
    v16f acc[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;
    const int my_key = 16 * (col / 4 % 2) + 4 * (col / 8) + col % 4; // K's row at this lane's place of the operand
    int k_from = my_key * DP * 2 + kColumn<DP>(my_key, half) * 16;
    int v_from = Sh::kV + col * kStep * 2 + vColumn(col, 2 * half) * 16;
    int s_from = Sh::kScales;

    // The next step's codes are staged beside the first product, and those of the one after it asked for.
    const auto compute = [&](int step) {
        const Place place = placeOf(step + 2);
        v4u info[4];
        v16f sc[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[0][i] = sc[1][i] = 0.0f;
        float best[2] = {-INFINITY, -INFINITY};
        // operands three products ahead, half a piece of the staging before each; the first 32 keys' maximum beside the
        // product of the others
        constexpr int kRingK = 4;
        v8h k[kRingK];
        const auto readK = [&](int n) {
            if (n < 2 * kSteps) k[n % kRingK] = get16((k_from ^ (n % kSteps * 32)) + n / kSteps * 32 * DP * 2);
        };
#pragma unroll
        for (int n = 0; n < kRingK - 1; ++n) readK(n);
#pragma unroll
        for (int g = 0; g < 4; ++g) info[g] = *reinterpret_cast<const v4u *>(sh.in + s_from + 16 * g);
#pragma unroll
        for (int n = 0; n < 2 * kSteps; ++n) {
            const int t = n / kSteps, x = n % kSteps;
            readK(n + kRingK - 1);
#pragma unroll
            for (int j = n * kHalves / (2 * kSteps); j < (n + 1) * kHalves / (2 * kSteps); ++j) stageHalf(j);
            if (t == 1) {
#pragma unroll
                for (int i = x * 16 / kSteps; i < (x + 1) * 16 / kSteps; ++i) best[0] = fmaxf(best[0], sc[0][i]);
            }
            __builtin_amdgcn_sched_barrier(0);
            sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n % kRingK], q[x], sc[t], 0, 0, 0);
            if constexpr (kTwoQ) sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n % kRingK], ql[x], sc[t], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        stageScales();
        fetch(step + 2, place);
#pragma unroll
        for (int i = 0; i < 16; ++i) best[1] = fmaxf(best[1], sc[1][i]);
        const bool hide = (step + 1) * kStep > wave_first || uniform(int(info[0].w | info[1].w | info[2].w | info[3].w)) != 0;
        // this lane's keys: 32 t + 16 half + 0..15
        float c[2], vscale[2], shift[2];
        bool sees[2] = {true, true};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            c[t] = row_scale * __uint_as_float(half ? info[2 * t + 1].x : info[2 * t].x);
            vscale[t] = __uint_as_float(half ? info[2 * t + 1].y : info[2 * t].y);
            shift[t] = __uint_as_float(half ? info[2 * t + 1].z : info[2 * t].z);
        }
        if (hide) {
            // a hidden key's score is so low that its weight is 0 for any factor from 1e-30 on; a smaller factor makes every
            // score 0 as 1e-30 does, and where no key of the 16 is seen neither scale may speak (they may be NaN)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const bool none = (half ? info[2 * t + 1].w : info[2 * t].w) != 0;
                const int left = none ? 0 : limit - (step * kStep + 32 * t + 16 * half); // keys seen of the 16
                sees[t] = left > 0;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i >= left) sc[t][i] = -3e38f;
                best[t] = sc[t][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) best[t] = fmaxf(best[t], sc[t][i]);
                if (c[t] < 1e-30f || !sees[t]) c[t] = 1e-30f;
            }
        }
        float top = -INFINITY, vtop = vref;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            top = sees[t] ? fmaxf(top, best[t] * c[t]) : top;
            vtop = sees[t] ? fmaxf(vtop, vscale[t]) : vtop;
        }
        top = butterflyStep<32, MaxOp>(top);
        vtop = butterflyStep<32, MaxOp>(vtop);
        if (__any(top > mx + kLazy || vtop > vref || (mx == -INFINITY && top > mx))) {
            const float m = fmaxf(mx, top), keep = mergeWeight(mx, m);
            const float f = vtop > vref ? keep * (vref / vtop) : keep;
            l *= keep;
#pragma unroll
            for (int k = 0; k < kTiles; ++k) acc[k] *= f;
            mx = m;
            vref = vtop;
            lref = vref > 0.0f ? __builtin_amdgcn_logf(vref) : 0.0f;
        }
        const float base = (mx == -INFINITY ? 0.0f : mx) - kManyBits;
        float to[2], w[2], sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            to[t] = base;
            if constexpr (kTwoQ) {
                w[t] = !sees[t] ? 0.0f : vref > 0.0f ? vscale[t] / vref : vscale[t]; // 0, or NaN, where no scale was above 0
            } else {
                // the value scale's ratio goes into the exponent, and out of the sum at once; below 2^-100 (or 0) the
                // weights are 0 as f16
                const float d = shift[t] - lref;
                shift[t] = !sees[t] ? 0.0f : d < -100.0f ? -100.0f : d;
                to[t] = base - shift[t];
            }
        }
        // eight weights at a time, those of the next eight keys computed between the products of these
        float f[2][8];
        v8h v[2][kTiles];
        const auto weight = [&](int g, int e) {
            const int t = g / 2;
            float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * (g % 2) + e], c[t], -to[t]));
            sum[t] += x;
            if constexpr (kTwoQ) x *= w[t];
            f[g % 2][e] = x;
        };
        const auto readV = [&](int g, int k) { v[g % 2][k] = get16((v_from ^ ((g / 2 * 4 + g % 2) * 16)) + k * 32 * kStep * 2); };
#pragma unroll
        for (int k = 0; k < kTiles; ++k) readV(0, k);
#pragma unroll
        for (int e = 0; e < 8; ++e) weight(0, e);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            v8h p, r;
            if constexpr (kTwoP) split8(f[g % 2], p, r);
            else p = narrow8(f[g % 2]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < kTiles; ++k) {
                acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[g % 2][k], p, acc[k], 0, 0, 0);
                if constexpr (kTwoP) acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[g % 2][k], r, acc[k], 0, 0, 0);
                if (g < 3) {
                    readV(g + 1, k);
#pragma unroll
                    for (int e = k * 8 / kTiles; e < (k + 1) * 8 / kTiles; ++e) weight(g + 1, e);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if constexpr (!kTwoQ) sum[t] *= __builtin_amdgcn_exp2f(-shift[t]);
            l += sum[t];
        }
    };

    if (it.step0 < end) {
        stage();
        fetch(it.step0 + 1, placeOf(it.step0 + 1));
        ldsBarrier();
        for (int step = it.step0; step < end; ++step) {
            if (step * kStep < wave_last) {
                compute(step);
            } else {
                stage();
                fetch(step + 2, placeOf(step + 2));
            }
            k_from ^= Sh::kBuffer;
            v_from ^= Sh::kBuffer;
            s_from ^= 64;
            ldsBarrier();
        }
        if (any_bad && lane == 0) atomicOr(a.err, kErrPagedIndex);
    }

    // ---- outputs through LDS: row, 8 channels
    l = butterflyStep<32, SumOp>(l);
    const float unit = vref * (1.0f / kCodeUnit);
    const int mine = 32 * wave + col;
#pragma unroll
    for (int k = 0; k < kTiles; ++k)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int ch = 32 * k + 8 * (i / 4) + 4 * half;
            *reinterpret_cast<v4f *>(&sh.out[mine][ch]) = v4f{acc[k][i] * unit, acc[k][i + 1] * unit, acc[k][i + 2] * unit, acc[k][i + 3] * unit};
        }
    if (half == 0) {
        sh.m[mine] = mx;
        sh.l[mine] = l;
        sh.at[mine] = out_row;
    }
    __syncthreads();
    finishItem<T, kManyTile>(
        a, it, head, rows, dim, &arrived, [&](int r) { return (out0 + unsigned(sh.at[r])) * dim; },
        [&](int r, int c, float *o, float &m, float &sum) {
            m = sh.m[r];
            sum = sh.l[r];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = sh.out[r][c + e];
        });
}

template <typename T>
void launchPagedMany(const PagedAttnArgs &a, unsigned items, hipStream_t s) {
    const unsigned grid = items * unsigned(a.heads);
    if (a.dim == 128) pagedMany<T, 128, 128><<<grid, kPagedThreads, 0, s>>>(a);
    else if (a.dim == 64) pagedMany<T, 64, 64><<<grid, kPagedThreads, 0, s>>>(a);
    else if (a.dim < 64) pagedMany<T, 64, 0><<<grid, kPagedThreads, 0, s>>>(a);
    else if (a.dim < 128) pagedMany<T, 128, 0><<<grid, kPagedThreads, 0, s>>>(a);
    else pagedMany<T, 256, 0><<<grid, kPagedThreads, 0, s>>>(a);
}

} // namespace llaisys::kernels
