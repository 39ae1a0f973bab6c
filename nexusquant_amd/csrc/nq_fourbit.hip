// Attention of packed queries over a cache held in 4 bits (nq_fourbit.h): decode steps, several new tokens of a sequence
// over its past and themselves, and queries that see all of another sequence's tokens.
//
// With q~ = H q, a token's codes n and scales s:
//   logit = scale * s_k sum q~ (n - 8)         out = H sum p s_v (n - 8)
// so nothing is undone a token: codes go to fp16 (exactly) and into the matrix cores, the transform is applied to a query
// before and to its output after.
//
// The host cuts each sequence's queries into tiles of rows (a row: a query token and one of the kv head's query heads)
// and its tokens into chunks.  A workgroup takes a tile, a chunk and a kv head: up to 16 rows few_kernel, more wide_kernel.
// A partial (maximum, sum, value sum) per row and chunk goes to the workspace; join_kernel joins a row's, transforms and
// rounds.
#include "nq_flash.h"
#include "nq_fourbit.h"

namespace nq {

using namespace flash;

constexpr int kItemInts = 12;

struct FourBitArgs {
    const uint16_t* query;
    uint16_t* out;
    FourBitRows pool;
    const int32_t* items;     // [n_items * kItemInts], see nq_fourbit_desc
    const int32_t* pages;
    const int32_t* joins;     // [n_joins * 4]: query token, its first slot, slots, 0
    float* part_y;            // [slots, q_heads, D]
    float* part_ml;           // [slots, q_heads, 2]
    int64_t q_row, q_head, o_row, o_head;  // strides, elements
    uint32_t q_heads, kv_heads, group, tokens;
    FastDiv by_tokens, by_group, by_kv;
    int32_t window;           // 0: none
    int32_t step;             // 1: query i sees the tokens up to last + i; 0: up to last
    float c;                  // scale * log2(e) * h
    float hscale;
};

struct Item {
    const int32_t* pages;
    int tok0, n_tok, q_row0, r0, n_rows, slot0, slots, last;
};
__device__ __forceinline__ Item item_of(const FourBitArgs& a, uint32_t i, int most_rows, int most_tokens) {
    const int32_t* const it = a.items + (size_t)kItemInts * i;
    Item x;
    x.pages = a.pages + it[0];
    x.tok0 = it[1];
    x.n_tok = min(max(it[2], 1), most_tokens);  // what LDS is sized for, whatever a plan from elsewhere holds
    x.q_row0 = it[3];
    x.r0 = it[4];
    x.n_rows = min(max(it[5], 1), most_rows);
    x.slot0 = it[6];
    x.slots = it[7];
    x.last = it[8];
    return x;
}

// a.group rows a query token: which token and head row r is
struct RowAt {
    uint32_t token, head;
};
__device__ __forceinline__ RowAt row_at(const FourBitArgs& a, uint32_t r, uint32_t kh) {
    const uint32_t t = div(r, a.by_group);
    return {t, kh * a.group + (r - t * a.group)};
}
// row's first and last token seen, counted from the chunk's first
__device__ __forceinline__ void seen_by(const FourBitArgs& a, const Item& it, uint32_t token, int& lo, int& hi) {
    const int last = it.last + a.step * (int)token;
    lo = a.window ? max(last - a.window + 1 - it.tok0, 0) : 0;
    hi = min(last - it.tok0, it.n_tok - 1);
}

__device__ __forceinline__ f32x2 rows16(float v) {  // lanes l and l ^ 16: the one with bit 4 clear first
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return {__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ float four_max(float v) {
    const f32x2 h = rows16(v);
    return both_max(__builtin_fmaxf(h.x, h.y));
}
__device__ __forceinline__ float four_sum(float v) {
    const f32x2 h = rows16(v);
    return both_sum(h.x + h.y);
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A scale, or 0 for one that is not finite: what those who see it get of it must not change what others get.
__device__ __forceinline__ float finite_scale(uint16_t bits) { return (bits & 0x7c00u) == 0x7c00u ? 0.0f : f16_bits_to_f32(bits); }

// The power of two that takes a row's largest |v| into [2^14, 2^15), as an exponent; 0 for what has none.
__device__ __forceinline__ int row_exponent(float big) {
    int e = 0;
    if (big > 0.0f && big < __builtin_inff()) (void)__builtin_frexpf(big, &e);
    return min(max(15 - e, -126), 126);
}

// ------------------------------------------------------------------- few rows ----

// A wave takes 32 tokens at a time through 16x16x32 MFMAs, from their codes to the output without LDS between:
//   S = K q~^T     A: lane (token m, kg) the D / 32 words of its row from D / 32 kg on, a word a step; B: queries alike
//   O^T = V^T P^T  S came out as lane (query, kg) with tokens 4 kg + 0..3 of either half, which is the B operand as it
//                  stands; A: lane (m, kg) the D / 16 nibbles from D / 16 m on of these eight tokens, nibble j of all of
//                  them the operand of output tile j
// Codes stand in the operands as 16 + n.  The 24 too much of each comes off by the logits' first accumulator,
// -24 sum q~, and by one more tile of ones, which sums the weights.  Queries and weights go in twice, as fp16 and what
// that rounds off: 22 bits.
template <int D>
struct FewShape {
    static constexpr int WAVES = 4, ROWS = 16;
    static constexpr int CHUNK = 1024;  // most tokens of a chunk
    static constexpr int PER_SIMD = D == 256 ? 2 : 4;
};

template <int D>
struct FewLds {
    f32x4 o[FewShape<D>::WAVES / 2][D / 16][64];
    uint32_t row[FewShape<D>::CHUNK];  // a token's row of this head
    uint16_t ks[FewShape<D>::CHUNK], vs[FewShape<D>::CHUNK];  // its scales (fp16)
    float max[FewShape<D>::WAVES], m[FewShape<D>::WAVES / 2][16], l[FewShape<D>::WAVES / 2][16];
};

template <int D, int QDT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(FewShape<D>::PER_SIMD))) void few_kernel(FourBitArgs a) {
    using F = FewShape<D>;
    constexpr int KS = D / 32, TILES = D / 16, NW = F::WAVES, NT = 64 * NW, RB = D / 2;
    constexpr int VW = D == 256 ? 2 : 1;  // words of a token's values a lane (head_dim 64: half of one)
    __shared__ __align__(16) FewLds<D> lds;
    const int lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t item = div(blockIdx.x, a.by_kv), kh = blockIdx.x - item * a.kv_heads;
    const Item it = item_of(a, item, F::ROWS, F::CHUNK);
    const int n_units = (it.n_tok + 31) / 32, last_place = 32 * n_units - 1;

    // ---- the chunk's tokens: places past it repeat its last (no row sees them) ----
    uint32_t kcode[2][KS], vcode[8][VW];
    auto row_of = [&](int i) {
        const uint32_t t = (uint32_t)(it.tok0 + min(i, it.n_tok - 1)), p = div(t, a.by_tokens);
        return ((uint32_t)it.pages[p] * a.kv_heads + kh) * a.tokens + (t - p * a.tokens);
    };
    auto load_keys = [&](int half, uint32_t row) {
        const uint32_t* const p = reinterpret_cast<const uint32_t*>(a.pool.codes[0] + (size_t)row * RB + 4 * KS * kg);
        if constexpr (KS == 2) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p);
            kcode[half][0] = w.x;
            kcode[half][1] = w.y;
        } else {
#pragma unroll
            for (int s = 0; s < KS; s += 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(p + s);
#pragma unroll
                for (int i = 0; i < 4; ++i) kcode[half][s + i] = w[i];
            }
        }
    };
    auto load_values = [&](int i, uint32_t row) {
        const uint8_t* const p = a.pool.codes[1] + (size_t)row * RB;
        if constexpr (D == 64) vcode[i][0] = *reinterpret_cast<const uint32_t*>(p + 4 * (n16 >> 1));
        else if constexpr (D == 128) vcode[i][0] = *reinterpret_cast<const uint32_t*>(p + 4 * n16);
        else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p + 8 * n16);
            vcode[i][0] = w.x;
            vcode[i][VW - 1] = w.y;
        }
    };
#pragma unroll
    for (int t = 0; t < 2; ++t) load_keys(t, row_of(32 * wave + 16 * t + n16));

    // ---- queries: lane (query n16, kg) coordinates D / 4 kg .. + D / 4 - 1 ----
    const RowAt my = row_at(a, (uint32_t)(it.r0 + min(n16, it.n_rows - 1)), kh);
    float x[KS][8];
    {
        const uint16_t* const p = a.query + (int64_t)(it.q_row0 + (int)my.token) * a.q_row + my.head * a.q_head + (D / 4) * kg;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p + 8 * s);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[s][2 * k] = unpack<QDT>(w[k] & 0xffffu);
                x[s][2 * k + 1] = unpack<QDT>(w[k] >> 16);
            }
        }
    }
    float vmax = 0.0f;
    for (int i = threadIdx.x; i <= last_place; i += NT) {
        const uint32_t row = row_of(i);
        lds.row[i] = row;
        lds.ks[i] = a.pool.scales[0][row];
        const uint16_t vs = a.pool.scales[1][row];
        lds.vs[i] = vs;
        vmax = __builtin_fmaxf(vmax, finite_scale(vs));
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) vmax = __builtin_fmaxf(vmax, __shfl_xor(vmax, o, 64));
    if (lane == 0) lds.max[wave] = vmax;

    // the transform over coordinate bits 0..2 (in a step), then the steps, then kg
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int len = 1; len < 8; len <<= 1)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i & len) continue;
                const float u = x[s][i], v = x[s][i + len];
                x[s][i] = u + v;
                x[s][i + len] = u - v;
            }
#pragma unroll
    for (int len = 1; len < KS; len <<= 1)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s & len) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = x[s][i], v = x[s + len][i];
                x[s][i] = u + v;
                x[s + len][i] = u - v;
            }
        }
    const float sign16 = (lane & 16) ? -1.0f : 1.0f, sign32 = (lane & 32) ? -1.0f : 1.0f;
    float big = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const f32x2 h = rows16(x[s][i]);
            const f32x2 g = halves(__builtin_fmaf(h.y, sign16, h.x));
            x[s][i] = __builtin_fmaf(g.y, sign32, g.x);
            big = __builtin_fmaxf(big, __builtin_fabsf(x[s][i]));
        }
    const int qexp = row_exponent(four_max(big));
    u32x4 qh[KS], ql[KS];
    float qsum = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // the pair (j, j + 4) of a word's nibbles
            const float u = __builtin_ldexpf(x[s][j], qexp), v = __builtin_ldexpf(x[s][j + 4], qexp);
            qh[s][j] = pack2<NQ_F16>(u, v);
            const float uh = f16_bits_to_f32(qh[s][j] & 0xffffu), vh = f16_bits_to_f32(qh[s][j] >> 16);
            ql[s][j] = pack2<NQ_F16>(u - uh, v - vh);
            qsum += (uh + vh) + (f16_bits_to_f32(ql[s][j] & 0xffffu) + f16_bits_to_f32(ql[s][j] >> 16));
        }
    const float s_first = -kNibbleBias * four_sum(qsum);
    const float c = __builtin_ldexpf(a.c, -qexp);
    int lo, hi;
    seen_by(a, it, my.token, lo, hi);
    __syncthreads();
    // The values' scales go with the weights: times 2^vexp the chunk's largest is in [64, 128), so weights (2^kSlack at
    // most) stay below 2^15.
    float vall = lds.max[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) vall = __builtin_fmaxf(vall, lds.max[w]);
    int vexp = 0;
    if (vall > 0.0f) {
        (void)__builtin_frexpf(vall, &vexp);
        vexp = 7 - vexp;
    }
    const float vmul = __builtin_ldexpf(1.0f, vexp);
    auto values_at = [&](int first) {
        const uint32_t* const r = lds.row + first + 4 * kg;
        const u32x4 r0 = *reinterpret_cast<const u32x4*>(r), r1 = *reinterpret_cast<const u32x4*>(r + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_values(i, r0[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_values(4 + i, r1[i]);
    };
    values_at(min(32 * wave, 32 * (n_units - 1)));

    f32x4 o[TILES], wsum = {};
#pragma unroll
    for (int j = 0; j < TILES; ++j) o[j] = f32x4{};
    float m = kNoMax, l = 0.0f;
    const uint32_t pick_lo = D == 64 && (n16 & 1) ? 0x07060302u : 0x05040100u;
    const u32x4 ones = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
#pragma unroll 1
    for (int u = wave; u < n_units; u += NW) {
        const int next = 32 * min(u + NW, n_units - 1);
        // ---- logits of 16 tokens twice ----
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = f32x4{s_first, s_first, s_first, s_first};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint32_t w = kcode[t][k];
                const u32x4 v = {nibble_pair<0>(w), nibble_pair<1>(w), nibble_pair<2>(w), nibble_pair<3>(w)};
                s[t] = mfma16(v, qh[k], mfma16(v, ql[k], s[t]));
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) load_keys(t, lds.row[next + 16 * t + n16]);
        // ---- weights ----
        float p[8], mx = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int at = 32 * u + 16 * t + 4 * kg;
            const u32x2 kw = *reinterpret_cast<const u32x2*>(lds.ks + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = s[t][i] * f16_bits_to_f32((i & 1) ? kw[i / 2] >> 16 : kw[i / 2] & 0xffffu) * c;
                const bool seen = at + i >= lo && at + i <= hi;
                p[4 * t + i] = seen ? v : -__builtin_inff();
                mx = __builtin_fmaxf(mx, p[4 * t + i]);
            }
        }
        if (__any(mx > m + kSlack)) {
            const float to = __builtin_fmaxf(m, four_max(mx));
            const float f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
            wsum *= f;
#pragma unroll
            for (int j = 0; j < TILES; ++j) o[j] *= f;
        }
        u32x4 w, rest;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int at = 32 * u + 16 * t + 4 * kg;
            const u32x2 vw = *reinterpret_cast<const u32x2*>(lds.vs + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(p[4 * t + i] - m);
                l += e;
                const float v = e * f16_bits_to_f32((i & 1) ? vw[i / 2] >> 16 : vw[i / 2] & 0xffffu) * vmul;
                p[4 * t + i] = at + i >= lo && at + i <= hi ? v : 0.0f;  // (a scale that is not seen may be NaN)
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = pack2<NQ_F16>(p[2 * i], p[2 * i + 1]);
            rest[i] = pack2<NQ_F16>(p[2 * i] - f16_bits_to_f32(w[i] & 0xffffu), p[2 * i + 1] - f16_bits_to_f32(w[i] >> 16));
        }
        // ---- values: nibble j of eight tokens ----
        wsum = mfma16(ones, rest, mfma16(ones, w, wsum));
#pragma unroll
        for (int k = 0; k < VW; ++k)
#pragma unroll
            for (int half = 0; half < (D == 64 ? 1 : 2); ++half) {
                uint32_t x4[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x4[i] = __builtin_amdgcn_perm(vcode[2 * i + 1][k], vcode[2 * i][k], half ? 0x07060302u : pick_lo);
                auto tile = [&](int j, u32x4 v) {
                    f32x4& to = o[8 * k + 4 * half + j];
                    to = mfma16(v, rest, mfma16(v, w, to));
                };
                tile(0, u32x4{nibble_pair<0>(x4[0]), nibble_pair<0>(x4[1]), nibble_pair<0>(x4[2]), nibble_pair<0>(x4[3])});
                tile(1, u32x4{nibble_pair<1>(x4[0]), nibble_pair<1>(x4[1]), nibble_pair<1>(x4[2]), nibble_pair<1>(x4[3])});
                tile(2, u32x4{nibble_pair<2>(x4[0]), nibble_pair<2>(x4[1]), nibble_pair<2>(x4[2]), nibble_pair<2>(x4[3])});
                tile(3, u32x4{nibble_pair<3>(x4[0]), nibble_pair<3>(x4[1]), nibble_pair<3>(x4[2]), nibble_pair<3>(x4[3])});
            }
        values_at(next);
    }
#pragma unroll
    for (int j = 0; j < TILES; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] = __builtin_fmaf(-kNibbleBias, wsum[i], o[j][i]);

    // ---- the waves' sums joined: the upper half's into the lower half's, twice ----
    l = four_sum(l);
#pragma unroll
    for (int step = NW / 2; step >= 1; step >>= 1) {
        if (wave >= step && wave < 2 * step) {
#pragma unroll
            for (int j = 0; j < TILES; ++j) lds.o[wave - step][j][lane] = o[j];
            if (kg == 0) {
                lds.m[wave - step][n16] = m;
                lds.l[wave - step][n16] = l;
            }
        }
        __syncthreads();
        if (wave < step) {
            const float mo = lds.m[wave][n16], to = __builtin_fmaxf(m, mo);
            const float f = __builtin_amdgcn_exp2f(m - to), fo = __builtin_amdgcn_exp2f(mo - to);
            m = to;
            l = l * f + lds.l[wave][n16] * fo;
#pragma unroll
            for (int j = 0; j < TILES; ++j) {
                const f32x4 y = lds.o[wave][j][lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j][i] = __builtin_fmaf(y[i], fo, o[j][i] * f);
            }
        }
        __syncthreads();
    }
    if (wave > 0 || n16 >= it.n_rows) return;
    const size_t slot = (size_t)(uint32_t)(it.slot0 + (int)my.token * it.slots) * a.q_heads + my.head;
    if (kg == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * slot) = f32x2{m, l};
    const float f = __builtin_ldexpf(1.0f, -vexp);
    // lane (n, kg), register i of tile j: coordinate D / 16 (4 kg + i) + j
    float* const y = a.part_y + slot * D + TILES * 4 * kg;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < TILES; j += 4)
            *reinterpret_cast<f32x4*>(y + TILES * i + j) = f32x4{o[j][i] * f, o[j + 1][i] * f, o[j + 2][i] * f, o[j + 3][i] * f};
}

// One (query token, head) a workgroup: its chunks' sums weighted and added in a fixed order, then the transform, h and the
// softmax's sum.  A row that saw nothing is zero.
template <int D, int QDT>
__global__ __launch_bounds__(256) void fourbit_join_kernel(FourBitArgs a) {
    constexpr int V = D / 4, NG = 256 / V;  // lanes of a chunk's row, chunks at a time
    __shared__ f32x4 s_y[NG][V];
    __shared__ float s_l[NG];
    const uint32_t which = blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads;
    const int32_t row = a.joins[4 * which], c0 = a.joins[4 * which + 1], c1 = c0 + a.joins[4 * which + 2];
    const int tid = threadIdx.x, grp = tid / V, at = tid % V;
    float m = kNoMax;
    for (int s = c0 + (tid & 63); s < c1; s += 64) m = __builtin_fmaxf(m, a.part_ml[2 * ((size_t)s * a.q_heads + head)]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, o, 64));
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int s = c0 + grp; s < c1; s += NG) {
        const size_t i = (size_t)s * a.q_heads + head;
        const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * i] - m);
        l = __builtin_fmaf(f, a.part_ml[2 * i + 1], l);
        const f32x4 p = *reinterpret_cast<const f32x4*>(a.part_y + i * D + 4 * at);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = __builtin_fmaf(f, p[k], y[k]);
    }
    s_y[grp][at] = y;
    if (at == 0) s_l[grp] = l;
    __syncthreads();
    if (tid >= 64) return;
    // the first wave: lane's coordinates 4 at .. 4 at + 3 (head_dim 64 and 128: several times over)
    y = s_y[0][at];
    l = s_l[0];
    for (int i = 1; i < NG; ++i) {
        y += s_y[i][at];
        l += s_l[i];
    }
    const float p0 = y[0] + y[1], p1 = y[0] - y[1], p2 = y[2] + y[3], p3 = y[2] - y[3];
    y = f32x4{p0 + p2, p1 + p3, p0 - p2, p1 - p3};
#pragma unroll
    for (int o = 1; o < V; o <<= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float mine = y[k], other = __shfl_xor(mine, o, 64);
            y[k] = (at & o) ? other - mine : mine + other;
        }
    if (tid >= V) return;
    const float f = l == 0.0f ? 0.0f : a.hscale / l;
    *reinterpret_cast<u32x2*>(a.out + (int64_t)row * a.o_row + head * a.o_head + 4 * at) =
        u32x2{pack2<QDT>(y[0] * f, y[1] * f), pack2<QDT>(y[2] * f, y[3] * f)};
}

// ------------------------------------------------------------------ many rows ----

// 32 rows a wave (nq_flash.h), 64 tokens a stage in one of two LDS buffers: codes come into registers a stage ahead, go to
// LDS as fp16 (n - 8, exactly) while the other buffer is attended to, and their scales as fp32: the keys' times the
// logits, the values' times the weights.  With few rows several waves share them and split a stage's two tiles; their sums
// are joined in LDS.
// A stage's words are kept in the order of nibble_pair: place 2 j of 8 is coordinate j, place 2 j + 1 coordinate j + 4.
constexpr int kWideStage = 64;

template <int D, int NW>
struct WideShape {
    static constexpr int THREADS = 64 * NW, ROWS = 32 * NW;
    static constexpr int UNITS = 4 * D;                            // 16-byte pieces of a stage's codes
    static constexpr int PER = (UNITS + THREADS - 1) / THREADS;    // a thread
    static constexpr int LOOKUPS = UNITS / 2 > THREADS ? UNITS / 2 / THREADS : 1;  // rows of a thread's pieces
    static constexpr int PER_SIMD = D == 256 ? 1 : NW / 4 > 2 ? NW / 4 : 2;
};

template <int D, int QDT, int NW>
__global__ __launch_bounds__((WideShape<D, NW>::THREADS)) __attribute__((amdgpu_waves_per_eu(WideShape<D, NW>::PER_SIMD))) void
wide_kernel(FourBitArgs a) {
    using T = Tile<D>;
    using W = WideShape<D, NW>;
    constexpr int ROWB = T::ROWB, NT = W::THREADS, RB = D / 2, PR = D / 32;  // pieces a row
    static_assert(W::LOOKUPS == 1 || W::PER == 2 * W::LOOKUPS, "keys' and values' pieces of a thread are of the same rows");
    __shared__ __align__(16) char s_kv[2][2 * kWideStage * ROWB];
    __shared__ __align__(16) float s_k[2][kWideStage], s_v[2][kWideStage];
    __shared__ int s_exp[2];
    __shared__ float s_m[NW][32], s_l[NW][32];
    static_assert(sizeof(s_kv) >= NW * 32 * D * 4, "the waves' sums must fit the stage buffers");

    const int lane = threadIdx.x & 63, n = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t item = div(blockIdx.x, a.by_kv), kh = blockIdx.x - item * a.kv_heads;
    const Item it = item_of(a, item, W::ROWS, 0x7fffffff);
    const int n_stages = (it.n_tok + kWideStage - 1) / kWideStage;

    // ---- tokens: places past the chunk repeat its last (no row sees them) ----
    auto page_of = [&](int i, uint32_t& off) {
        const uint32_t t = (uint32_t)(it.tok0 + min(i, it.n_tok - 1)), p = div(t, a.by_tokens);
        off = t - p * a.tokens;
        return (uint32_t)it.pages[p];
    };
    // a thread's pieces: piece u = NT i + thread, keys first; row u % (UNITS / 2) / PR of the stage
    auto piece_row = [&](int i) { return ((i * NT + (int)threadIdx.x) % (W::UNITS / 2)) / PR; };
    uint32_t page[W::LOOKUPS], off[W::LOOKUPS], s_page = 0, s_off = 0;
    auto look_up = [&](int stage) {
#pragma unroll
        for (int i = 0; i < W::LOOKUPS; ++i) page[i] = page_of(kWideStage * stage + piece_row(i), off[i]);
        if (wave == 0) s_page = page_of(kWideStage * stage + lane, s_off);
    };
    u32x4 code[W::PER];
    uint16_t ks = 0, vs = 0;
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < W::PER; ++i) {
            const int u = i * NT + (int)threadIdx.x, k = i % W::LOOKUPS;
            if (W::UNITS % NT == 0 || u < W::UNITS) {
                const bool value = u >= W::UNITS / 2;
                const size_t row = ((size_t)page[k] * a.kv_heads + kh) * a.tokens + off[k];
                code[i] = *reinterpret_cast<const u32x4*>((value ? a.pool.codes[1] : a.pool.codes[0]) + row * RB + 16 * (u % PR));
            }
        }
        if (wave == 0) {
            const size_t row = ((size_t)s_page * a.kv_heads + kh) * a.tokens + s_off;
            ks = a.pool.scales[0][row];
            vs = a.pool.scales[1][row];
        }
    };
    // The values' scales times 2^(7 - e), e the exponent of the largest so far: weights (2^kSlack at most) stay below 2^15.
    // e grows seldom; the sums are then rescaled.
    int vexp = -40;
    auto store = [&](int buf) {
        char* const kv = s_kv[buf];
#pragma unroll
        for (int i = 0; i < W::PER; ++i) {
            const int u = i * NT + (int)threadIdx.x;
            if (W::UNITS % NT == 0 || u < W::UNITS) {
                const bool value = u >= W::UNITS / 2;
                const int r = piece_row(i), f = value ? T::value_swizzle(r) : T::key_swizzle(r);
                char* const to = kv + (value ? kWideStage * ROWB : 0) + r * ROWB;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t x = code[i][w];
                    const f16x2 bias = {(_Float16)-kNibbleBias, (_Float16)-kNibbleBias};
                    const f16x2 p[4] = {__builtin_bit_cast(f16x2, nibble_pair<0>(x)) + bias, __builtin_bit_cast(f16x2, nibble_pair<1>(x)) + bias,
                                        __builtin_bit_cast(f16x2, nibble_pair<2>(x)) + bias, __builtin_bit_cast(f16x2, nibble_pair<3>(x)) + bias};
                    *reinterpret_cast<u32x4*>(to + 16 * ((4 * (u % PR) + w) ^ f)) =
                        u32x4{__builtin_bit_cast(uint32_t, p[0]), __builtin_bit_cast(uint32_t, p[1]), __builtin_bit_cast(uint32_t, p[2]),
                              __builtin_bit_cast(uint32_t, p[3])};
                }
            }
        }
        if (wave == 0) {
            const float v = f16_bits_to_f32(vs);
            float big = finite_scale(vs);
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) big = __builtin_fmaxf(big, __shfl_xor(big, o, 64));
            if (big > 0.0f) {
                int e;
                (void)__builtin_frexpf(big, &e);
                vexp = max(vexp, e);
            }
            s_k[buf][lane] = f16_bits_to_f32(ks);
            s_v[buf][lane] = __builtin_ldexpf(v, 7 - vexp);
            if (lane == 0) s_exp[buf] = vexp;
        }
    };
    look_up(0);
    load();
    look_up(1);

    // ---- this wave's queries ----
    int rw = 1;  // waves with rows of their own; the others share these rows and take the other tile of a stage
    while (rw < NW && it.n_rows > 32 * rw) rw *= 2;
    const int r0 = 32 * (wave % rw), tile0 = rw == NW ? 0 : wave / rw, tiles = rw == NW ? 2 : 1;
    const bool live = r0 < it.n_rows && tile0 < 2;
    Rows<NQ_F16, D> rows;
    float c;
    int lo, hi;
    {
        const RowAt my = row_at(a, (uint32_t)(it.r0 + min(r0 + n, it.n_rows - 1)), kh);
        seen_by(a, it, my.token, lo, hi);
        const uint16_t* const p = a.query + (int64_t)(it.q_row0 + (int)my.token) * a.q_row + my.head * a.q_head + 8 * g;
        float x[T::KS][8];
#pragma unroll
        for (int s = 0; s < T::KS; ++s) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p + 16 * s);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[s][2 * k] = unpack<QDT>(w[k] & 0xffffu);
                x[s][2 * k + 1] = unpack<QDT>(w[k] >> 16);
            }
        }
        // the transform: coordinate bits 0..2 (in a lane's eight), 4.. (the steps), 3 (the other half of the wave)
#pragma unroll
        for (int s = 0; s < T::KS; ++s)
#pragma unroll
            for (int len = 1; len < 8; len <<= 1)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (i & len) continue;
                    const float u = x[s][i], v = x[s][i + len];
                    x[s][i] = u + v;
                    x[s][i + len] = u - v;
                }
#pragma unroll
        for (int len = 1; len < T::KS; len <<= 1)
#pragma unroll
            for (int s = 0; s < T::KS; ++s) {
                if (s & len) continue;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = x[s][i], v = x[s + len][i];
                    x[s][i] = u + v;
                    x[s + len][i] = u - v;
                }
            }
        const float sign = g ? -1.0f : 1.0f;
        float big = 0.0f;
#pragma unroll
        for (int s = 0; s < T::KS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x2 h = halves(x[s][i]);
                x[s][i] = __builtin_fmaf(h.y, sign, h.x);
                big = __builtin_fmaxf(big, __builtin_fabsf(x[s][i]));
            }
        const int qexp = row_exponent(both_max(big));
        c = __builtin_ldexpf(a.c, -qexp);
        rows.init(lane);
#pragma unroll
        for (int s = 0; s < T::KS; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                rows.q[s][j] = pack2<NQ_F16>(__builtin_ldexpf(x[s][j], qexp), __builtin_ldexpf(x[s][j + 4], qexp));
    }
    store(0);
    load();
    look_up(2);
    __syncthreads();
    int cur = s_exp[0];

    auto scaled = [&](f32x16& s, const float* k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 f = *reinterpret_cast<const f32x4*>(k + 8 * i + 4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[4 * i + j] *= f[j];
        }
    };
    auto begin = [&](int buf) {
        const int e = s_exp[buf];
        if (e != cur) {
            const float f = __builtin_ldexpf(1.0f, cur - e);
            cur = e;
#pragma unroll
            for (int b = 0; b < T::DB; ++b) rows.o[b] *= f;
        }
    };
    // a stage that every row of the workgroup sees whole
    auto whole = [&](int buf) {
        if (!live) return;
        const char* const kbuf = s_kv[buf];
        const char* const vbuf = kbuf + kWideStage * ROWB;
#pragma unroll 1
        for (int t = tile0; t < tile0 + tiles; ++t) {
            f32x16 s = rows.logits(kbuf, t);
            scaled(s, s_k[buf] + 32 * t);
            float mx = s[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) mx = __builtin_fmaxf(mx, s[j]);
            rows.template raise<true>(mx, c);
            uint32_t p[8];
            rows.template weights<true>(s, c, p, s_v[buf] + 32 * t, g);
            rows.add_values(p, vbuf, t);
        }
    };
    // one that hides tokens from some rows: what they do not see enters neither their maximum nor their sums, whatever it holds
    auto masked = [&](int buf, int first) {
        if (!live) return;
        const char* const kbuf = s_kv[buf];
        const char* const vbuf = kbuf + kWideStage * ROWB;
#pragma unroll 1
        for (int t = tile0; t < tile0 + tiles; ++t) {
            const int from = lo - (first + 32 * t), to = hi - (first + 32 * t);
            if (!__any(from < 32 && to >= 0)) continue;
            f32x16 s = rows.logits(kbuf, t);
            scaled(s, s_k[buf] + 32 * t);
            float mx = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int key = acc_row(j, g);
                s[j] = key >= from && key <= to ? s[j] : -__builtin_inff();
                mx = __builtin_fmaxf(mx, s[j]);
            }
            rows.template raise<true>(mx, c);
            uint32_t p[8];
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 f = *reinterpret_cast<const f32x4*>(s_v[buf] + 32 * t + 8 * i + 4 * g);
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int key = 8 * i + 4 * g + k;
                    x[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + k], c, -rows.m));
                    sum += x[k];
                    x[k] = key >= from && key <= to ? x[k] * f[k] : 0.0f;
                }
                p[2 * i] = pack2<NQ_F16>(x[0], x[1]);
                p[2 * i + 1] = pack2<NQ_F16>(x[2], x[3]);
            }
            rows.l += sum;
            rows.add_values(p, vbuf, t);
        }
    };
    auto end = [&](int stage) {  // the next stage to the other buffer, the one after it into registers
        if (stage + 1 < n_stages) store((stage + 1) & 1);
        if (stage + 2 < n_stages) {
            load();
            look_up(stage + 3);
        }
        __syncthreads();
    };
    // Whole stages are [it0, it1): from the last row's window on, up to the first row's last token.
    int it0, it1;
    {
        int a0, a1, b0, b1;
        seen_by(a, it, div((uint32_t)it.r0, a.by_group), a0, a1);
        seen_by(a, it, div((uint32_t)(it.r0 + it.n_rows - 1), a.by_group), b0, b1);
        it0 = min((b0 + kWideStage - 1) / kWideStage, n_stages);
        it1 = max(min((a1 + 1) / kWideStage, n_stages), it0);
    }
    int at = 0;
#pragma unroll 1
    for (; at < it0; ++at) {
        begin(at & 1);
        masked(at & 1, kWideStage * at);
        end(at);
    }
#pragma unroll 1
    for (; at < it1; ++at) {
        begin(at & 1);
        whole(at & 1);
        end(at);
    }
#pragma unroll 1
    for (; at < n_stages; ++at) {
        begin(at & 1);
        masked(at & 1, kWideStage * at);
        end(at);
    }

    // ---- the waves' sums joined, and written ----
    const float lsum = both_sum(rows.l);
    if (g == 0) {
        s_m[wave][n] = rows.m;
        s_l[wave][n] = lsum;
    }
    __syncthreads();
    {
        float m = kNoMax;
        for (int w = wave % rw; w < NW; w += rw) m = __builtin_fmaxf(m, s_m[w][n]);
        const float f = __builtin_ldexpf(__builtin_amdgcn_exp2f(rows.m - m), cur - 7);
        // [wave][row][place], 16-byte chunks at chunk ^ row
        float* const area = reinterpret_cast<float*>(&s_kv[0][0]) + (wave * 32 + n) * D;
#pragma unroll
        for (int b = 0; b < T::DB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int to = (8 * b + 2 * i + g) ^ (n & 15);
                *reinterpret_cast<f32x4*>(area + 4 * to) = f32x4{rows.o[b][4 * i] * f, rows.o[b][4 * i + 1] * f,
                                                                 rows.o[b][4 * i + 2] * f, rows.o[b][4 * i + 3] * f};
            }
    }
    __syncthreads();
    auto slot_of = [&](int r) {
        const RowAt my = row_at(a, (uint32_t)(it.r0 + r), kh);
        return (size_t)(uint32_t)(it.slot0 + (int)my.token * it.slots) * a.q_heads + my.head;
    };
    for (int r = threadIdx.x; r < it.n_rows; r += NT) {
        const int w0 = r >> 5, q = r & 31;
        float m = kNoMax, l = 0.0f;
        for (int w = w0; w < NW; w += rw) m = __builtin_fmaxf(m, s_m[w][q]);
        for (int w = w0; w < NW; w += rw) l += s_l[w][q] * __builtin_amdgcn_exp2f(s_m[w][q] - m);
        *reinterpret_cast<f32x2*>(a.part_ml + 2 * slot_of(r)) = f32x2{m, l};
    }
    const float* const sums = reinterpret_cast<const float*>(&s_kv[0][0]);
    for (int i = threadIdx.x; i < it.n_rows * (D / 8); i += NT) {
        const int r = i / (D / 8), j = i % (D / 8), w0 = r >> 5, q = r & 31;
        f32x4 y0 = {}, y1 = {};
        for (int w = w0; w < NW; w += rw) {
            y0 += *reinterpret_cast<const f32x4*>(sums + (w * 32 + q) * D + 4 * ((2 * j) ^ (q & 15)));
            y1 += *reinterpret_cast<const f32x4*>(sums + (w * 32 + q) * D + 4 * ((2 * j + 1) ^ (q & 15)));
        }
        float* const to = a.part_y + slot_of(r) * D + 8 * j;  // places to coordinates
        *reinterpret_cast<f32x4*>(to) = f32x4{y0[0], y0[2], y1[0], y1[2]};
        *reinterpret_cast<f32x4*>(to + 4) = f32x4{y0[1], y0[3], y1[1], y1[3]};
    }
}

template <int D, int QDT>
static hipError_t launch_fourbit(FourBitArgs a, uint32_t n_wide, uint32_t n_few, uint32_t n_joins, hipStream_t s) {
    if (n_wide > 0) hipLaunchKernelGGL((wide_kernel<D, QDT, 4>), dim3(n_wide * a.kv_heads), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.items += (size_t)kItemInts * n_wide;
    if (n_few > 0) hipLaunchKernelGGL((few_kernel<D, QDT>), dim3(n_few * a.kv_heads), dim3(256), 0, s, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (n_joins > 0) hipLaunchKernelGGL((fourbit_join_kernel<D, QDT>), dim3(n_joins * a.q_heads), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int QDT>
static hipError_t fourbit_dims(int32_t d, const FourBitArgs& a, uint32_t n_wide, uint32_t n_few, uint32_t n_joins, hipStream_t s) {
    switch (d) {
        case 64: return launch_fourbit<64, QDT>(a, n_wide, n_few, n_joins, s);
        case 128: return launch_fourbit<128, QDT>(a, n_wide, n_few, n_joins, s);
        default: return launch_fourbit<256, QDT>(a, n_wide, n_few, n_joins, s);
    }
}

}  // namespace nq

extern "C" int32_t nq_fourbit_rows(int32_t kind) { return kind == 0 ? nq::WideShape<128, 4>::ROWS : nq::FewShape<128>::ROWS; }

extern "C" int32_t nq_fourbit_chunk_tokens(void) { return nq::FewShape<128>::CHUNK; }

extern "C" int64_t nq_fourbit_workspace(int32_t n_slots, int32_t q_heads, int32_t head_dim) {
    if (n_slots <= 0 || q_heads <= 0 || head_dim <= 0) return 0;
    return (int64_t)n_slots * q_heads * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int nq_fourbit_attention(const nq_fourbit_desc* d, void* stream) {
    using namespace nq;
    NQ_CHECK_ARG(d != nullptr, "nq_fourbit_attention: desc is NULL");
    if (int st = check_fourbit_pool(d->pool, d->layer, "nq_fourbit_attention")) return st;
    const nq_pool* p = d->pool;
    const int32_t dim = p->head_dim;
    NQ_CHECK_ARG(d->q_dtype == NQ_F16 || d->q_dtype == NQ_BF16, "nq_fourbit_attention: queries must be fp16 or bf16");
    NQ_CHECK_ARG(d->q_heads > 0 && d->q_heads % p->heads == 0, "nq_fourbit_attention: q_heads %d must be a positive multiple of the pool's %d",
                 d->q_heads, p->heads);
    NQ_CHECK_ARG(d->n_wide >= 0 && d->n_few >= 0 && d->n_joins >= 0 && d->n_slots >= 0 && d->sliding_window >= 0,
                 "nq_fourbit_attention: n_wide %d, n_few %d, n_joins %d, n_slots %d, sliding_window %d", d->n_wide, d->n_few, d->n_joins,
                 d->n_slots, d->sliding_window);
    NQ_CHECK_ARG(d->scale > 0.0f && d->scale < 1e30f, "nq_fourbit_attention: scale must be positive");
    const int64_t n_items = (int64_t)d->n_wide + d->n_few;
    if (n_items == 0 && d->n_joins == 0) return NQ_OK;
    NQ_CHECK_ARG(d->query && d->out && (n_items == 0 || (d->items && d->pages)) && (d->n_joins == 0 || d->joins),
                 "nq_fourbit_attention: query, out and the plan's arrays are required");
    NQ_CHECK_ARG(((uintptr_t)d->query & 15u) == 0 && ((uintptr_t)d->out & 7u) == 0 && ((d->q_stride[0] | d->q_stride[1]) & 7) == 0 &&
                     ((d->out_stride[0] | d->out_stride[1]) & 3) == 0,
                 "nq_fourbit_attention: query rows must be 16-byte aligned, out's 8-byte");
    NQ_CHECK_ARG((uint64_t)n_items * p->heads <= max_blocks(256) && (uint64_t)d->n_joins * d->q_heads <= max_blocks(256),
                 "nq_fourbit_attention: grid too large");
    NQ_CHECK_ARG((uint64_t)d->n_slots * d->q_heads < (1ull << 32), "nq_fourbit_attention: too many partial sums");
    const int64_t need = nq_fourbit_workspace(d->n_slots, d->q_heads, dim);
    NQ_CHECK_ARG(need == 0 || (d->workspace != nullptr && d->workspace_bytes >= need && ((uintptr_t)d->workspace & 15u) == 0),
                 "nq_fourbit_attention: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
    FourBitArgs a = {};
    a.query = static_cast<const uint16_t*>(d->query);
    a.out = static_cast<uint16_t*>(d->out);
    a.pool = fourbit_rows(p, d->layer);
    a.items = d->items;
    a.pages = d->pages;
    a.joins = d->joins;
    a.part_y = static_cast<float*>(d->workspace);
    a.part_ml = a.part_y + (size_t)d->n_slots * d->q_heads * dim;
    a.q_row = d->q_stride[0];
    a.q_head = d->q_stride[1];
    a.o_row = d->out_stride[0];
    a.o_head = d->out_stride[1];
    a.q_heads = (uint32_t)d->q_heads;
    a.kv_heads = (uint32_t)p->heads;
    a.group = a.q_heads / a.kv_heads;
    a.tokens = (uint32_t)p->tokens;
    a.by_tokens = fast_div(a.tokens);
    a.by_group = fast_div(a.group);
    a.by_kv = fast_div(a.kv_heads);
    a.window = d->sliding_window;
    a.step = d->causal ? 1 : 0;
    a.hscale = d->hadamard_scale;
    a.c = d->scale * 1.44269504088896340736f * d->hadamard_scale;
    hipStream_t s = (hipStream_t)stream;
    NQ_CHECK_HIP(d->q_dtype == NQ_F16 ? fourbit_dims<NQ_F16>(dim, a, (uint32_t)d->n_wide, (uint32_t)d->n_few, (uint32_t)d->n_joins, s)
                                      : fourbit_dims<NQ_BF16>(dim, a, (uint32_t)d->n_wide, (uint32_t)d->n_few, (uint32_t)d->n_joins, s));
    return NQ_OK;
}
