// Attention of packed queries over a cache held in 4 bits (nq_fourbit.h): decode steps, several new tokens of a sequence
// over its past and themselves, and queries that see all of another sequence's tokens.
//
// With q~ = H q, a token's codes n and scales s:
//   logit = scale * s_k sum q~ (n - 8)         out = H sum p s_v (n - 8)
// so nothing is undone a token: keys' codes go into int8 products with the query's two digits, values' into fp16 products with
// the weights, both exactly, and the transform is applied to a query before and to its output after.
//
// The host cuts each sequence's queries into tiles of rows (a row: a query token and one of the kv head's query heads) and its
// tokens into chunks.  A workgroup takes a tile, a chunk and a kv head: up to 16 rows few_kernel, bound by the codes' bytes or,
// where there are few, by launches; up to 128 or 256 rows wide_kernel, bound by instructions issued.  A chunk with all that a
// tile's rows see goes to the output as it is; of others a partial (maximum, sum, value sum) a row goes to the workspace, and
// fourbit_join_kernel joins a row's, transforms and rounds.
#include <type_traits>

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
__device__ __forceinline__ Item item_of(const FourBitArgs& a, uint32_t i, int most_rows) {
    const int32_t* const it = a.items + (size_t)kItemInts * i;
    Item x;
    x.pages = a.pages + it[0];
    x.tok0 = it[1];
    x.n_tok = max(it[2], 1);
    x.q_row0 = it[3];
    x.r0 = it[4];
    x.n_rows = min(max(it[5], 1), most_rows);  // what registers and LDS are for, whatever a plan from elsewhere holds
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

// Weights go into their products as fp16 numbers, times the values' scales and 2^lift, lift such that the largest scale that a
// row has seen is in [64, 128) then: with weights of 2^kSlack at most that is below 2^15, and what counts keeps its bits.  It is
// a row's own.  Scales that all of a workgroup's rows see lower it for all of them at once, as they come to LDS; others in the
// tiles that hide tokens, for those who see them: a token's scale changes nothing for a row before it.  (With one for all
// rows, a hidden token's scale 2^24 times the others' left an output 8e-3 from 64 bits, 2^28 times 0.1; 2.1e-4 and 2.6e-4 now.)
// One that is not finite lowers nothing.
constexpr float kMostLift = 31.0f;
__device__ __forceinline__ float scale_size(uint16_t bits) { return (bits & 0x7c00u) == 0x7c00u ? 0.0f : f16_bits_to_f32(bits & 0x7fffu); }
__device__ __forceinline__ float scale_size(float scale) {
    const float x = __builtin_fabsf(scale);
    return x <= 65504.0f ? x : 0.0f;
}
__device__ __forceinline__ float lift_of(float big) {
    int e = -24;
    if (big > 0.0f) (void)__builtin_frexpf(big, &e);
    return (float)(7 - e);
}

// ----------------------------------------------------------------------- queries ----

// A query's transform as whole numbers of 16 bits, 32512 its largest coordinate, in two int8 digits of base 256 (high: -127
// .. 127, low: -128 .. 127).  Codes are whole numbers too, so a logit's sum is exact in 32 bits, and what is rounded off of a
// coordinate, 2^-16 of the largest, is the only error.
constexpr float kQueryMax = 32512.0f;

// What multiplies a row's coordinates, and what then multiplies its logits, from its largest |coordinate| as bits (an
// infinity or a NaN is larger than any number: its row's logits are NaN).
__device__ __forceinline__ void query_scale(uint32_t big, float& to_int, float& from_int) {
    const float b = __builtin_bit_cast(float, max(big, 0x0da24260u));  // 1e-30
    to_int = kQueryMax / b;
    from_int = b / (16.0f * kQueryMax);  // (levels come 16 times as large)
}

// 16 coordinates in the order in which the codes' bytes come out of two words (Bytes): the high and the low digits' bytes.
__device__ __forceinline__ void query_digits(const float (&x)[16], float to_int, u32x4& high, u32x4& low) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            uint32_t h = 0, l = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int q = (int)__builtin_rintf(x[8 * w + 2 * k + odd] * to_int);
                const int hi = (q + 128) >> 8;
                h |= (uint32_t)(hi & 0xff) << (8 * k);
                l |= (uint32_t)(q & 0xff) << (8 * k);  // q - 256 hi
            }
            high[2 * w + odd] = h;
            low[2 * w + odd] = l;
        }
}

// Constants in registers that the compiler must not know: a VALU instruction takes no two literals, and with them a mask and
// what follows it are two.
struct Bytes {  // the levels of a word's nibbles as int8, times 16: coordinates 0, 2, 4, 6 and 1, 3, 5, 7
    uint32_t mask, sign;
    __device__ __forceinline__ void init() {
        mask = 0xf0f0f0f0u;
        sign = 0x80808080u;
        asm volatile("" : "+s"(mask));
        asm volatile("" : "+v"(sign));
    }
    __device__ __forceinline__ uint32_t even(uint32_t w) const { return ((w << 4) & mask) ^ sign; }
    __device__ __forceinline__ uint32_t odd(uint32_t w) const { return (w & mask) ^ sign; }
};
struct Pairs {  // nibbles j and j + 4 of a word as fp16 values 16 + n (nq_fourbit.h)
    uint32_t mask, sixteens;
    __device__ __forceinline__ void init() {
        mask = kNibbleMask;
        sixteens = kSixteens;
        asm volatile("" : "+s"(mask));
        asm volatile("" : "+v"(sixteens));
    }
    template <int J>
    __device__ __forceinline__ uint32_t get(uint32_t w) const { return nibble_pair<J>(w, mask, sixteens); }
};

// What a row's logits are multiplied by: above zero (what is not seen is -infinity, times zero a NaN), or NaN.
__device__ __forceinline__ float logit_factor(float c) { return c < 1.2e-38f ? 1.2e-38f : c; }

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

template <int N>
__device__ __forceinline__ void butterflies(float (&x)[N]) {
#pragma unroll
    for (int len = 1; len < N; len <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i & len) continue;
            const float u = x[i], v = x[i + len];
            x[i] = u + v;
            x[i + len] = u - v;
        }
}

// ------------------------------------------------------------------- few rows ----

// A wave takes 32 tokens at a time, from their codes to the output without LDS between:
//   S = K q~^T     16x16x64 int8 products, A: lane (token m, kg) the D / 32 words of its row from D / 32 kg on; B: queries'
//                  digits alike
//   O^T = V^T P^T  16x16x32 fp16 products; S came out as lane (query, kg) with tokens 4 kg + 0..3 of either half, which is
//                  the B operand as it stands; A: lane (m, kg) the D / 16 nibbles from D / 16 m on of these eight tokens,
//                  nibble j of all of them the operand of output tile j
// Values' codes stand in the operand as 16 + n; the 24 too much of each comes off by one more tile of ones, which sums the
// weights (n alone, as a subnormal number, would need fewer instructions, but the matrix cores then add to some 20 bits: one row
// of 131072 tokens is 5.4e-4 off for 2.1e-4).  Weights go in twice, as fp16 and what that rounds off: 22 bits.
//
// Where a section's tokens are and their scales stand in LDS, in one of three places: the next section's are written in the
// middle of this one, behind a barrier there a wave's last unit asks for the next section's first codes, and a wave that is
// ahead writes the section after that one, which no wave reads yet.
//
// Measured (a copy of 2 GiB reads and writes 4.9 TB/s): 64 rows up to 8192 tokens of 8 x 128 (335 MB) 64 us, 5.2 TB/s, and 4.8
// for the join; one row of 131072 (138 MB) 28 and 5.4; four rows of 1000 6.2 and 3.8.  Eight waves a workgroup were no faster where
// one takes a whole sequence (24 of up to 1500 tokens) and 5 to 10 % slower in the others.
template <int D>
struct FewShape {
    static constexpr int WAVES = 4, ROWS = 16;
    static constexpr int SECTION = 512, UNITS = SECTION / 32;  // tokens, and units of 32
    static constexpr int PER_SIMD = D == 256 ? 2 : 4;
};

template <int D>
struct FewLds {
    using F = FewShape<D>;
    f32x4 o[F::WAVES / 2][D / 16][64];
    uint32_t row[3][F::SECTION];                 // a token's row of this head
    float ks[3][F::SECTION], vs[3][F::SECTION];  // its scales
    uint8_t q[2][16][D + 16];                    // the queries' digits, high and low
    float factor[16], max[3][F::WAVES], m[F::WAVES / 2][16], l[F::WAVES / 2][16];
};

// The transform of 16 rows, four a wave: lane (bits 2, 3: row; 0, 1 and 4, 5: j) coordinates D / 16 j .. of one, so that all
// exchanges are lane permutations.  Digits and factors go to LDS.
template <int D, int QDT>
__device__ __forceinline__ void few_queries(const FourBitArgs& a, const Item& it, uint32_t kh, FewLds<D>& lds, int lane, int wave) {
    constexpr int N = D / 16;
    const int r = 4 * wave + ((lane >> 2) & 3), j = (lane & 3) | ((lane >> 4) << 2);
    const RowAt at = row_at(a, (uint32_t)(it.r0 + min(r, it.n_rows - 1)), kh);
    const uint16_t* const p = a.query + (int64_t)(it.q_row0 + (int)at.token) * a.q_row + at.head * a.q_head + N * j;
    float x[N];
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(p + i);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t both = w[k];
            x[i + 2 * k] = unpack<QDT>(both & 0xffffu);
            x[i + 2 * k + 1] = unpack<QDT>(both >> 16);
        }
    }
    butterflies(x);
    const float s0 = (lane & 1) ? -1.0f : 1.0f, s1 = (lane & 2) ? -1.0f : 1.0f, s4 = (lane & 16) ? -1.0f : 1.0f, s5 = (lane & 32) ? -1.0f : 1.0f;
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = __builtin_fmaf(x[i], s0, dpp_f32<kQuadXor1>(x[i]));
        x[i] = __builtin_fmaf(x[i], s1, dpp_f32<kQuadXor2>(x[i]));
        const f32x2 h = rows16(x[i]);
        const f32x2 g = halves(__builtin_fmaf(h.y, s4, h.x));
        x[i] = __builtin_fmaf(g.y, s5, g.x);
        big = max(big, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
    }
    big = max(big, dpp_u32<kQuadXor1>(big));
    big = max(big, dpp_u32<kQuadXor2>(big));
    big = max(big, (uint32_t)__shfl_xor((int)big, 16, 64));
    big = max(big, (uint32_t)__shfl_xor((int)big, 32, 64));
    float to_int, from_int;
    query_scale(big, to_int, from_int);
    if (j == 0) lds.factor[r] = from_int;
    // places of a word's coordinates: the even ones' bytes, then the odd ones'
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        int q[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) q[k] = (int)__builtin_rintf(x[i + k] * to_int);
        const int coordinate = N * j + i, word = coordinate & ~7, place = (coordinate & 7) >> 1;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            lds.q[0][r][word + 4 * k + place] = (uint8_t)((q[k] + 128) >> 8);
            lds.q[1][r][word + 4 * k + place] = (uint8_t)q[k];
        }
    }
}

// FAR: a layer's codes take more than 4 GiB.  Else an offset has 32 bits, and a load one instruction for its address, where three
// are needed for 64 (ten loads a unit of some 240): 2 to 5 % less time (64 rows up to 8192 tokens 73.9 and 72.3 us).
template <int D, int QDT, bool FAR>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(FewShape<D>::PER_SIMD))) void few_kernel(FourBitArgs a) {
    using F = FewShape<D>;
    constexpr int KW = D / 32, KS = D / 64, TILES = D / 16, NW = F::WAVES, NT = 64 * NW, RB = D / 2;
    constexpr int VW = D == 256 ? 2 : 1;  // words of a token's values a lane (head_dim 64: half of one)
    __shared__ __align__(16) FewLds<D> lds;
    const int lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t item = div(blockIdx.x, a.by_kv), kh = blockIdx.x - item * a.kv_heads;
    const Item it = item_of(a, item, F::ROWS);
    const int n_units = (it.n_tok + 31) / 32, n_sections = (n_units + F::UNITS - 1) / F::UNITS;

    // ---- tokens: places past the chunk repeat its last (no row sees them) ----
    uint32_t kcode[2][KW], vcode[8][VW];
    auto page_of = [&](int i, uint32_t& off) {
        const uint32_t t = (uint32_t)(it.tok0 + min(i, it.n_tok - 1)), p = div(t, a.by_tokens);
        off = t - p * a.tokens;
        return (uint32_t)it.pages[p];
    };
    auto row_in = [&](uint32_t page, uint32_t off) { return (page * a.kv_heads + kh) * a.tokens + off; };
    const uint32_t k_at = 4 * KW * kg, v_at = D == 64 ? 4 * (n16 >> 1) : 4 * VW * n16;
    auto code_at = [&](const uint8_t* base, uint32_t row, uint32_t at) {
        if constexpr (FAR) return reinterpret_cast<const uint32_t*>(base + ((size_t)row * RB + at));
        else return reinterpret_cast<const uint32_t*>(base + (row * RB + at));
    };
    auto load_keys = [&](int half, uint32_t row) {
        const uint32_t* const p = code_at(a.pool.codes[0], row, k_at);
        if constexpr (KW == 2) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p);
            kcode[half][0] = w.x;
            kcode[half][1] = w.y;
        } else {
#pragma unroll
            for (int s = 0; s < KW; s += 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(p + s);
#pragma unroll
                for (int i = 0; i < 4; ++i) kcode[half][s + i] = w[i];
            }
        }
    };
    auto load_values = [&](int i, uint32_t row) {
        const uint32_t* const p = code_at(a.pool.codes[1], row, v_at);
        if constexpr (VW == 1) vcode[i][0] = *p;
        else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p);
            vcode[i][0] = w.x;
            vcode[i][VW - 1] = w.y;
        }
    };
    // What every row sees are the chunk's tokens [whole0, whole1].
    int whole0, whole1;
    {
        int unused;
        seen_by(a, it, div((uint32_t)it.r0, a.by_group), unused, whole1);
        seen_by(a, it, div((uint32_t)(it.r0 + it.n_rows - 1), a.by_group), whole0, unused);
    }
    // A section's places, two a thread: pages, then rows and scales, then LDS, each asked for before it is needed.
    constexpr int PER = F::SECTION / NT;
    uint32_t page[PER], off[PER], row[PER];
    uint16_t ks[PER], vs[PER];
    auto look_up = [&](int section) {
#pragma unroll
        for (int i = 0; i < PER; ++i) page[i] = page_of(F::SECTION * section + NT * i + (int)threadIdx.x, off[i]);
    };
    auto load_scales = [&] {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            row[i] = row_in(page[i], off[i]);
            ks[i] = a.pool.scales[0][row[i]];
            vs[i] = a.pool.scales[1][row[i]];
        }
    };
    auto write = [&](int section, int place) {
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = NT * i + (int)threadIdx.x;
            lds.row[place][at] = row[i];
            lds.ks[place][at] = f16_bits_to_f32(ks[i]);
            lds.vs[place][at] = f16_bits_to_f32(vs[i]);
            const int t = F::SECTION * section + at;
            big = __builtin_fmaxf(big, t >= whole0 && t <= whole1 ? scale_size(vs[i]) : 0.0f);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) big = __builtin_fmaxf(big, __shfl_xor(big, o, 64));
        if (lane == 0) lds.max[place][wave] = big;
    };
    look_up(0);
    {
        uint32_t first_page[2], first_off[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) first_page[t] = page_of(32 * wave + 16 * t + n16, first_off[t]);
        load_scales();
#pragma unroll
        for (int t = 0; t < 2; ++t) load_keys(t, row_in(first_page[t], first_off[t]));
    }
    few_queries<D, QDT>(a, it, kh, lds, lane, wave);
    write(0, 0);
    look_up(1);
    const RowAt my = row_at(a, (uint32_t)(it.r0 + min(n16, it.n_rows - 1)), kh);
    int lo, hi;
    seen_by(a, it, my.token, lo, hi);
    __syncthreads();
    u32x4 qh[KS], ql[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        qh[s] = *reinterpret_cast<const u32x4*>(&lds.q[0][n16][(D / 4) * kg + 16 * s]);
        ql[s] = *reinterpret_cast<const u32x4*>(&lds.q[1][n16][(D / 4) * kg + 16 * s]);
    }
    const float c = logit_factor(a.c * lds.factor[n16]);
    auto values_at = [&](const uint32_t* first) {
        const u32x4 r0 = *reinterpret_cast<const u32x4*>(first + 4 * kg), r1 = *reinterpret_cast<const u32x4*>(first + 16 + 4 * kg);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_values(i, r0[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_values(4 + i, r1[i]);
    };
    values_at(lds.row[0] + 32 * min(wave, n_units - 1));
    load_scales();
    look_up(2);

    f32x4 o[TILES], wsum = {};
#pragma unroll
    for (int j = 0; j < TILES; ++j) o[j] = f32x4{};
    // m: c * (lagging) maximum - lift.  The power of two is in the sum of weights as well.
    float m = kNoMax, l = 0.0f, lift = kMostLift;
    Bytes bytes;
    Pairs pairs;
    bytes.init();
    pairs.init();
    const uint32_t pick_lo = D == 64 && (n16 & 1) ? 0x07060302u : 0x05040100u;
    const u32x4 ones = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
    auto rescale = [&](float f) {
        l *= f;
        wsum *= f;
#pragma unroll
        for (int j = 0; j < TILES; ++j) o[j] *= f;
    };
    auto lower = [&](float big) {  // scales that come may be larger than those before
        const float to = __builtin_fminf(lift, lift_of(big));
        if (__any(to < lift)) {
            rescale(__builtin_amdgcn_exp2f(to - lift));
            m += lift - to;
            lift = to;
        }
    };
    auto section_max = [&](int place) {
        float big = lds.max[place][0];
#pragma unroll
        for (int w = 1; w < NW; ++w) big = __builtin_fmaxf(big, lds.max[place][w]);
        return big;
    };
    // The 24 too much of each code, taken off once a section: sums of codes as they stand are up to 24 times the sum of weights,
    // and what their additions round off is of that size, however near to zero the values' sum is.  Taken off at the end
    // alone, an output was 2.7e-4 from 64 bits after 32768 tokens in a workgroup and 5.4e-4 after 131072, where fp16's own
    // rounding is 2.1e-4; now it is 2.1e-4 in all, and no case takes longer than by 1 in 100.
    auto fold = [&] {
#pragma unroll
        for (int j = 0; j < TILES; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = __builtin_fmaf(-kNibbleBias, wsum[i], o[j][i]);
        wsum = f32x4{};
    };
    int place = 0, next_place = 1;  // of this section and the next
    lower(section_max(0));
    auto unit = [&](int u, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const int in = u % F::UNITS, first = 32 * in;  // within the section; its last unit of this wave is UNITS - NW + wave
        const bool last = in >= F::UNITS - NW;
        const int ahead = u + NW < n_units ? (last ? 32 * wave : first + 32 * NW) : first;
        const uint32_t* const next = lds.row[last && u + NW < n_units ? next_place : place] + ahead;
        if (MASKED && (32 * u < whole0 || min(32 * u + 31, it.n_tok - 1) > whole1)) {
            float big = 0.0f;
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                const int at = 32 * u + 16 * t + 4 * kg;
                const f32x4 scale = *reinterpret_cast<const f32x4*>(lds.vs[place] + first + 16 * t + 4 * kg);
#pragma unroll
                for (int i = 0; i < 4; ++i) big = __builtin_fmaxf(big, at + i >= lo && at + i <= hi ? scale_size(scale[i]) : 0.0f);
            }
            lower(four_max(big));
            __builtin_amdgcn_sched_barrier(0);  // (or the logits' registers are taken beside these)
        }
        // ---- logits of 16 tokens twice ----
        float p[8], mx = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            i32x4 sh = {}, sl = {};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint32_t w0 = kcode[t][2 * k], w1 = kcode[t][2 * k + 1];
                const i32x4 v = {(int)bytes.even(w0), (int)bytes.odd(w0), (int)bytes.even(w1), (int)bytes.odd(w1)};
                sh = __builtin_amdgcn_mfma_i32_16x16x64_i8(v, __builtin_bit_cast(i32x4, qh[k]), sh, 0, 0, 0);
                sl = __builtin_amdgcn_mfma_i32_16x16x64_i8(v, __builtin_bit_cast(i32x4, ql[k]), sl, 0, 0, 0);
            }
            const int at = 32 * u + 16 * t + 4 * kg;
            const f32x4 scale = *reinterpret_cast<const f32x4*>(lds.ks[place] + first + 16 * t + 4 * kg);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = (float)((sh[i] << 8) + sl[i]) * scale[i];
                if constexpr (MASKED) v = at + i >= lo && at + i <= hi ? v : -__builtin_inff();
                p[4 * t + i] = v;
                mx = __builtin_fmaxf(mx, v);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) load_keys(t, next[16 * t + n16]);
        if constexpr (FAR) __builtin_amdgcn_sched_barrier(0);  // (20 bytes of scratch at head_dim 128 otherwise)
        // ---- weights ----
        mx *= c;
        if (__any(mx > m + lift + kSlack)) {
            const float to = __builtin_fmaxf(m, four_max(mx) - lift);
            rescale(__builtin_amdgcn_exp2f(m - to));
            m = to;
        }
        u32x4 w, rest;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int at = 32 * u + 16 * t + 4 * kg;
            const f32x4 scale = *reinterpret_cast<const f32x4*>(lds.vs[place] + first + 16 * t + 4 * kg);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(p[4 * t + i], c, -m));
                l += e;
                const float v = e * scale[i];
                p[4 * t + i] = !MASKED || (at + i >= lo && at + i <= hi) ? v : 0.0f;  // (a scale that is not seen may be NaN)
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
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    y[i] = __builtin_amdgcn_perm(vcode[2 * i + 1][k], vcode[2 * i][k], half ? 0x07060302u : pick_lo);
                auto tile = [&](int j, u32x4 v) {
                    f32x4& to = o[8 * k + 4 * half + j];
                    to = mfma16(v, rest, mfma16(v, w, to));
                };
                tile(0, u32x4{pairs.get<0>(y[0]), pairs.get<0>(y[1]), pairs.get<0>(y[2]), pairs.get<0>(y[3])});
                tile(1, u32x4{pairs.get<1>(y[0]), pairs.get<1>(y[1]), pairs.get<1>(y[2]), pairs.get<1>(y[3])});
                tile(2, u32x4{pairs.get<2>(y[0]), pairs.get<2>(y[1]), pairs.get<2>(y[2]), pairs.get<2>(y[3])});
                tile(3, u32x4{pairs.get<3>(y[0]), pairs.get<3>(y[1]), pairs.get<3>(y[2]), pairs.get<3>(y[3])});
            }
        values_at(next);
        if (last && u + NW < n_units) {  // the next section's scales
            fold();
            place = next_place;
            next_place = next_place == 2 ? 0 : next_place + 1;
            lower(section_max(place));
        }
    };
    // In the middle of a section that another one follows (so that every wave has all its units of it): the next one to LDS.
    auto middle = [&](int u) {
        const int section = u / F::UNITS;
        if (u % F::UNITS / NW != F::UNITS / NW / 2 || section + 1 >= n_sections) return;
        write(section + 1, next_place);
        load_scales();
        look_up(section + 3);
        __syncthreads();
    };
    const int u0 = (whole0 + 31) / 32, u1 = (whole1 + 1) / 32;  // units that every row sees whole: [u0, u1)
    int u = wave;
#pragma unroll 1
    for (; u < min(u0, n_units); u += NW) {
        middle(u);
        unit(u, std::true_type{});
    }
#pragma unroll 1
    for (; u < u1; u += NW) {
        middle(u);
        unit(u, std::false_type{});
    }
#pragma unroll 1
    for (; u < n_units; u += NW) {
        middle(u);
        unit(u, std::true_type{});
    }
    fold();

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
        if (step > 1) __syncthreads();
    }
    if (wave > 0) return;
    // lane (n, kg), register i of tile j: coordinate TILES (4 kg + i) + j
    if (it.slots == 0) {  // the row's only chunk: transformed and rounded here
        float y[4 * TILES];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < TILES; ++j) y[TILES * i + j] = o[j][i];
        butterflies(y);
        const float f = l == 0.0f ? 0.0f : a.hscale / l;
        const float sign16 = (lane & 16) ? -1.0f : 1.0f, sign32 = (lane & 32) ? -1.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < 4 * TILES; ++i) {
            const f32x2 h = rows16(y[i]);
            const f32x2 g = halves(__builtin_fmaf(h.y, sign16, h.x));
            y[i] = __builtin_fmaf(g.y, sign32, g.x) * f;
        }
        if (n16 >= it.n_rows) return;
        uint16_t* const to = a.out + (int64_t)(it.q_row0 + (int)my.token) * a.o_row + my.head * a.o_head + 4 * TILES * kg;
#pragma unroll
        for (int i = 0; i < 4 * TILES; i += 4)
            *reinterpret_cast<u32x2*>(to + i) = u32x2{pack2<QDT>(y[i], y[i + 1]), pack2<QDT>(y[i + 2], y[i + 3])};
        return;
    }
    if (n16 >= it.n_rows) return;
    const size_t slot = (size_t)(uint32_t)(it.slot0 + (int)my.token * it.slots) * a.q_heads + my.head;
    if (kg == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * slot) = f32x2{m, l};
    float* const y = a.part_y + slot * D + TILES * 4 * kg;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < TILES; j += 4)
            *reinterpret_cast<f32x4*>(y + TILES * i + j) = f32x4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]};
}

// ----------------------------------------------------------------------- joins ----

// The chunks' sums of a (query token, head) weighted and added in a fixed order, then the transform, h and the softmax's sum.
// A row that saw nothing is zero.  WIDE: a workgroup for it, D / 4 lanes a chunk; else a wave, all lanes a chunk (2900 tokens
// of 20 heads x 64 in one to three chunks: 59 us with workgroups, 9 with waves).  985 tokens of 32 x 128 in 2500 slots (41 MB)
// 15 us; a decode step's 3.3 to 5, a launch and two loads that wait for each other.
template <int D, int QDT, bool WIDE>
__global__ __launch_bounds__(256) void fourbit_join_kernel(FourBitArgs a, uint32_t n) {
    constexpr int V = WIDE ? 4 : D / 64, LANES = D / V, NG = (WIDE ? 256 : 64) / LANES;  // chunks at a time
    __shared__ float s_y[WIDE ? NG : 1][WIDE ? D : 1], s_l[NG];
    const uint32_t unit = WIDE ? blockIdx.x : 4u * blockIdx.x + (threadIdx.x >> 6);
    if (unit >= n) return;  // whole wave, and not WIDE's
    const uint32_t which = unit / a.q_heads, head = unit - which * a.q_heads;
    const int32_t row = a.joins[4 * which], c0 = a.joins[4 * which + 1], c1 = c0 + a.joins[4 * which + 2];
    const int tid = WIDE ? (int)threadIdx.x : (int)(threadIdx.x & 63), grp = tid / LANES, at = tid % LANES;
    float m = kNoMax;
    for (int s = c0 + (tid & 63); s < c1; s += 64) m = __builtin_fmaxf(m, a.part_ml[2 * ((size_t)s * a.q_heads + head)]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, o, 64));
    float y[V] = {}, l = 0.0f;
#pragma unroll 4
    for (int s = c0 + grp; s < c1; s += NG) {
        const size_t i = (size_t)s * a.q_heads + head;
        const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * i] - m);
        l = __builtin_fmaf(f, a.part_ml[2 * i + 1], l);
        const float* const p = a.part_y + i * D + V * at;
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = __builtin_fmaf(f, p[k], y[k]);
    }
    if constexpr (WIDE) {
#pragma unroll
        for (int k = 0; k < V; ++k) s_y[grp][V * at + k] = y[k];
        if (at == 0) s_l[grp] = l;
        __syncthreads();
        if (tid >= 64) return;
        // the first wave: lane's coordinates 4 at .. 4 at + 3 (head_dim 64 and 128: several times over)
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = 0.0f;
        for (int i = 0; i < NG; ++i) {
            l += s_l[i];
#pragma unroll
            for (int k = 0; k < V; ++k) y[k] += s_y[i][V * at + k];
        }
    }
    butterflies(y);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float mine = y[k], other = __shfl_xor(mine, o, 64);
            y[k] = (at & o) ? other - mine : mine + other;
        }
    if (tid >= LANES) return;
    const float f = l == 0.0f ? 0.0f : a.hscale / l;
    uint16_t* const to = a.out + (int64_t)row * a.o_row + head * a.o_head + V * at;
    if constexpr (V == 1) *to = (uint16_t)pack2<QDT>(y[0] * f, 0.0f);
#pragma unroll
    for (int k = 0; k + 1 < V; k += 2) *reinterpret_cast<uint32_t*>(to + k) = pack2<QDT>(y[k] * f, y[k + 1] * f);
}

// ------------------------------------------------------------------ many rows ----

// 32 rows a wave, 64 tokens a stage in one of two LDS buffers: codes come into registers a stage ahead and go to LDS while the
// other buffer is attended to, keys as int8 levels times 16, values as fp16 levels, exactly.  S^T = K q~^T on 32x32x32 int8
// products of two digits, O^T += V^T P^T as in nq_flash.h (Rows).  Scales go to LDS as fp32: the keys' times the logits, the
// values' times the weights.  With few rows several waves share them and split a stage's two tiles; the upper tile's sums are
// then joined to the lower's in LDS.
//
// Bound by instructions issued: 2048 query tokens x 4 heads over 32768 tokens of 8 x 128 take 1215 us, 872 TFLOP/s where a
// library product of 8192^3 reaches 1340; a CU issues in 81 % of its cycles, the matrix cores are busy in 40, the vector units
// in 65, LDS in 34, with nearly a cycle of bank conflicts for each of its instructions (which of them was not counted).  With
// head_dim 64 (850 us) half as much is done for a softmax's weight, with 256 (1024 tokens over 16384, 902 us) a wave a SIMD
// hides less.  Tried: scaled keys and values in fp16 for exact codes (no faster), two halves of a workgroup in opposite order
// (11 % slower), waves' priorities (0 to 6 % slower).
//
// Weights, times their values' scales, are rounded to fp16 once: with 11 bits an fp16 output is 2.6e-4 from 64 bits where its
// own rounding is 2.1e-4, and a bf16 output as near as without (1.7e-3).  A second product for the rest, as few rows have it,
// would be half as many matrix instructions again in a kernel that is bound by issue.
constexpr int kWideStage = 64;

template <int D, int NW>
struct WideShape {
    static constexpr int THREADS = 64 * NW, ROWS = 32 * NW;
    static constexpr int UNITS = 4 * D;                            // 16-byte pieces of a stage's codes
    static constexpr int PER = (UNITS + THREADS - 1) / THREADS;    // a thread
    static constexpr int LOOKUPS = UNITS / 2 > THREADS ? UNITS / 2 / THREADS : 1;  // rows of a thread's pieces
    static constexpr int KEYS = kWideStage * D, BUF = KEYS + 2 * kWideStage * D;   // bytes
    static constexpr int JOIN = NW / 2 * 32 * D * 4;
    static constexpr int LDS = 2 * BUF > JOIN ? 2 * BUF : JOIN;
    static constexpr int PER_SIMD = D == 256 ? 1 : 2;
};
// 16-byte chunk c of key row r stands at c ^ key_place(r): 16 rows at one chunk lie in all 64 banks.
template <int D>
__device__ __forceinline__ constexpr int key_place(int r) {
    return D == 64 ? (r >> 2) & 3 : D == 128 ? (r >> 1) & 7 : r & 15;
}

template <int D, int QDT, int NW>
__global__ __launch_bounds__((WideShape<D, NW>::THREADS)) __attribute__((amdgpu_waves_per_eu(WideShape<D, NW>::PER_SIMD))) void
wide_kernel(FourBitArgs a) {
    using T = Tile<D>;
    using W = WideShape<D, NW>;
    constexpr int ROWB = T::ROWB, NT = W::THREADS, RB = D / 2, PR = D / 32;  // pieces a row
    constexpr int QS = D / 32;                                               // steps of a logit
    static_assert(W::LOOKUPS == 1 || W::PER == 2 * W::LOOKUPS, "keys' and values' pieces of a thread are of the same rows");
    __shared__ __align__(16) char s_kv[W::LDS];
    __shared__ __align__(16) float s_k[2][kWideStage], s_v[2][kWideStage];
    __shared__ float s_lift[2];
    __shared__ float s_m[NW / 2][32], s_l[NW / 2][32];

    const int lane = threadIdx.x & 63, n = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t item = div(blockIdx.x, a.by_kv), kh = blockIdx.x - item * a.kv_heads;
    const Item it = item_of(a, item, W::ROWS);
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
    Bytes bytes;
    Pairs pairs;
    bytes.init();
    pairs.init();
    auto store = [&](int buf) {
        char* const kv = s_kv + buf * W::BUF;
#pragma unroll
        for (int i = 0; i < W::PER; ++i) {
            const int u = i * NT + (int)threadIdx.x;
            if (W::UNITS % NT == 0 || u < W::UNITS) {
                const int r = piece_row(i);
                if (u < W::UNITS / 2) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t w0 = code[i][2 * h], w1 = code[i][2 * h + 1];
                        *reinterpret_cast<u32x4*>(kv + r * D + 16 * ((2 * (u % PR) + h) ^ key_place<D>(r))) =
                            u32x4{bytes.even(w0), bytes.odd(w0), bytes.even(w1), bytes.odd(w1)};
                    }
                } else {
                    char* const to = kv + W::KEYS + r * ROWB;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t x = code[i][w];
                        const f16x2 bias = {(_Float16)-kNibbleBias, (_Float16)-kNibbleBias};
                        const uint32_t p[4] = {__builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, pairs.get<0>(x)) + bias),
                                               __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, pairs.get<1>(x)) + bias),
                                               __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, pairs.get<2>(x)) + bias),
                                               __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, pairs.get<3>(x)) + bias)};
                        // (0, 4), (1, 5), (2, 6), (3, 7) to (0, 1), (2, 3), (4, 5), (6, 7)
                        *reinterpret_cast<u32x4*>(to + 16 * ((4 * (u % PR) + w) ^ T::value_swizzle(r))) =
                            u32x4{__builtin_amdgcn_perm(p[1], p[0], 0x05040100u), __builtin_amdgcn_perm(p[3], p[2], 0x05040100u),
                                  __builtin_amdgcn_perm(p[1], p[0], 0x07060302u), __builtin_amdgcn_perm(p[3], p[2], 0x07060302u)};
                    }
                }
            }
        }
        if (wave == 0) {
            float big = scale_size(vs);
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) big = __builtin_fmaxf(big, __shfl_xor(big, o, 64));
            s_k[buf][lane] = f16_bits_to_f32(ks);
            s_v[buf][lane] = f16_bits_to_f32(vs);
            if (lane == 0) s_lift[buf] = lift_of(big);
        }
    };
    look_up(0);
    load();
    look_up(1);

    // ---- this wave's queries: lane (n, g) coordinates 32 s + 16 g .. + 15 ----
    int rw = 1;  // waves with rows of their own; the others share these rows and take the other tile of a stage
    while (rw < NW && it.n_rows > 32 * rw) rw *= 2;
    const int r0 = 32 * (wave % rw), tile0 = rw == NW ? 0 : wave / rw, tiles = rw == NW ? 2 : 1;
    const bool live = r0 < it.n_rows && tile0 < 2;
    Rows<NQ_F16, D> rows;  // its queries: the high digits, then the low ones
    float c;
    int lo, hi;
    {
        const RowAt my = row_at(a, (uint32_t)(it.r0 + min(r0 + n, it.n_rows - 1)), kh);
        seen_by(a, it, my.token, lo, hi);
        const uint16_t* const p = a.query + (int64_t)(it.q_row0 + (int)my.token) * a.q_row + my.head * a.q_head + 16 * g;
        float x[16 * QS];
#pragma unroll
        for (int s = 0; s < 2 * QS; ++s) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p + 32 * (s >> 1) + 8 * (s & 1));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[8 * s + 2 * k] = unpack<QDT>(w[k] & 0xffffu);
                x[8 * s + 2 * k + 1] = unpack<QDT>(w[k] >> 16);
            }
        }
        butterflies(x);
        const float sign = g ? -1.0f : 1.0f;
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < 16 * QS; ++i) {
            const f32x2 h = halves(x[i]);
            x[i] = __builtin_fmaf(h.y, sign, h.x);
            big = max(big, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
        }
        big = max(big, (uint32_t)__shfl_xor((int)big, 32, 64));
        float to_int, from_int;
        query_scale(big, to_int, from_int);
        c = logit_factor(a.c * from_int);
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            float part[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) part[i] = x[16 * s + i];
            query_digits(part, to_int, rows.q[s], rows.q[QS + s]);
        }
    }
    rows.init(lane);
    // A lane's places in a tile: of row n of the keys its chunks 2 s + g, of the values' rows block b's coordinates.  With the
    // buffer and the tile known when this is compiled the rest of an address is in the instruction.
    uint32_t k_at[QS], v_at[T::DB];
#pragma unroll
    for (int s = 0; s < QS; ++s) k_at[s] = (uint32_t)(n * D + 16 * ((2 * s + g) ^ key_place<D>(n)));
#pragma unroll
    for (int b = 0; b < T::DB; ++b) v_at[b] = (rows.v_at + 64u * (uint32_t)b) ^ rows.v_xor;
    store(0);
    load();
    look_up(2);
    __syncthreads();
    float lift = kMostLift;  // rows.m: c * (lagging) maximum - lift; the power of two is in the sum of weights as well

    auto logits = [&](const char* kbuf, const float* scales) {
        i32x16 sh = {}, sl = {};
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            const i32x4 k = *reinterpret_cast<const i32x4*>(kbuf + k_at[s]);
            sh = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, __builtin_bit_cast(i32x4, rows.q[s]), sh, 0, 0, 0);
            sl = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, __builtin_bit_cast(i32x4, rows.q[QS + s]), sl, 0, 0, 0);
        }
        f32x16 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 scale = *reinterpret_cast<const f32x4*>(scales + 8 * i + 4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)((sh[4 * i + j] << 8) + sl[4 * i + j]) * scale[j];
        }
        return x;
    };
    auto add_values = [&](const uint32_t (&p)[8], const char* vbuf) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const u32x4 w = {p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]};
#pragma unroll
            for (int b = 0; b < T::DB; ++b) {
                const char* const from = vbuf + 16 * s * ROWB + v_at[b];
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)from);
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)(from + 8 * ROWB));
                const u32x2 u = __builtin_bit_cast(u32x2, x), v = __builtin_bit_cast(u32x2, y);
                rows.o[b] = mfma<NQ_F16>(u32x4{u.x, u.y, v.x, v.y}, w, rows.o[b]);
            }
        }
    };
    auto lower = [&](float most) {
        const float to = __builtin_fminf(lift, most);
        if (__any(to < lift)) {
            const float f = __builtin_amdgcn_exp2f(to - lift);
            rows.m += lift - to;
            lift = to;
            rows.l *= f;
#pragma unroll
            for (int b = 0; b < T::DB; ++b) rows.o[b] *= f;
        }
    };
    // Where a stage has scales larger than those before, lift follows for all rows at once, and in a stage that hides tokens
    // from some by what a row sees of it.
    float top = kMostLift;  // no row's lift is more
    auto larger = [&](int buf, float& most) {
        most = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, s_lift[buf])));
        return most < top;
    };
    auto begin = [&](int buf) {
        float most;
        if (__builtin_expect(larger(buf, most), 0)) {
            top = most;
            lower(most);
        }
    };
    auto begin_masked = [&](int buf, int first) {
        float most, big = 0.0f;
        if (__builtin_expect(!live || !larger(buf, most), 1)) return;
#pragma unroll 1
        for (int i = 32 * tile0 + 4 * g; i < 32 * (tile0 + tiles); i += 8) {
            const f32x4 f = *reinterpret_cast<const f32x4*>(s_v[buf] + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) big = __builtin_fmaxf(big, first + i + k >= lo && first + i + k <= hi ? scale_size(f[k]) : 0.0f);
        }
        lower(lift_of(both_max(big)));
    };
    auto raise = [&](float mx) {
        mx = both_max(mx) * c;
        if (__any(mx > rows.m + lift + kSlack)) {
            const float to = __builtin_fmaxf(rows.m, mx - lift), f = __builtin_amdgcn_exp2f(rows.m - to);
            rows.m = to;
            rows.l *= f;
#pragma unroll
            for (int b = 0; b < T::DB; ++b) rows.o[b] *= f;
        }
    };
    // tile t of a stage that every row of the workgroup sees whole
    auto whole_tile = [&](const char* kv, const float* sk, const float* sv, int t) {
        const f32x16 s = logits(kv + 32 * D * t, sk + 32 * t);
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) mx = __builtin_fmaxf(mx, s[j]);
        raise(mx);
        uint32_t p[8];
        rows.template weights<true>(s, c, p, sv + 32 * t, g);
        add_values(p, kv + W::KEYS + 32 * ROWB * t);
    };
    auto whole = [&](int buf) {
        if (!live) return;
#pragma unroll 1
        for (int t = tile0; t < tile0 + tiles; ++t) whole_tile(s_kv + buf * W::BUF, s_k[buf], s_v[buf], t);
    };
    // one that hides tokens from some rows: what they do not see enters neither their maximum nor their sums, whatever it holds
    auto masked = [&](int buf, int first) {
        if (!live) return;
#pragma unroll 1
        for (int t = tile0; t < tile0 + tiles; ++t) {
            const int from = lo - (first + 32 * t), to = hi - (first + 32 * t);
            if (!__any(from < 32 && to >= 0)) continue;
            f32x16 s = logits(s_kv + buf * W::BUF + 32 * D * t, s_k[buf] + 32 * t);
            float mx = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int key = acc_row(j, g);
                s[j] = key >= from && key <= to ? s[j] : -__builtin_inff();
                mx = __builtin_fmaxf(mx, s[j]);
            }
            raise(mx);
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
            add_values(p, s_kv + buf * W::BUF + W::KEYS + 32 * ROWB * t);
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
        begin_masked(at & 1, kWideStage * at);
        masked(at & 1, kWideStage * at);
        end(at);
    }
    if (tiles == 2 && r0 < it.n_rows) {
        if ((at & 1) && at < it1) {
            begin(1);
            whole(1);
            end(at);
            ++at;
        }
#pragma unroll 1
        for (; at + 1 < it1; at += 2) {
            begin(0);
            whole_tile(s_kv, s_k[0], s_v[0], 0);
            whole_tile(s_kv, s_k[0], s_v[0], 1);
            end(at);
            begin(1);
            whole_tile(s_kv + W::BUF, s_k[1], s_v[1], 0);
            whole_tile(s_kv + W::BUF, s_k[1], s_v[1], 1);
            end(at + 1);
        }
    }
#pragma unroll 1
    for (; at < it1; ++at) {
        begin(at & 1);
        whole(at & 1);
        end(at);
    }
#pragma unroll 1
    for (; at < n_stages; ++at) {
        begin_masked(at & 1, kWideStage * at);
        masked(at & 1, kWideStage * at);
        end(at);
    }

    // ---- the upper tile's sums joined to the lower's (the stages' last barrier is behind all reads of them) ----
    float l = both_sum(rows.l), m = rows.m;
    uint32_t end_lane = threadIdx.x;  // what follows from the lane is worked out again: nothing of it is kept over the loops
    asm volatile("" : "+v"(end_lane));
    const int n2 = end_lane & 31, g2 = (end_lane >> 5) & 1;
    const RowAt to_row = row_at(a, (uint32_t)(it.r0 + min(r0 + n2, it.n_rows - 1)), kh);
    if (rw < NW) {
        // [wave][row][coordinate], 16-byte chunks at chunk ^ row
        float* const area = reinterpret_cast<float*>(s_kv) + ((wave % rw) * 32 + n2) * D;
        if (live && tile0 == 1) {
            if (g2 == 0) {
                s_m[wave % rw][n2] = m;
                s_l[wave % rw][n2] = l;
            }
#pragma unroll
            for (int b = 0; b < T::DB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(area + 4 * ((8 * b + 2 * i + g2) ^ (n2 & 15))) =
                        f32x4{rows.o[b][4 * i], rows.o[b][4 * i + 1], rows.o[b][4 * i + 2], rows.o[b][4 * i + 3]};
        }
        __syncthreads();
        if (tile0 != 0) return;
        const float mo = s_m[wave][n2], to = __builtin_fmaxf(m, mo);
        const float f = __builtin_amdgcn_exp2f(m - to), fo = __builtin_amdgcn_exp2f(mo - to);
        m = to;
        l = l * f + s_l[wave][n2] * fo;
#pragma unroll
        for (int b = 0; b < T::DB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(area + 4 * ((8 * b + 2 * i + g2) ^ (n2 & 15)));
#pragma unroll
                for (int k = 0; k < 4; ++k) rows.o[b][4 * i + k] = __builtin_fmaf(y[k], fo, rows.o[b][4 * i + k] * f);
            }
    }
    // lane (n, g), register 4 i + k of block b: coordinate 32 b + 8 i + 4 g + k
    if (it.slots == 0) {  // the row's only chunk: transformed and rounded here
        float y[16 * T::DB];
#pragma unroll
        for (int b = 0; b < T::DB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) y[16 * b + j] = rows.o[b][j];
        butterflies(y);
        const float sign = g2 ? -1.0f : 1.0f, f = l == 0.0f ? 0.0f : a.hscale / l;
#pragma unroll
        for (int i = 0; i < 16 * T::DB; ++i) {
            const f32x2 h = halves(y[i]);
            y[i] = __builtin_fmaf(h.y, sign, h.x) * f;
        }
        if (r0 + n2 >= it.n_rows) return;
        uint16_t* const to = a.out + (int64_t)(it.q_row0 + (int)to_row.token) * a.o_row + to_row.head * a.o_head + 4 * g2;
#pragma unroll
        for (int b = 0; b < T::DB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float* const v = y + 16 * b + 4 * i;
                *reinterpret_cast<u32x2*>(to + 32 * b + 8 * i) = u32x2{pack2<QDT>(v[0], v[1]), pack2<QDT>(v[2], v[3])};
            }
        return;
    }
    if (r0 + n2 >= it.n_rows) return;
    const size_t slot = (size_t)(uint32_t)(it.slot0 + (int)to_row.token * it.slots) * a.q_heads + to_row.head;
    if (g2 == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * slot) = f32x2{m, l};
    float* const to = a.part_y + slot * D + 4 * g2;
#pragma unroll
    for (int b = 0; b < T::DB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(to + 32 * b + 8 * i) =
                f32x4{rows.o[b][4 * i], rows.o[b][4 * i + 1], rows.o[b][4 * i + 2], rows.o[b][4 * i + 3]};
}

// Waves of a workgroup of many rows: at head_dim 256 registers leave one wave a SIMD.
template <int D>
constexpr int kManyWaves = D == 256 ? 4 : 8;

// Rows of at most this many chunks are joined a wave each.
constexpr uint32_t kWaveChunks = 16;

template <int D, int QDT>
static hipError_t launch_fourbit(FourBitArgs a, const uint32_t (&n_items)[3], uint32_t n_joins, uint32_t most_chunks, bool far, hipStream_t s) {
    for (int k = 0; k < 3; ++k) {
        if (n_items[k] == 0) continue;
        const dim3 grid(n_items[k] * a.kv_heads);
        if (k == 0) hipLaunchKernelGGL((wide_kernel<D, QDT, kManyWaves<D>>), grid, dim3(64 * kManyWaves<D>), 0, s, a);
        else if (k == 1) hipLaunchKernelGGL((wide_kernel<D, QDT, 4>), grid, dim3(256), 0, s, a);
        else if (far) hipLaunchKernelGGL((few_kernel<D, QDT, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((few_kernel<D, QDT, false>), grid, dim3(256), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        a.items += (size_t)kItemInts * n_items[k];
    }
    if (n_joins > 0) {
        const uint32_t n = n_joins * a.q_heads;
        if (most_chunks > kWaveChunks) hipLaunchKernelGGL((fourbit_join_kernel<D, QDT, true>), dim3(n), dim3(256), 0, s, a, n);
        else hipLaunchKernelGGL((fourbit_join_kernel<D, QDT, false>), dim3((n + 3) / 4), dim3(256), 0, s, a, n);
    }
    return hipGetLastError();
}

template <int QDT>
static hipError_t fourbit_dims(int32_t d, const FourBitArgs& a, const uint32_t (&n_items)[3], uint32_t n_joins, uint32_t most_chunks, bool far, hipStream_t s) {
    switch (d) {
        case 64: return launch_fourbit<64, QDT>(a, n_items, n_joins, most_chunks, far, s);
        case 128: return launch_fourbit<128, QDT>(a, n_items, n_joins, most_chunks, far, s);
        default: return launch_fourbit<256, QDT>(a, n_items, n_joins, most_chunks, far, s);
    }
}

}  // namespace nq

extern "C" int32_t nq_fourbit_rows(int32_t head_dim, int32_t kind) {
    if (kind == 2) return nq::FewShape<128>::ROWS;
    return kind == 0 && head_dim <= 128 ? 32 * nq::kManyWaves<128> : nq::WideShape<128, 4>::ROWS;
}

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
    NQ_CHECK_ARG(d->n_items[0] >= 0 && d->n_items[1] >= 0 && d->n_items[2] >= 0 && d->n_joins >= 0 && d->n_slots >= 0 && d->most_chunks >= 0 && d->sliding_window >= 0,
                 "nq_fourbit_attention: n_items %d, %d, %d, n_joins %d, n_slots %d, most_chunks %d, sliding_window %d", d->n_items[0],
                 d->n_items[1], d->n_items[2], d->n_joins, d->n_slots, d->most_chunks, d->sliding_window);
    NQ_CHECK_ARG(d->scale > 0.0f && d->scale < 1e30f, "nq_fourbit_attention: scale must be positive");
    const int64_t n_items = (int64_t)d->n_items[0] + d->n_items[1] + d->n_items[2];
    if (n_items == 0 && d->n_joins == 0) return NQ_OK;
    NQ_CHECK_ARG(d->query && d->out && (n_items == 0 || (d->items && d->pages)) && (d->n_joins == 0 || d->joins),
                 "nq_fourbit_attention: query, out and the plan's arrays are required");
    NQ_CHECK_ARG(((uintptr_t)d->query & 15u) == 0 && ((uintptr_t)d->out & 7u) == 0 && ((d->q_stride[0] | d->q_stride[1]) & 7) == 0 &&
                     ((d->out_stride[0] | d->out_stride[1]) & 3) == 0,
                 "nq_fourbit_attention: query rows must be 16-byte aligned, out's 8-byte");
    NQ_CHECK_ARG((uint64_t)n_items * p->heads <= max_blocks(512) && (uint64_t)d->n_joins * d->q_heads <= max_blocks(256),
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
    const uint32_t n[3] = {(uint32_t)d->n_items[0], (uint32_t)d->n_items[1], (uint32_t)d->n_items[2]};
    const bool far = (uint64_t)p->pages * p->heads * p->tokens * (uint64_t)(dim / 2) > 1ull << 32;
    NQ_CHECK_HIP(d->q_dtype == NQ_F16 ? fourbit_dims<NQ_F16>(dim, a, n, (uint32_t)d->n_joins, (uint32_t)d->most_chunks, far, s)
                                      : fourbit_dims<NQ_BF16>(dim, a, n, (uint32_t)d->n_joins, (uint32_t)d->most_chunks, far, s));
    return NQ_OK;
}
