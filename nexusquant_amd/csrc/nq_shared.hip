// Decode attention over a pool's pages for rows that share pages: what several rows begin
// with is read and decoded once for all of them.
//
// The host cuts the rows' tokens into segments: a run of pages and the batch rows that see all its
// tokens (a shared prefix: many rows; a row's own rest: one).  A workgroup takes a chunk of a segment's
// tokens, one kv head, and the segment's query rows (batch rows x the kv head's query heads), up to 16 of
// them (few_attn_kernel, below), 128 or 256 (shared_attn_kernel, two shapes).  The latter, stage by stage
// (128 tokens; 64),
//  1. decodes keys and values into LDS as fp16, all waves together: keys through the int8
//     matrix cores (nq_keymfma.h), scaled and rotated in fp32; values as their codes: their
//     scales go with the softmax weights, and the transform, which is linear, with a row's
//     sum (combine kernel);
//  2. attends (nq_flash.h): 32 query rows a wave and all tiles of the stage; with fewer rows
//     several waves share them and split the tiles, and their sums are joined in LDS at the end.
// A partial (maximum, sum, value sum) per query row and chunk goes to the workspace; the
// combine kernel joins a row's chunks.
//
// What bounds it: 512 query rows of 8 kv heads x 128 over 32768 tokens, a call 107 to 112 us by card (610 to 640
// TFLOP/s): 92 without the decoding (every wave reads every key and value from LDS), 67 without the attention, and they
// run under each other only in part.  Few rows: see there.
//
// Weights times scales keep fp16's 11 bits here; twice as many, as few rows have, are a second product for the values.
// us and error of fp16 outputs (2.1e-4 is their own rounding) with 11 and with 22, head_dim 128: 32 query rows x 32768
// tokens 34.2, 3.3e-4 and 34.7, 2.6e-4; 128 x 4096 24.8, 3.3e-4 and 26.1, 2.7e-4; 512 x 32768 107, 3.4e-4 and 129,
// 2.7e-4.  The other half of what is above 2.1e-4 is the keys'.
#include "nq_flash.h"
#include "nq_keymfma.h"
#include "nq_rowmath.h"

namespace nq {

using namespace flash;

// The shape of a workgroup.  MANY: rows count, so as many as the registers hold (32 a wave) share what is decoded,
// and a stage is decoded under the attention to the one before it; two stage buffers, 128 KB of LDS at head_dim
// 128 and 256, so one workgroup on a CU.  Not MANY: decoding counts, and several small workgroups on a CU hide
// each other's loads.  8 kv heads x 128, us a call: 512 query rows x 32768 tokens 107 (MANY) and 146; 128 rows x
// 16384 31.1 and 34.4, x 4096 21.7 and 24.0; 64 rows x 8192 21.2 and 24.5, x 4096 19.5 and 18.1.
template <int D, bool MANY>
struct Shape {
    static constexpr int WAVES = MANY && D <= 128 ? 8 : 4;
    static constexpr int STAGE = MANY && D > 128 ? 64 : 128;  // tokens
    static constexpr int BUFS = MANY ? 2 : 1;
    static constexpr int CHUNK = MANY ? 2048 : 1024;   // most tokens of a chunk: their places and scales stay in LDS
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int TILES = STAGE / 32;
    static constexpr int ROWS = 32 * WAVES;            // query rows
    static constexpr int UNITS = STAGE / 16 / WAVES;   // 16-token units a wave decodes
    static_assert(BUFS * 2 * STAGE * 2 * D >= WAVES * 32 * D * 4, "the waves' sums must fit the stage buffers");
    static constexpr int PER_SIMD = MANY ? WAVES / 4 : D == 64 ? 3 : D == 128 ? 2 : 1;  // waves
};
struct SharedArgs {
    const uint16_t* query;
    void* out;
    const int8_t* kc;
    const int8_t* vc;
    const uint16_t* ks;
    const uint16_t* vs;
    const int32_t* positions;
    const int32_t* items;     // [n_items * 8]: pages, first token, tokens, rows, batch rows, chunk
    const int32_t* pages;     // the segments' page numbers
    const int32_t* seg_rows;  // per segment and row: batch row, its first slot there
    const int32_t* row_slots; // [batch + 1]
    float* part_y;            // [slots, q_heads, D]
    float* part_ml;           // [slots, q_heads, 2]
    const float* rope_dm;
    const float* rope_dp;
    uint32_t q_heads, kv_heads, rope_n_pos, n_items, tokens;  // n_items: of the launch, from `items` on
    FastDiv by_tokens, by_group;
    float c;                  // log2(e) / scale_divisor
    float hscale;
};

// bf16 queries of a row to fp16, and the power of two taken out of them: scaled so that the row's
// largest is in [2^14, 2^15), where all of it that counts is exact in fp16 (8 bits of 11; what falls
// below 2^-24 is 2^-38 of the largest).
template <typename Words, typename Max>
__device__ __forceinline__ float bf16_queries(Words& q, Max row_max) {
    constexpr int N = sizeof(Words) / 4;
    uint32_t* const words = reinterpret_cast<uint32_t*>(&q);
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t w = words[i];
        big = __builtin_fmaxf(big, __builtin_fmaxf(__builtin_fabsf(bf16_bits_to_f32(w & 0xffffu)),
                                                   __builtin_fabsf(bf16_bits_to_f32(w >> 16))));
    }
    big = row_max(big);
    int e = 0;
    if (big > 0.0f && big < __builtin_inff()) (void)__builtin_frexpf(big, &e);
    e = max(e - 15, -126);  // bf16's subnormals: scaled as far as fp32 reaches
    const float f = __builtin_ldexpf(1.0f, -e);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t w = words[i];
        words[i] = pack2<NQ_F16>(bf16_bits_to_f32(w & 0xffffu) * f, bf16_bits_to_f32(w >> 16) * f);
    }
    return __builtin_ldexpf(1.0f, e);
}

// The values' scales go with the weights, so that the codes are exact in fp16 and one rounding is left.
// Times 2^vexp the chunk's largest is in [64, 128): weights (at most 2^kSlack) stay below 2^15, and keep
// their 11 bits down to 2^-20 of that.
template <int NW>
__device__ __forceinline__ int value_exponent(const float (&wave_max)[NW]) {
    float m = wave_max[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = __builtin_fmaxf(m, wave_max[w]);
    int e = 0;
    if (!(m > 0.0f && m < __builtin_inff())) return 0;
    (void)__builtin_frexpf(m, &e);
    return 7 - e;
}

// ------------------------------------------------------------------- few rows ----

// Up to 16 query rows of a kv head: a wave takes 16 tokens at a time through 16x16x16 MFMAs, from their codes to the
// output without LDS between.  The int8 products leave a key's coordinates 16 t + 4 kg + i with lane (token, kg), which is
// how the next product takes its A operand: S = K q^T comes out as lane (query, kg) with tokens 4 kg + i, which is how
// P^T goes into O^T += V^T P^T.  For V^T lane (n, kg) reads the D / 16 bytes from D / 16 n on of tokens 4 kg + i and
// turns them four by four, so tile j of the output is coordinates D / 16 r + j.  Keys stay without scales, which go with
// the logits (sums of codes are below 2 D 127: they fit fp16).  Waves need no barriers; what a wave's next 16 tokens need
// is loaded into registers as soon as they are free, without a branch, so that the waits count only what they must.
//
// us a call here and in the small shape above: 2 rows x 2 heads of 32 kv heads x 128 over 6352 own tokens 33.8 and 43.5
// (3.1 TB/s of codes and scales), 64 x 8 of 8 over 512 27.4 and 33.4, 3 x 8 of 8 x 256 over 9184 38.3 and 66.2, 1 x 8 of 8
// x 128 over 131072 97 and 107.  Loads alone take some 70 % of the first's; the rest is conversions (some 280 vector
// instructions for 16 tokens of a head) and rows of the rotation table, twice the bytes of the codes, from L2.
template <int D>
struct Few {
    static constexpr int WAVES = 4, ROWS = 16;
    static constexpr int CHUNK = 1024;  // most tokens of a chunk
    static constexpr int PER_SIMD = D == 64 ? 4 : D == 128 ? 3 : 2;
};

// over the lanes n, n + 16, n + 32, n + 48
__device__ __forceinline__ f32x2 rows16(float v) {  // the values of lanes n and n ^ 16
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

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}

template <int D>
struct FewLds {
    float vs[Few<D>::CHUNK];     // a token's value scale
    uint32_t row[Few<D>::CHUNK]; // its row of this head
    uint32_t pos[Few<D>::CHUNK]; // its rotation table row, in bytes
    f32x4 o[Few<D>::WAVES / 2][D / 16][64];
    uint16_t ks[Few<D>::CHUNK];  // its key scale (fp16)
    float max[Few<D>::WAVES], m[Few<D>::WAVES / 2][16], l[Few<D>::WAVES / 2][16];
};

template <int D, int QDT>
__device__ __forceinline__ void few_chunk(const SharedArgs& a, FewLds<D>& lds, const int32_t* it, uint32_t kh) {
    using KM = KeyMfma<D>;
    using F = Few<D>;
    constexpr int T = KM::T, NW = F::WAVES, NT = 64 * NW;
    constexpr int TILES = D / 16, VW = D / 64;  // tiles of the output; dwords of a token's values a lane
    auto& s_row = lds.row;
    auto& s_pos = lds.pos;
    auto& s_vs = lds.vs;
    auto& s_ks = lds.ks;
    auto& s_max = lds.max;
    auto& s_m = lds.m;
    auto& s_l = lds.l;
    auto& s_o = lds.o;

    const int lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int32_t* const pages = a.pages + it[0];
    const uint32_t tok0 = (uint32_t)it[1];
    const int32_t* const seg_rows = a.seg_rows + 2 * it[3];
    const int G = (int)(a.q_heads / a.kv_heads), chunk = it[5];
    // what LDS is sized for, whatever a plan from elsewhere holds
    const int n_tok = (int)min(max((uint32_t)it[2], 1u), (uint32_t)F::CHUNK);
    const int n_q = (int)min(max((uint32_t)it[4] * (uint32_t)G, 1u), (uint32_t)F::ROWS);
    const int n_units = (n_tok + 15) / 16, last = 16 * n_units - 1;

    // ---- queries: B operands of coordinates 16 t + 4 kg + 0..3 of either half ----
    u32x2 q[2][T];
    {
        const uint32_t my_r = (uint32_t)min(n16, n_q - 1), my_br = div(my_r, a.by_group), my_head = kh * G + (my_r - my_br * G);
        const uint16_t* const p = a.query + ((size_t)(uint32_t)seg_rows[2 * my_br] * a.q_heads + my_head) * D + 4 * kg;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int t = 0; t < T; ++t) q[hf][t] = *reinterpret_cast<const u32x2*>(p + hf * (D / 2) + 16 * t);
    }

    // ---- the chunk's tokens; places past it repeat its last (with weight 0) ----
    auto row_of = [&](int i, uint32_t& page, uint32_t& off) {
        const uint32_t t = tok0 + min(i, n_tok - 1), p = div(t, a.by_tokens);
        off = t - p * a.tokens;
        page = (uint32_t)pages[p];
        return (page * a.kv_heads + kh) * a.tokens + off;
    };
    // Key codes a quad per token, 64 consecutive bytes, tables likewise: the operands want lane (token, kg), so the lanes
    // exchange them when they are used.
    uint32_t kcode[2][KM::NK][KM::W], vcode[4][VW];
    constexpr int DEPTH = T <= 4 ? T : 2;  // tiles of the tables on their way (registers)
    static_assert(T % DEPTH == 0, "a tile keeps its registers from token to token");
    f32x4 tm[DEPTH], tp[DEPTH];
    auto load_keys = [&](uint32_t lane, uint32_t row) {  // row: of token lane / 4
        const int8_t* const p = a.kc + (size_t)row * D + KM::KPL * (lane & 3u);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int s = 0; s < KM::NK; ++s) {
                const uint32_t* const w = reinterpret_cast<const uint32_t*>(p + hf * KM::HALF + s * KM::KB);
#pragma unroll
                for (int i = 0; i < KM::W; ++i) kcode[hf][s][i] = w[i];
            }
    };
    auto load_table = [&](int t, uint32_t tab) {
        tm[t % DEPTH] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(a.rope_dm) + (tab + 64u * t));
        tp[t % DEPTH] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(a.rope_dp) + (tab + 64u * t));
    };
    auto load_values = [&](uint32_t n16, int i, uint32_t row) {  // row: of token 4 kg + i
        const uint32_t* const w = reinterpret_cast<const uint32_t*>(a.vc + (size_t)row * D + (D / 16) * n16);
#pragma unroll
        for (int k = 0; k < VW; ++k) vcode[i][k] = w[k];
    };
    {
        uint32_t page, off;
        load_keys(lane, row_of(16 * wave + (lane >> 2), page, off));
    }
    float vmax = 0.0f;
    for (int i = threadIdx.x; i <= last; i += NT) {
        uint32_t page, off;
        const uint32_t row = row_of(i, page, off);
        const int32_t pos = a.positions[page * a.tokens + off];
        const float vs = i < n_tok ? f16_bits_to_f32(a.vs[row]) : 0.0f;
        s_row[i] = row;
        s_pos[i] = (pos < 0 ? 0u : ((uint32_t)pos >= a.rope_n_pos ? a.rope_n_pos - 1u : (uint32_t)pos)) * (2u * D);
        s_ks[i] = a.ks[row];
        s_vs[i] = vs;
        vmax = __builtin_fmaxf(vmax, __builtin_fabsf(vs));
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) vmax = __builtin_fmaxf(vmax, __shfl_xor(vmax, o, 64));
    if (lane == 0) s_max[wave] = vmax;
    float c = a.c * (0.5f * a.hscale);
    if constexpr (QDT == NQ_BF16) c *= bf16_queries(q, [](float v) { return four_max(v); });
    KM signs;
    signs.init(lane);
    __syncthreads();
    const int vexp = value_exponent<NW>(s_max);  // used with the weights, not in place: no second pass over s_vs

    uint32_t tab;
    {
        const int first = min(16 * wave, last - 15);
        tab = s_pos[first + (lane >> 2)] + 16u * (lane & 3);
#pragma unroll
        for (int t = 0; t < DEPTH; ++t) load_table(t, tab);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_values(n16, i, s_row[first + 4 * kg + i]);
        __builtin_amdgcn_sched_barrier(0);
    }

    f32x4 o[TILES];
#pragma unroll
    for (int j = 0; j < TILES; ++j) o[j] = f32x4{};
    float m = kNoMax, l = 0.0f;
    const float vmul = __builtin_ldexpf(1.0f, vexp);
#pragma unroll 1
    for (int u = wave; u < n_units; u += NW) {
        // what follows from the lane alone is worked out again each time, as in decode
        uint32_t lane = threadIdx.x;
        asm volatile("" : "+v"(lane));
        lane &= 63u;
        const uint32_t n16 = lane & 15u, kg = lane >> 4;
        const int from_quad = (int)(4 * (4 * n16 + kg));  // byte address of the lane that loaded this lane's block
        KM km = signs;
#pragma unroll
        for (int w = 0; w < KM::W; ++w) asm volatile("" : "+v"(km.h[w]));
        const int next = 16 * min(u + NW, n_units - 1);
        uint32_t code[2][KM::NK][KM::W];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int s = 0; s < KM::NK; ++s)
#pragma unroll
                for (int i = 0; i < KM::W; ++i) code[hf][s][i] = (uint32_t)__builtin_amdgcn_ds_bpermute(from_quad, (int)kcode[hf][s][i]);
        load_keys(lane, s_row[next + (lane >> 2)]);
        const uint32_t next_tab = s_pos[next + (lane >> 2)] + 16u * (lane & 3u);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 s = {};
#pragma unroll
        for (int t = 0; t < T; ++t) {
            f32x4 dm, dp;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = tm[t % DEPTH][i], y = tp[t % DEPTH][i];  // (an element is taken out before it is cast)
                dm[i] = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(from_quad, __builtin_bit_cast(int, x)));
                dp[i] = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(from_quad, __builtin_bit_cast(int, y)));
            }
            if (t + DEPTH < T) load_table(t + DEPTH, tab);
            else load_table(t + DEPTH - T, next_tab);
            int4v y0 = {0, 0, 0, 0}, y1 = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KM::NK; ++k) {
                y0 = km.mul(t, k, lane, code[0][k], y0);
                y1 = km.mul(t, k, lane, code[1][k], y1);
            }
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float lo = (float)y0[i], hi = (float)y1[i];
                x[i] = __builtin_fmaf(-lo, dm[i], hi * dp[i]);
                x[4 + i] = __builtin_fmaf(lo, dp[i], hi * dm[i]);
            }
            s = mfma16(u32x2{pack2<NQ_F16>(x[0], x[1]), pack2<NQ_F16>(x[2], x[3])}, q[0][t], s);
            s = mfma16(u32x2{pack2<NQ_F16>(x[4], x[5]), pack2<NQ_F16>(x[6], x[7])}, q[1][t], s);
            __builtin_amdgcn_sched_barrier(0);
        }
        tab = next_tab;
        // ---- weights ----
        const int at = 16 * u + 4 * (int)kg, left = n_tok - at;
        const u32x2 kw = *reinterpret_cast<const u32x2*>(s_ks + at);
        const f32x4 vs = *reinterpret_cast<const f32x4*>(s_vs + at);
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = s[i] * f16_bits_to_f32((i & 1) ? kw[i / 2] >> 16 : kw[i / 2] & 0xffffu);
            s[i] = i < left ? x * c : -__builtin_inff();
            mx = __builtin_fmaxf(mx, s[i]);
        }
        if (__any(mx > m + kSlack)) {
            const float to = __builtin_fmaxf(m, four_max(mx));
            const float f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int j = 0; j < TILES; ++j) o[j] *= f;
        }
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(s[i] - m);
            l += p[i];
            p[i] *= vs[i] * vmul;
        }
        // Weights in fp16 and what that rounds off of them, in fp16 too: 1 to 3 % of the time for an error of fp16 outputs
        // of 2.7e-4 instead of 3.1e-4 (2.1e-4 is their own rounding; the rest is the keys').
        const u32x2 w = {pack2<NQ_F16>(p[0], p[1]), pack2<NQ_F16>(p[2], p[3])};
        const u32x2 rest = {pack2<NQ_F16>(p[0] - f16_bits_to_f32(w.x & 0xffffu), p[1] - f16_bits_to_f32(w.x >> 16)),
                            pack2<NQ_F16>(p[2] - f16_bits_to_f32(w.y & 0xffffu), p[3] - f16_bits_to_f32(w.y >> 16))};
        // ---- values: bytes to fp16 as codes_to_f16, four tokens of a coordinate together ----
#pragma unroll
        for (int k = 0; k < VW; ++k) {
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = vcode[i][k] ^ 0x80808080u;
            const uint32_t pairs[2][2] = {{__builtin_amdgcn_perm(x[1], x[0], 0x05010400u), __builtin_amdgcn_perm(x[3], x[2], 0x05010400u)},
                                          {__builtin_amdgcn_perm(x[1], x[0], 0x07030602u), __builtin_amdgcn_perm(x[3], x[2], 0x07030602u)}};
            const half2v bias = {(__fp16)-1152.0f, (__fp16)-1152.0f};
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t sel = (b & 1) ? 0x00070006u : 0x00050004u;
                const half2v v0 = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(pairs[b / 2][0], 0x64646464u, sel)) + bias;
                const half2v v1 = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(pairs[b / 2][1], 0x64646464u, sel)) + bias;
                const u32x2 v = {__builtin_bit_cast(uint32_t, v0), __builtin_bit_cast(uint32_t, v1)};
                o[4 * k + b] = mfma16(v, rest, mfma16(v, w, o[4 * k + b]));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_values(n16, i, s_row[next + 4 * kg + i]);
    }

    // ---- the waves' sums joined: the upper half's into the lower half's, twice ----
    uint32_t end_lane = threadIdx.x;  // as in the loop: nothing of the lane is kept over it
    asm volatile("" : "+v"(end_lane));
    const int lane2 = end_lane & 63, n = lane2 & 15, g = lane2 >> 4;
    l = four_sum(l);
#pragma unroll
    for (int step = NW / 2; step >= 1; step >>= 1) {
        if (wave >= step && wave < 2 * step) {
#pragma unroll
            for (int j = 0; j < TILES; ++j) s_o[wave - step][j][lane2] = o[j];
            if (g == 0) {
                s_m[wave - step][n] = m;
                s_l[wave - step][n] = l;
            }
        }
        __syncthreads();
        if (wave < step) {
            const float mo = s_m[wave][n], to = __builtin_fmaxf(m, mo);
            const float f = __builtin_amdgcn_exp2f(m - to), fo = __builtin_amdgcn_exp2f(mo - to);
            m = to;
            l = l * f + s_l[wave][n] * fo;
#pragma unroll
            for (int j = 0; j < TILES; ++j) {
                const f32x4 y = s_o[wave][j][lane2];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j][i] = __builtin_fmaf(y[i], fo, o[j][i] * f);
            }
        }
        __syncthreads();
    }
    if (wave > 0 || n >= n_q) return;
    const uint32_t my_br = div((uint32_t)n, a.by_group), my_head = kh * G + ((uint32_t)n - my_br * G);
    const size_t slot = (size_t)(uint32_t)(seg_rows[2 * my_br + 1] + chunk) * a.q_heads + my_head;
    if (g == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * slot) = f32x2{m, l};
    const float f = __builtin_ldexpf(0.5f, -vexp);
    float* const y = a.part_y + slot * D + (D / 16) * 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < VW; ++k)
            *reinterpret_cast<f32x4*>(y + (D / 16) * i + 4 * k) = f32x4{o[4 * k][i] * f, o[4 * k + 1][i] * f, o[4 * k + 2][i] * f, o[4 * k + 3][i] * f};
}

template <int D, int QDT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Few<D>::PER_SIMD))) void few_attn_kernel(SharedArgs a) {
    __shared__ __align__(16) FewLds<D> lds;
    const uint32_t in_xcd = blockIdx.x >> 3, item = (blockIdx.x & 7u) + 8u * (in_xcd / a.kv_heads);  // as in shared_attn_kernel
    if (item < a.n_items) few_chunk<D, QDT>(a, lds, a.items + 8 * item, in_xcd % a.kv_heads);
}

// -------------------------------------------------------------- some rows, many ----

template <int D, int QDT, bool MANY>
__global__ __launch_bounds__((Shape<D, MANY>::THREADS)) __attribute__((amdgpu_waves_per_eu(Shape<D, MANY>::PER_SIMD))) void
shared_attn_kernel(SharedArgs a) {
    using T = Tile<D>;
    using KM = KeyMfma<D>;
    using SH = Shape<D, MANY>;
    constexpr int ROWB = T::ROWB, NT = SH::THREADS, NW = SH::WAVES, STAGE = SH::STAGE;
    __shared__ __align__(16) char s_kv[SH::BUFS][2 * STAGE * ROWB];  // stages of keys and values; at the end the waves' sums
    __shared__ uint32_t s_row[SH::CHUNK];    // a token's row of head 0
    __shared__ uint32_t s_pos[SH::CHUNK];    // its rotation table row, in bytes
    __shared__ __align__(16) float s_vs[SH::CHUNK];  // its value scale times 2^vexp
    __shared__ uint16_t s_ks[SH::CHUNK];     // its key scale (fp16)
    __shared__ float s_max[NW], s_m[NW][32], s_l[NW][32];
    __shared__ uint32_t s_slot[SH::ROWS];       // a query row's place among the partial sums

    const int lane = threadIdx.x & 63, n = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // block 8 i + x runs on XCD x: the kv heads of an item there, one after another, share its rows of
    // the rotation table in that XCD's L2 (the host puts items of one chunk 8 apart, for its codes)
    const uint32_t in_xcd = blockIdx.x >> 3, item = (blockIdx.x & 7u) + 8u * (in_xcd / a.kv_heads), kh = in_xcd % a.kv_heads;
    if (item >= a.n_items) return;  // whole block
    const int32_t* const it = a.items + 8 * item;
    if constexpr (!MANY) {
        static_assert(sizeof(FewLds<D>) <= sizeof(s_kv) && 64 * Few<D>::WAVES == NT, "a chunk of few rows in this launch");
        if (it[6] != 0) {
            few_chunk<D, QDT>(a, *reinterpret_cast<FewLds<D>*>(&s_kv), it, kh);
            return;
        }
    }
    const int32_t* const pages = a.pages + it[0];
    const uint32_t tok0 = (uint32_t)it[1];
    const int32_t* const seg_rows = a.seg_rows + 2 * it[3];
    const int G = (int)(a.q_heads / a.kv_heads), chunk = it[5];
    // what LDS is sized for, whatever a plan from elsewhere holds
    const int n_tok = (int)min(max((uint32_t)it[2], 1u), (uint32_t)SH::CHUNK);
    const int n_q = (int)min(max((uint32_t)it[4] * (uint32_t)G, 1u), (uint32_t)SH::ROWS);

    // The three chains of loads that the first stage waits for run at once: rows -> queries, pages -> codes,
    // pages -> positions and scales (-> rotation tables).
    // ---- this wave's queries ----
    int rw = 1;  // waves with rows of their own; the others share these rows and take other tiles
    while (rw < NW && n_q > 32 * rw) rw *= 2;
    const int per_wave = SH::TILES * rw < NW ? 1 : SH::TILES * rw / NW;   // tiles of a stage
    const int r0 = 32 * (wave % rw), tile0 = wave / rw * per_wave;
    const bool live = r0 < n_q && tile0 < SH::TILES;
    Rows<NQ_F16, D> rows;
    rows.init(lane);
    {
        const uint32_t r = (uint32_t)min(r0 + n, n_q - 1), br = div(r, a.by_group);
        const uint32_t head = kh * G + (r - br * G);
        const uint16_t* const q = a.query + ((size_t)(uint32_t)seg_rows[2 * br] * a.q_heads + head) * D + 8 * g;
#pragma unroll
        for (int i = 0; i < T::KS; ++i) rows.q[i] = *reinterpret_cast<const u32x4*>(q + 16 * i);
    }

    // ---- the codes of a unit, 16 tokens, to registers ----
    // Keys a quad per token, 64 consecutive bytes; the MFMA operands want token n16 and 16-byte block kg in
    // lane 16 kg + n16, so the lanes exchange them when they decode.
    constexpr int PIECES = D / 64;  // 16-byte pieces of a unit's values a lane
    uint32_t kcode[SH::UNITS][2][KM::NK][KM::W];
    u32x4 vcode[SH::UNITS][PIECES];
    auto load = [&](int s0, auto&& row_of) {
#pragma unroll
        for (int u = 0; u < SH::UNITS; ++u) {
            const int first = s0 + 16 * (SH::UNITS * wave + u);
            const int8_t* const p = a.kc + (size_t)row_of(first + (lane >> 2)) * D + KM::KPL * (lane & 3);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int s = 0; s < KM::NK; ++s) {
                    const uint32_t* const w = reinterpret_cast<const uint32_t*>(p + hf * KM::HALF + s * KM::KB);
#pragma unroll
                    for (int i = 0; i < KM::W; ++i) kcode[u][hf][s][i] = w[i];
                }
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const uint32_t j = 64u * i + lane;
                vcode[u][i] = *reinterpret_cast<const u32x4*>(a.vc + (size_t)row_of(first + j / (D / 16)) * D + 16 * (j % (D / 16)));
            }
        }
    };
    for (int r = threadIdx.x; r < n_q; r += NT) {
        const uint32_t br = div((uint32_t)r, a.by_group);
        s_slot[r] = (uint32_t)(seg_rows[2 * br + 1] + chunk) * a.q_heads + kh * G + ((uint32_t)r - br * G);
    }
    // a slot's place: slots past the chunk repeat its last token (with weight 0)
    const uint32_t head_rows = kh * a.tokens;
    auto page_of = [&](int i, uint32_t& off) {
        const uint32_t t = tok0 + min(i, n_tok - 1), p = div(t, a.by_tokens);
        off = t - p * a.tokens;
        return (uint32_t)pages[p];
    };
    load(0, [&](int i) {
        uint32_t off;
        const uint32_t page = page_of(i, off);
        return page * a.kv_heads * a.tokens + head_rows + off;
    });

    // ---- the chunk's tokens ----
    float vmax = 0.0f;
    const int n_slots = (n_tok + STAGE - 1) / STAGE * STAGE;
    for (int i = threadIdx.x; i < n_slots; i += NT) {
        uint32_t off;
        const uint32_t page = page_of(i, off), row = page * a.kv_heads * a.tokens + head_rows + off;
        const int32_t pos = a.positions[page * a.tokens + off];
        const float vs = i < n_tok ? f16_bits_to_f32(a.vs[row]) : 0.0f;
        s_row[i] = row;
        s_pos[i] = (pos < 0 ? 0u : ((uint32_t)pos >= a.rope_n_pos ? a.rope_n_pos - 1u : (uint32_t)pos)) * (2u * D);
        s_ks[i] = a.ks[row];
        s_vs[i] = vs;
        vmax = __builtin_fmaxf(vmax, __builtin_fabsf(vs));
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) vmax = __builtin_fmaxf(vmax, __shfl_xor(vmax, o, 64));
    if (lane == 0) s_max[wave] = vmax;
    float c = a.c;
    if constexpr (QDT == NQ_BF16) c *= bf16_queries(rows.q, [](float v) { return both_max(v); });
    KM signs;
    signs.init(lane);
    __syncthreads();
    const int vexp = value_exponent<NW>(s_max);
    for (int i = threadIdx.x; i < n_slots; i += NT) s_vs[i] = __builtin_ldexpf(s_vs[i], vexp);
    // Other waves use them: MANY behind the barrier after its first decode, the others' waves may go on by themselves.
    if constexpr (!MANY) __syncthreads();

    // The stage at s0 to LDS: its codes are in registers, and those of the stage after it follow.
    auto decode = [&](int s0, char* kbuf) {
        // what follows from the lane alone (operand signs, addresses) is worked out again in each stage:
        // kept across stages it would take 40 registers that the attention needs
        uint32_t lane = threadIdx.x;
        asm volatile("" : "+v"(lane));
        lane &= 63u;
        const uint32_t n16 = lane & 15u, kg = lane >> 4;
        const int from_quad = (int)(4 * (4 * n16 + kg));  // byte address of the lane that loaded this lane's block
        KM km = signs;
#pragma unroll
        for (int w = 0; w < KM::W; ++w) asm volatile("" : "+v"(km.h[w]));
        // The units' rows of the rotation tables, by way of the LDS that their keys and values will take:
        // they arrive a row per 16 lanes, and every lane then reads its own coordinates.
#pragma unroll
        for (int u = 0; u < SH::UNITS; ++u) {
            const int row0 = 16 * (SH::UNITS * wave + u);
            char* const krows = kbuf + row0 * ROWB;
            char* const vrows = krows + STAGE * ROWB;
#pragma unroll
            for (int i = 0; i < T::UPR / 4; ++i) {
                const uint32_t slot = 64u * i + lane, r = slot / T::UPR;
                const uint32_t tab = s_pos[s0 + row0 + r] + 16u * ((slot % T::UPR) ^ T::key_swizzle(r));
                __builtin_amdgcn_global_load_lds((global_void*)(reinterpret_cast<const char*>(a.rope_dm) + tab),
                                                 (lds_void*)(krows + 1024 * i), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((global_void*)(reinterpret_cast<const char*>(a.rope_dp) + tab),
                                                 (lds_void*)(vrows + 1024 * i), 16, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < SH::UNITS; ++u) {
            const int row0 = 16 * (SH::UNITS * wave + u);
            char* const krows = kbuf + row0 * ROWB;
            char* const vrows = krows + STAGE * ROWB;
            const float k_scale = (0.5f * f16_bits_to_f32(s_ks[s0 + row0 + n16])) * a.hscale;
            uint32_t code[2][KM::NK][KM::W];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int s = 0; s < KM::NK; ++s)
#pragma unroll
                    for (int i = 0; i < KM::W; ++i)
                        code[hf][s][i] = (uint32_t)__builtin_amdgcn_ds_bpermute(from_quad, (int)kcode[u][hf][s][i]);
            if (u == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tables are this wave's own: no barrier
            f32x4 tm[KM::T], tp[KM::T];
#pragma unroll
            for (int t = 0; t < KM::T; ++t) {
                const uint32_t at = n16 * ROWB + 16u * ((4u * t + kg) ^ (uint32_t)T::key_swizzle(n16));
                tm[t] = *reinterpret_cast<const f32x4*>(krows + at);
                tp[t] = *reinterpret_cast<const f32x4*>(vrows + at);
            }
            asm volatile("" ::: "memory");  // a wave's LDS accesses run in order: read before they are written over
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const uint32_t j = 64u * i + lane, r = j / (D / 16), piece = j % (D / 16);
                u32x4 o[2];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    half2v lo, hi;
                    codes_to_f16(vcode[u][i][k], lo, hi);
                    o[k / 2][2 * (k & 1)] = __builtin_bit_cast(uint32_t, lo);
                    o[k / 2][2 * (k & 1) + 1] = __builtin_bit_cast(uint32_t, hi);
                }
                const uint32_t f = T::value_swizzle(r);
                *reinterpret_cast<u32x4*>(vrows + r * ROWB + 16 * ((2 * piece) ^ f)) = o[0];
                *reinterpret_cast<u32x4*>(vrows + r * ROWB + 16 * ((2 * piece + 1) ^ f)) = o[1];
            }
            char* const to = krows + n16 * ROWB + 8 * (kg & 1);
#pragma unroll
            for (int t = 0; t < KM::T; ++t) {
                int4v y0 = {0, 0, 0, 0}, y1 = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < KM::NK; ++s) {
                    y0 = km.mul(t, s, lane, code[0][s], y0);
                    y1 = km.mul(t, s, lane, code[1][s], y1);
                }
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float lo = (float)y0[i] * k_scale, hi = (float)y1[i] * k_scale;
                    x[i] = __builtin_fmaf(-lo, tm[t][i], hi * tp[t][i]);
                    x[4 + i] = __builtin_fmaf(lo, tp[t][i], hi * tm[t][i]);
                }
                // coordinates 16 t + 4 kg + 0..3 and those D / 2 on: half a 16-byte chunk each
                const uint32_t chunk16 = 2u * t + (kg >> 1), f = T::key_swizzle(n16);
                *reinterpret_cast<u32x2*>(to + 16 * (chunk16 ^ f)) = u32x2{pack2<NQ_F16>(x[0], x[1]), pack2<NQ_F16>(x[2], x[3])};
                *reinterpret_cast<u32x2*>(to + 16 * ((chunk16 + D / 16) ^ f)) =
                    u32x2{pack2<NQ_F16>(x[4], x[5]), pack2<NQ_F16>(x[6], x[7])};
            }
            if constexpr (SH::UNITS > 1) __builtin_amdgcn_sched_barrier(0);  // one unit at a time in registers
        }
        if (s0 + STAGE < n_tok) load(s0 + STAGE, [&](int i) { return s_row[i]; });
    };
    auto attend = [&](int s0, const char* kbuf) {
        if (!live) return;
        asm volatile("" : "+v"(rows.k_at), "+v"(rows.v_at));  // its addresses, as in decode
        const char* const vbuf = kbuf + STAGE * ROWB;
        const int left = n_tok - s0;
        const int t1 = min(tile0 + per_wave, (min(left, STAGE) + 31) / 32);
        int t = tile0;
        if constexpr (MANY)
#pragma unroll 1
        for (; t + 1 < t1 && 32 * (t + 2) <= left; t += 2)
            rows.template two_tiles<true>(kbuf, vbuf, t, c, g, s_vs + s0 + 32 * t);
#pragma unroll 1
        for (; t < t1; ++t) rows.template masked_tile<true>(kbuf, vbuf, t, c, 0, left - 32 * t, g, s_vs + s0 + 32 * t);
    };

    if constexpr (MANY) {
        // ---- the stages: one is decoded while the one before it is attended to ----
        // A SIMD's two waves do these in opposite order, so that one's matrix products run under the other's
        // conversions.
        decode(0, s_kv[0]);
        __syncthreads();
        const bool decode_first = wave >= NW / 2;
        int at = 0;
        for (int s0 = 0; s0 < n_tok; s0 += STAGE, at ^= 1) {
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
                if ((part == 0) == decode_first) {
                    if (s0 + STAGE < n_tok) decode(s0 + STAGE, s_kv[(at ^ 1) % SH::BUFS]);
                } else {
                    attend(s0, s_kv[at % SH::BUFS]);
                }
            }
            __syncthreads();
        }
    } else {
        // Up to 32 rows: every wave has all of them and attends to the tokens that it decoded itself.  Its LDS accesses
        // run in order, so the waves need no barriers and drift apart, one's loads under another's work (3 to 5 %).
        const bool alone = rw == 1;
        for (int s0 = 0; s0 < n_tok; s0 += STAGE) {
            decode(s0, s_kv[0]);
            if (alone) asm volatile("" ::: "memory");
            else __syncthreads();
            attend(s0, s_kv[0]);
            // the next stage's tables come by DMA into the rows that were read here, in no order with these reads
            if (alone) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            else __syncthreads();
        }
        if (alone) __syncthreads();  // the sums go over the other waves' stages
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
        const float f = __builtin_ldexpf(__builtin_amdgcn_exp2f(rows.m - m), -1 - vexp);
        // [wave][query][coordinate], 16-byte chunks at chunk ^ query
        float* const area = reinterpret_cast<float*>(s_kv) + (wave * 32 + n) * D;
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
    for (int r = threadIdx.x; r < n_q; r += NT) {
        const int w0 = r >> 5, q = r & 31;
        float m = kNoMax, l = 0.0f;
        for (int w = w0; w < NW; w += rw) m = __builtin_fmaxf(m, s_m[w][q]);
        for (int w = w0; w < NW; w += rw) l += s_l[w][q] * __builtin_amdgcn_exp2f(s_m[w][q] - m);
        *reinterpret_cast<f32x2*>(a.part_ml + 2 * (size_t)s_slot[r]) = f32x2{m, l};
    }
    const float* const sums = reinterpret_cast<const float*>(s_kv);
#pragma unroll 4
    for (int i = threadIdx.x; i < n_q * (D / 4); i += NT) {
        const int r = i / (D / 4), j = i % (D / 4), w0 = r >> 5, q = r & 31;
        f32x4 y = *reinterpret_cast<const f32x4*>(sums + r * D + 4 * (j ^ (q & 15)));
        for (int w = w0 + rw; w < NW; w += rw) y += *reinterpret_cast<const f32x4*>(sums + (w * 32 + q) * D + 4 * (j ^ (q & 15)));
        f32x4* const to = reinterpret_cast<f32x4*>(a.part_y + (size_t)s_slot[r] * D + 4 * j);
        // many rows: more bytes than the next kernel finds in its XCD's L2 (32 rows x 4 heads over 4096 tokens,
        // 27.7 -> 25.2 us); few: 16.1 us kept there, 16.4 not
        if constexpr (MANY) __builtin_nontemporal_store(y, to);
        else *to = y;
    }
}

// One (row, query head) a workgroup: its chunks' sums weighted and added in a fixed order, then the
// Walsh-Hadamard transform, h_D and the softmax's sum.  Every wave finds the maximum for itself and one of them
// transforms, over its lanes: one barrier in all (with nine of them 0.1 to 0.3 us more of 10 to 15 a call).
template <int D, int QDT>
__global__ __launch_bounds__(256) void shared_combine_kernel(SharedArgs a) {
    constexpr int V = D / 4, NG = 256 / V;  // lanes of a chunk's row, chunks at a time
    __shared__ f32x4 s_y[NG][V];
    __shared__ float s_l[NG];
    const uint32_t row = blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads;
    const int c0 = a.row_slots[row], c1 = a.row_slots[row + 1];
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
    const float f = c1 > c0 ? a.hscale : 0.0f;  // a row without tokens is zero
    if (c1 <= c0) l = 1.0f;
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + (size_t)blockIdx.x * D + 4 * at) =
        u32x2{pack2<QDT>(y[0] * f / l, y[1] * f / l), pack2<QDT>(y[2] * f / l, y[3] * f / l)};
}

// items: those of segments of many query rows first, those of few last
template <int D, int QDT>
static hipError_t launch_shared(SharedArgs a, const uint32_t (&n)[3], uint32_t batch, hipStream_t s) {
    for (int k = 0; k < 3; ++k) {
        if (n[k] == 0) continue;
        a.n_items = n[k];
        const dim3 grid((n[k] + 7u) / 8u * 8u * a.kv_heads);
        if (k == 0) hipLaunchKernelGGL((shared_attn_kernel<D, QDT, true>), grid, dim3(Shape<D, true>::THREADS), 0, s, a);
        else if (k == 1) hipLaunchKernelGGL((shared_attn_kernel<D, QDT, false>), grid, dim3(Shape<D, false>::THREADS), 0, s, a);
        else hipLaunchKernelGGL((few_attn_kernel<D, QDT>), grid, dim3(64 * Few<D>::WAVES), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        a.items += 8 * (size_t)n[k];
    }
    hipLaunchKernelGGL((shared_combine_kernel<D, QDT>), dim3(batch * a.q_heads), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int QDT>
static hipError_t shared_dims(int32_t d, const SharedArgs& a, const uint32_t (&n)[3], uint32_t batch, hipStream_t s) {
    switch (d) {
        case 64: return launch_shared<64, QDT>(a, n, batch, s);
        case 128: return launch_shared<128, QDT>(a, n, batch, s);
        default: return launch_shared<256, QDT>(a, n, batch, s);
    }
}

}  // namespace nq

extern "C" int32_t nq_shared_attention_chunk_tokens(int32_t kind) {
    return kind == 0 ? nq::Shape<128, true>::CHUNK : kind == 1 ? nq::Shape<128, false>::CHUNK : nq::Few<128>::CHUNK;
}
extern "C" int32_t nq_shared_attention_rows(int32_t head_dim, int32_t kind) {
    if (kind == 0) return head_dim <= 128 ? nq::Shape<128, true>::ROWS : nq::Shape<256, true>::ROWS;
    return kind == 1 ? nq::Shape<128, false>::ROWS : nq::Few<128>::ROWS;
}

extern "C" int64_t nq_shared_attention_workspace(int32_t n_slots, int32_t q_heads, int32_t head_dim) {
    if (n_slots <= 0 || q_heads <= 0 || head_dim <= 0) return 0;
    return (int64_t)n_slots * q_heads * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int nq_shared_attention(const nq_shared_desc* d, void* stream) {
    using namespace nq;
    NQ_CHECK_ARG(d != nullptr && d->pool != nullptr, "nq_shared_attention: desc and pool are required");
    const nq_pool* p = d->pool;
    NQ_CHECK_ARG(p->head_dim == 64 || p->head_dim == 128 || p->head_dim == 256,
                 "nq_shared_attention: head_dim %d unsupported (64, 128, 256)", p->head_dim);
    NQ_CHECK_ARG(p->layers > 0 && p->pages > 0 && p->heads > 0 && p->tokens > 0 && d->layer >= 0 && d->layer < p->layers,
                 "nq_shared_attention: bad pool geometry, or layer %d of %d", d->layer, p->layers);
    NQ_CHECK_ARG((uint64_t)p->pages * p->heads * p->tokens < (1ull << 31),
                 "nq_shared_attention: a layer must have less than 2^31 token rows");
    NQ_CHECK_ARG(d->q_dtype == NQ_F16 || d->q_dtype == NQ_BF16, "nq_shared_attention: queries must be fp16 or bf16");
    NQ_CHECK_ARG(d->batch >= 0 && d->q_heads > 0 && d->q_heads % p->heads == 0 &&
                     d->q_heads / p->heads <= nq_shared_attention_rows(p->head_dim, 0),
                 "nq_shared_attention: q_heads %d must be a multiple of the pool's %d heads, at most %d times", d->q_heads,
                 p->heads, nq_shared_attention_rows(p->head_dim, 0));
    NQ_CHECK_ARG(d->n_items >= 0 && d->n_slots >= 0 && d->n_many >= 0 && d->n_few >= 0 &&
                     (int64_t)d->n_many + d->n_few <= d->n_items,
                 "nq_shared_attention: n_items %d, n_many %d, n_few %d, n_slots %d", d->n_items, d->n_many, d->n_few, d->n_slots);
    for (int k = 1; k < 3; ++k)
        NQ_CHECK_ARG((k == 1 ? d->n_items - d->n_many - d->n_few : d->n_few) == 0 ||
                         d->q_heads / p->heads <= nq_shared_attention_rows(p->head_dim, k),
                     "nq_shared_attention: %d query heads per kv head are too many for items of kind %d", d->q_heads / p->heads, k);
    if (d->batch == 0) return NQ_OK;
    NQ_CHECK_ARG(d->query && d->out && d->row_slots, "nq_shared_attention: query, out and row_slots are required");
    NQ_CHECK_ARG(((uintptr_t)d->query & 15u) == 0 && ((uintptr_t)d->out & 7u) == 0,
                 "nq_shared_attention: query must be 16-byte aligned, out 8-byte");
    NQ_CHECK_ARG((uint64_t)d->batch * d->q_heads <= max_blocks(256) &&
                     ((uint64_t)d->n_items + 7) * p->heads <= max_blocks(512), "nq_shared_attention: grid too large");
    SharedArgs a = {};
    if (d->n_items > 0) {
        NQ_CHECK_ARG(d->items && d->pages && d->seg_rows, "nq_shared_attention: the plan's arrays are required");
        NQ_CHECK_ARG(p->key_codes && p->value_codes && p->key_scales && p->value_scales && p->positions,
                     "nq_shared_attention: the pool's arrays are required");
        NQ_CHECK_ARG((((uintptr_t)p->key_codes | (uintptr_t)p->value_codes | (uintptr_t)p->key_scales |
                       (uintptr_t)p->value_scales) & 15u) == 0 && ((uintptr_t)p->positions & 3u) == 0,
                     "nq_shared_attention: the pool's codes and scales must be 16-byte aligned");
        NQ_CHECK_ARG(d->rope_sin_minus_cos && d->rope_cos_plus_sin && d->rope_n_pos > 0 && d->rope_n_pos < (1ll << 31) / p->head_dim,
                     "nq_shared_attention: keys need RoPE tables, of less than 4 GB each");
        NQ_CHECK_ARG((uint64_t)d->n_slots * d->q_heads < (1ull << 32), "nq_shared_attention: too many partial sums");
        const int64_t need = nq_shared_attention_workspace(d->n_slots, d->q_heads, p->head_dim);
        NQ_CHECK_ARG(d->n_slots > 0 && d->workspace != nullptr && d->workspace_bytes >= need &&
                         ((uintptr_t)d->workspace & 15u) == 0,
                     "nq_shared_attention: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
        NQ_CHECK_ARG(d->scale_divisor > 0.0f, "nq_shared_attention: scale_divisor must be positive");
    }
    const size_t rows = (size_t)d->layer * p->pages * p->heads * p->tokens;
    a.query = static_cast<const uint16_t*>(d->query);
    a.out = d->out;
    a.kc = p->key_codes + rows * p->head_dim;
    a.vc = p->value_codes + rows * p->head_dim;
    a.ks = static_cast<const uint16_t*>(p->key_scales) + rows;
    a.vs = static_cast<const uint16_t*>(p->value_scales) + rows;
    a.positions = p->positions;
    a.items = d->items;
    a.pages = d->pages;
    a.seg_rows = d->seg_rows;
    a.row_slots = d->row_slots;
    a.part_y = static_cast<float*>(d->workspace);
    a.part_ml = a.part_y + (size_t)d->n_slots * d->q_heads * p->head_dim;
    a.rope_dm = d->rope_sin_minus_cos;
    a.rope_dp = d->rope_cos_plus_sin;
    a.q_heads = (uint32_t)d->q_heads;
    a.kv_heads = (uint32_t)p->heads;
    a.rope_n_pos = (uint32_t)(d->rope_n_pos > 0 ? d->rope_n_pos : 1);
    a.tokens = (uint32_t)p->tokens;
    a.by_tokens = fast_div(a.tokens);
    a.by_group = fast_div(a.q_heads / a.kv_heads);
    a.c = 1.44269504088896340736f / (d->scale_divisor > 0.0f ? d->scale_divisor : 1.0f);
    a.hscale = d->hadamard_scale;
    hipStream_t s = (hipStream_t)stream;
    const uint32_t n[3] = {(uint32_t)d->n_many, (uint32_t)(d->n_items - d->n_many - d->n_few), (uint32_t)d->n_few};
    NQ_CHECK_HIP(d->q_dtype == NQ_F16 ? shared_dims<NQ_F16>(p->head_dim, a, n, (uint32_t)d->batch, s)
                                      : shared_dims<NQ_BF16>(p->head_dim, a, n, (uint32_t)d->batch, s));
    return NQ_OK;
}
