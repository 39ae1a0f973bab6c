// Decode attention over a pool's pages for rows that share pages: what several rows begin
// with is read and decoded once for all of them.
//
// The host cuts the rows' tokens into segments: a run of pages and the batch rows that see
// all its tokens (a shared prefix: many rows; a row's own rest: one).  A workgroup takes a
// chunk of a segment's tokens, one kv head, and up to 256 (head_dim 256: 128) of the segment's
// query rows (batch rows x the kv head's query heads).  Stage by stage (128 tokens; 64) it
//  1. decodes keys and values into LDS as fp16, all waves together: keys through the int8
//     matrix cores (nq_keymfma.h), scaled and rotated in fp32; values as their codes: their
//     scales go with the softmax weights, and the transform, which is linear, with a row's
//     sum (combine kernel);
//  2. attends (nq_flash.h): 32 query rows a wave and all tiles of the stage; with fewer rows
//     several waves share them and split the tiles, and their sums are joined in LDS at the end.
// A partial (maximum, sum, value sum) per query row and chunk goes to the workspace; the
// combine kernel joins a row's chunks.
#include "nq_flash.h"
#include "nq_keymfma.h"
#include "nq_rowmath.h"

namespace nq {

using namespace flash;

// The shape of a workgroup.  MANY: rows count, so as many as the registers hold (32 a wave) share what is decoded,
// and a stage is decoded under the attention to the one before it; two stage buffers, 128 KB of LDS at head_dim
// 128 and 256, so one workgroup on a CU.  Not MANY: decoding counts, and several small workgroups on a CU hide
// each other's loads.  8 kv heads x 128, us: 512 query rows x 32768 tokens 122 (MANY) and 230; 128 rows x
// 16384 35.0 and 38.9, x 4096 24.8 and 25.5; 64 rows x 8192 23.4 and 23.8; 8 rows (32 heads x 64) 63.6 and 41.
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
template <int KS>
__device__ __forceinline__ float bf16_queries(u32x4 (&q)[KS]) {
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w = q[i][k];
            big = __builtin_fmaxf(big, __builtin_fmaxf(__builtin_fabsf(bf16_bits_to_f32(w & 0xffffu)),
                                                       __builtin_fabsf(bf16_bits_to_f32(w >> 16))));
        }
    big = both_max(big);
    int e = 0;
    if (big > 0.0f && big < __builtin_inff()) (void)__builtin_frexpf(big, &e);
    e = max(e - 15, -126);  // bf16's subnormals: scaled as far as fp32 reaches
    const float f = __builtin_ldexpf(1.0f, -e);
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w = q[i][k];
            q[i][k] = pack2<NQ_F16>(bf16_bits_to_f32(w & 0xffffu) * f, bf16_bits_to_f32(w >> 16) * f);
        }
    return __builtin_ldexpf(1.0f, e);
}

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
            const int first = s0 + 16 * (NW * u + wave);
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
    if constexpr (QDT == NQ_BF16) c *= bf16_queries(rows.q);
    KM signs;
    signs.init(lane);
    __syncthreads();
    // The values' scales go with the weights, so that the codes are exact in fp16 and one rounding is left.
    // Times 2^vexp the chunk's largest is in [64, 128): weights (at most 2^kSlack) stay below 2^15, and keep
    // their 11 bits down to 2^-20 of that.
    int vexp = 0;
    {
        float m = s_max[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) m = __builtin_fmaxf(m, s_max[w]);
        if (m > 0.0f && m < __builtin_inff()) {
            (void)__builtin_frexpf(m, &vexp);
            vexp = 7 - vexp;
        }
    }
    for (int i = threadIdx.x; i < n_slots; i += NT) s_vs[i] = __builtin_ldexpf(s_vs[i], vexp);  // used after the next barrier

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
            const int row0 = 16 * (NW * u + wave);
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
            const int row0 = 16 * (NW * u + wave);
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
        for (int s0 = 0; s0 < n_tok; s0 += STAGE) {
            decode(s0, s_kv[0]);
            __syncthreads();
            attend(s0, s_kv[0]);
            __syncthreads();
        }
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
// Walsh-Hadamard transform, h_D and the softmax's sum.
template <int D, int QDT>
__global__ __launch_bounds__(256) void shared_combine_kernel(SharedArgs a) {
    constexpr int V = D / 4, NG = 256 / V;  // lanes of a chunk's row, chunks at a time
    __shared__ f32x4 s_y[NG][V];
    __shared__ float s_l[NG], s_x[D], s_mw[4];
    const uint32_t row = blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads;
    const int c0 = a.row_slots[row], c1 = a.row_slots[row + 1];
    const int tid = threadIdx.x, grp = tid / V, at = tid % V;
    float m = kNoMax;
    for (int s = c0 + tid; s < c1; s += 256) m = __builtin_fmaxf(m, a.part_ml[2 * ((size_t)s * a.q_heads + head)]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, o, 64));
    if ((tid & 63) == 0) s_mw[tid >> 6] = m;
    __syncthreads();
    m = __builtin_fmaxf(__builtin_fmaxf(s_mw[0], s_mw[1]), __builtin_fmaxf(s_mw[2], s_mw[3]));
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
    if (grp == 0) {
        for (int i = 1; i < NG; ++i) y += s_y[i][at];
        const float p0 = y[0] + y[1], p1 = y[0] - y[1], p2 = y[2] + y[3], p3 = y[2] - y[3];
        *reinterpret_cast<f32x4*>(&s_x[4 * at]) = f32x4{p0 + p2, p1 + p3, p0 - p2, p1 - p3};
    }
    __syncthreads();
#pragma unroll
    for (int len = 4; len < D; len <<= 1) {
        if (tid < D / 2) {
            const int i = (tid / len) * 2 * len + tid % len;
            const float x0 = s_x[i], x1 = s_x[i + len];
            s_x[i] = x0 + x1;
            s_x[i + len] = x0 - x1;
        }
        __syncthreads();
    }
    if (tid >= D) return;
    l = s_l[0];
    for (int i = 1; i < NG; ++i) l += s_l[i];
    const float v = c1 > c0 ? s_x[tid] * a.hscale / l : 0.0f;  // a row without tokens is zero
    static_cast<uint16_t*>(a.out)[(size_t)blockIdx.x * D + tid] = (uint16_t)(pack2<QDT>(v, 0.0f) & 0xffffu);
}

// items: those of segments of many query rows first, then the others
template <int D, int QDT>
static hipError_t launch_shared(SharedArgs a, uint32_t n_many, uint32_t n_items, uint32_t batch, hipStream_t s) {
    const int32_t* const items = a.items;
    if (n_many > 0) {
        a.n_items = n_many;
        hipLaunchKernelGGL((shared_attn_kernel<D, QDT, true>), dim3((n_many + 7u) / 8u * 8u * a.kv_heads),
                           dim3(Shape<D, true>::THREADS), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (n_items > n_many) {
        a.items = items + 8 * (size_t)n_many;
        a.n_items = n_items - n_many;
        hipLaunchKernelGGL((shared_attn_kernel<D, QDT, false>), dim3((a.n_items + 7u) / 8u * 8u * a.kv_heads),
                           dim3(Shape<D, false>::THREADS), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((shared_combine_kernel<D, QDT>), dim3(batch * a.q_heads), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int QDT>
static hipError_t shared_dims(int32_t d, const SharedArgs& a, uint32_t n_many, uint32_t n_items, uint32_t batch, hipStream_t s) {
    switch (d) {
        case 64: return launch_shared<64, QDT>(a, n_many, n_items, batch, s);
        case 128: return launch_shared<128, QDT>(a, n_many, n_items, batch, s);
        default: return launch_shared<256, QDT>(a, n_many, n_items, batch, s);
    }
}

}  // namespace nq

extern "C" int32_t nq_shared_attention_chunk_tokens(int32_t many) {
    return many ? nq::Shape<128, true>::CHUNK : nq::Shape<128, false>::CHUNK;
}
extern "C" int32_t nq_shared_attention_rows(int32_t head_dim) {
    return head_dim <= 128 ? nq::Shape<128, true>::ROWS : nq::Shape<256, true>::ROWS;
}

extern "C" int32_t nq_shared_attention_few_rows(void) { return nq::Shape<128, false>::ROWS; }

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
                     d->q_heads / p->heads <= nq_shared_attention_rows(p->head_dim),
                 "nq_shared_attention: q_heads %d must be a multiple of the pool's %d heads, at most %d times", d->q_heads,
                 p->heads, nq_shared_attention_rows(p->head_dim));
    NQ_CHECK_ARG(d->n_items >= 0 && d->n_slots >= 0 && d->n_many >= 0 && d->n_many <= d->n_items,
                 "nq_shared_attention: n_items %d, n_many %d, n_slots %d", d->n_items, d->n_many, d->n_slots);
    NQ_CHECK_ARG(d->n_many == d->n_items || d->q_heads / p->heads <= nq_shared_attention_few_rows(),
                 "nq_shared_attention: over %d query heads per kv head, every item belongs to the n_many of many rows",
                 nq_shared_attention_few_rows());
    if (d->batch == 0) return NQ_OK;
    NQ_CHECK_ARG(d->query && d->out && d->row_slots, "nq_shared_attention: query, out and row_slots are required");
    NQ_CHECK_ARG(((uintptr_t)d->query & 15u) == 0, "nq_shared_attention: query must be 16-byte aligned");
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
    NQ_CHECK_HIP(d->q_dtype == NQ_F16 ? shared_dims<NQ_F16>(p->head_dim, a, (uint32_t)d->n_many, (uint32_t)d->n_items, (uint32_t)d->batch, s)
                                      : shared_dims<NQ_BF16>(p->head_dim, a, (uint32_t)d->n_many, (uint32_t)d->n_items, (uint32_t)d->batch, s));
    return NQ_OK;
}
