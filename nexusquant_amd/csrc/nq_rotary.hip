// Rotary positions with one or several axes, and new tokens into a cache held in 4 bits with their rotation on the way.
//
//   angles   cos, sin of pos[axis(i)] * inv_freq[i], once for all layers of a step
//   rotate   (a, b) = (x[i], x[i + d / 2]) -> (a c - b s, b c + a s); the inverse, its gradient, with -s
//   append   queries rotated; keys rotated, transformed, encoded and stored in their slots; values likewise, unrotated
//   read     what slots hold, as values again
// Bytes bound all of them where there are many rows, the launch where there are few.
#include "nq_fourbit.h"
#include "nq_rowmath.h"

namespace nq {

// ----------------------------------------------------------------- angles ----

struct AngleArgs {
    const void* positions;  // [axes, rows], int32 or int64
    float* out;             // [rows, 2, half]: cosines, sines
    int64_t stride;         // of an axis, elements
    uint32_t rows, half;
    FastDiv by_half;
    int32_t wide;           // int64 positions
    float freq[128];
    uint8_t axis[128];
};

// The angle is the fp32 product of fp32 numbers, as models form it; its cosine and sine are taken in 64 bits and rounded
// once (an angle of 10^5 has no digit to lose to a reduction in fp32).
//
// Up to 2^31: k quarter turns are taken off with pi / 2 as two 64-bit numbers (the first product is exact within the fma, the
// second's error is 2^-53 of what is left at most), and Taylor's series to the 13th and 14th power has 4e-14 left at pi / 4.
__device__ __forceinline__ void sincos_exactly(float angle, float& sine, float& cosine) {
    if (__builtin_fabsf(angle) >= 0x1p31f) {
        double s, c;
        sincos((double)angle, &s, &c);
        sine = (float)s;
        cosine = (float)c;
        return;
    }
    const double k = rint((double)angle * 0.6366197723675814), q = fma(-k, 6.123233995736766e-17, fma(-k, 1.5707963267948966, (double)angle));
    const double q2 = q * q;
    double s = 1.0 / 6227020800.0, c = -1.0 / 87178291200.0;
    s = fma(s, q2, -1.0 / 39916800.0);
    s = fma(s, q2, 1.0 / 362880.0);
    s = fma(s, q2, -1.0 / 5040.0);
    s = fma(s, q2, 1.0 / 120.0);
    s = fma(s, q2, -1.0 / 6.0);
    c = fma(c, q2, 1.0 / 479001600.0);
    c = fma(c, q2, -1.0 / 3628800.0);
    c = fma(c, q2, 1.0 / 40320.0);
    c = fma(c, q2, -1.0 / 720.0);
    c = fma(c, q2, 1.0 / 24.0);
    c = fma(c, q2, -0.5);
    const float sq = (float)fma(q * q2, s, q), cq = (float)fma(q2, c, 1.0);
    const int turns = (int)k;
    const float a = turns & 1 ? cq : sq, b = turns & 1 ? sq : cq;
    sine = turns & 2 ? -a : a;
    cosine = (turns + 1) & 2 ? -b : b;
}

__global__ __launch_bounds__(256) void rotation_kernel(AngleArgs a) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= a.rows * a.half) return;
    const uint32_t r = div(u, a.by_half), i = u - r * a.half;
    const int64_t at = (int64_t)a.axis[i] * a.stride + r;
    const float pos = a.wide ? (float)static_cast<const int64_t*>(a.positions)[at] : (float)static_cast<const int32_t*>(a.positions)[at];
    float s, c;
    sincos_exactly(pos * a.freq[i], s, c);
    float* const o = a.out + (size_t)r * 2u * a.half + i;
    o[0] = c;
    o[a.half] = s;
}

// ----------------------------------------------------------------- rotate ----

struct RotateArgs {
    const uint8_t* x[2];    // queries, keys
    uint8_t* y[2];
    int64_t x_row[2], x_head[2], y_row[2], y_head[2];  // strides, bytes
    const float* angles;    // [rows, 2, d / 2]
    uint32_t rows, heads[2], parts;  // waves that share a row's heads
    float sign;             // -1: the inverse
    uint32_t stream;
};

// STREAM: past the caches (kStreamBytes, nq_rowmath.h).
template <int DT, bool STREAM>
__device__ __forceinline__ void store8(uint8_t* p, const float (&x)[8]) {
    NQ_GLOBAL u32x4* const to = (NQ_GLOBAL u32x4*)(uint64_t)p;
    auto put = [&](int i, u32x4 v) {
        if constexpr (STREAM) __builtin_nontemporal_store(v, to + i);
        else to[i] = v;
    };
    if constexpr (DT == NQ_F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __builtin_bit_cast(uint32_t, x[4 * i + k]);
            put(i, v);
        }
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const f32x2 v = {x[2 * k], x[2 * k + 1]};
            if constexpr (DT == NQ_F16) w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
            else w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
        }
        put(0, w);
    }
}

// A wave takes a token's heads h = first, first + step, .., D / 16 lanes a head and eight pairs a lane, 1024 / D heads one after
// another in memory at a time: the angles stay in registers, and N steps' inputs are read before their outputs are written.
// 16384 tokens of 32 + 8 heads of 128 (336 MB) with their angles: a wave on eight tokens of one head at a time 83 us, on eight
// heads of a token 71, with stores past the caches 58, reading ahead the same (51 and 6 for the angles: 6.6 TB/s, the inputs
// being in the last-level cache still from the call before; 67 where they are not); 8188 tokens in fp32, forward and back (671
// MB), 139 to 146, of which it keeps nothing.
template <int DT, int D, bool STREAM, typename Where>
__device__ __forceinline__ void rotate_heads(const float* angles, float sign, uint32_t first, uint32_t step, uint32_t heads, int at, Where where) {
    constexpr int SIZE = DT == NQ_F32 ? 4 : 2, N = DT == NQ_F32 ? 2 : 4;
    float c[8], s[8];
    load8f(angles + 8 * at, c);
    load8f(angles + D / 2 + 8 * at, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= sign;
    for (uint32_t h = first; h < heads; h += N * step) {
        float lo[N][8], hi[N][8];
        uint8_t* to[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint8_t* from;
            where(min(h + n * step, heads - 1u), from, to[n]);
            load8<DT>(from + 8 * SIZE * at, 0, lo[n]);
            load8<DT>(from + 8 * SIZE * at, D / 2, hi[n]);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (h + n * step >= heads) continue;
            float u[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                u[i] = __builtin_fmaf(lo[n][i], c[i], -(hi[n][i] * s[i]));
                v[i] = __builtin_fmaf(hi[n][i], c[i], lo[n][i] * s[i]);
            }
            store8<DT, STREAM>(to[n] + 8 * SIZE * at, u);
            store8<DT, STREAM>(to[n] + (8 * at + D / 2) * SIZE, v);
        }
    }
}

template <int DT, int D>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
    constexpr int LANES = D / 16, HEADS = 64 / LANES;
    const uint32_t wave = blockIdx.x * 4u + (threadIdx.x >> 6), row = wave / a.parts, lane = threadIdx.x & 63u;
    if (row >= a.rows) return;  // whole wave
    auto where = [&](uint32_t h, const uint8_t*& from, uint8_t*& to) {
        const bool key = h >= a.heads[0];
        const uint32_t head = key ? h - a.heads[0] : h;
        from = (key ? a.x[1] : a.x[0]) + row * (key ? a.x_row[1] : a.x_row[0]) + head * (key ? a.x_head[1] : a.x_head[0]);
        to = (key ? a.y[1] : a.y[0]) + row * (key ? a.y_row[1] : a.y_row[0]) + head * (key ? a.y_head[1] : a.y_head[0]);
    };
    const float* const angles = a.angles + (size_t)row * D;
    const uint32_t first = wave % a.parts * HEADS + lane / LANES, heads = a.heads[0] + a.heads[1];
    if (a.stream) rotate_heads<DT, D, true>(angles, a.sign, first, a.parts * HEADS, heads, lane % LANES, where);
    else rotate_heads<DT, D, false>(angles, a.sign, first, a.parts * HEADS, heads, lane % LANES, where);
}

// ----------------------------------------------------------------- append ----

struct AppendArgs {
    const uint8_t* x[3];                // keys, values, queries
    int64_t row[3], head[3];            // strides, bytes
    uint8_t* out;                       // rotated queries
    int64_t out_row, out_head;
    const float* angles;                // [rows, 2, d / 2], or NULL
    const int32_t* slots;               // [rows]
    FourBitRows pool;
    uint32_t rows, q_heads, kv_heads;
    uint32_t batches, waves;            // of 16 keys and values of a token; waves that share a token's heads
    uint32_t stream;
    uint32_t tokens, slot_end;
    FastDiv by_tokens;
    float hscale;
};

// One row encoded in 64 bits by a whole wave, from its input on: lane l coordinates D / 64 l .. .
template <int DT, int D>
__device__ __forceinline__ void encode_exactly(const uint8_t* from, const float* angles, int lane, uint32_t* codes, uint16_t* scale) {
    constexpr int V = D / 64;
    double x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if constexpr (DT == NQ_F16) x[k] = (double)f16_bits_to_f32(reinterpret_cast<const uint16_t*>(from)[V * lane + k]);
        else x[k] = (double)bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(from)[V * lane + k]);
    }
    if (angles) {
        const int half = V * (lane & 31);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const double other = __shfl_xor(x[k], 32, 64), c = angles[half + k], s = angles[D / 2 + half + k];
            x[k] = x[k] * c + (lane < 32 ? -other : other) * s;
        }
    }
#pragma unroll
    for (int len = 1; len < V; len <<= 1)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (k & len) continue;
            const double u = x[k], v = x[k + len];
            x[k] = u + v;
            x[k + len] = u - v;
        }
    double most = 0.0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double other = __shfl_xor(x[k], o, 64);
            x[k] = (lane & o) ? other - x[k] : x[k] + other;
        }
        most = fmax(most, fabs(x[k]));
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = fmax(most, __shfl_xor(most, o, 64));
    const double h = D == 64 ? 0.125 : D == 256 ? 0.0625 : 0.08838834764831844;  // 1 / sqrt(D)
    const uint32_t s16 = f32_to_f16_bits((float)fmin(most * h / 7.5, 65504.0));  // by way of fp32, as where 32 bits suffice
    const double scale64 = s16 ? (double)f16_bits_to_f32(s16) : 1.0;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) w |= (uint32_t)fmin(fmax(floor(x[k] * h / scale64 + 8.5), 0.0), 15.0) << (4 * ((V * lane + k) & 7));
#pragma unroll
    for (int o = 1; o < 8 / V; o <<= 1) w |= (uint32_t)__shfl_xor((int)w, o, 64);
    if ((V * lane & 7) == 0) codes[V * lane >> 3] = w;
    if (lane == 0) *scale = (uint16_t)s16;
}

// A wave takes a token: its keys and values sixteen at a time, a quad a head (nq_rowmath.h), then its queries.  Bound by bytes:
// 10149 tokens of 32, 8 and 8 heads of 128 (224 MB) 35 us, 6.4 TB/s (inputs in the last-level cache, queries stored past it);
// a decode step of 32 tokens 6.2, a launch and three loads that wait for each other.
//
// 32 bits decide a level, or the scale, wrongly where it lies next to a border: of 10 K prompt tokens' keys and values of
// 8 x 128 some 30 coordinates in 21 M were a whole step off, and what is read back was 5.1e-4 from 64 bits where fp16's own
// rounding is 2.1e-4.  So a row with a coordinate within kNear of a border, or a scale next to one of fp16's, is encoded
// again in 64 bits from its cosines and sines on, by the whole wave: some 4 rows in 1000, 2.8e-4, 2 us of 60.  Sixteen
// rows at a time, a quad a row, it took 256 registers and 26 more at head_dim 256 (one wave a SIMD for two).
constexpr float kNear = 0x1p-17f;

template <int DT, int D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    constexpr int C = D / 32, HC = C / 2;
    const int lane = threadIdx.x & 63, q = lane & 3;
    const uint32_t wave = blockIdx.x * 4u + (threadIdx.x >> 6), token = wave / a.waves;
    if (token >= a.rows) return;  // whole wave
    float cs[HC][8], sn[HC][8];
    if (a.angles) {
#pragma unroll
        for (int c = 0; c < HC; ++c) {
            const float* const t = a.angles + (size_t)token * D + 32 * c + 8 * q;
            load8f(t, cs[c]);
            load8f(t + D / 2, sn[c]);
        }
    }
    const int32_t slot = a.slots[token];
    const bool stored = slot >= 0 && (uint32_t)slot < a.slot_end;
    const uint32_t page = stored ? div((uint32_t)slot, a.by_tokens) : 0u, off = stored ? (uint32_t)slot - page * a.tokens : 0u;
    uint32_t batch = wave % a.waves;
    for (; batch < a.batches; batch += a.waves) {
        const uint32_t want = 16u * batch + ((uint32_t)lane >> 2), h = min(want, 2u * a.kv_heads - 1u);
        const uint32_t role = h < a.kv_heads ? 0u : 1u, head = h - role * a.kv_heads;
        const uint8_t* const x = (role ? a.x[1] : a.x[0]) + token * (role ? a.row[1] : a.row[0]) + head * (role ? a.head[1] : a.head[0]);
        float v[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) load8<DT>(x, 32 * c + 8 * q, v[c]);
        if (role == 0 && a.angles) {
#pragma unroll
            for (int c = 0; c < HC; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float lo = v[c][i], hi = v[c + HC][i];
                    v[c][i] = __builtin_fmaf(lo, cs[c][i], -(hi * sn[c][i]));
                    v[c + HC][i] = __builtin_fmaf(hi, cs[c][i], lo * sn[c][i]);
                }
        }
        fwht_row<C>(v, q);
        // the largest |t| as an integer: infinities and NaNs are larger than any number
        uint32_t big = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[c][i] *= a.hscale;
                big = max(big, __builtin_bit_cast(uint32_t, v[c][i]) & 0x7fffffffu);
            }
        big = max(big, dpp_u32<kQuadXor1>(big));
        big = max(big, dpp_u32<kQuadXor2>(big));
        const bool finite = big < 0x7f800000u;
        const float amax = finite ? __builtin_bit_cast(float, big) : 0.0f;
        const float s32 = __builtin_fminf(amax / 7.5f, 65504.0f);
        const uint32_t s16 = f32_to_f16_bits(s32);
        const float s = f16_bits_to_f32(s16);
        const float inv = (s > 0.0f ? 1.0f / s : 0.0f) * quad_sign(q);  // the transform's sign (nq_rowmath.h)
        uint32_t w[C];
        float far = 0.0f;  // from the nearest level
#pragma unroll
        for (int c = 0; c < C; ++c) {
            w[c] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = v[c][i] * inv, level = __builtin_rintf(y);
                far = __builtin_fmaxf(far, __builtin_fabsf(y - level));
                w[c] |= (uint32_t)(int)__builtin_fminf(__builtin_fmaxf(level + 8.0f, 0.0f), 15.0f) << (4 * i);
            }
        }
        far = __builtin_fmaxf(far, dpp_f32<kQuadXor1>(far));
        far = __builtin_fmaxf(far, dpp_f32<kQuadXor2>(far));
        const bool mine = stored && want == h;
        const bool near = mine && finite && (far > 0.5f - kNear || f32_to_f16_bits(s32 * (1.0f - 0x1p-21f)) != f32_to_f16_bits(s32 * (1.0f + 0x1p-21f)));
        for (uint64_t todo = __ballot(near && q == 0); todo; todo &= todo - 1) {
            const int from = __builtin_ctzll(todo);
            const uint32_t value = (uint32_t)__builtin_amdgcn_readlane((int)role, from), of = (uint32_t)__builtin_amdgcn_readlane((int)head, from);
            const size_t to = ((size_t)page * a.kv_heads + of) * a.tokens + off;
            encode_exactly<DT, D>((value ? a.x[1] : a.x[0]) + token * (value ? a.row[1] : a.row[0]) + of * (value ? a.head[1] : a.head[0]),
                                  value || !a.angles ? nullptr : a.angles + (size_t)token * D, lane,
                                  reinterpret_cast<uint32_t*>((value ? a.pool.codes[1] : a.pool.codes[0]) + to * (D / 2)),
                                  (value ? a.pool.scales[1] : a.pool.scales[0]) + to);
        }
        if (mine && !near) {
            const size_t to = ((size_t)page * a.kv_heads + head) * a.tokens + off;
            uint32_t* const codes = reinterpret_cast<uint32_t*>((role ? a.pool.codes[1] : a.pool.codes[0]) + to * (D / 2)) + q;
#pragma unroll
            for (int c = 0; c < C; ++c) codes[4 * c] = w[c];
            if (q == 0) (role ? a.pool.scales[1] : a.pool.scales[0])[to] = finite ? (uint16_t)s16 : (uint16_t)0x7e00u;
        }
    }
    if (a.q_heads == 0) return;
    constexpr int LANES = D / 16, HEADS = 64 / LANES;
    auto where = [&](uint32_t head, const uint8_t*& from, uint8_t*& to) {
        from = a.x[2] + token * a.row[2] + head * a.head[2];
        to = a.out + token * a.out_row + head * a.out_head;
    };
    const float* const angles = a.angles + (size_t)token * D;
    const uint32_t first = (batch - a.batches) * HEADS + (uint32_t)lane / LANES;
    if (a.stream) rotate_heads<DT, D, true>(angles, 1.0f, first, a.waves * HEADS, a.q_heads, lane % LANES, where);
    else rotate_heads<DT, D, false>(angles, 1.0f, first, a.waves * HEADS, a.q_heads, lane % LANES, where);
}

// ------------------------------------------------------------------- read ----

struct ReadArgs {
    uint8_t* out[2];        // [rows, kv_heads, d]
    const int32_t* slots;
    FourBitRows pool;
    uint32_t rows, kv_heads, tokens, slot_end, stream;
    FastDiv by_tokens, by_heads;
    float hscale;
};

// A quad a row, its keys and then its values; sums of n - 8 are whole numbers of at most 2048, so fp16 holds them exactly, and
// each coordinate is rounded by its scale and by its type.  10149 tokens of 8 heads of 128 (11 MB to 42 MB) 11 us, 4.8 TB/s.
template <int DT, int D, bool STREAM>
__device__ __forceinline__ void read_rows(const ReadArgs& a) {
    constexpr int C = D / 32, SIZE = DT == NQ_F32 ? 4 : 2;
    const int q = threadIdx.x & 3;
    const uint32_t u = blockIdx.x * 64u + (threadIdx.x >> 2), n = a.rows * a.kv_heads, r = min(u, n - 1u);
    const uint32_t token = div(r, a.by_heads), head = r - token * a.kv_heads;
    const int32_t slot = a.slots[token];
    const bool stored = slot >= 0 && (uint32_t)slot < a.slot_end;
    const uint32_t page = stored ? div((uint32_t)slot, a.by_tokens) : 0u, off = stored ? (uint32_t)slot - page * a.tokens : 0u;
    const size_t at = ((size_t)page * a.kv_heads + head) * a.tokens + off;
#pragma unroll
    for (int role = 0; role < 2; ++role) {
        const uint32_t* const codes = reinterpret_cast<const uint32_t*>(a.pool.codes[role] + at * (D / 2)) + q;
        half2v h[C][4];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t w = codes[4 * c];
            const half2v bias = {(__fp16)-kNibbleBias, (__fp16)-kNibbleBias};
            const uint32_t p[4] = {nibble_pair<0>(w), nibble_pair<1>(w), nibble_pair<2>(w), nibble_pair<3>(w)};
            // (0, 4), (1, 5), (2, 6), (3, 7) to (0, 1), (2, 3), (4, 5), (6, 7)
            h[c][0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(p[1], p[0], 0x05040100u)) + bias;
            h[c][1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(p[3], p[2], 0x05040100u)) + bias;
            h[c][2] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(p[1], p[0], 0x07060302u)) + bias;
            h[c][3] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(p[3], p[2], 0x07060302u)) + bias;
        }
        const float f = f16_bits_to_f32(a.pool.scales[role][at]) * a.hscale * quad_sign(q);
        fwht_row_f16<C>(h, q);
        if (u >= n) continue;
        uint8_t* const o = a.out[role] + (size_t)r * D * SIZE;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[2 * k] = stored ? (float)h[c][k].x * f : 0.0f;
                x[2 * k + 1] = stored ? (float)h[c][k].y * f : 0.0f;
            }
            store8<DT, STREAM>(o + SIZE * (32 * c + 8 * q), x);
        }
    }
}

template <int DT, int D>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
    if (a.stream) read_rows<DT, D, true>(a);
    else read_rows<DT, D, false>(a);
}

int check_fourbit_pool(const nq_pool* p, int32_t layer, const char* who) {
    NQ_CHECK_ARG(p != nullptr, "%s: pool is NULL", who);
    NQ_CHECK_ARG(four_bit(p), "%s: the pool holds 8 bits a coordinate", who);
    NQ_CHECK_ARG(p->head_dim == 64 || p->head_dim == 128 || p->head_dim == 256, "%s: head_dim %d unsupported (64, 128, 256)", who, p->head_dim);
    NQ_CHECK_ARG(p->layers > 0 && p->pages > 0 && p->heads > 0 && p->tokens > 0 && layer >= 0 && layer < p->layers,
                 "%s: bad pool geometry, or layer %d of %d", who, layer, p->layers);
    NQ_CHECK_ARG((uint64_t)p->pages * p->heads * p->tokens < (1ull << 31), "%s: a layer must have less than 2^31 token rows", who);
    NQ_CHECK_ARG(p->key_codes && p->value_codes && p->key_scales && p->value_scales, "%s: the pool's arrays are required", who);
    NQ_CHECK_ARG((((uintptr_t)p->key_codes | (uintptr_t)p->value_codes | (uintptr_t)p->key_scales | (uintptr_t)p->value_scales) & 15u) == 0,
                 "%s: the pool's codes and scales must be 16-byte aligned", who);
    return NQ_OK;
}

FourBitRows fourbit_rows(const nq_pool* p, int32_t layer) {
    const size_t rows = (size_t)layer * p->pages * p->heads * p->tokens;
    FourBitRows r = {};
    r.codes[0] = reinterpret_cast<uint8_t*>(p->key_codes) + rows * (p->head_dim / 2);
    r.codes[1] = reinterpret_cast<uint8_t*>(p->value_codes) + rows * (p->head_dim / 2);
    r.scales[0] = static_cast<uint16_t*>(p->key_scales) + rows;
    r.scales[1] = static_cast<uint16_t*>(p->value_scales) + rows;
    return r;
}

#define NQ_BY_DIM(KERNEL, DT, d, ...)                                                     \
    switch (d) {                                                                          \
        case 64: hipLaunchKernelGGL((KERNEL<DT, 64>), __VA_ARGS__); break;                \
        case 128: hipLaunchKernelGGL((KERNEL<DT, 128>), __VA_ARGS__); break;              \
        default: hipLaunchKernelGGL((KERNEL<DT, 256>), __VA_ARGS__); break;               \
    }

// Waves that share a row's heads: one until the launch has fewer than 1024 workgroups.
static uint32_t share(uint64_t blocks, uint32_t most) {
    uint32_t n = 1;
    while (n < most && blocks * n < 1024) n *= 2;
    return n < most ? n : most;
}

}  // namespace nq

extern "C" int nq_rotation(const void* positions, int32_t int64_positions, int32_t axes, int64_t axis_stride, int64_t rows,
                           int32_t half, const float* inv_freq, const uint8_t* axis_of, float* out, void* stream) {
    using namespace nq;
    NQ_CHECK_ARG(axes >= 1 && axes <= 255 && rows >= 0 && half >= 1 && half <= 128, "nq_rotation: axes %d, rows %lld, half %d", axes,
                 (long long)rows, half);
    NQ_CHECK_ARG((uint64_t)rows * half < (1ull << 32) - 256, "nq_rotation: %lld rows are too many", (long long)rows);
    if (rows == 0) return NQ_OK;
    NQ_CHECK_ARG(positions && inv_freq && axis_of && out, "nq_rotation: positions, inv_freq, axis_of and out are required");
    AngleArgs a = {};
    a.positions = positions;
    a.out = out;
    a.stride = axis_stride;
    a.rows = (uint32_t)rows;
    a.half = (uint32_t)half;
    a.by_half = fast_div((uint32_t)half);
    a.wide = int64_positions;
    for (int32_t i = 0; i < half; ++i) {
        NQ_CHECK_ARG(axis_of[i] < axes, "nq_rotation: frequency %d is of axis %d of %d", i, axis_of[i], axes);
        a.freq[i] = inv_freq[i];
        a.axis[i] = axis_of[i];
    }
    hipLaunchKernelGGL(rotation_kernel, dim3((uint32_t)(((uint64_t)rows * half + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
    NQ_CHECK_HIP(hipGetLastError());
    return NQ_OK;
}

extern "C" int nq_rotate(const nq_rotate_desc* d, void* stream) {
    using namespace nq;
    NQ_CHECK_ARG(d != nullptr, "nq_rotate: desc is NULL");
    NQ_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "nq_rotate: head_dim %d unsupported (64, 128, 256)", d->head_dim);
    NQ_CHECK_ARG(d->dtype == NQ_F16 || d->dtype == NQ_BF16 || d->dtype == NQ_F32, "nq_rotate: unknown dtype %d", d->dtype);
    NQ_CHECK_ARG(d->rows >= 0 && d->q_heads >= 0 && d->k_heads >= 0, "nq_rotate: rows %d, q_heads %d, k_heads %d", d->rows, d->q_heads, d->k_heads);
    if (d->rows == 0 || d->q_heads + (int64_t)d->k_heads == 0) return NQ_OK;
    NQ_CHECK_ARG((int64_t)d->q_heads + d->k_heads < (1ll << 31), "nq_rotate: too many heads");
    NQ_CHECK_ARG(d->angles && (d->q_heads == 0 || (d->q && d->q_out)) && (d->k_heads == 0 || (d->k && d->k_out)),
                 "nq_rotate: angles, and inputs and outputs of all heads, are required");
    const int64_t size = d->dtype == NQ_F32 ? 4 : 2;
    const int64_t all = (d->q_stride[0] | d->q_stride[1] | d->k_stride[0] | d->k_stride[1] | d->q_out_stride[0] | d->q_out_stride[1] |
                         d->k_out_stride[0] | d->k_out_stride[1]) * size;
    NQ_CHECK_ARG(((all | (int64_t)(uintptr_t)d->q | (int64_t)(uintptr_t)d->k | (int64_t)(uintptr_t)d->q_out | (int64_t)(uintptr_t)d->k_out |
                   (int64_t)(uintptr_t)d->angles) & 15) == 0,
                 "nq_rotate: head vectors and angles must be 16-byte aligned");
    RotateArgs a = {};
    a.x[0] = static_cast<const uint8_t*>(d->q);
    a.x[1] = static_cast<const uint8_t*>(d->k);
    a.y[0] = static_cast<uint8_t*>(d->q_out);
    a.y[1] = static_cast<uint8_t*>(d->k_out);
    a.x_row[0] = d->q_stride[0] * size;
    a.x_head[0] = d->q_stride[1] * size;
    a.x_row[1] = d->k_stride[0] * size;
    a.x_head[1] = d->k_stride[1] * size;
    a.y_row[0] = d->q_out_stride[0] * size;
    a.y_head[0] = d->q_out_stride[1] * size;
    a.y_row[1] = d->k_out_stride[0] * size;
    a.y_head[1] = d->k_out_stride[1] * size;
    a.angles = d->angles;
    a.rows = (uint32_t)d->rows;
    a.heads[0] = (uint32_t)d->q_heads;
    a.heads[1] = (uint32_t)d->k_heads;
    a.sign = d->inverse ? -1.0f : 1.0f;
    const uint32_t per = 1024u / (uint32_t)d->head_dim;
    a.parts = share(((uint64_t)d->rows + 3) / 4, (a.heads[0] + a.heads[1] + per - 1) / per);
    a.stream = (uint64_t)d->rows * (a.heads[0] + (uint64_t)a.heads[1]) * d->head_dim * size >= kStreamBytes;
    const uint64_t blocks = ((uint64_t)d->rows * a.parts + 3) / 4;
    NQ_CHECK_ARG(blocks <= max_blocks(256) && (uint64_t)d->rows * a.parts < (1ull << 32), "nq_rotate: grid too large");
    const dim3 grid((uint32_t)blocks);
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == NQ_F16) NQ_BY_DIM(rotate_kernel, NQ_F16, d->head_dim, grid, dim3(256), 0, s, a)
    else if (d->dtype == NQ_BF16) NQ_BY_DIM(rotate_kernel, NQ_BF16, d->head_dim, grid, dim3(256), 0, s, a)
    else NQ_BY_DIM(rotate_kernel, NQ_F32, d->head_dim, grid, dim3(256), 0, s, a)
    NQ_CHECK_HIP(hipGetLastError());
    return NQ_OK;
}

extern "C" int nq_fourbit_append(const nq_fourbit_append_desc* d, void* stream) {
    using namespace nq;
    NQ_CHECK_ARG(d != nullptr, "nq_fourbit_append: desc is NULL");
    if (int st = check_fourbit_pool(d->pool, d->layer, "nq_fourbit_append")) return st;
    const nq_pool* p = d->pool;
    const int32_t dim = p->head_dim;
    NQ_CHECK_ARG(d->dtype == NQ_F16 || d->dtype == NQ_BF16, "nq_fourbit_append: dtype must be fp16 or bf16");
    NQ_CHECK_ARG(d->rows >= 0 && d->q_heads >= 0, "nq_fourbit_append: rows %d, q_heads %d", d->rows, d->q_heads);
    if (d->rows == 0) return NQ_OK;
    NQ_CHECK_ARG(d->k && d->v && d->slots && (d->q_heads == 0 || (d->q && d->q_out && d->angles)),
                 "nq_fourbit_append: keys, values, slots, and for queries an output and angles, are required");
    const int64_t all = d->k_stride[0] | d->k_stride[1] | d->v_stride[0] | d->v_stride[1] | d->q_stride[0] | d->q_stride[1] |
                        d->q_out_stride[0] | d->q_out_stride[1];
    NQ_CHECK_ARG(((2 * all | (int64_t)(uintptr_t)d->k | (int64_t)(uintptr_t)d->v | (int64_t)(uintptr_t)d->q | (int64_t)(uintptr_t)d->q_out |
                   (int64_t)(uintptr_t)d->angles) & 15) == 0,
                 "nq_fourbit_append: head vectors and angles must be 16-byte aligned");
    AppendArgs a = {};
    a.x[0] = static_cast<const uint8_t*>(d->k);
    a.x[1] = static_cast<const uint8_t*>(d->v);
    a.x[2] = static_cast<const uint8_t*>(d->q);
    const int64_t* const strides[3] = {d->k_stride, d->v_stride, d->q_stride};
    for (int i = 0; i < 3; ++i) {
        a.row[i] = 2 * strides[i][0];
        a.head[i] = 2 * strides[i][1];
    }
    a.out = static_cast<uint8_t*>(d->q_out);
    a.out_row = 2 * d->q_out_stride[0];
    a.out_head = 2 * d->q_out_stride[1];
    a.angles = d->angles;
    a.slots = d->slots;
    a.pool = fourbit_rows(p, d->layer);
    a.rows = (uint32_t)d->rows;
    a.q_heads = (uint32_t)d->q_heads;
    a.kv_heads = (uint32_t)p->heads;
    NQ_CHECK_ARG(2ll * p->heads + d->q_heads < (1ll << 30), "nq_fourbit_append: too many heads");
    a.batches = (2u * a.kv_heads + 15u) / 16u;
    const uint32_t per = 1024u / (uint32_t)dim;  // queries at a time
    a.waves = share(((uint64_t)d->rows + 3) / 4, a.batches + (a.q_heads + per - 1u) / per);
    a.stream = (uint64_t)d->rows * a.q_heads * dim * 2 >= kStreamBytes;
    a.tokens = (uint32_t)p->tokens;
    a.slot_end = (uint32_t)p->pages * (uint32_t)p->tokens;
    a.by_tokens = fast_div(a.tokens);
    a.hscale = d->hadamard_scale;
    const uint64_t blocks = ((uint64_t)d->rows * a.waves + 3) / 4;
    NQ_CHECK_ARG(blocks <= max_blocks(256) && (uint64_t)d->rows * a.waves < (1ull << 32), "nq_fourbit_append: grid too large");
    const dim3 grid((uint32_t)blocks);
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == NQ_F16) NQ_BY_DIM(append_kernel, NQ_F16, dim, grid, dim3(256), 0, s, a)
    else NQ_BY_DIM(append_kernel, NQ_BF16, dim, grid, dim3(256), 0, s, a)
    NQ_CHECK_HIP(hipGetLastError());
    return NQ_OK;
}

extern "C" int nq_fourbit_read(const nq_pool* p, int32_t layer, const int32_t* slots, int32_t n, int32_t dtype, float hadamard_scale,
                               void* keys, void* values, void* stream) {
    using namespace nq;
    if (int st = check_fourbit_pool(p, layer, "nq_fourbit_read")) return st;
    NQ_CHECK_ARG(dtype == NQ_F16 || dtype == NQ_BF16 || dtype == NQ_F32, "nq_fourbit_read: unknown dtype %d", dtype);
    NQ_CHECK_ARG(n >= 0 && (uint64_t)n * p->heads < (1ull << 32) - 64, "nq_fourbit_read: %d rows of %d heads", n, p->heads);
    if (n == 0) return NQ_OK;
    NQ_CHECK_ARG(slots && keys && values, "nq_fourbit_read: slots, keys and values are required");
    NQ_CHECK_ARG((((uintptr_t)keys | (uintptr_t)values) & 15u) == 0, "nq_fourbit_read: keys and values must be 16-byte aligned");
    ReadArgs a = {};
    a.out[0] = static_cast<uint8_t*>(keys);
    a.out[1] = static_cast<uint8_t*>(values);
    a.slots = slots;
    a.pool = fourbit_rows(p, layer);
    a.rows = (uint32_t)n;
    a.kv_heads = (uint32_t)p->heads;
    a.tokens = (uint32_t)p->tokens;
    a.slot_end = (uint32_t)p->pages * (uint32_t)p->tokens;
    a.by_tokens = fast_div(a.tokens);
    a.by_heads = fast_div(a.kv_heads);
    a.hscale = hadamard_scale;
    a.stream = 2ull * n * p->heads * p->head_dim * (dtype == NQ_F32 ? 4 : 2) >= kStreamBytes;
    const uint64_t blocks = ((uint64_t)n * p->heads + 63) / 64;
    NQ_CHECK_ARG(blocks <= max_blocks(256), "nq_fourbit_read: grid too large");
    const dim3 grid((uint32_t)blocks);
    const int32_t dim = p->head_dim;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == NQ_F16) NQ_BY_DIM(read_kernel, NQ_F16, dim, grid, dim3(256), 0, s, a)
    else if (dtype == NQ_BF16) NQ_BY_DIM(read_kernel, NQ_BF16, dim, grid, dim3(256), 0, s, a)
    else NQ_BY_DIM(read_kernel, NQ_F32, dim, grid, dim3(256), 0, s, a)
    NQ_CHECK_HIP(hipGetLastError());
    return NQ_OK;
}
