// One pass of softmax attention over tiles of keys and values in LDS: 32 query rows a
// wave, running maximum and sum, matrix cores for both products.
//
// With q the wave's 32 queries, a tile of 32 keys K and its values V:
//   S^T = K q^T      32x32x16 MFMAs, keys the A operand: lane (n, g) gets its query n's
//                    logits at the keys acc_row(j, g) = 8 (j / 4) + 4 g + j % 4
//   p   = 2^(c s - m)  c = scale * log2(e), m >= c max s - kSlack - LIFT: lane-local
//   O^T += V^T P^T   P^T is the B operand as it stands (an MFMA's k order is free as long
//                    as both operands share it: slot (g, i) of step s is key
//                    16 s + 8 (i / 4) + 4 g + i % 4), V^T the A operand by transposing
//                    LDS reads (ds_read_b64_tr_b16: 4 keys x 16 coordinates of 16 lanes)
// so a query's maximum, sum and output stay in the two lanes (n, 0) and (n, 1).
#pragma once

#include "nq_common.h"
#include "nq_tile.h"

namespace nq {
namespace flash {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// A running maximum may lag the true one by 2^kSlack before the output is rescaled: weights stay at
// most 256 times what they are at the maximum (sums in fp32, weights in fp16 or bf16 have the room), and
// the 16 D / 32 multiplies of a rescale run in the first stages of a row only.
constexpr float kSlack = 8.0f;
constexpr float kNoMax = -3.0e38f;  // finite, so that a row that has seen no key forms no inf - inf

template <int DT>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == NQ_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two floats rounded to nearest even, packed
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == NQ_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
template <int DT>
__device__ __forceinline__ float unpack(uint32_t bits16) {
    if constexpr (DT == NQ_F16) return f16_bits_to_f32(bits16);
    else return bf16_bits_to_f32(bits16);
}

// The values of lanes l and l + 32, in either.  (Elements are taken out before they are cast: a bit
// cast of a vector's element reads the first one.)
__device__ __forceinline__ f32x2 halves(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return {__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ float both_max(float v) {
    const f32x2 h = halves(v);
    return __builtin_fmaxf(h.x, h.y);
}
__device__ __forceinline__ float both_sum(float v) {
    const f32x2 h = halves(v);
    return h.x + h.y;
}

__device__ __forceinline__ int acc_row(int j, int g) { return 8 * (j >> 2) + 4 * g + (j & 3); }

template <int DT, int D>
struct Rows {
    using T = Tile<D>;
    u32x4 q[T::KS];       // lane (n, g): query n, coordinates 16 s + 8 g + 0..7
    f32x16 o[T::DB];      // lane (n, g): query n, coordinates 32 b + acc_row(j, g)
    float m, l;           // c * (lagging) maximum - LIFT; this lane's part of the sum
    uint32_t k_at, v_at, v_xor;

    __device__ __forceinline__ void init(int lane) {
        const int n = lane & 31, g = lane >> 5;
#pragma unroll
        for (int b = 0; b < T::DB; ++b) o[b] = f32x16{};
        m = kNoMax;
        l = 0.0f;
        // keys: row n of a tile, chunk (2 s + g) ^ swizzle(n); swizzles of rows n and n + 32 agree
        k_at = (uint32_t)(n * T::ROWB + 16 * (g ^ T::key_swizzle(n)));
        // values: row 4 g + r of a step, r = lane / 4 % 4; chunk 4 b + 2 (lane / 16 % 2) + lane / 2 % 2
        const int r = 4 * g + ((lane >> 2) & 3);
        v_at = (uint32_t)(r * T::ROWB + 16 * (2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 8 * (lane & 1));
        v_xor = (uint32_t)(16 * T::value_swizzle(r));
    }

    __device__ __forceinline__ f32x16 logits(const char* kbuf, int t) const {
        f32x16 s = {};
        const char* const base = kbuf + t * 32 * T::ROWB;
#pragma unroll
        for (int i = 0; i < T::KS; ++i)
            s = mfma<DT>(*reinterpret_cast<const u32x4*>(base + (k_at ^ (uint32_t)(32 * i))), q[i], s);
        return s;
    }

    __device__ __forceinline__ u32x4 value_operand(const char* vbuf, int t, int s, int b) const {
        const uint32_t at = (uint32_t)((t * 32 + 16 * s) * T::ROWB) + ((v_at + 64u * (uint32_t)b) ^ v_xor);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)(vbuf + at));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)(vbuf + at + 8 * T::ROWB));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), c = __builtin_bit_cast(u32x2, hi);
        return u32x4{a.x, a.y, c.x, c.y};
    }

    // What m is below the maximum.  fp16 weights are up to 2^(kSlack + LIFT) = 2^15 then, and keep their 11 bits down to
    // 2^-21 of a row's largest; without it 2^-14: a first token that takes nearly all of the weight leaves little above
    // that to the others, and where its values are near zero they are the output.  (Scales of their own, SCALED, do this.)
    template <bool SCALED>
    static constexpr float LIFT = DT == NQ_F16 && !SCALED ? 7.0f : 0.0f;

    // the maximum of the stage's logits (c > 0), and the output rescaled where it passes the slack
    template <bool SCALED>
    __device__ __forceinline__ void raise(float mx, float c) {
        mx = both_max(mx) * c;
        if (__any(mx > m + (kSlack + LIFT<SCALED>))) {
            const float to = __builtin_fmaxf(m, mx - LIFT<SCALED>);
            const float f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int b = 0; b < T::DB; ++b) o[b] *= f;
        }
    }

    // SCALED: the weights of the sum of values are times v[key of the tile], in LDS
    template <bool SCALED>
    __device__ __forceinline__ void weights(const f32x16& s, float c, uint32_t (&p)[8], const float* v, int g) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 f = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (SCALED) f = *reinterpret_cast<const f32x4*>(v + 8 * i + 4 * g);
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + k], c, -m));
                float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + k + 1], c, -m));
                sum += x;
                sum += y;
                if constexpr (SCALED) {
                    x *= f[k];
                    y *= f[k + 1];
                }
                p[2 * i + k / 2] = pack2<DT>(x, y);
            }
        }
        l += sum;
    }

    __device__ __forceinline__ void add_values(const uint32_t (&p)[8], const char* vbuf, int t) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const u32x4 w = {p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]};
#pragma unroll
            for (int b = 0; b < T::DB; ++b) o[b] = mfma<DT>(value_operand(vbuf, t, s, b), w, o[b]);
        }
    }

    // tiles t and t + 1, which every query sees whole
    template <bool SCALED = false>
    __device__ __forceinline__ void two_tiles(const char* kbuf, const char* vbuf, int t, float c, int g, const float* v = nullptr) {
        f32x16 s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i] = f32x16{};
#pragma unroll
        for (int k = 0; k < T::KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                s[i] = mfma<DT>(*reinterpret_cast<const u32x4*>(kbuf + (t + i) * 32 * T::ROWB + (k_at ^ (uint32_t)(32 * k))), q[k], s[i]);
        float mx = s[0][0];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = __builtin_fmaxf(mx, s[i][j]);
        // the wave that is past its logits goes first, so that a SIMD's waves fall out of step and one's
        // exponentials run under the other's products
        __builtin_amdgcn_s_setprio(1);
        raise<SCALED>(mx, c);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t p[8];
            weights<SCALED>(s[i], c, p, v + 32 * i, g);
            add_values(p, vbuf, t + i);
        }
        __builtin_amdgcn_s_setprio(0);
    }

    // tile t, of which this lane's query sees the keys lo <= key < hi (of 32)
    template <bool SCALED = false>
    __device__ __forceinline__ void masked_tile(const char* kbuf, const char* vbuf, int t, float c, int lo, int hi, int g,
                                                const float* v = nullptr) {
        f32x16 s = logits(kbuf, t);
        float mx = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int key = acc_row(j, g);
            s[j] = key >= lo && key < hi ? s[j] : -__builtin_inff();
            mx = __builtin_fmaxf(mx, s[j]);
        }
        raise<SCALED>(mx, c);
        uint32_t p[8];
        weights<SCALED>(s, c, p, v, g);
        add_values(p, vbuf, t);
    }
};

}  // namespace flash
}  // namespace nq
