// The Walsh-Hadamard stages of a page's keys below the top one, as int8 matrix products
// (decode attention from compressed pages).
#pragma once

#include "nq_common.h"

namespace nq {

typedef int int4v __attribute__((ext_vector_type(4)));

// The half-row Walsh-Hadamard matrix as int8 MFMA A operands.  Rows are output
// coordinates m = 16 t + r (r = lane % 16), columns the codes k = KB u + KPL kg + j
// (kg = lane / 16, j the lane's byte): entry (-1)^popcount(m & k), which is the
// entry of tile 0 and step 0 with its sign set by a parity of t, u and kg alone.
template <int D>
struct KeyMfma {
    static constexpr int HALF = D / 2;
    static constexpr int KB = HALF < 64 ? 32 : 64;  // codes per MFMA
    static constexpr int KPL = KB / 4;              // of them per lane
    static constexpr int NK = HALF / KB;            // MFMAs per tile
    static constexpr int T = HALF / 16;             // tiles per half row
    static constexpr int W = KPL / 4;               // operand dwords
    uint32_t h[W];

    __device__ __forceinline__ void init(int lane) {
        const uint32_t r = lane & 15, kg = lane >> 4;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            uint32_t v = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t k = KPL * kg + 4 * w + b;
                v |= (uint32_t)((__builtin_popcount(r & k & 15u) & 1) ? 0xff : 0x01) << (8 * b);
            }
            h[w] = v;
        }
    }
    // acc += (tile t, step u) x the codes
    __device__ __forceinline__ int4v mul(int t, int u, int lane, const uint32_t (&c)[W], int4v acc) const {
        const uint32_t kg = lane >> 4;
        const uint32_t hi = (KB == 64 ? 4u * u + kg : kg >> 1) & (uint32_t)t;  // the bits of k from 16 on
        const uint32_t flip = (__builtin_popcount(hi) & 1) ? 0xfefefefeu : 0u; // +1 <-> -1
        if constexpr (KB == 64) {
            const int4v a = {(int)(h[0] ^ flip), (int)(h[1] ^ flip), (int)(h[2] ^ flip), (int)(h[3] ^ flip)};
            const int4v b = {(int)c[0], (int)c[1], (int)c[2], (int)c[3]};
            return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
        } else {
            const uint64_t a = (uint64_t)(h[0] ^ flip) | (uint64_t)(h[1] ^ flip) << 32;
            const uint64_t b = (uint64_t)c[0] | (uint64_t)c[1] << 32;
            return __builtin_amdgcn_mfma_i32_16x16x32_i8((long)a, (long)b, acc, 0, 0, 0);
        }
    }
};

}  // namespace nq
