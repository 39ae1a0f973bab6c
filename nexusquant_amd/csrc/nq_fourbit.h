// A cache held in 4 bits: what its kernels share.
//
// A token's vector x of one head, d coordinates, is held as its Walsh-Hadamard transform t = H x (H orthonormal) in 16
// levels: s = fp16(max |t| / 7.5), n = clamp(floor(t / s + 8.5), 0, 15); it stands for H ((n - 8) s).  No coordinate is off by
// more than s / 2 (and what fp16 takes from s: 2^-11 of the largest, which is 7.5 s and held as 7 s or -7 s; -8 s stands only
// where fp16 rounded s down).  Zero is a level: with odd halves for levels a vector whose transform has one coordinate would
// get the others' halves on top of it.  The 8-bit pages' lattice in 4 bits a coordinate would lower the squared error by 0.65
// dB, and cost a coset to be found out for each 8 nibbles.
// Coordinate i of a row is nibble i % 2 of byte i / 2.  Keys are transformed after their rotation, so a product with a
// query needs neither: q . x = s (H q) . (n - 8).
//
// A row whose transform holds an infinity or a NaN has a NaN scale; scales past 65504 are held as that.
#pragma once

#include "nq_common.h"

namespace nq {

// The pool as kernels see it: a layer's rows are [pages, heads, tokens].
struct FourBitRows {
    uint8_t* codes[2];    // keys, values: d / 2 bytes a row
    uint16_t* scales[2];  // fp16
};

// A pool of 4 bits a coordinate has no positions; one that has them holds 8 bits, whatever `reserved` (which the entry points
// of such pools never read) is.
inline bool four_bit(const nq_pool* p) { return p->reserved == 4 && p->positions == nullptr; }

int check_fourbit_pool(const nq_pool* p, int32_t layer, const char* who);
FourBitRows fourbit_rows(const nq_pool* p, int32_t layer);

// Nibbles of a word in pairs (j, j + 4), j = 0 .. 3, as fp16 values 16 + n: the nibble under the exponent of 16.
constexpr uint32_t kNibbleMask = 0x03C003C0u, kSixteens = 0x4C004C00u;
template <int J>
__device__ __forceinline__ uint32_t nibble_pair(uint32_t w, uint32_t mask = kNibbleMask, uint32_t sixteens = kSixteens) {
    constexpr int at = 6 - 4 * J;  // where the nibble goes, from where it is
    const uint32_t x = at >= 0 ? w << (at >= 0 ? at : 0) : w >> (at < 0 ? -at : 0);
    return (x & mask) | sixteens;
}
constexpr float kNibbleBias = 24.0f;  // (16 + n) - kNibbleBias = n - 8

}  // namespace nq
