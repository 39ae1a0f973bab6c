// Layout of the attention kernels' tiles of keys and values in LDS, and where a lane's pieces of a stage come from.
// Plain C++ without HIP: the host's tests replay it.
#pragma once

#include <stdint.h>

namespace nq {
namespace flash {

// A tile's LDS layout: row r (a key) at byte r * 2 D, its 16-byte chunk c at chunk place
// c ^ f(r).  Keys are read 32 rows at one chunk (ds_read_b128), values 4 rows at 64 bytes
// (transposing ds_read_b64); each f spreads its read over all 64 banks.
template <int D>
struct Tile {
    static constexpr int ROWB = 2 * D;
    static constexpr int UPR = D / 8;           // 16-byte chunks a row
    static constexpr int KS = D / 16;           // MFMA steps of a logit
    static constexpr int DB = D / 32;           // 32-coordinate blocks of the output
    static constexpr int key_swizzle(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
    // (its bit 0 is for writers of two chunks a lane: half of their rows then take the odd one first)
    static constexpr int value_swizzle(int r) {
        return (D == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3)) ^ ((r >> 2) & 1);
    }
};

// Rows to LDS in Tile's layout, 16 bytes a lane, 256 lanes: load i fills the places from 256 i on, so lane
// (thread) s the place s % UPR of row s / UPR + STEP i.  Which chunk stands there repeats after PERIOD loads.
template <int D, bool VALUES>
struct StagePieces {
    using T = Tile<D>;
    static constexpr int STEP = 256 / T::UPR;   // rows of a load
    static constexpr int PERIOD = !VALUES && D == 256 ? 2 : 1;
    static constexpr int row(int s, int i) { return s / T::UPR + STEP * i; }
    static constexpr int chunk(int s, int i) {
        const int r = row(s, i % PERIOD);
        return (s % T::UPR) ^ (VALUES ? T::value_swizzle(r) : T::key_swizzle(r));
    }
    // bytes from row STEP i (rows `stride` elements apart) to the lane's piece of load i: the same after PERIOD loads
    static constexpr uint32_t offset(int s, int i, int64_t stride) {
        return (uint32_t)row(s, 0) * (uint32_t)(2 * stride) + 16u * (uint32_t)chunk(s, i);
    }
};

}  // namespace flash
}  // namespace nq
