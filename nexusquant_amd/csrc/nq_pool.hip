// Pages of a compressed cache moved within their pool: whole pages copied
// (branches of a sequence), kept tokens compacted into fewer pages (eviction),
// newly encoded tokens written to their slots.
//
// A pool holds, per layer and page, int8 codes [heads, tokens, d] and fp16 scales
// [heads, tokens] of keys and values, and int32 positions [tokens] per page for all
// layers.  Nothing is computed: every operator is bytes read once and written once,
// so HBM's copy rate bounds the large ones and the launch the small ones.
#include "nq_fourbit.h"

#include <stdlib.h>

namespace nq {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct PoolPtrs {
    char* codes[2];   // keys, values: [layers, pages, heads * tokens * d] bytes
    char* scales[2];  // [layers, pages, heads * tokens * 2] bytes
    int32_t* positions;
    uint32_t pages;
};

// ----------------------------------------------------------------- copies ----

// The page pairs of a launch travel in its arguments (a kernel's arguments take 4 KB):
// no copy to the device ahead of it, and nothing that must outlive it.
constexpr int kCopyPairs = 448;
// Copies of fewer bytes stay in the 8 L2s of 4 MB: a branch's last page is read by its next step.
constexpr uint64_t kStreamBytes = 32ull << 20;

struct CopyArgs {
    PoolPtrs p;
    uint32_t code_bytes, scale_bytes, tokens;   // a page's, in one layer
    uint32_t code_units, scale_units;           // in all: pairs * layers * 2 * bytes / width
    uint32_t code_blocks, scale_blocks, pos_units;
    uint32_t pairs;
    FastDiv code_page, scale_page, by_pairs, by_tokens;
    int32_t src[kCopyPairs], dst[kCopyPairs];
};

// `Unit`-sized pieces first .. first + 4 * 256 of all pairs and layers: piece u of page x,
// x = ((role * layers) + layer) * pairs + pair.
template <typename Unit, bool STREAM>
__device__ __forceinline__ void copy_units(const CopyArgs& a, char* const (&base)[2], uint32_t bytes, const FastDiv& per_page,
                                           uint32_t units, uint32_t layers, uint32_t first) {
    Unit v[4];
    char* to[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = first + 256u * i + threadIdx.x;
        to[i] = nullptr;
        if (u < units) {
            const uint32_t x = div(u, per_page), at = (u - x * per_page.d) * (uint32_t)sizeof(Unit);
            const uint32_t lr = div(x, a.by_pairs), pair = x - lr * a.pairs;
            const uint32_t role = lr >= layers, layer = role ? lr - layers : lr;
            char* const b = base[role] + (size_t)layer * a.p.pages * bytes + at;
            const Unit* const from = reinterpret_cast<const Unit*>(b + (size_t)a.src[pair] * bytes);
            if constexpr (STREAM) v[i] = __builtin_nontemporal_load(from);
            else v[i] = *from;
            to[i] = b + (size_t)a.dst[pair] * bytes;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (to[i]) {
            if constexpr (STREAM) __builtin_nontemporal_store(v[i], reinterpret_cast<Unit*>(to[i]));
            else *reinterpret_cast<Unit*>(to[i]) = v[i];
        }
}

// A thread moves four 16-byte pieces, all loads ahead of the stores: 1024 pages of 16 layers (8 heads x 16 x 128,
// 1.09 GB read and written) 212 us, 5.14 TB/s, a large copy's rate.  STREAM, from kStreamBytes on: codes past the
// caches (233 us without).
template <typename ScaleUnit, bool STREAM>
__global__ __launch_bounds__(256) void pool_copy_kernel(CopyArgs a, uint32_t layers) {
    uint32_t blk = blockIdx.x;
    if (blk < a.code_blocks) {
        copy_units<u32x4, STREAM>(a, a.p.codes, a.code_bytes, a.code_page, a.code_units, layers, blk * 1024u);
        return;
    }
    blk -= a.code_blocks;
    if (blk < a.scale_blocks) {
        copy_units<ScaleUnit, false>(a, a.p.scales, a.scale_bytes, a.scale_page, a.scale_units, layers, blk * 1024u);
        return;
    }
    blk -= a.scale_blocks;
    const uint32_t u = blk * 256u + threadIdx.x;
    if (u < a.pos_units) {
        const uint32_t pair = div(u, a.by_tokens), t = u - pair * a.tokens;
        a.p.positions[(size_t)a.dst[pair] * a.tokens + t] = a.p.positions[(size_t)a.src[pair] * a.tokens + t];
    }
}

// ------------------------------------------------------------ token moves ----

constexpr int kMoveTokens = 64;  // tokens of a workgroup

// A compaction's plan, or a write's slots, of at most this many integers travel in the launch's arguments: the copy to
// the device ahead of it and what it waits for were 11 us of a call of 8191 tokens in one layer (90 us with it, 81 without).
constexpr int kPlanInts = 896;

// A source of token rows: pages of `tokens` rows a head.
struct MoveArgs {
    PoolPtrs src, dst;
    uint32_t src_tokens, dst_tokens;  // tokens a page
    uint32_t heads, d;
    uint32_t head_split;              // workgroups that share a tile's heads
    uint32_t n;                       // writes: tokens in all
    int32_t renumber;
    // compaction: per tile its sequence, per sequence {first tile, tokens kept, tokens it had, src table, dst table},
    // and from there on the tables; writes: the slot of each token, negative: none
    const int32_t* plan;
    uint32_t seq_at, tables_at;
    const int32_t* kept;
    uint32_t kept_stride;
    uint32_t slot_end;                // writes: of the pool
};
struct InlineArgs : MoveArgs {
    int32_t ints[kPlanInts];
};
__device__ __forceinline__ int32_t plan_at(const MoveArgs& a, uint32_t i) { return a.plan[i]; }
__device__ __forceinline__ int32_t plan_at(const InlineArgs& a, uint32_t i) { return a.ints[i]; }

// Rows of D bytes: D / 16 lanes a row.  The workgroup's token slots are worked out once, into
// LDS, and serve every head of its share: keys and values of a head are 2 * 64 rows, moved as
// 16-byte pieces with all of a thread's loads ahead of its stores.
template <int D, bool COMPACT, typename Args>
__global__ __launch_bounds__(256) void pool_move_kernel(Args a) {
    constexpr int UR = D / 16;                    // 16-byte units a row
    constexpr int PER = (kMoveTokens * UR + 255) / 256;  // of a role and head, per thread (D 32: half of the threads have one)
    __shared__ uint64_t s_src[kMoveTokens], s_dst[kMoveTokens];  // row index of head 0, page by page
    const uint32_t tile = blockIdx.x / a.head_split, part = blockIdx.x % a.head_split;
    const uint32_t layer = blockIdx.y;
    uint32_t n_tok;
    if constexpr (COMPACT) {
        const int32_t sq = plan_at(a, tile);
        const uint32_t s = a.seq_at + 5u * (uint32_t)sq;
        const uint32_t first = (tile - (uint32_t)plan_at(a, s)) * kMoveTokens;
        n_tok = min((uint32_t)plan_at(a, s + 1) - first, (uint32_t)kMoveTokens);
        if (threadIdx.x < n_tok) {
            const uint32_t j = first + threadIdx.x;
            const int32_t had = plan_at(a, s + 2);
            int32_t i = a.kept[(size_t)sq * a.kept_stride + j];
            i = i < 0 ? 0 : (i >= had ? had - 1 : i);  // the caller's list; clamped, so no page is read past its sequence
            const uint32_t sp = (uint32_t)i / a.src_tokens, so = (uint32_t)i % a.src_tokens;
            const uint32_t dp = j / a.dst_tokens, d0 = j % a.dst_tokens;
            const uint64_t spage = (uint32_t)plan_at(a, a.tables_at + (uint32_t)plan_at(a, s + 3) + sp);
            const uint64_t dpage = (uint32_t)plan_at(a, a.tables_at + (uint32_t)plan_at(a, s + 4) + dp);
            s_src[threadIdx.x] = spage * a.heads * a.src_tokens + so;
            s_dst[threadIdx.x] = dpage * a.heads * a.dst_tokens + d0;
            if (layer == 0 && part == 0 && a.dst.positions)
                a.dst.positions[dpage * a.dst_tokens + d0] =
                    a.renumber ? (int32_t)j : a.src.positions[spage * a.src_tokens + so];
        }
    } else {
        const uint32_t first = tile * kMoveTokens;
        n_tok = min(a.n - first, (uint32_t)kMoveTokens);
        if (threadIdx.x < n_tok) {
            const uint32_t j = first + threadIdx.x;
            const int32_t slot = plan_at(a, j);
            const bool ok = slot >= 0 && (uint32_t)slot < a.slot_end;
            const uint64_t dp = ok ? (uint32_t)slot / a.dst_tokens : 0u, d0 = ok ? (uint32_t)slot % a.dst_tokens : 0u;
            s_src[threadIdx.x] = j;  // one page of n tokens a head
            s_dst[threadIdx.x] = ok ? dp * a.heads * a.dst_tokens + d0 : ~0ull;
            if (ok && part == 0) a.dst.positions[slot] = a.src.positions[j];
        }
    }
    __syncthreads();
    const size_t src_layer = (size_t)layer * a.src.pages * a.heads * a.src_tokens;
    const size_t dst_layer = (size_t)layer * a.dst.pages * a.heads * a.dst_tokens;
    for (uint32_t h = part; h < a.heads; h += a.head_split) {
        const size_t src_head = src_layer + (size_t)h * a.src_tokens, dst_head = dst_layer + (size_t)h * a.dst_tokens;
        u32x4 v[2][PER];
#pragma unroll
        for (int role = 0; role < 2; ++role)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t u = 256u * i + threadIdx.x, t = u / UR;
                if (t < n_tok)
                    v[role][i] = *reinterpret_cast<const u32x4*>(a.src.codes[role] + (src_head + s_src[t]) * D + 16u * (u % UR));
            }
#pragma unroll
        for (int role = 0; role < 2; ++role)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t u = 256u * i + threadIdx.x, t = u / UR;
                if (t < n_tok && (COMPACT || s_dst[t] != ~0ull))
                    *reinterpret_cast<u32x4*>(a.dst.codes[role] + (dst_head + s_dst[t]) * D + 16u * (u % UR)) = v[role][i];
            }
        const uint32_t t = threadIdx.x & 63u, role = threadIdx.x >> 6;
        if (role < 2 && t < n_tok && (COMPACT || s_dst[t] != ~0ull))
            reinterpret_cast<uint16_t*>(a.dst.scales[role])[dst_head + s_dst[t]] =
                reinterpret_cast<const uint16_t*>(a.src.scales[role])[src_head + s_src[t]];
    }
}

// Workgroups that share a tile's heads: one until the launch has fewer than 2048 (eight a CU).
static uint32_t head_split(uint32_t heads, uint64_t tiles) {
    uint32_t split = 1;
    while (split < heads && tiles * split < 2048) split *= 2;
    return split < heads ? split : heads;
}

template <bool COMPACT, typename Args>
static hipError_t launch_move(const Args& a, uint32_t tiles, uint32_t layers, hipStream_t s) {
    const dim3 grid(tiles * a.head_split, layers);
    switch (a.d) {
        case 32:
            if constexpr (COMPACT) hipLaunchKernelGGL((pool_move_kernel<32, COMPACT, Args>), grid, dim3(256), 0, s, a);
            break;
        case 64: hipLaunchKernelGGL((pool_move_kernel<64, COMPACT, Args>), grid, dim3(256), 0, s, a); break;
        case 128: hipLaunchKernelGGL((pool_move_kernel<128, COMPACT, Args>), grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((pool_move_kernel<256, COMPACT, Args>), grid, dim3(256), 0, s, a); break;
    }
    return hipGetLastError();
}

template <bool COMPACT>
static hipError_t launch_plan(const MoveArgs& a, bool on_host, uint32_t ints, uint32_t tiles, uint32_t layers, hipStream_t s) {
    if (!on_host) return launch_move<COMPACT>(a, tiles, layers, s);
    InlineArgs in = {};
    static_cast<MoveArgs&>(in) = a;
    memcpy(in.ints, a.plan, (size_t)ints * sizeof(int32_t));
    return launch_move<COMPACT>(in, tiles, layers, s);
}

template <typename ScaleUnit>
static void launch_copy(dim3 grid, hipStream_t s, const CopyArgs& a, uint32_t layers) {
    if (16ull * a.code_units >= kStreamBytes) hipLaunchKernelGGL((pool_copy_kernel<ScaleUnit, true>), grid, dim3(256), 0, s, a, layers);
    else hipLaunchKernelGGL((pool_copy_kernel<ScaleUnit, false>), grid, dim3(256), 0, s, a, layers);
}

// A row's bytes of codes: a pool of 4 bits a coordinate has half of them, and no positions.
static uint32_t row_bytes(const nq_pool* p) { return (uint32_t)(four_bit(p) ? p->head_dim / 2 : p->head_dim); }

static int check_pool(const nq_pool* p, const char* who) {
    NQ_CHECK_ARG(p != nullptr, "%s: pool is NULL", who);
    NQ_CHECK_ARG(p->head_dim == 64 || p->head_dim == 128 || p->head_dim == 256,
                 "%s: head_dim %d unsupported (64, 128, 256)", who, p->head_dim);
    NQ_CHECK_ARG(p->layers > 0 && p->layers <= 65535 && p->pages > 0 && p->heads > 0 && p->tokens > 0,
                 "%s: bad geometry (%d layers, %d pages, %d heads, %d tokens)", who, p->layers, p->pages, p->heads,
                 p->tokens);
    NQ_CHECK_ARG((uint64_t)p->heads * p->tokens * p->head_dim < (1ull << 31) &&
                     (uint64_t)p->pages * p->tokens < (1ull << 31),
                 "%s: a page's codes and the pool's slots must each stay below 2^31", who);
    NQ_CHECK_ARG(p->key_codes && p->value_codes && p->key_scales && p->value_scales && (p->positions || four_bit(p)),
                 "%s: the pool's arrays are required", who);
    NQ_CHECK_ARG((((uintptr_t)p->key_codes | (uintptr_t)p->value_codes | (uintptr_t)p->key_scales |
                   (uintptr_t)p->value_scales) & 15u) == 0 && ((uintptr_t)p->positions & 3u) == 0,
                 "%s: the pool's codes and scales must be 16-byte aligned", who);
    return NQ_OK;
}

static PoolPtrs pool_ptrs(const nq_pool* p) {
    PoolPtrs x = {};
    x.codes[0] = reinterpret_cast<char*>(p->key_codes);
    x.codes[1] = reinterpret_cast<char*>(p->value_codes);
    x.scales[0] = static_cast<char*>(p->key_scales);
    x.scales[1] = static_cast<char*>(p->value_scales);
    x.positions = p->positions;
    x.pages = (uint32_t)p->pages;
    return x;
}

}  // namespace nq

extern "C" int nq_pool_copy_pages(const nq_pool* p, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
    using namespace nq;
    if (int st = check_pool(p, "nq_pool_copy_pages")) return st;
    NQ_CHECK_ARG(n >= 0, "nq_pool_copy_pages: n %d", n);
    if (n == 0) return NQ_OK;
    NQ_CHECK_ARG(src && dst, "nq_pool_copy_pages: src and dst are required");
    // one bit a page: every page is written at most once, and none that is read
    uint8_t* const written = static_cast<uint8_t*>(calloc((size_t)(p->pages + 7) / 8, 1));
    if (written == nullptr) {
        set_error("nq_pool_copy_pages: out of host memory");
        return NQ_EHIP;
    }
    const char* bad = nullptr;
    int32_t at = 0;
    for (int32_t i = 0; i < n && !bad; ++i) {
        at = i;
        if (src[i] < 0 || src[i] >= p->pages || dst[i] < 0 || dst[i] >= p->pages) bad = "is not a page of the pool";
        else if (written[dst[i] >> 3] >> (dst[i] & 7) & 1) bad = "names a destination twice";
        else written[dst[i] >> 3] |= (uint8_t)(1u << (dst[i] & 7));
    }
    for (int32_t i = 0; i < n && !bad; ++i) {
        at = i;
        if (written[src[i] >> 3] >> (src[i] & 7) & 1) bad = "reads a page that the call writes";
    }
    free(written);
    NQ_CHECK_ARG(!bad, "nq_pool_copy_pages: pair %d (%d to %d) %s", at, src[at], dst[at], bad);

    CopyArgs a = {};
    a.p = pool_ptrs(p);
    a.code_bytes = (uint32_t)p->heads * p->tokens * row_bytes(p);
    a.scale_bytes = (uint32_t)p->heads * p->tokens * 2u;
    a.tokens = (uint32_t)p->tokens;
    // scales in the widest pieces that every page's offset allows
    const uint32_t width = a.scale_bytes % 16 == 0 ? 16u : a.scale_bytes % 4 == 0 ? 4u : 2u;
    a.code_page = fast_div(a.code_bytes / 16);
    a.scale_page = fast_div(a.scale_bytes / width);
    a.by_tokens = fast_div(a.tokens);
    // pairs a launch: what its arguments hold, and what 32-bit piece indices reach
    const uint64_t per_pair = 2ull * p->layers * (a.code_bytes / 16 > a.scale_bytes / width ? a.code_bytes / 16 : a.scale_bytes / width);
    NQ_CHECK_ARG(per_pair < (1ull << 31), "nq_pool_copy_pages: a page of all layers is too large");
    uint64_t most = ((1ull << 31) - 1) / per_pair;
    if (most > kCopyPairs) most = kCopyPairs;
    hipStream_t s = (hipStream_t)stream;
    for (int32_t i = 0; i < n; i += (int32_t)most) {
        a.pairs = (uint32_t)((uint64_t)(n - i) < most ? (uint64_t)(n - i) : most);
        memcpy(a.src, src + i, a.pairs * sizeof(int32_t));
        memcpy(a.dst, dst + i, a.pairs * sizeof(int32_t));
        a.by_pairs = fast_div(a.pairs);
        const uint32_t pages = 2u * (uint32_t)p->layers * a.pairs;
        a.code_units = pages * (a.code_bytes / 16);
        a.scale_units = pages * (a.scale_bytes / width);
        a.pos_units = four_bit(p) ? 0u : a.pairs * a.tokens;
        a.code_blocks = (a.code_units + 1023u) / 1024u;
        a.scale_blocks = (a.scale_units + 1023u) / 1024u;
        const dim3 grid(a.code_blocks + a.scale_blocks + (a.pos_units + 255u) / 256u);
        const uint32_t layers = (uint32_t)p->layers;
        if (width == 16) launch_copy<u32x4>(grid, s, a, layers);
        else if (width == 4) launch_copy<uint32_t>(grid, s, a, layers);
        else launch_copy<uint16_t>(grid, s, a, layers);
        NQ_CHECK_HIP(hipGetLastError());
    }
    return NQ_OK;
}

extern "C" int32_t nq_pool_move_tokens(void) { return nq::kMoveTokens; }

extern "C" int32_t nq_pool_host_ints(void) { return nq::kPlanInts; }

extern "C" int nq_pool_compact(const nq_pool* p, const int32_t* plan, int32_t plan_ints, int32_t plan_on_host, int32_t n_tiles,
                               int32_t n_seq, const int32_t* kept, int32_t kept_stride, int32_t renumber, void* stream) {
    using namespace nq;
    if (int st = check_pool(p, "nq_pool_compact")) return st;
    NQ_CHECK_ARG(n_tiles >= 0 && kept_stride >= 0, "nq_pool_compact: n_tiles %d, kept_stride %d", n_tiles, kept_stride);
    if (n_tiles == 0) return NQ_OK;
    NQ_CHECK_ARG(plan && kept, "nq_pool_compact: the plan and the kept list are required");
    NQ_CHECK_ARG(!four_bit(p) || !renumber, "nq_pool_compact: a pool of 4 bits a coordinate stores keys rotated and cannot renumber");
    NQ_CHECK_ARG(n_seq > 0 && plan_ints > 0 && (int64_t)n_tiles + 5ll * n_seq <= plan_ints,
                 "nq_pool_compact: %d integers hold no plan of %d tiles and %d sequences", plan_ints, n_tiles, n_seq);
    NQ_CHECK_ARG(!plan_on_host || plan_ints <= kPlanInts, "nq_pool_compact: a host plan has at most %d integers, got %d",
                 kPlanInts, plan_ints);
    MoveArgs a = {};
    a.src = a.dst = pool_ptrs(p);
    a.src_tokens = a.dst_tokens = (uint32_t)p->tokens;
    a.heads = (uint32_t)p->heads;
    a.d = row_bytes(p);
    a.renumber = renumber;
    a.plan = plan;
    a.seq_at = (uint32_t)n_tiles;
    a.tables_at = (uint32_t)n_tiles + 5u * (uint32_t)n_seq;
    a.kept = kept;
    a.kept_stride = (uint32_t)kept_stride;
    a.head_split = head_split(a.heads, (uint64_t)n_tiles * p->layers);
    NQ_CHECK_ARG((uint64_t)n_tiles * a.head_split <= max_blocks(256), "nq_pool_compact: grid too large");
    NQ_CHECK_HIP(launch_plan<true>(a, plan_on_host, (uint32_t)plan_ints, (uint32_t)n_tiles, (uint32_t)p->layers, (hipStream_t)stream));
    return NQ_OK;
}

extern "C" int nq_pool_write(const nq_pool* p, int32_t layer, const nq_pool* tokens, const int32_t* slots,
                             int32_t slots_on_host, int32_t n, void* stream) {
    using namespace nq;
    if (int st = check_pool(p, "nq_pool_write")) return st;
    NQ_CHECK_ARG(!four_bit(p), "nq_pool_write: a pool of 4 bits a coordinate is written by nq_fourbit_append");
    NQ_CHECK_ARG(n >= 0 && layer >= 0 && layer < p->layers, "nq_pool_write: n %d, layer %d of %d", n, layer, p->layers);
    if (n == 0) return NQ_OK;
    if (int st = check_pool(tokens, "nq_pool_write")) return st;
    NQ_CHECK_ARG(!four_bit(tokens) && tokens->layers == 1 && tokens->pages == 1 && tokens->tokens == n && tokens->heads == p->heads &&
                     tokens->head_dim == p->head_dim,
                 "nq_pool_write: the tokens must be one page of n tokens of the pool's heads and head_dim");
    NQ_CHECK_ARG(slots != nullptr, "nq_pool_write: slots are required");
    NQ_CHECK_ARG(!slots_on_host || n <= kPlanInts, "nq_pool_write: a host array has at most %d slots, got %d", kPlanInts, n);
    MoveArgs a = {};
    a.src = pool_ptrs(tokens);
    a.dst = pool_ptrs(p);
    const size_t rows = (size_t)layer * p->pages * p->heads * p->tokens;
    for (int role = 0; role < 2; ++role) {
        a.dst.codes[role] += rows * p->head_dim;
        a.dst.scales[role] += rows * 2;
    }
    a.src_tokens = (uint32_t)n;
    a.dst_tokens = (uint32_t)p->tokens;
    a.heads = (uint32_t)p->heads;
    a.d = (uint32_t)p->head_dim;
    a.n = (uint32_t)n;
    a.plan = slots;
    a.slot_end = (uint32_t)p->pages * (uint32_t)p->tokens;
    const uint32_t tiles = ((uint32_t)n + kMoveTokens - 1) / kMoveTokens;
    a.head_split = head_split(a.heads, tiles);
    NQ_CHECK_ARG((uint64_t)tiles * a.head_split <= max_blocks(256), "nq_pool_write: grid too large");
    NQ_CHECK_HIP(launch_plan<false>(a, slots_on_host, (uint32_t)n, tiles, 1u, (hipStream_t)stream));
    return NQ_OK;
}
