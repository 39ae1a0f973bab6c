// Causal attention over packed prompts (grouped heads, optional sliding window) on gfx950:
// query i of a sequence sees its keys j with i - window < j <= i.
//
// A workgroup of 4 waves owns 128 consecutive queries of one sequence and head, 32 a wave,
// and streams the 64-key stages that they see through two LDS buffers each for keys and
// values (direct-to-LDS loads, under way while the other buffer is computed on).  128 queries
// and 64 keys are what two workgroups on a CU leave of registers and LDS at head_dim 128.
//
// What bounds it: at 16384 tokens of 32 / 8 heads x 128, fp16, 2.15 to 2.26 ms by card (975 to 1020
// TFLOP/s; bf16 1090); with half of the LDS reads 6 % less, without exponentials 5 %, so nothing by
// itself.  At head_dim 64 exponentials take half of the products' time (890, bf16 940), at 256 a SIMD
// holds one wave (810; 4096 tokens 720).  A window of 1024 tokens leaves many of a workgroup's stages
// masked: 760 TFLOP/s of what is seen, 530 at 256.  Short prompts are bound by the latency of their
// few stages: 10.6 us for up to 190 tokens.
#include "nq_flash.h"

namespace nq {

using namespace flash;

struct PromptArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    const int32_t* tiles;  // [n_tiles * 4]: first row of the sequence, its length, the tile's first query, 0
    int64_t q_row, k_row, v_row, o_row;      // strides of a token, elements
    int64_t q_head, k_head, v_head, o_head;  // of a head
    uint32_t hq, hkv;
    int32_t window;        // 0: none
    float c;               // scale * log2(e)
    uint32_t n_split;      // workgroups that share a tile's keys
    float* part_o;         // [workgroups, 128, D]: their sums
    float* part_ml;        // [workgroups, 128, 2]: their maxima and sums of weights
};

constexpr int kWaitVm0 = 0x0f70;  // vmcnt(0), the other counters left open
constexpr int kPromptRows = 128;
constexpr int kStage = 64;        // keys of a stage: two tiles

// Rows row0 .. row0 + 63 of one head to LDS in Tile's layout (StagePieces), 16 bytes a lane.  A whole stage
// is a uniform address plus a lane's fixed offsets.  In the sequence's last stage rows past its end repeat
// its last one (their weights are zero, and what lies behind the sequence is never read).
template <int D, bool VALUES>
struct StageLoad {
    using T = Tile<D>;
    using P = StagePieces<D, VALUES>;
    int thread;
    uint32_t off[P::PERIOD];
    __device__ __forceinline__ void init(int wave, int lane, int64_t stride) {
        thread = 64 * wave + lane;
#pragma unroll
        for (int i = 0; i < P::PERIOD; ++i) off[i] = P::offset(thread, i, stride);
    }
    __device__ __forceinline__ void operator()(const uint16_t* base, int64_t stride, int row0, int n, char* buf, int wave) const {
        if (row0 + kStage <= n) {
            const char* const from = reinterpret_cast<const char*>(base + (int64_t)row0 * stride);
#pragma unroll
            for (int i = 0; i < T::UPR / 4; ++i)
                __builtin_amdgcn_global_load_lds((global_void*)(from + (int64_t)(P::STEP * i) * 2 * stride + off[i % P::PERIOD]),
                                                 (lds_void*)(buf + 1024 * (4 * i + wave)), 16, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < T::UPR / 4; ++i) {
                const uint16_t* const src = base + (int64_t)min(row0 + P::row(thread, i), n - 1) * stride + 8 * P::chunk(thread, i);
                __builtin_amdgcn_global_load_lds((global_void*)src, (lds_void*)(buf + 1024 * (4 * i + wave)), 16, 0, 0);
            }
        }
    }
};

// The output of a wave's queries again, key by key on the vector ALUs, each query over the keys
// it sees only: where an infinity or a NaN is among the sums of values.
// The maxima and sums of the fast pass hold (hidden logits never enter them).
template <int DT, int D>
__device__ __forceinline__ void sum_again(Rows<DT, D>& rows, const uint16_t* kb, int64_t k_row, const uint16_t* vb, int64_t v_row,
                                          float c, int key_first, int key_last, int lo, int hi, int g) {
    using T = Tile<D>;
#pragma unroll
    for (int b = 0; b < T::DB; ++b) rows.o[b] = f32x16{};
#pragma unroll 1
    for (int key = key_first; key <= key_last; ++key) {
        const uint16_t* const kr = kb + key * k_row + 8 * g;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < T::KS; ++i) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(kr + 16 * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s = __builtin_fmaf(unpack<DT>(x[k] & 0xffffu), unpack<DT>(rows.q[i][k] & 0xffffu), s);
                s = __builtin_fmaf(unpack<DT>(x[k] >> 16), unpack<DT>(rows.q[i][k] >> 16), s);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        s = both_sum(s);
        if (key < lo || key > hi) continue;
        const float p = unpack<DT>(pack2<DT>(__builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -rows.m)), 0.0f) & 0xffffu);
        const uint16_t* const vr = vb + key * v_row + 4 * g;
#pragma unroll
        for (int b = 0; b < T::DB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(vr + 32 * b + 8 * i);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    rows.o[b][4 * i + k] = __builtin_fmaf(p, unpack<DT>((k & 1) ? x[k / 2] >> 16 : x[k / 2] & 0xffffu), rows.o[b][4 * i + k]);
                __builtin_amdgcn_sched_barrier(0);
            }
    }
}

// SPLIT: a tile's stages go to n_split workgroups, whose sums prompt_join_kernel joins.
template <int DT, int D, bool SPLIT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void prompt_kernel(PromptArgs a) {
    using T = Tile<D>;
    __shared__ __align__(16) char k0[kStage * T::ROWB];
    __shared__ __align__(16) char k1[kStage * T::ROWB];
    __shared__ __align__(16) char v0[kStage * T::ROWB];
    __shared__ __align__(16) char v1[kStage * T::ROWB];
    const int lane = threadIdx.x & 63, n = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // kv heads fastest: blocks go to the XCDs in turn, so the query heads of a kv head meet in one
    // XCD's L2 when the kv heads are a multiple of 8
    const uint32_t part = blockIdx.x / a.hq, j = blockIdx.x % a.hq, tile = SPLIT ? part / a.n_split : part;
    const uint32_t kh = j % a.hkv, head = kh * (a.hq / a.hkv) + j / a.hkv;
    const int32_t first = a.tiles[4 * tile], len = a.tiles[4 * tile + 1], q0 = a.tiles[4 * tile + 2];
    const int q_last = min(q0 + kPromptRows, len) - 1;
    int key0 = a.window ? max(q0 - a.window + 1, 0) & ~(kStage - 1) : 0;
    int n_stages = (q_last - key0) / kStage + 1;
    if constexpr (SPLIT) {
        const int per = (n_stages + (int)a.n_split - 1) / (int)a.n_split, before = per * (int)(part - tile * a.n_split);
        key0 += kStage * before;
        n_stages = min(per, n_stages - before);
        if (n_stages <= 0) {  // whole block: no keys
            if (threadIdx.x < kPromptRows) *reinterpret_cast<f32x2*>(a.part_ml + 2 * ((size_t)blockIdx.x * kPromptRows + threadIdx.x)) = f32x2{kNoMax, 0.0f};
            return;
        }
    }
    const int my0 = q0 + 32 * wave;               // this wave's first query
    const bool live = my0 < len;
    const int my_q = min(my0 + n, len - 1);
    const int my_last = min(my0 + 31, len - 1);

    const uint16_t* const kb = a.k + first * a.k_row + kh * a.k_head;
    const uint16_t* const vb = a.v + first * a.v_row + kh * a.v_head;
    Rows<DT, D> rows;
    rows.init(lane);
    const uint16_t* const qp = a.q + (first + (int64_t)my_q) * a.q_row + head * a.q_head + 8 * g;
#pragma unroll
    for (int i = 0; i < T::KS; ++i) rows.q[i] = *reinterpret_cast<const u32x4*>(qp + 16 * i);

    StageLoad<D, false> load_k;
    StageLoad<D, true> load_v;
    load_k.init(wave, lane, a.k_row);
    load_v.init(wave, lane, a.v_row);
    load_k(kb, a.k_row, key0, len, k0, wave);
    load_v(vb, a.v_row, key0, len, v0, wave);
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    __syncthreads();
    auto fetch = [&](int it, char* nk, char* nv) {
        if (it + 1 < n_stages) {
            load_k(kb, a.k_row, key0 + kStage * (it + 1), len, nk, wave);
            load_v(vb, a.v_row, key0 + kStage * (it + 1), len, nv, wave);
        }
    };
    auto landed = [&] {  // the next stage is in LDS, and this one may be overwritten
        __builtin_amdgcn_s_waitcnt(kWaitVm0);
        __syncthreads();
    };
    // a stage that hides keys from some queries of the workgroup, or from all of a wave's
    auto masked = [&](int it, const char* ck, const char* cv, char* nk, char* nv) {
        fetch(it, nk, nv);
        const int key = key0 + kStage * it;
        int lo = a.window ? my_q - a.window + 1 - key : 0, hi = live ? my_q + 1 - key : 0;
#pragma unroll 1
        for (int t = 0; t < 2; ++t, lo -= 32, hi -= 32) {
            if (!__any(lo < 32 && hi > 0)) continue;
            rows.masked_tile(ck, cv, t, a.c, lo, hi, g);
        }
        landed();
    };
    // one that every query of the workgroup sees whole
    auto whole = [&](int it, const char* ck, const char* cv, char* nk, char* nv) {
        fetch(it, nk, nv);
        rows.two_tiles(ck, cv, 0, a.c, g);
        landed();
    };
    // Whole stages are [it0, it1): past every query's window start, before the first query.  They run in a
    // loop of their own, two a turn: a branch between the two kinds in every stage made the compiler move all
    // of the output's registers twice a stage (32/8 heads x 16384 x 128 fp16: 2.47 ms with it).
    const int it0 = a.window ? max((q_last - a.window - key0 + kStage) / kStage, 0) : 0;
    const int it1 = min((q0 - key0) / kStage, n_stages);  // (a part of the keys may end before the first query)
    int it = 0;
    while (it < n_stages) {
        if (!(it & 1) && it >= it0 && it + 1 < it1) {
#pragma unroll 1
            do {
                whole(it, k0, v0, k1, v1);
                whole(it + 1, k1, v1, k0, v0);
                it += 2;
            } while (it + 1 < it1);
        } else {
            if (it & 1) masked(it, k1, v1, k0, v0);
            else masked(it, k0, v0, k1, v1);
            ++it;
        }
    }
    // A hidden key's weight is zero, but zero times an infinity or a NaN among its values is NaN: then a sum is, too.
    // (Looking at the tiles' values in the loop instead: 12.0 us for prompts of up to 190 tokens, so 10.7.)
    float zero = 0.0f;
#pragma unroll
    for (int b = 0; b < T::DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(rows.o[b][i], 0.0f, zero);
    if (__any(!(zero == 0.0f))) sum_again<DT, D>(rows, kb, a.k_row, vb, a.v_row, a.c, key0, SPLIT ? min(my_last, key0 + kStage * n_stages - 1) : my_last, a.window ? my_q - a.window + 1 : 0, my_q, g);
    if (!live || my0 + n >= len) return;
    if constexpr (SPLIT) {
        const size_t at = (size_t)blockIdx.x * kPromptRows + 32 * wave + n;
        const float l = both_sum(rows.l);
        if (g == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * at) = f32x2{rows.m, l};
        float* const to = a.part_o + at * D + 4 * g;
#pragma unroll
        for (int b = 0; b < T::DB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(to + 32 * b + 8 * i) = f32x4{rows.o[b][4 * i], rows.o[b][4 * i + 1], rows.o[b][4 * i + 2], rows.o[b][4 * i + 3]};
        return;
    }
    const float r = 1.0f / both_sum(rows.l);
    uint16_t* const op = a.out + (first + (int64_t)my_q) * a.o_row + head * a.o_head + 4 * g;
#pragma unroll
    for (int b = 0; b < T::DB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x2 w = {pack2<DT>(rows.o[b][4 * i] * r, rows.o[b][4 * i + 1] * r),
                             pack2<DT>(rows.o[b][4 * i + 2] * r, rows.o[b][4 * i + 3] * r)};
            *reinterpret_cast<u32x2*>(op + 32 * b + 8 * i) = w;
        }
}

// The parts of a tile and head joined, in their order: 1024 / D rows a workgroup, four coordinates a lane.
template <int DT, int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a) {
    constexpr int LANES = D / 4, ROWS = 256 / LANES, BLOCKS = kPromptRows / ROWS;
    const uint32_t wg = blockIdx.x / BLOCKS, tile = wg / a.hq, j = wg % a.hq;
    const uint32_t head = j % a.hkv * (a.hq / a.hkv) + j / a.hkv;
    const int32_t first = a.tiles[4 * tile], len = a.tiles[4 * tile + 1], q0 = a.tiles[4 * tile + 2];
    const int r = (int)(blockIdx.x % BLOCKS) * ROWS + (int)threadIdx.x / LANES, at = threadIdx.x % LANES;
    if (q0 + r >= len) return;
    const size_t row0 = ((size_t)tile * a.n_split * a.hq + j) * kPromptRows + r, step = (size_t)a.hq * kPromptRows;
    float m = kNoMax, l = 0.0f;
#pragma unroll 4
    for (uint32_t s = 0; s < a.n_split; ++s) m = __builtin_fmaxf(m, a.part_ml[2 * (row0 + s * step)]);
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t s = 0; s < a.n_split; ++s) {
        const size_t row = row0 + s * step;
        const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * row);
        const f32x4 o = *reinterpret_cast<const f32x4*>(a.part_o + row * D + 4 * at);
        const float f = __builtin_amdgcn_exp2f(ml.x - m);
        l = __builtin_fmaf(ml.y, f, l);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = ml.y == 0.0f ? y[k] : __builtin_fmaf(o[k], f, y[k]);  // no keys: no sums are written
    }
    const float d = 1.0f / l;
    *reinterpret_cast<u32x2*>(a.out + (first + (int64_t)(q0 + r)) * a.o_row + head * a.o_head + 4 * at) =
        u32x2{pack2<DT>(y[0] * d, y[1] * d), pack2<DT>(y[2] * d, y[3] * d)};
}

template <int DT, int D>
static hipError_t launch_prompt(const PromptArgs& a, uint32_t blocks, hipStream_t s) {
    if (a.n_split <= 1) {
        hipLaunchKernelGGL((prompt_kernel<DT, D, false>), dim3(blocks), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((prompt_kernel<DT, D, true>), dim3(blocks * a.n_split), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((prompt_join_kernel<DT, D>), dim3(blocks * (kPromptRows * D / 1024)), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int DT>
static hipError_t prompt_dims(int32_t d, const PromptArgs& a, uint32_t blocks, hipStream_t s) {
    switch (d) {
        case 64: return launch_prompt<DT, 64>(a, blocks, s);
        case 128: return launch_prompt<DT, 128>(a, blocks, s);
        default: return launch_prompt<DT, 256>(a, blocks, s);
    }
}

}  // namespace nq

extern "C" int32_t nq_prompt_tile_rows(void) { return nq::kPromptRows; }

extern "C" int64_t nq_prompt_workspace(int32_t n_tiles, int32_t q_heads, int32_t head_dim, int32_t n_split) {
    if (n_tiles <= 0 || q_heads <= 0 || head_dim <= 0 || n_split <= 1) return 0;
    return (int64_t)n_tiles * q_heads * n_split * nq::kPromptRows * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int nq_prompt_attention(const nq_prompt_desc* d, void* stream) {
    using namespace nq;
    NQ_CHECK_ARG(d != nullptr, "nq_prompt_attention: desc is NULL");
    NQ_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256,
                 "nq_prompt_attention: head_dim %d unsupported (64, 128, 256)", d->head_dim);
    NQ_CHECK_ARG(d->dtype == NQ_F16 || d->dtype == NQ_BF16, "nq_prompt_attention: dtype must be fp16 or bf16");
    NQ_CHECK_ARG(d->q_heads > 0 && d->kv_heads > 0 && d->q_heads % d->kv_heads == 0,
                 "nq_prompt_attention: q_heads %d must be a positive multiple of kv_heads %d", d->q_heads, d->kv_heads);
    NQ_CHECK_ARG(d->n_tiles >= 0 && d->sliding_window >= 0, "nq_prompt_attention: n_tiles %d, sliding_window %d",
                 d->n_tiles, d->sliding_window);
    NQ_CHECK_ARG(d->scale > 0.0f && d->scale < 1e30f, "nq_prompt_attention: scale must be positive");
    if (d->n_tiles == 0) return NQ_OK;
    NQ_CHECK_ARG(d->q && d->k && d->v && d->out && d->tiles, "nq_prompt_attention: q, k, v, out and tiles are required");
    NQ_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v) & 15u) == 0 && ((uintptr_t)d->out & 7u) == 0,
                 "nq_prompt_attention: q, k and v must be 16-byte aligned, out 8-byte");
    NQ_CHECK_ARG(((d->q_stride[0] | d->q_stride[1] | d->k_stride[0] | d->k_stride[1] | d->v_stride[0] | d->v_stride[1]) & 7) == 0 &&
                     ((d->out_stride[0] | d->out_stride[1]) & 3) == 0,
                 "nq_prompt_attention: strides must keep rows 16-byte aligned (out: 8-byte)");
    NQ_CHECK_ARG(d->k_stride[0] >= 0 && d->k_stride[0] < (1 << 24) && d->v_stride[0] >= 0 && d->v_stride[0] < (1 << 24),
                 "nq_prompt_attention: rows of k and v must be less than 2^24 elements apart");
    NQ_CHECK_ARG(d->n_split >= 1 && d->n_split <= 64, "nq_prompt_attention: n_split %d (1 .. 64)", d->n_split);
    // the tiles' parts, and where there are several the workgroups that join them
    const uint64_t blocks64 = (uint64_t)d->n_tiles * d->q_heads;
    NQ_CHECK_ARG(blocks64 <= max_blocks(256) && blocks64 * d->n_split <= max_blocks(256) &&
                     (d->n_split == 1 || blocks64 * (kPromptRows * d->head_dim / 1024) <= max_blocks(256)),
                 "nq_prompt_attention: grid too large");
    const int64_t need = nq_prompt_workspace(d->n_tiles, d->q_heads, d->head_dim, d->n_split);
    NQ_CHECK_ARG(need == 0 || (d->workspace != nullptr && d->workspace_bytes >= need && ((uintptr_t)d->workspace & 15u) == 0),
                 "nq_prompt_attention: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
    PromptArgs a = {};
    a.q = static_cast<const uint16_t*>(d->q);
    a.k = static_cast<const uint16_t*>(d->k);
    a.v = static_cast<const uint16_t*>(d->v);
    a.out = static_cast<uint16_t*>(d->out);
    a.tiles = d->tiles;
    a.q_row = d->q_stride[0];
    a.q_head = d->q_stride[1];
    a.k_row = d->k_stride[0];
    a.k_head = d->k_stride[1];
    a.v_row = d->v_stride[0];
    a.v_head = d->v_stride[1];
    a.o_row = d->out_stride[0];
    a.o_head = d->out_stride[1];
    a.hq = (uint32_t)d->q_heads;
    a.hkv = (uint32_t)d->kv_heads;
    a.window = d->sliding_window;
    a.c = d->scale * 1.44269504088896340736f;
    const uint32_t blocks = (uint32_t)blocks64;
    a.n_split = (uint32_t)d->n_split;
    a.part_o = static_cast<float*>(d->workspace);
    a.part_ml = a.part_o + (size_t)blocks * a.n_split * kPromptRows * d->head_dim;
    hipStream_t s = (hipStream_t)stream;
    NQ_CHECK_HIP(d->dtype == NQ_F16 ? prompt_dims<NQ_F16>(d->head_dim, a, blocks, s)
                                    : prompt_dims<NQ_BF16>(d->head_dim, a, blocks, s));
    return NQ_OK;
}
