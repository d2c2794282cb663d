// pkv_prompt_mma.cuh -- causal attention of packed prompts on the tcgen05
// tensor cores.  Included by pkv_prompt.cu only.
#pragma once

#include "pkv_tcgen05.cuh"

namespace pkv {

struct PromptParams {
    const uint8_t* q;  // [Tq][Hq][128], token / head strides in bytes
    const uint8_t* k;  // [Tk][Hkv][128]
    const uint8_t* v;
    const int32_t* cu_q;  // [B + 1]
    const int32_t* cu_k;  // [B + 1]
    void* out;            // [Tq][Hq][128] contiguous
    float* lse;           // [Tq][Hq] or null
    unsigned* error;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head;
    int B, Tq, Tk, Hq, Hkv, G;
    float scale_log2;
};

constexpr int kPmTile = 128;                     // query rows of a tile, keys of a block
constexpr int kPmTileBytes = kPmTile * kRowBytes;  // 32 KB: two 64-element halves of 16 KB
constexpr int kPmHalfBytes = kPmTileBytes / 2;
constexpr int kPmStages = 4;                     // K/V tiles in flight
// 8 softmax warps (tile, 32 rows each), then one warp each for the products,
// the copies and the schedule (and the V tiles that hold keys which not every row
// sees), and one that looks the ranges over.
constexpr int kPmSoftmaxWarps = 8;
constexpr int kPmMmaWarp = 8, kPmLoadWarp = 9, kPmPlanWarp = 10, kPmCheckWarp = 11;
constexpr int kPmThreads = 384;
constexpr int kPmParts = 4;  // parts of a block's weights, 32 keys each, handed over one by one
constexpr int kPmStageOut = 32 * 128;  // a softmax warp's 32 rows x 64 output dims
constexpr size_t kPmSmemBytes = 1024 + (size_t)(2 + kPmStages) * kPmTileBytes +
                                kPmSoftmaxWarps * kPmStageOut + 640;
// TMEM columns: scores of tile t at 128 t (its weights, 16 bit, in the first
// 64 of them), output of tile t at 256 + 128 t.
constexpr uint32_t kPmTmemColumns = 512;  // all there are
// The running maximum that weights refer to is raised, and the output
// rescaled, only when a row's maximum has grown by more than this many powers
// of two; the division by the sum at the end takes the factor out again.  fp16
// weights stay below 2^14 (the type reaches 2^16); the largest is 1 at least, and
// those below 2^-14 are rounded to 2^-25 of it.  bf16 has fp32's range: the
// reference lies kPmLift above the running maximum, so that weights stay below 1 and
// no sum of weights times V overflows that would not with weights of at most 1; a
// weight's relative rounding is the same at any size.
// With 2^8 every fourth block of a 16384-token prompt had a row that moved, at
// about 1400 cycles each.
template <typename T>
constexpr float kPmLazy = std::is_same<T, __half>::value ? 14.0f : 32.0f;
template <typename T>
constexpr float kPmLift = std::is_same<T, __half>::value ? 0.0f : 32.0f;
// 2^kPmLift: takes a sum of weights to the running maximum, exactly, so that its
// logarithm is the small one.
template <typename T>
__device__ __forceinline__ float pm_unlift() {
    return std::is_same<T, __half>::value ? 1.0f : 0x1p32f;
}

// One item of work: two query tiles that read the same keys.
struct alignas(16) PmWork {
    int q0, k0, lq, lk;     // the sequence's first query row and key, and lengths
    int row0;               // first query row of the item in its sequence; -1: no more items
    int head0, kvh, n_tiles;
    int first, n_blocks;    // this CTA's key blocks
    int tail;               // keys of the last of them
    int clear;              // blocks before this one hold only keys that every row sees
    // keys that row i of the sequence sees
    __device__ __forceinline__ int visible(int i) const {
        return max(0, min(lk, i + 1 + lk - lq));
    }
};
// The present item and those to come: with two, an item's schedule waited for the
// end of the output of the last but one.
constexpr int kPmWorks = 4;

struct PmShared {
    uint4 launch;  // answer of the launch control
    PmWork work[kPmWorks];
    uint64_t work_full[kPmWorks], work_empty[kPmWorks], launch_bar, issued;
    uint64_t q_full, q_empty, kv_full[kPmStages], kv_empty[kPmStages];
    uint64_t s_full[2], p_full[2][kPmParts], o_full[2], o_empty[2], drained;
    uint64_t look[2], clean[2];  // of the two V stages
    int dropped[kPmWorks];       // the item's V had values that were taken out
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(PmShared) <= 640, "prompt CTA's shared state");

__device__ __forceinline__ int pm_rows_per_item(int G) { return G == 1 ? 2 * kPmTile : kPmTile; }

// What follows for every role from the sequence, the rows and the head or pair of
// heads.  kSplit: the CTAs of a cluster share the item, its key blocks in equal
// parts.
template <bool kSplit>
__device__ __forceinline__ void pm_item(const PromptParams& p, PmWork& w, int group) {
    w.head0 = p.G == 1 ? group : 2 * group;
    w.kvh = w.head0 / p.G;
    w.n_tiles = (p.G == 1 && w.row0 + kPmTile >= w.lq) ? 1 : 2;
    const int n_keys = w.visible(min(w.row0 + pm_rows_per_item(p.G), w.lq) - 1);
    w.first = 0;
    w.n_blocks = (n_keys + kPmTile - 1) / kPmTile;
    w.tail = n_keys - (w.n_blocks - 1) * kPmTile;
    if (kSplit) {
        const int all = w.n_blocks, rank = (int)cluster_rank(), n = (int)cluster_size();
        w.first = all * rank / n;
        w.n_blocks = all * (rank + 1) / n - w.first;
        if (w.first + w.n_blocks < all) w.tail = kPmTile;
    }
    w.clear = max(0, w.visible(w.row0) / kPmTile - w.first);
}

// Whole warp: the query tile number `rank`, counted from the end over all
// sequences' tiles of `rows` rows, so that the longest rows of a sequence start
// first.  Returns 1 with the work filled in, 0 if there are fewer tiles, -1
// for a tile of a sequence whose ranges are bad.  `seen` sequences hold the
// first `before` tiles: a CTA's items come in ascending order, so the search goes
// on where the last one ended.
__device__ __forceinline__ int pm_find(const PromptParams& p, int rank, int rows, PmWork& w,
                                       int& seen, int& before) {
    const int lane = threadIdx.x & 31;
    if (rank < before) seen = before = 0;
    for (; seen < p.B; seen += 32) {
        const int base = seen;
        const int b = p.B - 1 - base - lane;
        int q0 = 0, q1 = 0, n = 0;
        if (b >= 0) {
            q0 = __ldg(p.cu_q + b);
            q1 = __ldg(p.cu_q + b + 1);
            const long long len = (long long)q1 - q0;
            n = len > 0 ? (int)min((len + rows - 1) / rows, (long long)p.Tq) : 0;
        }
        int x = n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off) x += y;
        }
        const int first = before + x - n;
        const unsigned hit = __ballot_sync(0xffffffffu, rank >= first && rank < first + n);
        if (hit != 0u) {
            const int src = __ffs(hit) - 1;
            const int bb = __shfl_sync(0xffffffffu, b, src);
            w.q0 = __shfl_sync(0xffffffffu, q0, src);
            q1 = __shfl_sync(0xffffffffu, q1, src);
            w.row0 = __shfl_sync(0xffffffffu, n - 1 - (rank - first), src) * rows;
            w.k0 = __ldg(p.cu_k + bb);
            const int k1 = __ldg(p.cu_k + bb + 1);
            w.lq = q1 - w.q0;
            w.lk = k1 - w.k0;
            return (w.q0 < 0 || q1 > p.Tq || w.k0 < 0 || k1 < w.k0 || k1 > p.Tk) ? -1 : 1;
        }
        before = __shfl_sync(0xffffffffu, before + x, 31);
    }
    return 0;
}

// One wait of a converged warp: false after the time limit or once another
// thread of the CTA has given up.
__device__ __forceinline__ bool pm_wait_warp(const PromptParams& p, PmShared* sh, uint64_t* bar,
                                             uint32_t parity) {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) {
        ok = mbar_wait_bounded(bar, parity, &sh->abort);
        if (!ok && atomicExch(&sh->abort, 1) == 0) raise_error(p.error, kErrTimeout);
    }
    return __all_sync(0xffffffffu, ok);
}

// One thread's wait.
__device__ __forceinline__ bool pm_wait(const PromptParams& p, PmShared* sh, uint64_t* bar,
                                        uint32_t parity) {
    if (mbar_wait_bounded(bar, parity, &sh->abort)) return true;
    if (atomicExch(&sh->abort, 1) == 0) raise_error(p.error, kErrTimeout);
    return false;
}

// Waits for item number n: false if there are no more (or on abort).
__device__ __forceinline__ bool pm_wait_work(const PromptParams& p, PmShared* sh, uint32_t n) {
    return pm_wait_warp(p, sh, &sh->work_full[n % kPmWorks], (n / kPmWorks) & 1u) &&
           *(const volatile int*)&sh->work[n % kPmWorks].row0 >= 0;
}

// The warp needs item number n's place no longer.
__device__ __forceinline__ void pm_release_work(PmShared* sh, uint32_t n) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh->work_empty[n % kPmWorks]);
}

// Both, with the item copied.
__device__ __forceinline__ bool pm_next(const PromptParams& p, PmShared* sh, uint32_t n,
                                        PmWork& it) {
    if (!pm_wait_work(p, sh, n)) return false;
    it = sh->work[n % kPmWorks];
    pm_release_work(sh, n);
    return true;
}

// A key's V that holds an infinity or NaN reaches a row that does not see the key
// all the same, through a product with a weight of 0.  So such values are taken out
// of the tiles whose keys not every row sees (`clear` and later), and come back
// here, to the rows that do see them: output rows [row, row_end) of the sequence,
// already written, get the sum of the values taken out among their keys from
// `key` on.  Whole warp, lane l dims 4l .. 4l + 3.
template <typename T>
__device__ __forceinline__ void pm_restore(const PromptParams& p, const PmWork& it, int head,
                                           int key, int row, int row_end) {
    const int lane = threadIdx.x & 31;
    const uint8_t* v = p.v + it.k0 * p.v_tok + it.kvh * p.v_head;
    auto load = [&](int j) {
        return __ldg(reinterpret_cast<const uint2*>(v + (size_t)j * p.v_tok) + lane);
    };
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](uint2 u) {
        const unsigned b[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((b[i] & 0x7fffu) >= kInf16<T>) sum[i] += from_bits16<T>(b[i]);
    };
    for (; row < row_end; ++row) {
        const int n = it.visible(row);
        for (; key + 8 <= n; key += 8) {
            uint2 u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = load(key + i);
#pragma unroll
            for (int i = 0; i < 8; ++i) add(u[i]);
        }
        for (; key < n; ++key) add(load(key));
        // (an infinity or NaN is no zero)
        if (sum[0] != 0.f || sum[1] != 0.f || sum[2] != 0.f || sum[3] != 0.f) {
            uint2* at = reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) +
                                                 ((size_t)(it.q0 + row) * p.Hq + head) * kHeadDim) +
                        lane;
            const uint2 o = *at;
            const float2 a = to_float2<T>(o.x), b = to_float2<T>(o.y);
            *at = make_uint2(ElemOps<T>::pack(a.x + sum[0], a.y + sum[1]),
                             ElemOps<T>::pack(b.x + sum[2], b.y + sum[3]));
        }
    }
}

// The same for the rows of a softmax warp.
template <typename T>
__device__ __forceinline__ void pm_restore_rows(const PromptParams& p, const PmWork* work) {
    const PmWork it = *work;
    const int warp = threadIdx.x >> 5, t = warp >> 2;
    const int row = it.row0 + (p.G == 1 ? t * kPmTile : 0) + (warp & 3) * 32;
    pm_restore<T>(p, it, p.G == 1 ? it.head0 : it.head0 + t, it.clear * kPmTile, row,
                  min(row + 32, it.lq));
}

// Takes infinities and NaN out of the first `keys` rows of a V tile, and zeroes the
// rows behind them; true if there was any to take out.  Whole warp.
template <typename T>
__device__ __forceinline__ bool pm_clean(uint8_t* tile, int keys) {
    const int lane = threadIdx.x & 31;
    // a lane's pieces of 16 bytes: of every fourth row, in both halves
    constexpr int kPieces = kPmTile / 4;
    uint4* const mine = reinterpret_cast<uint4*>(tile) + lane;
    if (keys < kPmTile) {
        for (int i = max(0, (keys - (lane >> 3) + 3) >> 2); i < kPieces; ++i)
            mine[32 * i] = mine[32 * (kPieces + i)] = make_uint4(0u, 0u, 0u, 0u);
    }
    // x * 0 is NaN for those and 0 for all others
    typename ElemOps<T>::Pair none[4] = {};
#pragma unroll 1
    for (int i = 0; i < 2 * kPieces; i += 8) {
        uint4 u[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) u[x] = mine[32 * (i + x)];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            none[0] = ElemOps<T>::zero_times(u[x].x, none[0]);
            none[1] = ElemOps<T>::zero_times(u[x].y, none[1]);
            none[2] = ElemOps<T>::zero_times(u[x].z, none[2]);
            none[3] = ElemOps<T>::zero_times(u[x].w, none[3]);
        }
    }
    const auto sum = __hadd2(__hadd2(none[0], none[1]), __hadd2(none[2], none[3]));
    const bool found = __hisnan(sum.x) || __hisnan(sum.y);
    if (!__any_sync(0xffffffffu, found)) return false;
    if (found) {
        auto finite = [](unsigned w) {
            return ((w & 0x7fffu) >= kInf16<T> ? 0u : w & 0xffffu) |
                   ((w >> 16 & 0x7fffu) >= kInf16<T> ? 0u : w & 0xffff0000u);
        };
        for (int i = 0; i < 2 * kPieces; ++i) {
            const uint4 u = mine[32 * i];
            mine[32 * i] = make_uint4(finite(u.x), finite(u.y), finite(u.z), finite(u.w));
        }
    }
    return true;
}

// The cluster's parts of an item joined: softmax warp w of CTA `rank` takes every
// n-th of its rows, lane l dims 4l .. 4l + 3, and reads the n CTAs' states through
// their shared memory.
template <typename T>
__device__ __forceinline__ void pm_join(const PromptParams& p, PmShared* sh, uint8_t* s_kv,
                                        float2* s_state) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (*(const volatile int*)&sh->work[0].row0 < 0 || *(const volatile int*)&sh->abort != 0) return;
    const PmWork it = sh->work[0];
    const int n = (int)cluster_size();
    bool dropped = false;
    for (int c = 0; c < n; ++c)
        dropped = dropped || ld_cluster_u32(cluster_addr(smem_u32(&sh->dropped[0]), c)) != 0u;
    const uint32_t o_u32 = smem_u32(s_kv), st_u32 = smem_u32(s_state);
    for (int i = warp + kPmSoftmaxWarps * (int)cluster_rank(); i < it.n_tiles * kPmTile;
         i += kPmSoftmaxWarps * n) {
        const int t = i / kPmTile;
        const int row = it.row0 + (p.G == 1 ? i : i - t * kPmTile);  // of the sequence
        if (row >= it.lq) continue;
        const int head = p.G == 1 ? it.head0 : it.head0 + t;
        float2 st[8];
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            st[c] = c < n ? ld_cluster_f2(cluster_addr(st_u32 + i * 8, c))
                          : make_float2(-INFINITY, 0.f);
            top = fmaxf(top, st[c].x);
        }
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
        const uint32_t piece = o_u32 + i * (kHeadDim * 4) + ((lane ^ (i & 31)) << 4);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            // (a part that saw no key holds nothing; one whose scores are all NaN has
            // no maximum either, and its sum is NaN)
            if (c >= n || (st[c].x == -INFINITY && st[c].y == 0.f)) continue;
            const float f = fast_exp2((st[c].x - top) * p.scale_log2);
            const float4 x = ld_cluster_f4(cluster_addr(piece, c));
            l = fmaf(f, st[c].y, l);
            o.x = fmaf(f, x.x, o.x);
            o.y = fmaf(f, x.y, o.y);
            o.z = fmaf(f, x.z, o.z);
            o.w = fmaf(f, x.w, o.w);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const size_t at = (size_t)(it.q0 + row) * p.Hq + head;
        T* out = reinterpret_cast<T*>(p.out) + at * kHeadDim;
        reinterpret_cast<uint2*>(out)[lane] =
            make_uint2(ElemOps<T>::pack(o.x * inv, o.y * inv), ElemOps<T>::pack(o.z * inv, o.w * inv));
        if (lane == 0 && p.lse != nullptr)
            p.lse[at] =
                l == 0.f ? -INFINITY : top * p.scale_log2 * kLn2 + logf(l * pm_unlift<T>());
        if (dropped) {
            __syncwarp();
            pm_restore<T>(p, sh->work[0], head, it.visible(it.row0) / kPmTile * kPmTile, row,
                          row + 1);
        }
    }
}

// An item is two query tiles of 128 rows that read the same keys: two heads of
// one KV group at the same positions, or (G = 1) two successive tiles of one
// head.  K and V pass through shared memory in blocks of 128 keys (TMA, ring
// of kPmStages tiles).  For each block, tile t's scores S = Q K^T and output
// O += P V are tcgen05 products issued by one warp, with S, P and O in TMEM; 4
// softmax warps per tile turn S into P in place, running maximum and sum in 32
// bits, one row per thread.  The issue order
//   S0 S1 | O0 S0' O1 S1' | O0' ...
// keeps the tensor cores on one tile while the other's softmax runs, and the
// weights of a block are handed over 32 keys at a time, so that its output
// product starts before its last exponentials.
//
// The grid has one CTA per item; a resident CTA goes on with items whose CTA
// has not started yet (launch control), so the next item's schedule, Q and
// first keys arrive while the present one is computed, and its first scores
// while the present one's output is written.
//
// kSplit: few rows and many keys.  A cluster of 2 to 8 CTAs takes an item, each a
// part of its key blocks, and joins the parts through distributed shared memory,
// without a workspace.
//
// Bound: the card's power cap, and a tile's chain scores -> softmax -> output.  One
// prompt of 16384 tokens (32 heads, bf16) takes 2.05 ms, 1.07 PFLOP/s, 3750 cycles
// per pair of tiles and block at 1.67 GHz under the cap; the products alone take
// 2580, the exponentials 2050, and the tensor cores' nominal rate would be 2048.
// An item's end costs 5500 cycles more: 9 prompts of 70 to 1487 tokens take 92 us.
template <typename T, bool kSplit>
__global__ void __launch_bounds__(kPmThreads, 1)
    pkv_prompt_mma_kernel(const __grid_constant__ PromptParams p,
                          const __grid_constant__ CUtensorMap map_q,
                          const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v) {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* s_q = smem;                      // 2 tiles
    uint8_t* s_kv = smem + 2 * kPmTileBytes;  // kPmStages tiles
    uint8_t* s_out = s_kv + kPmStages * kPmTileBytes;
    PmShared* sh = reinterpret_cast<PmShared*>(s_out + kPmSoftmaxWarps * kPmStageOut);
    float2* s_state = reinterpret_cast<float2*>(s_out);  // [2][128] m and l (kSplit)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPmWorks; ++i) {
            mbar_init(&sh->work_full[i], 1);
            mbar_init(&sh->work_empty[i], kPmSoftmaxWarps + 2);  // one arrival per reading warp
            sh->dropped[i] = 0;
        }
        mbar_init(&sh->launch_bar, 1);
        mbar_init(&sh->issued, 1);
        mbar_init(&sh->q_full, 1);
        mbar_init(&sh->q_empty, 1);
        for (int i = 0; i < kPmStages; ++i) {
            mbar_init(&sh->kv_full[i], 1);
            mbar_init(&sh->kv_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sh->s_full[t], 1);
            for (int i = 0; i < kPmParts; ++i) mbar_init(&sh->p_full[t][i], 4);  // the warps
            mbar_init(&sh->o_full[t], 1);
            mbar_init(&sh->o_empty[t], 4);
            mbar_init(&sh->look[t], 1);
            mbar_init(&sh->clean[t], 1);
        }
        mbar_init(&sh->drained, 1);
        sh->abort = 0;
        fence_mbar_init();
    }
    if (warp == kPmMmaWarp) tmem_alloc(&sh->tmem, kPmTmemColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all of TMEM: it starts at lane 0, column 0, and addresses are constants

    if (warp == kPmPlanWarp) {
        // ------------------------------------------------------------ schedule
        const int groups = p.G == 1 ? p.Hq : p.Hq / 2;  // fastest: they share keys in L2
        int item = kSplit ? blockIdx.x / cluster_size() : blockIdx.x;
        int seen = 0, before = 0;
        uint32_t n = 0;   // items published
        uint32_t gb = 0;  // blocks of the items before
        uint32_t looks[2] = {0u, 0u};  // V tiles looked over, per stage
        bool ok = true, asked = false;
        // V rows behind the last key belong to other sequences or to nobody and
        // may hold anything, and so may the values of keys that a row does not
        // see; their weights are 0, but 0 * NaN is not.  While the block's scores
        // and weights are computed, this warp zeroes the rows behind the last
        // key of block j's V tile and takes infinities and NaN out (pm_restore).
        // 9 ragged prompts take 92 us with it and 89 with the rows behind the last
        // key alone, 16384 tokens the same.
        auto wait_copy = [&](int j) -> bool {  // started: the barrier is in its phase
            const int x = (int)((gb + j) & 1u);  // V stage 1 or 3
            return pm_wait_warp(p, sh, &sh->look[x], looks[x]++ & 1u);
        };
        auto clean = [&](const PmWork& w, int j) -> bool {
            const int x = (int)((gb + j) & 1u);
            if (!pm_wait_warp(p, sh, &sh->kv_full[2 * x + 1], ((gb + j) >> 1) & 1u)) return false;
            if (pm_clean<T>(s_kv + (2 * x + 1) * kPmTileBytes,
                            j + 1 == w.n_blocks ? w.tail : kPmTile) &&
                lane == 0)
                sh->dropped[(n - 1) % kPmWorks] = 1;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->clean[x]);
            return true;
        };
        // The next item is asked for once the copies of this one's last blocks are
        // under way: early enough that it is there when this one ends, late enough
        // to be the fair one to take.
        auto ask = [&]() {
            if (lane == 0) {
                mbar_arrive_expect_tx(&sh->launch_bar, 16);
                launch_cancel_async(&sh->launch, &sh->launch_bar);
            }
            __syncwarp();
            asked = true;
        };
        for (uint32_t round = 0; ok; ++round) {
            PmWork w;
            const int found = pm_find(p, item / groups, pm_rows_per_item(p.G), w, seen, before);
            asked = false;
            if (found > 0) {  // (a bad sequence is reported by the checking warp)
                pm_item<kSplit>(p, w, item % groups);
                if (n >= (uint32_t)kPmWorks)
                    ok = pm_wait_warp(p, sh, &sh->work_empty[n % kPmWorks],
                                      (n / kPmWorks - 1) & 1u);
                if (!ok) break;
                if (lane == 0) {
                    sh->work[n % kPmWorks] = w;
                    sh->dropped[n % kPmWorks] = 0;
                    mbar_arrive(&sh->work_full[n % kPmWorks]);
                }
                __syncwarp();
                ++n;
                for (int j = w.clear; ok && j < w.n_blocks; ++j) {
                    ok = wait_copy(j);
                    if (!kSplit && ok && j + 1 == w.n_blocks) {
                        ok = pm_wait_warp(p, sh, &sh->issued, (n - 1) & 1u);
                        if (ok) ask();
                    }
                    ok = ok && clean(w, j);
                }
                gb += w.n_blocks;
                if (kSplit) break;  // a cluster has one item
                if (ok && !asked) ok = pm_wait_warp(p, sh, &sh->issued, (n - 1) & 1u);
            }
            if (kSplit) break;
            if (ok && !asked) ask();
            // (the answer lands in this CTA: its wait heeds no abort)
            if (asked &&
                !__all_sync(0xffffffffu, mbar_wait_bounded(&sh->launch_bar, round & 1u, nullptr))) {
                if (lane == 0 && atomicExch(&sh->abort, 1) == 0) raise_error(p.error, kErrTimeout);
                ok = false;
            }
            ok = ok && launch_cancelled(&sh->launch, item);
            fence_proxy_async_smem();  // read before the next answer is written
            __syncwarp();
        }
        if (n >= (uint32_t)kPmWorks)
            pm_wait_warp(p, sh, &sh->work_empty[n % kPmWorks], (n / kPmWorks - 1) & 1u);
        if (lane == 0) {
            sh->work[n % kPmWorks].row0 = -1;
            mbar_arrive(&sh->work_full[n % kPmWorks]);
        }
        __syncwarp();
    } else if (warp == kPmCheckWarp) {
        // ------------------------------------------------------------ ranges
        if (blockIdx.x == 0) {
            bool bad = false;
            for (int b = lane; b < p.B; b += 32) {
                const int q0 = __ldg(p.cu_q + b), q1 = __ldg(p.cu_q + b + 1);
                const int k0 = __ldg(p.cu_k + b), k1 = __ldg(p.cu_k + b + 1);
                bad = bad || q0 < 0 || q1 < q0 || q1 > p.Tq || k0 < 0 || k1 < k0 || k1 > p.Tk;
            }
            if (bad) raise_error(p.error, kErrIndex);
        }
    } else if (warp == kPmLoadWarp) {
        // ------------------------------------------------------------ copies
        if (lane == 0) {
            tma_prefetch_map(&map_q);
            tma_prefetch_map(&map_k);
            tma_prefetch_map(&map_v);
        }
        auto load = [&](uint8_t* dst, const CUtensorMap& map, int head, int token, uint64_t* bar) {
            tma_load_3d(dst, &map, 0, head, token, bar);
            tma_load_3d(dst + kPmHalfBytes, &map, 64, head, token, bar);
        };
        PmWork it;
        uint32_t i = 0;      // K/V tiles issued: K0 V0 K1 V1 ... of each item
        uint32_t loads = 0;  // items with keys
        bool ok = true;
        for (uint32_t n = 0; ok && pm_next(p, sh, n, it); ++n) {
            if (it.n_blocks == 0) {
                if (lane == 0) mbar_arrive(&sh->issued);
                continue;
            }
            if (loads > 0) ok = pm_wait_warp(p, sh, &sh->q_empty, (loads - 1) & 1u);
            if (!ok) break;
            ++loads;
            if (lane == 0) {
                mbar_arrive_expect_tx(&sh->q_full, it.n_tiles * kPmTileBytes);
                for (int t = 0; t < it.n_tiles; ++t)
                    load(s_q + t * kPmTileBytes, map_q, p.G == 1 ? it.head0 : it.head0 + t,
                         it.q0 + it.row0 + (p.G == 1 ? t * kPmTile : 0), &sh->q_full);
                for (int c = 0; ok && c < 2 * it.n_blocks; ++c, ++i) {
                    const int st = i % kPmStages;
                    if (i >= (uint32_t)kPmStages)
                        ok = pm_wait(p, sh, &sh->kv_empty[st], (i / kPmStages - 1) & 1u);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&sh->kv_full[st], kPmTileBytes);
                    if (c & 1)
                        load(s_kv + st * kPmTileBytes, map_v, it.kvh, it.k0 + (it.first + (int)(c >> 1)) * kPmTile,
                             &sh->kv_full[st]);
                    else
                        load(s_kv + st * kPmTileBytes, map_k, it.kvh, it.k0 + (it.first + (int)(c >> 1)) * kPmTile,
                             &sh->kv_full[st]);
                    if ((c & 1) && (c >> 1) >= it.clear) mbar_arrive(&sh->look[st >> 1]);
                }
                mbar_arrive(&sh->issued);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        // copies in flight land before the CTA ends (bounded)
        if (lane == 0) {
            bool landed = loads == 0 || mbar_wait_bounded(&sh->q_full, (loads - 1) & 1u, nullptr);
            for (uint32_t c = i > (uint32_t)kPmStages ? i - kPmStages : 0u; landed && c < i; ++c)
                landed = mbar_wait_bounded(&sh->kv_full[c % kPmStages], (c / kPmStages) & 1u, nullptr);
        }
        __syncwarp();
    } else if (warp == kPmMmaWarp) {
        // ------------------------------------------------------------ products
        // The whole warp walks the loop, so that descriptors and addresses are
        // uniform values; one elected lane issues the products and commits.
        constexpr uint32_t kDescQk = mma_desc_f16(kPmTile, kPmTile, kBf16, false);
        constexpr uint32_t kDescPv = mma_desc_f16(kPmTile, kHeadDim, kBf16, true);
        const uint32_t q_desc = smem_desc_sw128(smem_u32(s_q), 16);
        const uint32_t k_desc = smem_desc_sw128(smem_u32(s_kv), 16);
        const uint32_t v_desc = smem_desc_sw128(smem_u32(s_kv), kPmHalfBytes);
        constexpr uint32_t kTileStep = kPmTileBytes >> 4;  // in descriptor units
        // S of tile t from the K tile in stage st
        auto scores = [&](int t, int st) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint32_t off = ((ks >> 2) * kPmHalfBytes + (ks & 3) * 32) >> 4;
                mma_f16_ss(t * 128, q_desc + (t * kTileStep + off), k_desc + (st * kTileStep + off),
                           kDescQk, ks > 0);
            }
        };
        // O of tile t plus keys 32 part .. 32 part + 31 of the V tile in stage st
        auto output = [&](int t, int st, int part, bool accumulate) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int ks = 2 * part + k;
                mma_f16_ts(256 + t * 128, t * 128 + ks * 8, v_desc + (st * kTileStep + ks * 128),
                           kDescPv, accumulate || ks > 0);
            }
        };
        PmWork it{};
        uint32_t gb = 0;               // blocks of the items before
        uint32_t items = 0;            // items with keys
        uint32_t blocks[2] = {0u, 0u}, outs[2] = {0u, 0u};  // each tile's blocks and items
        uint32_t cleaned[2] = {0u, 0u};  // V tiles looked over, per stage
        // Block j of the item; its K tile is in stage 0 or 2, V in the next: with
        // stages and tiles known at compile time every operand of a product is
        // a constant away from a loop invariant.
        auto block = [&](int j, auto odd) -> bool {
            constexpr int sv = decltype(odd)::value ? 3 : 1;
            constexpr int sk = decltype(odd)::value ? 0 : 2;
            const uint32_t g = gb + j;  // its V tile is number 2 g + 1 of the ring
            const bool more = j + 1 < it.n_blocks;
            // (a tile that is looked over has landed by then; one wait with either
            // barrier: a second one cost 2 % of every block)
            const bool looked = j >= it.clear;
            if (!pm_wait_warp(p, sh, looked ? &sh->clean[sv >> 1] : &sh->kv_full[sv],
                              (looked ? cleaned[sv >> 1] : g >> 1) & 1u))
                return false;
            cleaned[sv >> 1] += looked ? 1u : 0u;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (t >= it.n_tiles) break;
                const bool last = t == it.n_tiles - 1;
                // the item before has read its output
                if (j == 0 && outs[t] > 0 &&
                    !pm_wait_warp(p, sh, &sh->o_empty[t], (outs[t] - 1) & 1u))
                    return false;
#pragma unroll
                for (int i = 0; i + 1 < kPmParts; ++i) {
                    if (!pm_wait_warp(p, sh, &sh->p_full[t][i], blocks[t] & 1u)) return false;
                    tc_fence_after();
                    if (elect_one()) output(t, sv, i, j > 0);
                    __syncwarp();
                }
                if (!pm_wait_warp(p, sh, &sh->p_full[t][kPmParts - 1], blocks[t] & 1u)) return false;
                ++blocks[t];
                if (more && t == 0 && !pm_wait_warp(p, sh, &sh->kv_full[sk], ((g + 1) >> 1) & 1u))
                    return false;
                tc_fence_after();
                if (elect_one()) {
                    output(t, sv, kPmParts - 1, true);
                    tc_commit(&sh->o_full[t]);
                    if (last) tc_commit(&sh->kv_empty[sv]);
                    if (more) {
                        scores(t, sk);
                        tc_commit(&sh->s_full[t]);
                        if (last) {
                            tc_commit(&sh->kv_empty[sk]);
                            if (j + 2 == it.n_blocks) tc_commit(&sh->q_empty);
                        }
                    }
                }
                __syncwarp();
                if (!more) ++outs[t];
            }
            return true;
        };
        auto first = [&](auto odd) {
            constexpr int sk = decltype(odd)::value ? 2 : 0;
            if (elect_one()) {
                scores(0, sk);
                tc_commit(&sh->s_full[0]);
                if (it.n_tiles == 2) {
                    scores(1, sk);
                    tc_commit(&sh->s_full[1]);
                }
                tc_commit(&sh->kv_empty[sk]);
                if (it.n_blocks == 1) tc_commit(&sh->q_empty);
            }
            __syncwarp();
        };
        static_assert(kPmStages == 4, "the stages of a block's tiles");
        const std::integral_constant<bool, false> kEven{};
        const std::integral_constant<bool, true> kOdd{};
        bool ok = true;
        for (uint32_t n = 0; ok && pm_next(p, sh, n, it); ++n) {
            if (it.n_blocks == 0) continue;
            const bool odd = (gb & 1u) != 0u;
            ok = pm_wait_warp(p, sh, &sh->q_full, items & 1u) &&
                 pm_wait_warp(p, sh, &sh->kv_full[odd ? 2 : 0], (gb >> 1) & 1u);
            ++items;
            if (!ok) break;
            tc_fence_after();
            if (odd) first(kOdd); else first(kEven);
            for (int j = 0; ok && j < it.n_blocks; ++j) {
                if (((gb + j) & 1u) != 0u) ok = block(j, kOdd); else ok = block(j, kEven);
            }
            gb += it.n_blocks;
        }
        // the products in flight end before TMEM is freed (bounded)
        if (elect_one()) tc_commit(&sh->drained);
        __syncwarp();
        mbar_wait_bounded(&sh->drained, 0, nullptr);
    } else if (warp < kPmSoftmaxWarps) {
        // ------------------------------------------------------------ softmax
        const int t = warp >> 2;  // query tile
        const int r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // 32 * (warp % 4) in bits 31..16
        const uint32_t t_s = lanes + t * 128;
        const uint32_t t_o = lanes + 256 + t * 128;
        uint32_t blocks = 0;  // of this tile
        bool ok = true;
        for (uint32_t n = 0; ok && pm_wait_work(p, sh, n); ++n) {
            // what the loop over the blocks needs; the rest is taken from the
            // item again after it
            int n_blocks, keys, clear;
            bool mine;
            {
                const PmWork it = sh->work[n % kPmWorks];
                mine = t < it.n_tiles;
                const int tile0 = it.row0 + (p.G == 1 ? t * kPmTile : 0);
                keys = it.visible(tile0 + r) - it.first * kPmTile;
                // blocks below need no mask for any row of the tile
                clear = it.visible(tile0) / kPmTile - it.first;
                n_blocks = it.n_blocks;
            }
            if (!mine) {
                pm_release_work(sh, n);
                continue;
            }
            float m = -INFINITY;  // what the weights refer to (raw score units)
            float l = 0.f;
            for (int j = 0; j < n_blocks; ++j, ++blocks) {
                ok = pm_wait_warp(p, sh, &sh->s_full[t], blocks & 1u);
                if (!ok) break;
                tc_fence_after();
                uint32_t s[128];
                float mx[4] = {m, m, m, m};
                const int lim = keys - j * kPmTile;
                tmem_ld32(t_s, s);
                tmem_ld32(t_s + 32, s + 32);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tmem_wait_ld32(s + 64 * h);
                    tmem_wait_ld32(s + 64 * h + 32);
                    if (h == 0) {
                        tmem_ld32(t_s + 64, s + 64);
                        tmem_ld32(t_s + 96, s + 96);
                    }
                    if (j >= clear) {
                        // (32 keys that every row of the warp sees need no mask)
#pragma unroll
                        for (int c0 = 64 * h; c0 < 64 * h + 64; c0 += 32) {
                            if (__all_sync(0xffffffffu, lim >= c0 + 32)) continue;
#pragma unroll
                            for (int c = c0; c < c0 + 32; ++c)
                                if (c >= lim) s[c] = 0xff800000u;
                        }
                    }
#pragma unroll
                    for (int c = 64 * h; c < 64 * h + 64; c += 2)
                        mx[(c >> 1) & 3] = fmaxf(fmaxf(mx[(c >> 1) & 3], __uint_as_float(s[c])),
                                                 __uint_as_float(s[c + 1]));
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                // (a maximum of -inf: the difference is NaN, no move)
                const bool move = (top - m) * p.scale_log2 > kPmLazy<T>;
                if (__any_sync(0xffffffffu, move)) {
                    const float to = move ? top : m;
                    const float f = m == to ? 1.f : fast_exp2((m - to) * p.scale_log2);
                    m = to;
                    l *= f;
                    if (j > 0) {
                        ok = pm_wait_warp(p, sh, &sh->o_full[t], (blocks - 1) & 1u);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            uint32_t o[16];
                            tmem_ld16(t_o + 16 * c, o);
                            tmem_wait_ld16(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st16(t_o + 16 * c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : fmaf(m, p.scale_log2, kPmLift<T>);
                const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
                const uint64_t base2 = pack_f32x2(-base, -base);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < kPmParts; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint64_t x = fma_f32x2(
                            pack_f32x2(__uint_as_float(s[32 * c + 2 * i]),
                                       __uint_as_float(s[32 * c + 2 * i + 1])),
                            scale2, base2);
                        float a, d;
                        unpack_f32x2(x, a, d);
                        a = fast_exp2(a);
                        d = fast_exp2(d);
                        sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(a, d));
                        w[i] = ElemOps<T>::pack(a, d);
                    }
                    tmem_st16(t_s + 16 * c, w);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->p_full[t][c]);
                }
                float lo, hi;
                unpack_f32x2(add_f32x2(sum[0], sum[1]), lo, hi);
                l += lo + hi;
            }
            if (!ok) break;
            // ---- output rows
            const PmWork it = sh->work[n % kPmWorks];
            const int qrow = it.row0 + (p.G == 1 ? t * kPmTile : 0) + r;  // of the sequence
            const int head = p.G == 1 ? it.head0 : it.head0 + t;
            const bool real = qrow < it.lq;
            // (while the last product runs)
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (!kSplit && real && p.lse != nullptr)
                p.lse[(size_t)(it.q0 + qrow) * p.Hq + head] =
                    l == 0.f ? -INFINITY : m * p.scale_log2 * kLn2 + logf(l * pm_unlift<T>());
            if (it.n_blocks > 0) {
                ok = pm_wait_warp(p, sh, &sh->o_full[t], (blocks - 1) & 1u);
                if (!ok) break;
                tc_fence_after();
            }
            if (kSplit) {
                // this CTA's part of the rows, for the cluster: O in 32 bits where
                // the keys were (both tiles' products have read them), m and l
                if (it.n_blocks > 0 && it.n_tiles == 2) {
                    ok = pm_wait_warp(p, sh, &sh->o_full[t ^ 1], (blocks - 1) & 1u);
                    if (!ok) break;
                }
                if (it.n_blocks > 0) {
                    uint8_t* mine_o = s_kv + (t * kPmTile + r) * (kHeadDim * 4);
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tmem_ld32(t_o + 32 * c, o);
                        tmem_wait_ld32(o);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4*>(mine_o + (((8 * c + i) ^ lane) << 4)) =
                                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
                s_state[t * kPmTile + r] = make_float2(m, l);
                continue;  // (the item's place is not needed again)
            }
            const uint64_t inv2 = pack_f32x2(inv, inv);
            // Through shared memory, 64 dims at a time, so that a warp stores 128
            // bytes of 4 rows at once: a thread writing its own row touches 32
            // lines an instruction, and the stores took longer than a block.
            // 16-byte piece i of row r stands at i ^ (r % 8): no bank conflicts.
            uint8_t* stage = s_out + warp * kPmStageOut;
            const int srow = lane >> 3, spiece = lane & 7;  // row of 4 and piece it stores
            const int rows = it.lq - (qrow - lane);         // of the sequence, from the warp's first
            uint4* dst = reinterpret_cast<uint4*>(
                             reinterpret_cast<T*>(p.out) +
                             ((size_t)(it.q0 + qrow - lane + srow) * p.Hq + head) * kHeadDim) + spiece;
            const size_t step = (size_t)4 * p.Hq * (kRowBytes / 16);
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                uint32_t o[64];
                if (it.n_blocks > 0) {
                    tmem_ld32(t_o + 64 * c, o);
                    tmem_ld32(t_o + 64 * c + 32, o + 32);
                    tmem_wait_ld32(o);
                    tmem_wait_ld32(o + 32);
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] = 0u;
                }
                if (c == 1 && it.n_blocks > 0) {
                    // TMEM has been read: the next item's output may start
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->o_empty[t]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t u[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint64_t o2 = pack_f32x2(__uint_as_float(o[8 * i + 2 * x]),
                                                       __uint_as_float(o[8 * i + 2 * x + 1]));
                        float a, d;
                        unpack_f32x2(mul_f32x2(o2, inv2), a, d);
                        u[x] = ElemOps<T>::pack(a, d);
                    }
                    *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
                        make_uint4(u[0], u[1], u[2], u[3]);
                }
                __syncwarp();
                uint4 u[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {  // (all loads first: the stores may alias)
                    const int row = 4 * k + srow;  // of the warp
                    u[k] = *reinterpret_cast<const uint4*>(
                        stage + row * 128 + ((spiece ^ (row & 7)) << 4));
                }
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (4 * k + srow < rows) dst[k * step + 8 * c] = u[k];
                __syncwarp();
            }
            if (it.clear < it.n_blocks &&
                *(const volatile int*)&sh->dropped[n % kPmWorks] != 0) {
                __syncwarp();
                pm_restore_rows<T>(p, &sh->work[n % kPmWorks]);
            }
            pm_release_work(sh, n);
        }
        tc_fence_before();
    }
    if (kSplit) {
        // Every thread of every CTA of the cluster passes both barriers, whatever
        // happened before.
        __syncwarp();
        cluster_sync();
        if (warp < kPmSoftmaxWarps) pm_join<T>(p, sh, s_kv, s_state);
        __syncwarp();
        cluster_sync();  // the others' parts have been read
    }
    __syncthreads();
    if (warp == kPmMmaWarp) {
        tc_fence_after();
        tmem_dealloc(sh->tmem, kPmTmemColumns);
    }
}

}  // namespace pkv
