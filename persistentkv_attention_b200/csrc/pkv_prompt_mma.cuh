// pkv_prompt_mma.cuh -- causal attention of packed prompts on the tcgen05
// tensor cores.  Included by pkv_prompt.cu only.
#pragma once

#include "pkv_prompt_kernels.cuh"
#include "pkv_tcgen05.cuh"

namespace pkv {

constexpr int kPmTile = 128;                     // query rows of a tile, keys of a block
constexpr int kPmTileBytes = kPmTile * kRowBytes;  // 32 KB: two 64-element halves of 16 KB
constexpr int kPmHalfBytes = kPmTileBytes / 2;
constexpr int kPmStages = 4;                     // K/V tiles in flight
constexpr int kPmThreads = 320;  // 4 softmax warps per query tile, MMA warp, loader warp
constexpr size_t kPmSmemBytes = 1024 + (size_t)(2 + kPmStages) * kPmTileBytes + 256;
// TMEM columns: scores of tile t at 128 t (its weights, 16 bit, in the first
// 64 of them), output of tile t at 256 + 128 t.
constexpr uint32_t kPmTmemColumns = 512;  // all there are
// The running maximum that weights refer to is raised, and the output
// rescaled, only when a row's maximum has grown by more than this many powers
// of two: weights stay below 2^8, far inside both 16-bit types' range, and
// the division by the sum at the end takes the factor out again.
constexpr float kPmLazy = 8.0f;

struct PmShared {
    uint64_t q_full, kv_full[kPmStages], kv_empty[kPmStages];
    uint64_t s_full[2], p_full[2][2], o_full[2], tail, drained;
    uint32_t tmem;
    int abort;
    int seq, tile;  // this CTA's work
    int warp_sum[kPmThreads / 32];
};
static_assert(sizeof(PmShared) <= 256, "prompt CTA's shared state");

// The CTA's sequence and its query tile: tile number `rank` from the end over
// all sequences' tiles of `rows` query rows, so the longest rows of each
// sequence start first.  Whole CTA; seq = -1 if there are fewer tiles.
__device__ __forceinline__ void pm_find_tile(const PromptParams& p, PmShared* sh, int rank,
                                             int rows) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (t == 0) sh->seq = -1;
    int before = 0;
    for (int base = 0; base < p.B; base += kPmThreads) {
        const int b = p.B - 1 - base - t;
        int n = 0;
        if (b >= 0) {
            const long long len = (long long)__ldg(p.cu_q + b + 1) - __ldg(p.cu_q + b);
            n = len > 0 ? (int)min((len + rows - 1) / rows, (long long)p.Tq) : 0;
        }
        int x = n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off) x += y;
        }
        __syncthreads();
        if (lane == 31) sh->warp_sum[warp] = x;
        __syncthreads();
        int first = before + x - n;
#pragma unroll
        for (int w = 0; w < kPmThreads / 32; ++w) {
            const int s = sh->warp_sum[w];
            first += w < warp ? s : 0;
            before += s;
        }
        if (rank >= first && rank < first + n) {
            sh->seq = b;
            sh->tile = n - 1 - (rank - first);
        }
        if (rank < before) break;  // uniform
    }
    __syncthreads();
}

// One wait of the kernel: false after the time limit or once another thread
// of the CTA has given up.
__device__ __forceinline__ bool pm_wait(const PromptParams& p, PmShared* sh, uint64_t* bar,
                                        uint32_t parity) {
    if (mbar_wait_bounded(bar, parity, &sh->abort)) return true;
    if (atomicExch(&sh->abort, 1) == 0) raise_error(p.error, kErrTimeout);
    return false;
}

// A CTA owns two query tiles of 128 rows that read the same keys: two heads of
// one KV group at the same positions, or (G = 1) two successive tiles of one
// head.  K and V pass through shared memory in blocks of 128 keys (TMA, ring
// of kPmStages tiles).  For each block, tile t's scores S = Q K^T and output
// O += P V are tcgen05 products of one issuing thread with S, P and O in
// TMEM; 128 softmax threads per tile, one per row, turn S into P in place
// with the running maximum and sum in 32 bits.  The issue order
//   S0 S1 | O0 S0' O1 S1' | O0' ...
// keeps the tensor cores on one tile while the other's softmax runs.
// Bound: the tensor cores (4 * 128 flops per query, key and head) and, close
// behind, the 1 exponential per query and key of the special-function units.
template <typename T>
__global__ void __launch_bounds__(kPmThreads, 1)
    pkv_prompt_mma_kernel(const __grid_constant__ PromptParams p,
                          const __grid_constant__ CUtensorMap map_q,
                          const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v) {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* s_q = smem;                          // 2 tiles
    uint8_t* s_kv = smem + 2 * kPmTileBytes;      // kPmStages tiles
    PmShared* sh = reinterpret_cast<PmShared*>(s_kv + kPmStages * kPmTileBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int G = p.Hq / p.Hkv;
    const int rows_per_cta = G == 1 ? 2 * kPmTile : kPmTile;
    const int head_groups = G == 1 ? p.Hq : p.Hq / 2;  // fastest: they share keys in L2
    const int rank = (int)(blockIdx.x / head_groups), group = (int)(blockIdx.x % head_groups);
    pm_find_tile(p, sh, rank, rows_per_cta);
    const int b = sh->seq;
    if (b < 0) return;
    const int q0 = __ldg(p.cu_q + b), q1 = __ldg(p.cu_q + b + 1);
    const int k0 = __ldg(p.cu_k + b), k1 = __ldg(p.cu_k + b + 1);
    if (q0 < 0 || q1 > p.Tq || k0 < 0 || k1 < k0 || k1 > p.Tk) {
        if (threadIdx.x == 0) raise_error(p.error, kErrIndex);
        return;
    }
    const int lq = q1 - q0, lk = k1 - k0;
    const int row0 = sh->tile * rows_per_cta;  // first query row of the CTA in its sequence
    const int head0 = G == 1 ? group : 2 * group;
    const int kvh = head0 / G;
    const int n_tiles = (G == 1 && row0 + kPmTile >= lq) ? 1 : 2;
    // keys that row i of the sequence sees
    auto visible = [lq, lk](int i) { return max(0, min(lk, i + 1 + lk - lq)); };
    const int last_row = min(row0 + rows_per_cta, lq) - 1;
    const int n_keys = visible(last_row);
    const int n_blocks = (n_keys + kPmTile - 1) / kPmTile;
    const int tail = n_keys - (n_blocks - 1) * kPmTile;  // keys of the last block

    if (threadIdx.x == 0) {
        mbar_init(&sh->q_full, 1);
        for (int i = 0; i < kPmStages; ++i) {
            mbar_init(&sh->kv_full[i], 1);
            mbar_init(&sh->kv_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sh->s_full[t], 1);
            mbar_init(&sh->p_full[t][0], 4);  // one arrival per warp
            mbar_init(&sh->p_full[t][1], 4);
            mbar_init(&sh->o_full[t], 1);
        }
        mbar_init(&sh->tail, 1);
        mbar_init(&sh->drained, 1);
        sh->abort = 0;
        fence_mbar_init();
    }
    if (warp == 8) tmem_alloc(&sh->tmem, kPmTmemColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all of TMEM: it starts at lane 0, column 0, and addresses are constants
    constexpr uint32_t tmem = 0;

    if (warp == 9) {
        // ------------------------------------------------------------ loader
        if (lane == 0 && n_blocks > 0) {
            tma_prefetch_map(&map_q);
            tma_prefetch_map(&map_k);
            tma_prefetch_map(&map_v);
            auto load = [&](uint8_t* dst, const CUtensorMap* map, int head, int token,
                            uint64_t* bar) {
                tma_load_3d(dst, map, 0, head, token, bar);
                tma_load_3d(dst + kPmHalfBytes, map, 64, head, token, bar);
            };
            mbar_arrive_expect_tx(&sh->q_full, n_tiles * kPmTileBytes);
            for (int t = 0; t < n_tiles; ++t)
                load(s_q + t * kPmTileBytes, &map_q, G == 1 ? head0 : head0 + t,
                     q0 + row0 + (G == 1 ? t * kPmTile : 0), &sh->q_full);
            int issued = 0;
            bool ok = true;
            for (int i = 0; i < 2 * n_blocks; ++i) {  // K0 V0 K1 V1 ...
                const int st = i % kPmStages;
                if (i >= kPmStages) {
                    ok = pm_wait(p, sh, &sh->kv_empty[st], (i / kPmStages - 1) & 1);
                    if (!ok) break;
                }
                mbar_arrive_expect_tx(&sh->kv_full[st], kPmTileBytes);
                load(s_kv + st * kPmTileBytes, (i & 1) ? &map_v : &map_k, kvh,
                     k0 + (i >> 1) * kPmTile, &sh->kv_full[st]);
                ++issued;
            }
            // copies in flight land before the CTA ends (bounded)
            if (!ok) {
                mbar_wait_bounded(&sh->q_full, 0, nullptr);
                for (int i = max(0, issued - kPmStages); i < issued; ++i)
                    mbar_wait_bounded(&sh->kv_full[i % kPmStages], (i / kPmStages) & 1, nullptr);
            }
        }
        __syncwarp();
        if (n_blocks > 0 && tail < kPmTile) {
            // Rows of V behind the last key belong to other sequences or to
            // nobody and may hold anything; their weights are 0, and 0 * NaN
            // is not: zero them before the product reads the tile.
            const int i = 2 * n_blocks - 1;
            const int st = i % kPmStages;
            bool ok = pm_wait(p, sh, &sh->kv_full[st], (i / kPmStages) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                uint8_t* tile = s_kv + st * kPmTileBytes;
                for (int c = tail * 8 + lane; c < kPmTile * 8; c += 32) {
                    *reinterpret_cast<uint4*>(tile + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(tile + kPmHalfBytes + c * 16) =
                        make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->tail);
            }
        }
    } else if (warp == 8) {
        // ------------------------------------------------------------ products
        // The whole warp walks the loop, so that descriptors and addresses are
        // uniform values; one elected lane issues the products and commits.
        if (n_blocks > 0) {
            constexpr uint32_t kDescQk = mma_desc_f16(kPmTile, kPmTile, kBf16, false);
            constexpr uint32_t kDescPv = mma_desc_f16(kPmTile, kHeadDim, kBf16, true);
            const uint64_t q_desc = smem_desc_sw128(smem_u32(s_q), 16, 1024);
            const uint64_t k_desc = smem_desc_sw128(smem_u32(s_kv), 16, 1024);
            const uint64_t v_desc = smem_desc_sw128(smem_u32(s_kv), kPmHalfBytes, 1024);
            constexpr uint32_t kTileStep = kPmTileBytes >> 4;  // in descriptor units
            auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                return __all_sync(0xffffffffu, pm_wait(p, sh, bar, parity));
            };
            // S of tile t from the K tile in stage st
            auto scores = [&](int t, int st) {
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint32_t off = ((ks >> 2) * kPmHalfBytes + (ks & 3) * 32) >> 4;
                    mma_f16_ss(t * 128, q_desc + (t * kTileStep + off),
                               k_desc + (st * kTileStep + off), kDescQk, ks > 0);
                }
            };
            // O of tile t plus keys 64 half .. 64 half + 63 of the V tile in stage st
            auto output = [&](int t, int st, int half, bool accumulate) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int ks = 4 * half + k;
                    mma_f16_ts(256 + t * 128, t * 128 + ks * 8,
                               v_desc + (st * kTileStep + ks * 128), kDescPv, accumulate || ks > 0);
                }
            };
            bool ok = wait(&sh->q_full, 0) && wait(&sh->kv_full[0], 0);
            if (ok && elect_one()) {
                scores(0, 0);
                tc_commit(&sh->s_full[0]);
                if (n_tiles == 2) {
                    scores(1, 0);
                    tc_commit(&sh->s_full[1]);
                }
                tc_commit(&sh->kv_empty[0]);
            }
            __syncwarp();
            // One block; its V tile is in stage 1 or 3, the next block's K tile in
            // stage 2 or 0: with stages and tiles known at compile time every
            // operand of a product is a constant away from a loop invariant.
            auto block = [&](int j, auto odd) -> bool {
                constexpr int sv = decltype(odd)::value ? 3 : 1;
                constexpr int sk = decltype(odd)::value ? 0 : 2;
                const uint32_t ring = (uint32_t)(j >> 1) & 1u;  // (2 j + 1) / 4
                const uint32_t ring_k = (uint32_t)((j + 1) >> 1) & 1u;
                const bool more = j + 1 < n_blocks;
                if (!wait(&sh->kv_full[sv], ring)) return false;
                if (!more && tail < kPmTile && !wait(&sh->tail, 0)) return false;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t >= n_tiles) break;
                    const bool last = t == n_tiles - 1;
                    if (!wait(&sh->p_full[t][0], j & 1)) return false;
                    tc_fence_after();
                    if (elect_one()) output(t, sv, 0, j > 0);
                    __syncwarp();
                    if (!wait(&sh->p_full[t][1], j & 1)) return false;
                    if (more && t == 0 && !wait(&sh->kv_full[sk], ring_k)) return false;
                    tc_fence_after();
                    if (elect_one()) {
                        output(t, sv, 1, true);
                        tc_commit(&sh->o_full[t]);
                        if (last) tc_commit(&sh->kv_empty[sv]);
                        if (more) {
                            scores(t, sk);
                            tc_commit(&sh->s_full[t]);
                            if (last) tc_commit(&sh->kv_empty[sk]);
                        }
                    }
                    __syncwarp();
                }
                return true;
            };
            static_assert(kPmStages == 4, "the stages of a block's tiles");
            for (int j = 0; ok && j < n_blocks; j += 2) {
                ok = block(j, std::integral_constant<bool, false>{});
                if (ok && j + 1 < n_blocks) ok = block(j + 1, std::integral_constant<bool, true>{});
            }
            // the products in flight end before TMEM is freed (bounded)
            if (elect_one()) tc_commit(&sh->drained);
            __syncwarp();
            mbar_wait_bounded(&sh->drained, 0, nullptr);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax
        const int t = warp >> 2;  // query tile
        const int r = threadIdx.x & 127;
        const int qrow = row0 + (G == 1 ? t * kPmTile : 0) + r;  // row of the sequence
        const int head = G == 1 ? head0 : head0 + t;
        const bool real = t < n_tiles && qrow < lq;
        if (t < n_tiles) {
            const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // 32 * (warp % 4) in bits 31..16
            const uint32_t t_s = tmem + lanes + t * 128;
            const uint32_t t_o = tmem + lanes + 256 + t * 128;
            const int n = visible(qrow);
            // blocks below need no mask for any row of the tile
            const int clear = visible(qrow - r) / kPmTile;
            float m = -INFINITY;  // what the weights refer to (raw score units)
            float l = 0.f;
            bool ok = true;
            for (int j = 0; j < n_blocks; ++j) {
                ok = __all_sync(0xffffffffu, pm_wait(p, sh, &sh->s_full[t], j & 1));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, s + 32 * c);
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_wait_ld32(s + 32 * c);
                if (j >= clear) {
                    const int lim = n - j * kPmTile;
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c >= lim) s[c] = 0xff800000u;
                }
                float mx[4] = {m, m, m, m};
#pragma unroll
                for (int c = 0; c < 128; c += 2)
                    mx[(c >> 1) & 3] = fmaxf(fmaxf(mx[(c >> 1) & 3], __uint_as_float(s[c])),
                                             __uint_as_float(s[c + 1]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                // (a maximum of -inf: the difference is NaN, no move)
                const bool move = (top - m) * p.scale_log2 > kPmLazy;
                if (__any_sync(0xffffffffu, move)) {
                    const float to = move ? top : m;
                    const float f = m == to ? 1.f : fast_exp2((m - to) * p.scale_log2);
                    m = to;
                    l *= f;
                    if (j > 0) {
                        ok = __all_sync(0xffffffffu, pm_wait(p, sh, &sh->o_full[t], (j - 1) & 1));
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t o[32];
                            tmem_ld32(t_o + 32 * c, o);
                            tmem_wait_ld32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st32(t_o + 32 * c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m * p.scale_log2;
                const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
                const uint64_t base2 = pack_f32x2(-base, -base);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint64_t x = fma_f32x2(
                            pack_f32x2(__uint_as_float(s[64 * c + 2 * i]),
                                       __uint_as_float(s[64 * c + 2 * i + 1])),
                            scale2, base2);
                        float a, d;
                        unpack_f32x2(x, a, d);
                        a = fast_exp2(a);
                        d = fast_exp2(d);
                        sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(a, d));
                        w[i] = ElemOps<T>::pack(a, d);
                    }
                    tmem_st32(t_s + 32 * c, w);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->p_full[t][c]);
                }
                float lo, hi;
                unpack_f32x2(add_f32x2(sum[0], sum[1]), lo, hi);
                l += lo + hi;
            }
            // ---- output rows
            if (ok && n_blocks > 0)
                ok = __all_sync(0xffffffffu,
                                pm_wait(p, sh, &sh->o_full[t], (n_blocks - 1) & 1));
            tc_fence_after();
            if (ok) {
                T* out = reinterpret_cast<T*>(p.out) +
                         ((size_t)(q0 + min(qrow, lq - 1)) * p.Hq + head) * kHeadDim;
                float* lse =
                    p.lse != nullptr ? p.lse + (size_t)(q0 + min(qrow, lq - 1)) * p.Hq + head : nullptr;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                float worst = 0.f;  // NaN if any value of the row is not finite
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[32];
                    if (n_blocks > 0) {
                        tmem_ld32(t_o + 32 * c, o);
                        tmem_wait_ld32(o);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) worst = fmaf(__uint_as_float(o[i]), 0.f, worst);
                    if (real) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 u;
                            u.x = ElemOps<T>::pack(__uint_as_float(o[8 * i]) * inv,
                                                   __uint_as_float(o[8 * i + 1]) * inv);
                            u.y = ElemOps<T>::pack(__uint_as_float(o[8 * i + 2]) * inv,
                                                   __uint_as_float(o[8 * i + 3]) * inv);
                            u.z = ElemOps<T>::pack(__uint_as_float(o[8 * i + 4]) * inv,
                                                   __uint_as_float(o[8 * i + 5]) * inv);
                            u.w = ElemOps<T>::pack(__uint_as_float(o[8 * i + 6]) * inv,
                                                   __uint_as_float(o[8 * i + 7]) * inv);
                            reinterpret_cast<uint4*>(out)[4 * c + i] = u;
                        }
                    }
                }
                if (real && lse != nullptr)
                    *lse = l == 0.f ? -INFINITY : m * p.scale_log2 * kLn2 + logf(l);
                // A value that is not finite may come from a key the row does
                // not see (weight 0 times an infinite or NaN V): such a row is
                // computed again from its own keys alone.
                __syncwarp();
                unsigned again = __ballot_sync(0xffffffffu, real && worst != 0.f);
                while (again != 0u) {
                    const int i = __ffs(again) - 1;
                    again &= again - 1;
                    const int row = qrow - lane + i;  // of the sequence
                    const size_t at = (size_t)(q0 + row) * p.Hq + head;
                    prompt_row<T>(p, p.q + (q0 + row) * p.q_tok + head * p.q_head,
                                  p.k + k0 * p.k_tok + kvh * p.k_head,
                                  p.v + k0 * p.v_tok + kvh * p.v_head, visible(row),
                                  reinterpret_cast<T*>(p.out) + at * kHeadDim,
                                  p.lse != nullptr ? p.lse + at : nullptr, lane);
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, kPmTmemColumns);
    }
}

}  // namespace pkv
