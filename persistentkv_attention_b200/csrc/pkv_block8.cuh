// pkv_block8.cuh -- decode over an e4m3 cache with one scale per block of
// tokens and head.  Included by pkv_block8.cu only.
#pragma once

#include "pkv_kernels.cuh"

namespace pkv {

struct Block8Params {
    DecodeParams d;
    const float* k_scales;  // [P][Hkv][page / block]
    const float* v_scales;
    int block;     // tokens per scale, a multiple of 16 that divides page_size
};

// A ring slot holds 32 tokens of one KV head: 32 lines of 128 e4m3 values of K,
// then of V, 16-byte chunk c of line t at position c ^ (t & 7); its two K and
// two V scales sit beside the ring.
constexpr int kB8Tokens = 32;
constexpr int kB8Line = kHeadDim;              // bytes
constexpr int kB8Half = kB8Tokens * kB8Line;   // K part of a slot
static_assert(2 * kB8Half == kSlotBytes, "a slot is the 16-bit ring's slot");
constexpr int kB8Scale = 16;                   // tokens that share a scale at least

// The running maximum that weights refer to is raised only when a row's
// maximum has grown by more than this many powers of two: weights stay below
// 2^8 (fp16 holds 2^15), the accumulators are rescaled a few times per row
// instead of every stage, and the division by the sum takes the factor out.
constexpr float kB8Lazy = 8.0f;

// What the producer resolves a round at a time (up to 16 stages of one item,
// up to 32 page lookups): pool lines of the round's copies, and the scales of
// its stages, {K, K, V, V} each.  Several rounds' scales are kept, so that
// short rows do not wait for one another.
constexpr int kB8Round = 16;  // stages
constexpr int kB8Rounds = kDescSlots;
static_assert((kB8Rounds & (kB8Rounds - 1)) == 0, "rounds are counted by masks");
struct B8Lookups {
    float scales[kB8Rounds][kB8Round][4];
    int lines[kB8Rounds][32];  // -1: no page
    int stages[kB8Rounds];     // 0: the last round is over
    uint64_t scales_full[kB8Rounds], lines_full[kB8Rounds];
};

// Four consumer warps, one producer warp that resolves pages and copies K, one
// that copies V: the copies of a stage are four instructions of one thread with
// pages of 16 tokens, and one thread issuing all of them beside the consumers'
// math falls behind HBM (64 rows up to 32768 tokens: 197 us, two threads 175 us).
constexpr int kB8Threads = kThreads + 32;

// The sum is in 32 bits and may grow further before its reference moves.
constexpr float kB8LazySum = 32.0f;
// A state that leaves the CTA refers to the largest score or, where V scales are
// beyond this many powers of two, to the largest contribution less it, so that
// its accumulators stay far from fp32's largest.
constexpr float kB8Headroom = 60.0f;

template <int G, int NSLOTS>
constexpr size_t block8_smem_bytes() {
    return decode_smem_bytes<G, NSLOTS>() + sizeof(B8Lookups);
}

// Two e4m3 values (the low or high half of a word) as two fp16 values: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t word, bool high) {
    uint32_t out;
    const uint16_t h = (uint16_t)(high ? word >> 16 : word);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(out) : "h"(h));
    return out;
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr));
    return v;
}

__device__ __forceinline__ float fast_log2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A scale, copied asynchronously.
__device__ __forceinline__ void cp_async_4(uint32_t smem_dst, const void* src, bool valid) {
    const uint32_t bytes = valid ? 4u : 0u;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_dst), "l"(src),
                 "r"(bytes)
                 : "memory");
}

// Same work division as pkv_decode_kernel's device schedule: CTA g * Hkv + kvh
// streams the row pieces of group g for one KV head, one producer warp and
// four consumer warps, every 32-token stage to one warp.
//
// Mathematics.  With s_t the scaled score, b_t the V scale of token t's block and
// v_t the raw e4m3 values:  O = sum e^s_t b_t v_t / sum e^s_t.  A V scale costs
// one add in a weight's exponent (p_t = exp(s_t + ln b_t - m)) and never touches
// the accumulators, and their running maximum m is that of a token's contribution
// s_t + ln b_t, so no block's scale can push another's weights out of fp16's
// range.  The sum has a reference of its own, the largest score, since weights
// that hold b_t say nothing about it once scales are 2^126 apart.  A K scale is a
// factor of its 16 tokens' scores.
//
// Both products run as mma.sync m16n8k16 on fp16 (every e4m3 value is exact in
// it), 16 tokens x 8 heads and 128 dims x 8 heads.  A lane's 16-byte loads are
// the fragments: the dims of a product's k index may come in any order that K
// and Q share, and the dims of the output rows in any order at all, so chunk
// 2 * (lane % 4) + h of a K line serves four k steps and chunk lane / 4 of two V
// lines, bytes interleaved, eight output tiles.  No second pass over shared
// memory and no transpose; that pass is what bounds the per-tensor route.
// Bound: HBM, 256 bytes per token and KV head, for long batches (64 rows up to
// 32768 tokens, 983 MB: 172 us, 5.7 TB/s; pages of 32 tokens 160 us, 6.1 TB/s; 168
// and 157 without a reference of the sum's own); for short ones the launch, the
// schedule, the first copies and the merge (one row of 4096 tokens: 11.1 us, of
// which its bytes take 1.3).
template <int G, typename T, int BOX, int NSLOTS>
__global__ void __launch_bounds__(kB8Threads, PKV_MIN_CTAS_PER_SM)
    pkv_block8_kernel(const __grid_constant__ Block8Params bp,
                      const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v) {
    static_assert(BOX == 16 || BOX == 32, "box rows");
    // A slot belongs to one consumer warp for good: a barrier's parity cannot
    // tell a phase from the one two before it, so a warp must not wait for a
    // slot's next use while another still owes its last one.
    static_assert(NSLOTS % kConsumerWarps == 0, "every use of a slot is one warp's");
    const DecodeParams& p = bp.d;
    using Ops = ElemOps<T>;
    constexpr int kBoxesPerStage = kB8Tokens / BOX;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_u32 = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw_u32 + 1023u) & ~1023u) - raw_u32);
    uint8_t* ring = smem;
    uint8_t* s_q = ring + (size_t)NSLOTS * kSlotBytes;
    float* s_merge = reinterpret_cast<float*>(s_q + kDescSlots * kQSlotBytes);
    ItemDesc* s_desc = reinterpret_cast<ItemDesc*>(ring + merge_region_bytes<G, NSLOTS>());
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_desc + kDescSlots);
    uint64_t* empty_bar = full_bar + NSLOTS;
    uint64_t* desc_full = empty_bar + NSLOTS;
    uint64_t* desc_empty = desc_full + kDescSlots;
    uint64_t* merge_bar = desc_empty + kDescSlots;
    uint8_t* s_flag_bytes = reinterpret_cast<uint8_t*>(merge_bar + 2);
    volatile int* s_flags = reinterpret_cast<volatile int*>(s_flag_bytes);  // [0] abort
    float* s_mstat = reinterpret_cast<float*>(s_flag_bytes + 64);
    float* s_lstat = s_mstat + 2 * kConsumerWarps * 8;
    float* s_mw = s_lstat + 2 * kConsumerWarps * 8;
    PendingMerge* s_pend = reinterpret_cast<PendingMerge*>(s_mw + mw_floats<G>());
    B8Lookups* s_look = reinterpret_cast<B8Lookups*>(s_pend + kMaxPending);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    decode_params_touch(p);
    griddep_wait();
    AutoCursor acur;
    acur.b = acur.b_end = 0;
    Item first_item;
    int first_pid = -1;
    __shared__ int s_my_items;
    if (warp == kConsumerWarps) {
        acur = auto_init(p, lane);
        const int mine = acur.b >= 0 ? acur.b_end - acur.b : 0;
        if (mine > 0) first_item = auto_item<BOX>(p, acur, lane, lane == 0, first_pid);
        if (lane == 0) s_my_items = mine;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < NSLOTS; ++s) {
            mbar_init(&full_bar[s], 2);  // K and V copies
            mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < kDescSlots; ++s) {
            mbar_init(&desc_full[s], 33);  // 32 lanes' Q copies + the descriptor store
            mbar_init(&desc_empty[s], kConsumerWarps);
        }
        mbar_init(merge_bar, 1);
        for (int r = 0; r < kB8Rounds; ++r) {
            mbar_init(&s_look->scales_full[r], 32);
            mbar_init(&s_look->lines_full[r], 1);
        }
        s_flags[0] = 0;
        fence_mbar_init();
    }
    __syncthreads();
    const int my_items = s_my_items;

    // One pool's copies of a round's stages, by one thread: lines of the pool
    // to part `part` of the ring's slots.  False if a slot did not come free.
    const uint64_t policy = l2_evict_first_policy();
    auto copy_round = [&](const CUtensorMap& map, int part, const int* lines, int stages,
                          uint32_t& gs) -> bool {
        for (int st = 0; st < stages; ++st, ++gs) {
            const uint32_t slot = gs % NSLOTS;
            int line[kBoxesPerStage];
            uint32_t bytes = 0;
#pragma unroll
            for (int bx = 0; bx < kBoxesPerStage; ++bx) {
                line[bx] = lines[st * kBoxesPerStage + bx];
                bytes += line[bx] >= 0 ? (uint32_t)(BOX * kB8Line) : 0u;
            }
            if (gs >= (uint32_t)NSLOTS &&
                !mbar_wait_bounded(&empty_bar[slot], ((gs / NSLOTS) - 1u) & 1u, s_flags))
                return false;
            mbar_arrive_expect_tx(&full_bar[slot], bytes);
            uint8_t* dst = ring + (size_t)slot * kSlotBytes + part * kB8Half;
#pragma unroll
            for (int bx = 0; bx < kBoxesPerStage; ++bx)
                if (line[bx] >= 0)
                    tma_load_2d(dst + bx * BOX * kB8Line, &map, 0, line[bx], &full_bar[slot], policy);
        }
        return true;
    };
    // Every copy a thread issued lands before the CTA exits.
    auto drain = [&](uint32_t gs) {
        for (uint32_t g = gs > (uint32_t)NSLOTS ? gs - NSLOTS : 0u; g < gs; ++g) {
            if (!mbar_wait_bounded(&full_bar[g % NSLOTS], (g / NSLOTS) & 1u, nullptr)) {
                raise_error(p.error, kErrTimeout);
                break;
            }
        }
    };

    if (warp == kConsumerWarps + 1) {
        // ============================ V copies ============================
        if (lane == 0) {
            tma_prefetch_map(&tmap_v);
            uint32_t gs = 0;
            for (uint32_t r = 0;; ++r) {
                const int at = (int)(r & (kB8Rounds - 1));
                bool ok = mbar_wait_bounded(&s_look->lines_full[at], (r / kB8Rounds) & 1u, s_flags);
                const int stages = ok ? s_look->stages[at] : 0;
                if (ok && stages == 0) break;
                ok = ok && copy_round(tmap_v, 1, s_look->lines[at], stages, gs);
                if (!ok) {
                    s_flags[0] = 1;
                    raise_error(p.error, kErrTimeout);
                    break;
                }
            }
            drain(gs);
        }
        return;
    }
    if (warp == kConsumerWarps) {
        // ============================ producer warp ============================
        const uint32_t q_base = smem_u32(s_q);
        const int nblk = p.page_size / bp.block;
        if (lane == 0) tma_prefetch_map(&tmap_k);
        uint32_t gstage = 0, ground = 0;
        uint32_t round_end[kB8Rounds] = {0u, 0u, 0u, 0u};  // of the rounds before, oldest first
        uint32_t round_len[kB8Rounds] = {0u, 0u, 0u, 0u};
        bool aborted = false;
        int pid0 = first_pid;
        Item cur = first_item;
        auto give_up = [&]() {
            if (lane == 0) {
                s_flags[0] = 1;
                raise_error(p.error, kErrTimeout);
            }
            aborted = true;
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
            bool ok = true;
            if (lane == 0) ok = mbar_wait_bounded(bar, parity, s_flags);
            return __shfl_sync(0xffffffffu, ok, 0) && s_flags[0] == 0;
        };
        // The next round's place in the lookups: that of the round kB8Rounds
        // before, all of whose stages must have been consumed (one that the ring
        // has issued a successor of has been).
        auto round_free = [&]() -> bool {
            const uint32_t g = round_end[0] - 1u - (uint32_t)lane;
            bool free = true;
            if ((uint32_t)lane < round_len[0] && gstage <= g + NSLOTS)
                free = mbar_wait_bounded(&empty_bar[g % NSLOTS], (g / NSLOTS) & 1u, s_flags);
            return __all_sync(0xffffffffu, free);
        };
        for (int s = 0; s < my_items && !aborted; ++s) {
            if (s == my_items - 1) griddep_launch_dependents();
            const int e = s % kDescSlots;
            if (s >= kDescSlots && !wait(&desc_empty[e], ((s / kDescSlots) - 1) & 1)) {
                give_up();
                break;
            }
            {
                const bool qok = cur.q_row >= 0;
                const uint8_t* qsrc = reinterpret_cast<const uint8_t*>(p.q) +
                                      ((size_t)(qok ? cur.q_row : 0) * p.Hq + (size_t)cur.kvh * G) *
                                          kRowBytes;
#pragma unroll
                for (int c = lane; c < G * 16; c += 32)
                    cp_async_16(q_base + e * kQSlotBytes + c * 16, qsrc + c * 16, qok ? 16u : 0u,
                                policy);
                cp_async_mbar_arrive_noinc(&desc_full[e]);
                if (lane == 0) {
                    ItemDesc& d = s_desc[e];
                    d.row = cur.row;
                    d.kvh = cur.kvh;
                    d.split = cur.split;
                    d.tok_begin = cur.tok_begin;
                    d.tok_end = cur.tok_end;
                    d.slot = cur.slot;
                    d.row_splits = cur.row_splits;
                    d.out_row = cur.out_row;
                    mbar_arrive(&desc_full[e]);
                }
            }
            const Item it = cur;
            const int n_stages = ceil_div_i(it.tok_end - it.tok_begin, kB8Tokens);
            const int n_boxes = ceil_div_i(it.tok_end - it.tok_begin, BOX);
            const int32_t* bt_row = p.block_table + (size_t)it.row * p.max_pages;
            const bool has_next = s + 1 < my_items;
            bool fetched = !has_next;
            Item nxt = it;
            int nxt_pid = -1;
            int pid_next = pid0;
            // page lookups a round at a time, one per lane, one round ahead
            constexpr int kRoundBoxes = kB8Round * kBoxesPerStage;
            for (int base = 0; base < n_boxes && !aborted; base += kRoundBoxes) {
                const int box = base + lane;
                const int tok = it.tok_begin + box * BOX;
                const int pid = pid_next;
                if (base + kRoundBoxes < n_boxes)
                    pid_next = box + kRoundBoxes < n_boxes
                                   ? __ldg(bt_row + (tok + kRoundBoxes * BOX) / p.page_size)
                                   : -1;
                bool ok = lane < kRoundBoxes && box < n_boxes;
                int y = -1;               // line of the box in the pool
                int sc = 0, sc_step = 0;  // scales of the box's one or two 16-token parts
                if (ok) {
                    if (pid < 0 || pid >= p.num_pages) {
                        ok = false;
                        raise_error(p.error, kErrPageId);
                    } else {
                        const int head = pid * p.Hkv + it.kvh;
                        const int off = tok % p.page_size;
                        y = head * p.page_size + off;
                        const int blk = off / bp.block;
                        sc = head * nblk + blk;
                        // (a box lies within a page, so its second part's block does too)
                        if (BOX > kB8Scale) sc_step = (off + kB8Scale) / bp.block - blk;
                    }
                }
                if (!round_free()) {
                    give_up();
                    break;
                }
                const int at_round = (int)(ground & (kB8Rounds - 1));
                if (lane < kRoundBoxes) {
                    // a missing box has scale 0
                    const uint32_t at =
                        smem_u32(&s_look->scales[at_round][lane / kBoxesPerStage][0]) +
                        (lane % kBoxesPerStage) * (BOX / kB8Scale) * 4;
#pragma unroll
                    for (int h = 0; h < BOX / kB8Scale; ++h) {
                        cp_async_4(at + 4 * h, bp.k_scales + sc + h * sc_step, ok);
                        cp_async_4(at + 8 + 4 * h, bp.v_scales + sc + h * sc_step, ok);
                    }
                }
                cp_async_mbar_arrive_noinc(&s_look->scales_full[at_round]);
                ++ground;
                const int stages_here = min(kB8Round, n_stages - base / kBoxesPerStage);
                s_look->lines[at_round][lane] = y;
                if (lane == 0) s_look->stages[at_round] = stages_here;
                __syncwarp();
                bool ok_stages = true;
                if (lane == 0) {
                    mbar_arrive(&s_look->lines_full[at_round]);
                    uint32_t gs = gstage;
                    ok_stages = copy_round(tmap_k, 0, s_look->lines[at_round], stages_here, gs);
                    if (!ok_stages) gstage = gs;  // what was issued, for the drain
                }
                ok_stages = __shfl_sync(0xffffffffu, ok_stages, 0);
                if (!ok_stages) {
                    give_up();
                    break;
                }
                gstage += stages_here;
#pragma unroll
                for (int r = 0; r + 1 < kB8Rounds; ++r) {
                    round_end[r] = round_end[r + 1];
                    round_len[r] = round_len[r + 1];
                }
                round_end[kB8Rounds - 1] = gstage;
                round_len[kB8Rounds - 1] = stages_here;
                if (!fetched) {
                    fetched = true;
                    nxt = auto_item<BOX>(p, acur, lane, lane == 0, nxt_pid);
                }
            }
            if (!fetched) nxt = auto_item<BOX>(p, acur, lane, lane == 0, nxt_pid);
            cur = nxt;
            pid0 = nxt_pid;
        }
        // the V copies end with a round of no stages
        if (!aborted && round_free() && lane == 0) {
            const int at = (int)(ground & (kB8Rounds - 1));
            s_look->stages[at] = 0;
            mbar_arrive(&s_look->lines_full[at]);
        }
        cp_async_wait_all();
        if (lane == 0) drain(gstage);
        return;
    }

    // ============================== consumer warps ==============================
    const int g8 = lane >> 2;         // token row of score tiles / head of B fragments
    const int t4 = lane & 3;          // head pair of accumulators
    const uint32_t ring_u32 = smem_u32(ring);
    uint32_t gbase = 0;
    uint32_t ground = 0, seen_round = 0xffffffffu;  // rounds of scales
    int buf = 0;
    bool aborted = false;
    int n_pend = 0;
    int pend_old = 0;
    uint32_t merge_phase = 0u;
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const bool ok = mbar_wait_bounded(bar, parity, s_flags);
        if (__all_sync(0xffffffffu, ok) && s_flags[0] == 0) return true;
        if (lane == 0) {
            s_flags[0] = 1;
            raise_error(p.error, kErrTimeout);
        }
        return false;
    };

    for (int s = 0; s < my_items; ++s) {
        if (s == my_items - 1) griddep_launch_dependents();
        const int e = s % kDescSlots;
        Item it;
        it.tok_begin = it.tok_end = 0;
        it.row = it.kvh = it.split = 0;
        it.slot = -1;
        it.row_splits = 2;
        it.out_row = -1;
        uint32_t qf[8][2];
        float qs[2] = {0.f, 0.f};  // score factor of this lane's two heads
        if (!aborted) aborted = !wait(&desc_full[e], (s / kDescSlots) & 1);
        if (!aborted) {
            const ItemDesc& d = s_desc[e];
            it.row = d.row;
            it.kvh = d.kvh;
            it.split = d.split;
            it.tok_begin = d.tok_begin;
            it.tok_end = d.tok_end;
            it.slot = d.slot;
            it.row_splits = d.row_splits;
            it.out_row = d.out_row;
            // Q^T as the B operand: k step 4 h + u holds dims 16 (2 t4 + h) + 4 u + 0 .. 3
            // of head g8 (zeros beyond the G heads)
            const uint8_t* qrow = s_q + e * kQSlotBytes + (g8 < G ? g8 : 0) * kRowBytes;
            uint4 raw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                raw[i] = g8 < G ? *reinterpret_cast<const uint4*>(qrow + t4 * 64 + i * 16)
                                : make_uint4(0u, 0u, 0u, 0u);
            float unit = 1.f;
            if constexpr (Ops::kSplitP) {
                // bf16 queries in fp16: the head's row is brought to [2^8, 2^9) by
                // a power of two, so all 8 bits of every element that matters are
                // kept (one 2^32 below the largest underflows)
                float amax = 0.f;
                const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 f =
                        __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
                    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                int ex = (int)(__float_as_uint(amax) >> 23) - 127 - 8;
                if (!(amax > 0.f) || !(amax < INFINITY)) ex = 0;
                if (ex < -126) ex = -126;
                const float down = __uint_as_float((unsigned)(127 - ex) << 23);
                unit = __uint_as_float((unsigned)(127 + ex) << 23);
                uint32_t* wm = reinterpret_cast<uint32_t*>(raw);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 f =
                        __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&wm[i]));
                    wm[i] = ElemOps<__half>::pack(f.x * down, f.y * down);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 a = raw[2 * h], b = raw[2 * h + 1];
                qf[4 * h][0] = a.x;
                qf[4 * h][1] = a.y;
                qf[4 * h + 1][0] = a.z;
                qf[4 * h + 1][1] = a.w;
                qf[4 * h + 2][0] = b.x;
                qf[4 * h + 2][1] = b.y;
                qf[4 * h + 3][0] = b.z;
                qf[4 * h + 3][1] = b.w;
            }
            // the accumulators' heads are 2 t4 and 2 t4 + 1; head g sits in lanes 4 g
            qs[0] = p.scale_log2 * __shfl_sync(0xffffffffu, unit, 8 * t4);
            qs[1] = p.scale_log2 * __shfl_sync(0xffffffffu, unit, 8 * t4 + 4);
            __syncwarp();
            if (lane == 0) mbar_arrive(&desc_empty[e]);
        }
        const int n_stages = aborted ? 0 : ceil_div_i(it.tok_end - it.tok_begin, kB8Tokens);

        float m_run[2] = {-INFINITY, -INFINITY};  // what weights refer to, log2
        float m_sum[2] = {-INFINITY, -INFINITY};  // what this lane's sum refers to
        float l_run[2] = {0.f, 0.f};
        float acc[8][4];
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;

        // stage gs goes to warp gs % 4, whatever the item it belongs to
        for (int j = (int)((warp - gbase) & (kConsumerWarps - 1)); j < n_stages;
             j += kConsumerWarps) {
            const uint32_t gs = gbase + (uint32_t)j;
            const uint32_t slot = gs % NSLOTS;
            if (!aborted) aborted = !wait(&full_bar[slot], (gs / NSLOTS) & 1u);
            if (aborted) break;
            const int valid = min(kB8Tokens, it.tok_end - (it.tok_begin + j * kB8Tokens));
            const uint32_t kbase = ring_u32 + slot * kSlotBytes;
            // the stage's round and place in it (rounds count from the item's start)
            const uint32_t rnd = ground + (uint32_t)(j / kB8Round);
            if (rnd != seen_round) {
                aborted = !wait(&s_look->scales_full[rnd & (kB8Rounds - 1)],
                                (rnd / kB8Rounds) & 1u);
                if (aborted) break;
                seen_round = rnd;
            }
            const float4 scales =
                *reinterpret_cast<const float4*>(
                s_look->scales[rnd & (kB8Rounds - 1)][j % kB8Round]);
            if (valid < kB8Tokens || scales.z == 0.f || scales.w == 0.f) {
                // V lines past the row's end or of a scale of 0 (a page that is not
                // there has that scale too) may hold anything: zero them, so that a
                // weight of 0 never meets a NaN
                uint8_t* line0 = ring + (size_t)slot * kSlotBytes + kB8Half;
                for (int c = lane; c < kB8Tokens * 8; c += 32) {
                    const int line = c >> 3;
                    if (line >= valid || (line < kB8Scale ? scales.z : scales.w) == 0.f)
                        *reinterpret_cast<uint4*>(line0 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
                __syncwarp();
            }

            // ---- the stage into registers, and its slot back to the producer
            uint4 kr[2][2][2], vr[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t at =
                        kbase + (16 * i + g8) * kB8Line + (((2 * t4 + h) ^ g8) << 4);
                    kr[i][h][0] = lds128(at);                // token 16 i + g8
                    kr[i][h][1] = lds128(at + 8 * kB8Line);  // token 16 i + g8 + 8
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // tokens 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9
                const uint32_t at = kbase + kB8Half + (16 * i + 2 * t4) * kB8Line;
                const uint32_t x0 = (uint32_t)((g8 ^ (2 * t4)) << 4);
                const uint32_t x1 = (uint32_t)((g8 ^ (2 * t4 + 1)) << 4);
                vr[i][0] = lds128(at + x0);
                vr[i][1] = lds128(at + kB8Line + x1);
                vr[i][2] = lds128(at + 8 * kB8Line + x0);
                vr[i][3] = lds128(at + 9 * kB8Line + x1);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[slot]);

            // ---- S^T: 2 x [16 tokens x 8 heads]
            float raw[2][4];  // scores, log2
            float lg[2];      // log2 of the parts' V scales
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 lo = kr[i][h][0], hi = kr[i][h][1];
                    const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w};
                    const uint32_t wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t a[4] = {
                            e4m3x2_to_f16x2(wl[u], false), e4m3x2_to_f16x2(wh[u], false),
                            e4m3x2_to_f16x2(wl[u], true), e4m3x2_to_f16x2(wh[u], true)};
                        ElemOps<__half>::mma(c, a, qf[4 * h + u][0], qf[4 * h + u][1]);
                    }
                }
                const float ks = i == 0 ? scales.x : scales.y;
                const float vs = i == 0 ? scales.z : scales.w;
                // -inf for a block of zeros; that of a part behind the row's end may be
                // anything
                lg[i] = 16 * i < valid ? fast_log2(vs) : 0.f;
                const float f0 = qs[0] * ks, f1 = qs[1] * ks;
                if (ks == 0.f) c[0] = c[1] = c[2] = c[3] = 0.f;  // K = 0, whatever the codes
                const bool ok0 = 16 * i + g8 < valid, ok1 = 16 * i + g8 + 8 < valid;
                raw[i][0] = ok0 ? c[0] * f0 : -INFINITY;
                raw[i][1] = ok0 ? c[1] * f1 : -INFINITY;
                raw[i][2] = ok1 ? c[2] * f0 : -INFINITY;
                raw[i][3] = ok1 ? c[3] * f1 : -INFINITY;
            }
            // ---- running maxima (log2 domain) of heads 2 t4 and 2 t4 + 1: of the
            // contributions over the warp, of the scores for this lane's sum
            float top[2], largest[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float a = fmaxf(raw[0][h], raw[0][2 + h]);
                const float b = fmaxf(raw[1][h], raw[1][2 + h]);
                largest[h] = fmaxf(a, b);
                float mx = fmaxf(a + lg[0], b + lg[1]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                top[h] = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            }
            const bool move0 = top[0] - m_run[0] > kB8Lazy, move1 = top[1] - m_run[1] > kB8Lazy;
            const bool grow0 = largest[0] - m_sum[0] > kB8LazySum;
            const bool grow1 = largest[1] - m_sum[1] > kB8LazySum;
            if (__any_sync(0xffffffffu, move0 || move1 || grow0 || grow1)) {
                const float c0 = move0 ? fast_exp2(m_run[0] - top[0]) : 1.f;
                const float c1 = move1 ? fast_exp2(m_run[1] - top[1]) : 1.f;
                if (move0) m_run[0] = top[0];
                if (move1) m_run[1] = top[1];
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) {
                    acc[mt][0] *= c0;
                    acc[mt][1] *= c1;
                    acc[mt][2] *= c0;
                    acc[mt][3] *= c1;
                }
                if (grow0) {
                    l_run[0] *= fast_exp2(m_sum[0] - largest[0]);
                    m_sum[0] = largest[0];
                }
                if (grow1) {
                    l_run[1] *= fast_exp2(m_sum[1] - largest[1]);
                    m_sum[1] = largest[1];
                }
            }
            // ---- weights, and O^T[128 x 8 heads] += V^T . P^T
            const float b0 = m_run[0] == -INFINITY ? 0.f : m_run[0];
            const float b1 = m_run[1] == -INFINITY ? 0.f : m_run[1];
            const float r0 = m_sum[0] == -INFINITY ? 0.f : m_sum[0];
            const float r1 = m_sum[1] == -INFINITY ? 0.f : m_sum[1];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float pr[4];
                const float u0 = lg[i] - b0, u1 = lg[i] - b1;
                pr[0] = fast_exp2(raw[i][0] + u0);
                pr[1] = fast_exp2(raw[i][1] + u1);
                pr[2] = fast_exp2(raw[i][2] + u0);
                pr[3] = fast_exp2(raw[i][3] + u1);
                l_run[0] += fast_exp2(raw[i][0] - r0) + fast_exp2(raw[i][2] - r0);
                l_run[1] += fast_exp2(raw[i][1] - r1) + fast_exp2(raw[i][3] - r1);
                const uint32_t pb0 = movmatrix_trans(ElemOps<__half>::pack(pr[0], pr[1]));
                const uint32_t pb1 = movmatrix_trans(ElemOps<__half>::pack(pr[2], pr[3]));
                // chunk g8 holds the dims 16 g8 + 2 mt + (0, 1) of output tile mt's rows
                // g8 and g8 + 8
                const uint4 va = vr[i][0], vb = vr[i][1], vc = vr[i][2], vd = vr[i][3];
                const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
                const uint32_t wc[4] = {vc.x, vc.y, vc.z, vc.w}, wd[4] = {vd.x, vd.y, vd.z, vd.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        // bytes 2 o, 2 o + 1 of both tokens' words, interleaved
                        const uint32_t lo = __byte_perm(wa[u], wb[u], o == 0 ? 0x5140 : 0x7362);
                        const uint32_t hi = __byte_perm(wc[u], wd[u], o == 0 ? 0x5140 : 0x7362);
                        const uint32_t a[4] = {
                            e4m3x2_to_f16x2(lo, false), e4m3x2_to_f16x2(lo, true),
                            e4m3x2_to_f16x2(hi, false), e4m3x2_to_f16x2(hi, true)};
                        ElemOps<__half>::mma(acc[2 * u + o], a, pb0, pb1);
                    }
                }
            }
        }
        gbase += (uint32_t)n_stages;
        ground += (uint32_t)ceil_div_i(n_stages, kB8Round);

        // ---- combine the four warps' states of this item
        float* mbuf = s_merge + buf * DecodeSmem<G>::kMergeFloats;
        float* mstat = s_mstat + buf * kConsumerWarps * 8;
        float* lstat = s_lstat + buf * kConsumerWarps * 8;
        // one reference for the warp's sums and accumulators (a sum of NaN keeps
        // the reference -inf and stays)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float m = m_sum[h];
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            m = fmaxf(m, m_run[h] - kB8Headroom);
            if (m_sum[h] != -INFINITY) l_run[h] *= fast_exp2(m_sum[h] - m);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 4);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 8);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 16);
            const float f = m == -INFINITY ? 1.f : fast_exp2(m_run[h] - m);
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
                acc[mt][h] *= f;
                acc[mt][2 + h] *= f;
            }
            m_run[h] = m;
        }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int g = 2 * t4 + h;
                if (g < G)
                    *reinterpret_cast<float2*>(
                        mbuf + (warp * G + g) * DecodeSmem<G>::kMergeStride + 16 * g8 + 2 * mt) =
                        make_float2(acc[mt][h], acc[mt][2 + h]);
            }
        }
        if (lane < 4) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int g = 2 * lane + h;
                if (g < G) {
                    mstat[warp * 8 + g] = m_run[h];
                    lstat[warp * 8 + g] = l_run[h];
                }
            }
        }
        consumer_bar_sync();
        const bool direct = it.row_splits == 1;
#pragma unroll 1
        for (int idx = threadIdx.x; idx < G * kHeadDim; idx += kConsumerWarps * 32) {
            const int g = idx / kHeadDim;
            const int d = idx % kHeadDim;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kConsumerWarps; ++w) mx = fmaxf(mx, mstat[w * 8 + g]);
            float lsum = 0.f, osum = 0.f;
#pragma unroll
            for (int w = 0; w < kConsumerWarps; ++w) {
                const float mw = mstat[w * 8 + g];
                const float wt = mw == -INFINITY ? 0.f : fast_exp2(mw - mx);
                lsum = fmaf(wt, lstat[w * 8 + g], lsum);
                osum = fmaf(wt, mbuf[(w * G + g) * DecodeSmem<G>::kMergeStride + d], osum);
            }
            if (direct) {
                if (it.out_row >= 0 && !aborted) {
                    T* orow = reinterpret_cast<T*>(p.out) +
                              ((size_t)it.out_row * p.Hq + (size_t)it.kvh * G + g) * kHeadDim;
                    orow[d] = Ops::from_float(osum * (lsum == 0.f ? 0.f : 1.f / lsum));
                }
            } else if (it.slot >= 0) {
                const size_t si = ((size_t)it.kvh * p.total_slots + it.slot) * G + g;
                p.part_acc[si * kHeadDim + d] = osum;
                if (d == 0) {
                    p.part_m[si] = mx == -INFINITY ? kNegFltMax : mx * kLn2;
                    p.part_l[si] = lsum;
                }
            }
        }
        if (!direct && it.slot >= 0 && p.merge_counters != nullptr) {
            // fused merge, deferred to the CTA's end (a group holds at most two
            // split rows: its first and its last)
            int32_t* ctr = p.merge_counters + (size_t)it.row * p.Hkv + it.kvh;
            consumer_bar_sync();
            if (n_pend < kMaxPending) {
                if (threadIdx.x == 0) {
                    if (n_pend > 0) s_pend[n_pend - 1].old = pend_old;
                    PendingMerge& pe = s_pend[n_pend];
                    pe.row = it.row;
                    pe.kvh = it.kvh;
                    pe.s0 = it.slot - it.split;
                    pe.n = it.row_splits;
                    pe.out_row = it.out_row;
                    pend_old = atom_add_acq_rel_gpu(ctr, 1);
                }
                ++n_pend;
            } else if (threadIdx.x == 0) {
                raise_error(p.error, kErrSlot);
            }
        }
        buf ^= 1;
    }
    if (n_pend > 0) {
        if (threadIdx.x == 0) s_pend[n_pend - 1].old = pend_old;
        fence_proxy_async_smem();
        consumer_bar_sync();
#pragma unroll 1
        for (int k = 0; k < n_pend; ++k) {
            const PendingMerge pe = s_pend[k];
            if (pe.old != pe.n - 1) continue;
            if (threadIdx.x == 0) p.merge_counters[(size_t)pe.row * p.Hkv + pe.kvh] = 0;
            if (aborted || s_flags[0] != 0) continue;
            if (pe.n * G <= kMergeWeights) {
                merge_bulk<G, T>(p, pe, ring, (uint32_t)merge_region_bytes<G, NSLOTS>(), s_mw,
                                 merge_bar, merge_phase, s_flags);
            } else {
                // more slots than the weight buffer holds: the chunked merge
                MergeSmem ms{s_mw, s_mw + kMergeChunk * 8, s_merge};
                const size_t sb = ((size_t)pe.kvh * p.total_slots + pe.s0) * G;
                T* o = pe.out_row >= 0 ? reinterpret_cast<T*>(p.out) +
                                             ((size_t)pe.out_row * p.Hq + pe.kvh * G) * kHeadDim
                                       : nullptr;
                const XgSink unused{};
                merge_slots<G, T, kConsumerWarps, true, false>(
                    p.part_m + sb, p.part_l + sb, p.part_acc + sb * kHeadDim, 0, pe.n, G, 0, ms, o,
                    nullptr, unused);
                fence_proxy_async_smem();
                consumer_bar_sync();
            }
        }
    }
}

}  // namespace pkv
