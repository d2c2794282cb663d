// pkv_cache_kernels.cuh -- the prompt side of the paged cache: block tables
// and slot maps from request lengths, and the writes of packed K/V tokens
// into 16-bit pools and into e4m3 pools with one scale per block of tokens
// and head.  Included by pkv_prompt.cu only.
#pragma once

#include <climits>
#include <type_traits>

#include "pkv_device.cuh"

namespace pkv {

// ------------------------------------------------------------ prompt slots
struct SlotsParams {
    const int32_t* cached_lens;  // [B]
    const int32_t* new_lens;     // [B]
    int32_t* block_table;        // [B][max_pages]
    int32_t* slots;              // [num_slots]
    int32_t* cu_seqlens;         // [B + 1]
    int32_t* seq_lens;           // [B]
    const int32_t* free_pages;   // stack, or null (every page is already mapped)
    const int32_t* free_count;
    int32_t* free_left;          // may be free_count
    int32_t* counters;           // [1] zeroed; finished CTAs
    unsigned* error;
    int B, max_pages, page_size, num_slots, free_capacity;
};

constexpr int kSlotThreads = 256;
// 256 rows, 400k tokens: 8.5 us (with 1024: 7.8, 2048: 10.0); 8 rows, 3k tokens:
// 3.5 us (4.6, 6.9).
constexpr int kSlotTokensPerCta = 512;

// Exclusive prefix sums over the CTA of two non-negative values per thread, and
// their totals in `total`.  Sums stop at INT_MAX: lengths may hold anything, and
// a row behind so many tokens or pages is not served whatever their number.
__device__ __forceinline__ int2 slot_scan(int2 v, int2* s_warp, int2& total) {
    auto add = [](int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)INT_MAX); };
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    int2 x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int yx = __shfl_up_sync(0xffffffffu, x.x, off);
        const int yy = __shfl_up_sync(0xffffffffu, x.y, off);
        if (lane >= off) x = make_int2(add(x.x, yx), add(x.y, yy));
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int2 before = make_int2(0, 0);
    total = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < kSlotThreads / 32; ++w) {
        const int2 t = s_warp[w];
        if (w < warp) before = make_int2(add(before.x, t.x), add(before.y, t.y));
        total = make_int2(add(total.x, t.x), add(total.y, t.y));
    }
    __syncthreads();
    x.x = __shfl_up_sync(0xffffffffu, x.x, 1);
    x.y = __shfl_up_sync(0xffffffffu, x.y, 1);
    return lane > 0 ? make_int2(add(before.x, x.x), add(before.y, x.y)) : before;
}

// Everything a token's slot depends on is a prefix sum over the rows before
// its own: its first token, and the number of pages those rows take from the
// stack.  So each CTA scans all rows (256 at a time) and fills the slots of
// its own kSlotTokensPerCta tokens, and no CTA waits for another; the token's
// row comes from a binary search in the scanned prefixes.  New pages are read
// from the stack, never from block_table, where another CTA may still be
// writing them.  A thread finds the places of its tokens first, then loads
// their pages together.  Bound: the latency of the chain lengths -> pages ->
// slots, three trips to L2 (256 rows, 400k tokens: 8.5 us against 0.3 us for its
// bytes).
__global__ void __launch_bounds__(kSlotThreads)
    pkv_prompt_slots_kernel(const __grid_constant__ SlotsParams p) {
    __shared__ int2 s_warp[kSlotThreads / 32];
    __shared__ int s_start[kSlotThreads], s_cached[kSlotThreads], s_need[kSlotThreads];
    __shared__ int s_avail;
    constexpr int kMine = kSlotTokensPerCta / kSlotThreads;  // tokens of a thread
    const int t = threadIdx.x;
    const long long limit = (long long)p.max_pages * p.page_size;
    const bool stack = p.free_pages != nullptr;
    // A stack lowered in place: the CTA that counts last as having read it
    // writes what is left.  The count travels while the work is done.
    const bool in_place = stack && p.free_left == p.free_count;
    int counted = 0;
    if (stack && t == 0) {
        int n = *(const volatile int32_t*)p.free_count;
        if (in_place) counted = atom_add_acq_rel_gpu(p.counters, 1);
        if (n > p.free_capacity) {
            if (blockIdx.x == 0) raise_error(p.error, kErrIndex);
            n = p.free_capacity;
        }
        s_avail = max(n, 0);
    }
    const long long t0 = (long long)blockIdx.x * kSlotTokensPerCta;
    const long long t1 = min(t0 + kSlotTokensPerCta, (long long)p.num_slots);
    long long tokens = 0, pages = 0;  // of the rows before the current chunk
    int avail = 0, taken = 0;
    bool bad_len = false, no_page = false, bad_page = false, no_room = false;
    for (int base = 0; base < p.B; base += kSlotThreads) {
        const int b = base + t;
        int c = 0, n = 0, need = 0;
        bool valid = true;
        if (b < p.B) {
            c = __ldg(p.cached_lens + b);
            n = __ldg(p.new_lens + b);
            valid = c >= 0 && n >= 0 && (long long)c + n <= limit;
            if (n < 0) n = 0;
            if (!valid) bad_len = true;
            if (valid && stack)
                need = (c + n + p.page_size - 1) / p.page_size -
                       (c + p.page_size - 1) / p.page_size;
        }
        int2 total;
        const int2 pre = slot_scan(make_int2(n, need), s_warp, total);
        if (stack) avail = s_avail;  // (written before the scan's barriers)
        const long long start = tokens + pre.x;
        const long long before = pages + pre.y;
        const bool short_of = need > 0 && before + need > avail;
        const bool beyond = n > 0 && start + n > p.num_slots;
        const bool served = valid && !short_of && !beyond;
        if (short_of) no_page = true;
        if (beyond) no_room = true;
        if (served && need > 0) taken = max(taken, (int)(before + need));
        if (b < p.B && blockIdx.x == 0) {
            p.cu_seqlens[b] = (int)min(start, (long long)INT_MAX);
            p.seq_lens[b] = served ? c + n : max(c, 0);
        }
        // rows of this chunk for the token search; -1 marks a row not served
        s_start[t] = (int)min(start, (long long)INT_MAX);
        s_cached[t] = served ? c : -1;
        s_need[t] = (int)min(before, (long long)INT_MAX);
        __syncthreads();
        const long long end = tokens + total.x;
        const int rows = min(kSlotThreads, p.B - base);
        const long long lo = max(t0, tokens), hi = min(t1, end);
        // tokens t0 + t + 256 i of this chunk's rows
        const int32_t* from[kMine];  // where the page of the token stands
        int32_t* opened[kMine];      // block-table entry that the token opens
        int off[kMine];
        bool here[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const long long tok = t0 + t + i * kSlotThreads;
            here[i] = tok >= lo && tok < hi;
            from[i] = nullptr;
            opened[i] = nullptr;
            off[i] = 0;
            if (here[i]) {
                // the last row that starts at or before tok (rows of no tokens
                // that start there come before it)
                int a = 0, z = rows;
                while (z - a > 1) {
                    const int m = (a + z) >> 1;
                    if ((long long)s_start[m] <= tok) a = m; else z = m;
                }
                const int cached = s_cached[a];
                if (cached >= 0) {
                    const int pos = cached + (int)(tok - s_start[a]);
                    const int j = pos / p.page_size;
                    off[i] = pos - j * p.page_size;
                    int32_t* entry = p.block_table + (size_t)(base + a) * p.max_pages + j;
                    const int first = (cached + p.page_size - 1) / p.page_size;
                    if (stack && j >= first) {
                        from[i] = p.free_pages + (avail - 1 - s_need[a] - (j - first));
                        if (off[i] == 0) opened[i] = entry;
                    } else {
                        from[i] = entry;
                    }
                }
            }
        }
        int page[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            page[i] = from[i] != nullptr ? *(const volatile int32_t*)from[i] : 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            if (!here[i]) continue;
            int slot = -1;
            if (from[i] != nullptr) {
                if (opened[i] != nullptr) *opened[i] = page[i];
                if (page[i] < 0 || page[i] > (INT_MAX - p.page_size) / p.page_size)
                    bad_page = true;
                else
                    slot = page[i] * p.page_size + off[i];
            }
            p.slots[t0 + t + i * kSlotThreads] = slot;
        }
        tokens = end;
        pages += total.y;
        __syncthreads();
    }
    for (long long tok = max(t0, tokens) + t; tok < t1; tok += kSlotThreads) p.slots[tok] = -1;
    if (bad_page) raise_error(p.error, kErrPageId);
    if (blockIdx.x == 0) {
        if (bad_len) raise_error(p.error, kErrLogicalPage);
        if (no_page) raise_error(p.error, kErrNoPage);
        if (no_room) raise_error(p.error, kErrSlot);
        if (t == 0) p.cu_seqlens[p.B] = (int)min(tokens, (long long)INT_MAX);
    }
    if (stack && (in_place || blockIdx.x == 0)) {
        taken = __reduce_max_sync(0xffffffffu, taken);
        if ((t & 31) == 0) s_start[t >> 5] = taken;
        __syncthreads();
        if (t == 0 && (!in_place || counted == (int)gridDim.x - 1)) {
#pragma unroll
            for (int w = 1; w < kSlotThreads / 32; ++w) taken = max(taken, s_start[w]);
            if (in_place) *p.counters = 0;
            *p.free_left = s_avail - taken;
        }
    }
}

// ------------------------------------------------------------ 16-bit write
struct WriteParams {
    const uint8_t* k;  // [T][Hkv][128] 16-bit elements, token / head strides in bytes
    const uint8_t* v;
    uint8_t* k_pages;  // [P][Hkv][page][128], 16-bit or e4m3
    uint8_t* v_pages;
    float* k_scales;   // [P][Hkv][page / block] (e4m3 pools)
    float* v_scales;
    const int32_t* slots;  // [T]
    unsigned* error;
    long long k_tok, k_head, v_tok, v_head;
    long long num_slots;  // P * page
    int T, Hkv, page_size, block;
    int split_log2;  // warps that share a window of tokens (e4m3 write)
};

constexpr int kWriteThreads = 128;

// One thread moves one 16-byte piece of a token's K and the same piece of its
// V.  A copy: HBM-bound for long prompts (22.8k tokens of 8 heads, 187 MB: 31 us,
// 6.0 TB/s), launch latency for short ones (37 tokens: 1.6 us).
__global__ void __launch_bounds__(kWriteThreads)
    pkv_kv_write_kernel(const __grid_constant__ WriteParams p) {
    constexpr int kPieces = kRowBytes / 16;
    const int per_token = p.Hkv * kPieces;
    const long long i = (long long)blockIdx.x * kWriteThreads + threadIdx.x;
    const long long t = i / per_token;
    if (t >= p.T) return;
    const int r = (int)(i - t * per_token);
    const int h = r / kPieces, piece = r % kPieces;
    const int slot = __ldg(p.slots + t);
    if (slot < 0) return;  // padding
    if (slot >= p.num_slots) {
        if (r == 0) raise_error(p.error, kErrSlot);
        return;
    }
    const uint4 kv = __ldg(reinterpret_cast<const uint4*>(p.k + t * p.k_tok + h * p.k_head) + piece);
    const uint4 vv = __ldg(reinterpret_cast<const uint4*>(p.v + t * p.v_tok + h * p.v_head) + piece);
    const int page = slot / p.page_size;
    const size_t row = ((size_t)page * p.Hkv + h) * p.page_size + (slot - page * p.page_size);
    reinterpret_cast<uint4*>(p.k_pages + row * kRowBytes)[piece] = kv;
    reinterpret_cast<uint4*>(p.v_pages + row * kRowBytes)[piece] = vv;
}

// ------------------------------------------------------------ e4m3 block write
// The tokens of a call that fall into one block of the cache (`block` slots of
// one page) are a run of consecutive tokens.  A warp takes a run of one head's
// K or V: the block's scale is the least power of two, at least 2^-24,
// that brings the run's largest magnitude to e4m3's 448 or below, and, when
// the run starts inside the block, at least the block's old scale, whose
// earlier tokens stay.  A power of two makes x / scale and the move of old
// codes to a larger scale exact up to e4m3's own rounding, and costs no
// precision: e4m3 is a floating format, so a scale within a factor of two of
// the tightest one keeps the same 3 mantissa bits.
constexpr int kScaleExpMin = -24;

__device__ __forceinline__ float block_scale(float amax) {
    const unsigned bits = __float_as_uint(amax);
    // amax = 1.f * 2^(E - 127); 448 = 1.75 * 2^8
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    if (e < kScaleExpMin) e = kScaleExpMin;
    return __uint_as_float((unsigned)(e + 127) << 23);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// Four 16-bit values times a factor as e4m3 codes.
template <typename T>
__device__ __forceinline__ uint32_t e4m3x4(uint32_t lo, uint32_t hi, uint64_t factor2) {
    const float2 a = to_float2<T>(lo), b = to_float2<T>(hi);
    float ax, ay, bx, by;
    unpack_f32x2(mul_f32x2(pack_f32x2(a.x, a.y), factor2), ax, ay);
    unpack_f32x2(mul_f32x2(pack_f32x2(b.x, b.y), factor2), bx, by);
    return __byte_perm(e4m3x2(ax, ay), e4m3x2(bx, by), 0x5410);
}

// Two e4m3 codes times a power of two, rounded back to e4m3.
__device__ __forceinline__ uint32_t rescale_e4m3x2(uint32_t codes, float ratio) {
    const __half2_raw h =
        __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return e4m3x2(f.x * ratio, f.y * ratio);
}

constexpr int kRunRows = 16;  // tokens held in registers at a time

// A window of 16 tokens of one head's K or V belongs to 2^split_log2 warps: the
// runs that start in it go to them in turn.  Long prompts start about one run
// per window (one warp); the new tokens of a decode step are a run each, and
// one warp would take them one after another (64 rows: 27.9 us; with a warp
// each 4.7 us).  Lane l holds 16 bytes (8 elements) of tokens l / 16 + 2 i: 8 loads
// in flight, 4 KB a warp, 28 warps an SM (72 registers, 104 bytes of a thread spilled;
// at 24 or 32 warps it took 39 and 32 us where this takes 30).  Bound: issue slots,
// the spills and a shuffle per row for its slot among them, and HBM for long
// prompts (2 bytes read, 1 written per element; 23k tokens of 8 heads, 143 MB:
// 30.0 us, 4.75 TB/s), the chain slots -> tokens -> codes for short ones.
template <typename T>
__global__ void __launch_bounds__(kWriteThreads, 7)
    pkv_kv_write_block_kernel(const __grid_constant__ WriteParams p) {
    const int lane = threadIdx.x & 31;
    const long long t0 = (long long)blockIdx.x * kRunRows;
    const int role = blockIdx.y * (kWriteThreads / 32) + (threadIdx.x >> 5);
    if (role >= (2 * p.Hkv) << p.split_log2) return;
    const int split = 1 << p.split_log2;
    const int sub = role & (split - 1);
    const int r = role >> p.split_log2;
    const int h = r >> 1;
    const bool is_v = (r & 1) != 0;
    const uint8_t* src = is_v ? p.v + h * p.v_head : p.k + h * p.k_head;
    const long long tok_stride = is_v ? p.v_tok : p.k_tok;
    uint8_t* pool = is_v ? p.v_pages : p.k_pages;
    float* scales = is_v ? p.v_scales : p.k_scales;
    const int nblk = p.page_size / p.block;
    // slots and blocks of the tokens t0 - 1 .. t0 + 30; block -1 is padding
    auto slot_of = [&](long long t) -> int {
        return t >= 0 && t < p.T ? __ldg(p.slots + t) : -1;
    };
    auto block_of = [&](int slot) -> int {
        return slot >= 0 && slot < p.num_slots ? slot / p.block : -1;
    };
    if (lane >= 1 && lane <= kRunRows && t0 + lane - 1 < p.T) {
        // the window's tokens come to L2 while their slots are looked up
        const uint8_t* row = src + (t0 + lane - 1) * tok_stride;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(row));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(row + 128));
    }
    const int slot = slot_of(t0 + lane - 1);
    if (slot >= p.num_slots && r == 0) raise_error(p.error, kErrSlot);
    const int blk = block_of(slot);
    const int prev = __shfl_up_sync(0xffffffffu, blk, 1);
    unsigned starts = __ballot_sync(0xffffffffu, lane >= 1 && lane <= kRunRows && blk >= 0 &&
                                                     blk != prev);
    const int half = lane >> 4, piece = lane & 15;
    for (int turn = 0; starts != 0u; ++turn) {
        const int sl = __ffs(starts) - 1;
        starts &= starts - 1;
        if ((turn & (split - 1)) != sub) continue;
        const int run_blk = __shfl_sync(0xffffffffu, blk, sl);
        const int kept = __shfl_sync(0xffffffffu, slot, sl) - run_blk * p.block;
        const long long first = t0 + sl - 1;
        // length of the run: the tokens in hand hold any run of 16, longer ones
        // are followed
        int n = __ffs(~(__ballot_sync(0xffffffffu, blk == run_blk) >> sl)) - 1;
        if (n < 0 || n > 32 - sl) n = 32 - sl;
        if (n == 32 - sl && p.block > kRunRows) {
            while (true) {
                const unsigned same = __ballot_sync(
                    0xffffffffu, block_of(slot_of(first + n + lane)) == run_blk);
                const int more = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
                n += more;
                if (more < 32) break;
            }
        }
        const int page = run_blk / nblk, g = run_blk % nblk;
        float* scale_at = scales + ((size_t)page * p.Hkv + h) * nblk + g;
        uint8_t* block_base =
            pool + (((size_t)page * p.Hkv + h) * p.page_size + (size_t)g * p.block) * kHeadDim;
        float old = 0.f;
        if (kept > 0) old = *scale_at;
        uint4 x[kRunRows / 2];
        const uint8_t* from = src + (first + half) * tok_stride + 16 * piece;
        auto load = [&](int base) {
            const uint8_t* at = from + base * tok_stride;
#pragma unroll
            for (int i = 0; i < kRunRows / 2; ++i) {
                x[i] = base + half + 2 * i < n ? __ldg(reinterpret_cast<const uint4*>(at))
                                               : make_uint4(0u, 0u, 0u, 0u);
                at += 2 * tok_stride;
            }
        };
        // the largest magnitude, two elements at a time on their bits
        unsigned top2 = 0u;
        for (int base = 0; base < n; base += kRunRows) {
            load(base);
#pragma unroll
            for (int i = 0; i < kRunRows / 2; ++i) {
                top2 = __vmaxu2(top2, x[i].x & 0x7fff7fffu);
                top2 = __vmaxu2(top2, x[i].y & 0x7fff7fffu);
                top2 = __vmaxu2(top2, x[i].z & 0x7fff7fffu);
                top2 = __vmaxu2(top2, x[i].w & 0x7fff7fffu);
            }
        }
        unsigned top = __reduce_max_sync(0xffffffffu, max(top2 & 0xffffu, top2 >> 16));
        if (top >= kInf16<T>) {
            // infinities and NaN do not set a scale: again without them
            top = 0u;
            for (int row = half; row < n; row += 2) {
                const uint4 y = __ldg(reinterpret_cast<const uint4*>(from + (row - half) * tok_stride));
                const unsigned u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned lo = u[j] & 0x7fffu, hi = (u[j] >> 16) & 0x7fffu;
                    if (lo < kInf16<T>) top = max(top, lo);
                    if (hi < kInf16<T>) top = max(top, hi);
                }
            }
            __syncwarp();
            top = __reduce_max_sync(0xffffffffu, top);
        }
        float scale = block_scale(from_bits16<T>(top));
        if (kept > 0) {
            if (old > scale) {
                scale = old;
            } else if (old < scale) {
                // the earlier tokens move to the larger scale
                const float ratio = old / scale;
                for (int o = half; o < kept; o += 2) {
                    uint2* at = reinterpret_cast<uint2*>(block_base + (size_t)o * kHeadDim) + piece;
                    // (codes under a scale of 0 are zeros, whatever they hold)
                    uint2 c = old == 0.f ? make_uint2(0u, 0u) : *at;
                    c.x = rescale_e4m3x2(c.x, ratio) | (rescale_e4m3x2(c.x >> 16, ratio) << 16);
                    c.y = rescale_e4m3x2(c.y, ratio) | (rescale_e4m3x2(c.y >> 16, ratio) << 16);
                    *at = c;
                }
            }
        }
        __syncwarp();
        if (lane == 0) *scale_at = scale;
        // 1 / scale: exact for a power of two (an old scale may be any value)
        const uint64_t inv2 = pack_f32x2(1.0f / scale, 1.0f / scale);
        for (int base = 0; base < n; base += kRunRows) {
            if (n > kRunRows) load(base);
#pragma unroll
            for (int i = 0; i < kRunRows / 2; ++i) {
                const int row = base + half + 2 * i;
                const int near = __shfl_sync(0xffffffffu, slot, (sl + row) & 31);
                if (row >= n) continue;
                const int to = sl + row < 32 ? near : __ldg(p.slots + first + row);
                const uint2 out = make_uint2(e4m3x4<T>(x[i].x, x[i].y, inv2),
                                             e4m3x4<T>(x[i].z, x[i].w, inv2));
                *reinterpret_cast<uint2*>(block_base + (to - run_blk * p.block) * kHeadDim +
                                          8 * piece) = out;
            }
        }
    }
}

}  // namespace pkv
