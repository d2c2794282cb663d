// pkv_prompt.cu -- C ABI of the prompt side (declared in include/pkv_b200.h):
// block tables and slot maps, K/V writes by slot, attention of packed prompts.
// No counterpart in the reference, which decodes over pre-filled pools.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "../../include/pkv_b200.h"
#include "pkv_cache_kernels.cuh"
#include "pkv_internal.h"
#include "pkv_prompt_mma.cuh"

using namespace pkv;
using pkv_internal::device_state;
using pkv_internal::fail_fmt;
using pkv_internal::ok;

namespace {

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

pkv_status launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
        return fail_fmt(PKV_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return ok();
}

// Strides (in elements) of a [T][H][128] operand: 16-byte rows, forward.  The
// stride of a dimension of one entry means nothing and becomes a dense one.
pkv_status check_strides(const char* name, int T, int H, long long* tok, long long* head) {
    if (H <= 1) *head = kHeadDim;
    if (T <= 1) *tok = *head * H;
    if (*tok <= 0 || *head <= 0 || *tok % 8 != 0 || *head % 8 != 0)
        return fail_fmt(PKV_ERR_MISALIGNED, "%s strides must be positive multiples of 8 elements",
                        name);
    return PKV_OK;
}

// Key blocks that a CTA of a split item gets at the least (prompt attention).  A
// join costs about 8 us, a block 2: 16 queries over 8016 keys (32 heads) take
// 114 us in one CTA per item and 51 in eight, 256 over 256 keys 11 and, in two, 21.
constexpr int kPmSplitBlocks = 4;

// Shared checks of the two writes; fills everything but the scales.
pkv_status write_params(WriteParams& wp, const void* k, const void* v, void* k_pages,
                        void* v_pages, const int32_t* slots, int T, int Hkv, int head_dim,
                        long long k_stride, long long k_head_stride, long long v_stride,
                        long long v_head_stride, int physical_pages, int page_size,
                        pkv_dtype dtype) {
    // (tensors of no tokens have no address)
    if (T > 0 && (k == nullptr || v == nullptr))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "k and v must be CUDA tensors");
    if (k_pages == nullptr || v_pages == nullptr)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "k_pages and v_pages must be CUDA tensors");
    if (T > 0 && slots == nullptr)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "slots must be a CUDA tensor");
    if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
        return fail_fmt(PKV_ERR_UNSUPPORTED, "k has wrong dtype");
    if (head_dim != kHeadDim)
        return fail_fmt(PKV_ERR_UNSUPPORTED, "PersistentKV extension currently requires d=128");
    if (T < 0 || Hkv <= 0 || physical_pages <= 0 || page_size <= 0)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "invalid write shape");
    if ((long long)physical_pages * page_size >= (1ll << 31))
        return fail_fmt(PKV_ERR_UNSUPPORTED, "the pool holds %lld slots, beyond 32-bit slots",
                        (long long)physical_pages * page_size);
    pkv_status st = check_strides("k", T, Hkv, &k_stride, &k_head_stride);
    if (st == PKV_OK) st = check_strides("v", T, Hkv, &v_stride, &v_head_stride);
    if (st != PKV_OK) return st;
    if (misaligned(k) || misaligned(v) || misaligned(k_pages) || misaligned(v_pages))
        return fail_fmt(PKV_ERR_MISALIGNED, "k, v and the pools must be 16-byte aligned");
    wp.k = static_cast<const uint8_t*>(k);
    wp.v = static_cast<const uint8_t*>(v);
    wp.k_pages = static_cast<uint8_t*>(k_pages);
    wp.v_pages = static_cast<uint8_t*>(v_pages);
    wp.k_scales = wp.v_scales = nullptr;
    wp.slots = slots;
    wp.error = nullptr;
    wp.k_tok = 2 * k_stride;
    wp.k_head = 2 * k_head_stride;
    wp.v_tok = 2 * v_stride;
    wp.v_head = 2 * v_head_stride;
    wp.num_slots = (long long)physical_pages * page_size;
    wp.T = T;
    wp.Hkv = Hkv;
    wp.page_size = page_size;
    wp.block = page_size;
    wp.split_log2 = 0;
    return PKV_OK;
}

// The bytes of a [T][H][128] 16-bit operand, from its first element to its last.
struct Range {
    const char* begin;
    long long bytes;
};
Range operand_range(const void* base, int T, int H, long long tok_bytes, long long head_bytes) {
    return {static_cast<const char*>(base),
            T > 0 ? (T - 1) * tok_bytes + (H - 1) * head_bytes + kRowBytes : 0};
}
bool overlap(const Range& a, const Range& b) {
    return a.bytes > 0 && b.bytes > 0 && a.begin < b.begin + b.bytes && b.begin < a.begin + a.bytes;
}

// K and V go to pools of their own, apart from the tokens that are read.
pkv_status check_apart(const WriteParams& wp, int physical_pages, int elem_bytes) {
    if (wp.T == 0) return PKV_OK;
    const long long pool = (long long)physical_pages * wp.Hkv * wp.page_size * kHeadDim * elem_bytes;
    const Range kp{reinterpret_cast<const char*>(wp.k_pages), pool};
    const Range vp{reinterpret_cast<const char*>(wp.v_pages), pool};
    const Range k = operand_range(wp.k, wp.T, wp.Hkv, wp.k_tok, wp.k_head);
    const Range v = operand_range(wp.v, wp.T, wp.Hkv, wp.v_tok, wp.v_head);
    if (overlap(kp, vp) || overlap(kp, k) || overlap(kp, v) || overlap(vp, k) || overlap(vp, v))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT,
                        "k_pages, v_pages and the tokens written must not overlap");
    return PKV_OK;
}

pkv_status grid_of(long long threads, int per_cta, unsigned* grid) {
    const long long n = (threads + per_cta - 1) / per_cta;
    if (n > INT_MAX) return fail_fmt(PKV_ERR_UNSUPPORTED, "too many tokens for one launch");
    *grid = (unsigned)n;
    return PKV_OK;
}

// The checks that only the 16-bit write makes; gives the grid.
pkv_status copy_params(const WriteParams& wp, int physical_pages, unsigned* grid) {
    const pkv_status st = check_apart(wp, physical_pages, 2);
    if (st != PKV_OK) return st;
    return grid_of((long long)wp.T * wp.Hkv * (kRowBytes / 16), kWriteThreads, grid);
}

// Rows of the e4m3 write's grid: its warps are (head, K or V, share of a window).
long long block_rows(int Hkv, int split_log2) {
    return (((2ll * Hkv) << split_log2) + kWriteThreads / 32 - 1) / (kWriteThreads / 32);
}

// The checks that only the e4m3 write makes; fills the scales.
pkv_status block_params(WriteParams& wp, float* k_scales, float* v_scales, int physical_pages,
                        int block_tokens) {
    if (k_scales == nullptr || v_scales == nullptr)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "k_scales and v_scales must be CUDA tensors");
    if (block_tokens <= 0 || block_tokens % 16 != 0 || wp.page_size % block_tokens != 0)
        return fail_fmt(PKV_ERR_UNSUPPORTED,
                        "a scale block must be a multiple of 16 tokens that divides the page; "
                        "got %d tokens in pages of %d",
                        block_tokens, wp.page_size);
    // (a window is shared only while the whole grid is a few thousand warps)
    if (block_rows(wp.Hkv, 0) > 65535)
        return fail_fmt(PKV_ERR_UNSUPPORTED, "too many heads for one launch");
    wp.k_scales = k_scales;
    wp.v_scales = v_scales;
    wp.block = block_tokens;
    if (wp.T == 0) return PKV_OK;
    const pkv_status st = check_apart(wp, physical_pages, 1);
    if (st != PKV_OK) return st;
    const long long pool = (long long)physical_pages * wp.Hkv * wp.page_size * kHeadDim;
    const Range scales[2] = {
        {reinterpret_cast<const char*>(k_scales), pool / kHeadDim / block_tokens * 4},
        {reinterpret_cast<const char*>(v_scales), pool / kHeadDim / block_tokens * 4}};
    if (overlap(scales[0], scales[1]))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "k_scales and v_scales must not overlap");
    for (const Range& sc : scales)
        if (overlap(sc, {reinterpret_cast<const char*>(wp.k_pages), pool}) ||
            overlap(sc, {reinterpret_cast<const char*>(wp.v_pages), pool}) ||
            overlap(sc, operand_range(wp.k, wp.T, wp.Hkv, wp.k_tok, wp.k_head)) ||
            overlap(sc, operand_range(wp.v, wp.T, wp.Hkv, wp.v_tok, wp.v_head)))
            return fail_fmt(PKV_ERR_INVALID_ARGUMENT,
                            "the scales must not overlap the pools or the tokens written");
    return PKV_OK;
}

// The operand [T][H][128] as a 3-D tensor (element, head, token); one box is 64
// elements (one 128-byte line) of 128 tokens of one head.
pkv_status token_map(CUtensorMap* map, const void* base, int T, int H, long long tok_bytes,
                     long long head_bytes, pkv_dtype dtype) {
    const cuuint64_t dims[3] = {(cuuint64_t)kHeadDim, (cuuint64_t)H, (cuuint64_t)T};
    const cuuint64_t strides[2] = {(cuuint64_t)head_bytes, (cuuint64_t)tok_bytes};
    const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)kPmTile};
    const cuuint32_t elem[3] = {1u, 1u, 1u};
    const pkv_internal::EncodeTiledFn fn = pkv_internal::encode_tiled();
    if (fn == nullptr) return fail_fmt(PKV_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const CUresult r = fn(map,
                          dtype == PKV_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          3, const_cast<void*>(base), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail_fmt(PKV_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return PKV_OK;
}

// Items of the launch: one per pair of query tiles and KV head's pair of heads.
long long prompt_items(const PromptParams& pp) {
    const int rows = pp.G == 1 ? 2 * kPmTile : kPmTile;
    // every sequence has at most one tile that is not full
    const long long tiles = std::min<long long>((long long)pp.Tq / rows + pp.B, pp.Tq);
    return tiles * (pp.G == 1 ? pp.Hq : pp.Hq / 2);
}

// Shared checks of prompt attention; fills everything but the error word.  A
// call without rows or sequences (nothing to launch) may lack any operand.
pkv_status prompt_params(PromptParams& pp, const void* q, const void* k, const void* v,
                         const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, void* output,
                         float* lse, int B, int q_tokens, int k_tokens, int Hq, int Hkv,
                         int head_dim, long long q_stride, long long q_head_stride,
                         long long k_stride, long long k_head_stride, long long v_stride,
                         long long v_head_stride, pkv_dtype dtype) {
    if (q_tokens > 0 && (q == nullptr || output == nullptr))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "q and output must be CUDA tensors");
    if (k_tokens > 0 && (k == nullptr || v == nullptr))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "k and v must be CUDA tensors");
    if (cu_seqlens_q == nullptr)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "cu_seqlens_q must be a CUDA tensor");
    if (cu_seqlens_k == nullptr) cu_seqlens_k = cu_seqlens_q;
    if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
        return fail_fmt(PKV_ERR_UNSUPPORTED, "q has wrong dtype");
    if (head_dim != kHeadDim)
        return fail_fmt(PKV_ERR_UNSUPPORTED, "PersistentKV extension currently requires d=128");
    if (Hkv <= 0) return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "Hkv must be positive");
    if (Hq <= 0 || Hq % Hkv != 0)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "Hq must be divisible by Hkv");
    const int G = Hq / Hkv;
    if (!(G == 1 || G == 2 || G == 4 || G == 8))
        return fail_fmt(PKV_ERR_UNSUPPORTED,
                        "PersistentKV supports G=Hq/Hkv in {1,2,4,8}; got G=%d from Hq=%d Hkv=%d",
                        G, Hq, Hkv);
    if (B < 0 || q_tokens < 0 || k_tokens < 0)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "invalid prompt shape");
    pkv_status st = check_strides("q", q_tokens, Hq, &q_stride, &q_head_stride);
    if (st == PKV_OK) st = check_strides("k", k_tokens, Hkv, &k_stride, &k_head_stride);
    if (st == PKV_OK) st = check_strides("v", k_tokens, Hkv, &v_stride, &v_head_stride);
    if (st != PKV_OK) return st;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(output))
        return fail_fmt(PKV_ERR_MISALIGNED, "q, k, v and output must be 16-byte aligned");
    if (B == 0 || q_tokens == 0) return PKV_OK;
    pp.q = static_cast<const uint8_t*>(q);
    pp.k = static_cast<const uint8_t*>(k);
    pp.v = static_cast<const uint8_t*>(v);
    pp.cu_q = cu_seqlens_q;
    pp.cu_k = cu_seqlens_k;
    pp.out = output;
    pp.lse = lse;
    pp.q_tok = 2 * q_stride;
    pp.q_head = 2 * q_head_stride;
    pp.k_tok = 2 * k_stride;
    pp.k_head = 2 * k_head_stride;
    pp.v_tok = 2 * v_stride;
    pp.v_head = 2 * v_head_stride;
    pp.B = B;
    pp.Tq = q_tokens;
    pp.Tk = k_tokens;
    pp.Hq = Hq;
    pp.Hkv = Hkv;
    pp.G = G;
    pp.scale_log2 = (1.0f / sqrtf((float)kHeadDim)) * kLog2e;
    const Range o = operand_range(output, q_tokens, Hq, (long long)Hq * kRowBytes, kRowBytes);
    if (overlap(o, operand_range(q, q_tokens, Hq, pp.q_tok, pp.q_head)) ||
        overlap(o, operand_range(k, k_tokens, Hkv, pp.k_tok, pp.k_head)) ||
        overlap(o, operand_range(v, k_tokens, Hkv, pp.v_tok, pp.v_head)))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "output must not overlap q, k or v");
    const Range l{reinterpret_cast<const char*>(lse), lse ? (long long)q_tokens * Hq * 4 : 0};
    if (overlap(l, o) || overlap(l, operand_range(q, q_tokens, Hq, pp.q_tok, pp.q_head)) ||
        overlap(l, operand_range(k, k_tokens, Hkv, pp.k_tok, pp.k_head)) ||
        overlap(l, operand_range(v, k_tokens, Hkv, pp.v_tok, pp.v_head)))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "lse must not overlap output, q, k or v");
    if (prompt_items(pp) > INT_MAX)
        return fail_fmt(PKV_ERR_UNSUPPORTED, "too many tokens for one launch");
    return PKV_OK;
}

// Shared-memory limit of a kernel, once per device.
template <typename K>
pkv_status set_smem(K kern, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(
            kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPmSmemBytes);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return fail_fmt(PKV_ERR_CUDA, "cudaFuncSetAttribute failed: %s",
                            cudaGetErrorString(e));
        }
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    return PKV_OK;
}

template <typename T>
pkv_status launch_prompt(const PromptParams& pp, pkv_dtype dtype, int sms, cudaStream_t stream) {
    CUtensorMap mq, mk, mv;
    pkv_status st = token_map(&mq, pp.q, pp.Tq, pp.Hq, pp.q_tok, pp.q_head, dtype);
    // without keys no block is ever loaded: any valid map does
    if (st == PKV_OK)
        st = pp.Tk > 0 ? token_map(&mk, pp.k, pp.Tk, pp.Hkv, pp.k_tok, pp.k_head, dtype)
                       : token_map(&mk, pp.q, pp.Tq, pp.Hq, pp.q_tok, pp.q_head, dtype);
    if (st == PKV_OK)
        st = pp.Tk > 0 ? token_map(&mv, pp.v, pp.Tk, pp.Hkv, pp.v_tok, pp.v_head, dtype)
                       : token_map(&mv, pp.q, pp.Tq, pp.Hq, pp.q_tok, pp.q_head, dtype);
    if (st != PKV_OK) return st;
    const long long items = prompt_items(pp);
    // A cluster per item where that still leaves SMs free and each CTA gets
    // at least kPmSplitBlocks key blocks of an average sequence.
    int split = 1;
    while (split < 8 && items * split * 2 <= sms &&
           (long long)pp.Tk / pp.B >= (long long)kPmTile * kPmSplitBlocks * split * 2)
        split *= 2;
    const unsigned grid = (unsigned)(items * split);
    if (split == 1) {
        static std::atomic<unsigned long long> done{0ull};
        auto kern = pkv_prompt_mma_kernel<T, false>;
        st = set_smem(kern, done);
        if (st != PKV_OK) return st;
        kern<<<grid, kPmThreads, kPmSmemBytes, stream>>>(pp, mq, mk, mv);
        return launched("prompt attention");
    }
    static std::atomic<unsigned long long> done{0ull};
    auto kern = pkv_prompt_mma_kernel<T, true>;
    st = set_smem(kern, done);
    if (st != PKV_OK) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kPmThreads);
    cfg.dynamicSmemBytes = kPmSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, pp, mq, mk, mv);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail_fmt(PKV_ERR_CUDA, "prompt attention launch failed: %s", cudaGetErrorString(e));
    }
    return ok();
}

}  // namespace

extern "C" {

pkv_status pkv_prompt_slots(const int32_t* cached_lens, const int32_t* new_lens,
                            int32_t* block_table, int32_t* slots, int32_t* cu_seqlens,
                            int32_t* seq_lens, const int32_t* free_pages,
                            const int32_t* free_count, int32_t* free_left, int32_t* counters,
                            int B, int max_pages, int page_size, int num_slots,
                            int free_capacity, void* stream) {
    if (B > 0 && (cached_lens == nullptr || new_lens == nullptr))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "cached_lens and new_lens must be CUDA tensors");
    if (cu_seqlens == nullptr || (B > 0 && (block_table == nullptr || seq_lens == nullptr)))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT,
                        "block_table, cu_seqlens and seq_lens must be CUDA tensors");
    if (slots == nullptr && num_slots > 0)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "slots must be a CUDA tensor");
    if (free_pages != nullptr &&
        (free_count == nullptr || free_left == nullptr || counters == nullptr))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT,
                        "a free-page list needs free_count, free_left and zeroed counters");
    if (B > 0 && (seq_lens == cached_lens || seq_lens == new_lens || cu_seqlens == cached_lens ||
                  cu_seqlens == new_lens))
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT,
                        "seq_lens and cu_seqlens must not be the tensors they are made from");
    if (B < 0 || max_pages <= 0 || page_size <= 0 || num_slots < 0 || free_capacity < 0)
        return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "invalid slot map shape");
    // (a length rounded up to pages fits into 32 bits too)
    if (((long long)max_pages + 1) * page_size > (1ll << 31))
        return fail_fmt(PKV_ERR_UNSUPPORTED, "max_pages * page_size exceeds 32-bit positions");
    auto words = [](const int32_t* p, long long n) -> Range {
        return {reinterpret_cast<const char*>(p), p != nullptr ? 4 * n : 0};
    };
    const bool stack = free_pages != nullptr;
    const bool in_place = stack && free_left == free_count;
    // what is written, the first stack ? 6 : 3 of them, then what is only read
    const Range used[] = {words(slots, num_slots),
                          words(cu_seqlens, B + 1ll),
                          words(seq_lens, B),
                          words(block_table, (long long)B * max_pages),
                          words(free_left, stack ? 1 : 0),
                          words(counters, stack ? 1 : 0),
                          words(cached_lens, B),
                          words(new_lens, B),
                          words(free_pages, free_capacity),
                          words(free_count, stack && !in_place ? 1 : 0)};
    constexpr int kUsed = sizeof(used) / sizeof(used[0]);
    for (int i = 0; i < (stack ? 6 : 3); ++i)
        for (int j = i + 1; j < kUsed; ++j)
            if (overlap(used[i], used[j]))
                return fail_fmt(PKV_ERR_INVALID_ARGUMENT,
                                "the buffers that a slot map writes must not overlap each other or "
                                "those it reads");
    int sms = 0;
    unsigned* error = nullptr;
    pkv_status st = device_state(&sms, &error);
    if (st != PKV_OK) return st;
    const SlotsParams sp{cached_lens, new_lens,  block_table, slots,     cu_seqlens,
                         seq_lens,    free_pages, free_count, free_left, counters,
                         error,       B,          max_pages,  page_size, num_slots,
                         free_capacity};
    const int grid = num_slots > 0 ? (int)(((long long)num_slots + kSlotTokensPerCta - 1) /
                                           kSlotTokensPerCta)
                                   : 1;
    pkv_prompt_slots_kernel<<<grid, kSlotThreads, 0, static_cast<cudaStream_t>(stream)>>>(sp);
    return launched("slot map");
}

pkv_status pkv_kv_write(const void* k, const void* v, void* k_pages, void* v_pages,
                        const int32_t* slots, int T, int Hkv, int head_dim, long long k_stride,
                        long long k_head_stride, long long v_stride, long long v_head_stride,
                        int physical_pages, int page_size, pkv_dtype dtype, void* stream) {
    WriteParams wp;
    pkv_status st = write_params(wp, k, v, k_pages, v_pages, slots, T, Hkv, head_dim, k_stride,
                                 k_head_stride, v_stride, v_head_stride, physical_pages,
                                 page_size, dtype);
    if (st != PKV_OK) return st;
    unsigned grid = 0;
    st = copy_params(wp, physical_pages, &grid);
    if (st != PKV_OK) return st;
    if (T == 0) return ok();
    int sms = 0;
    st = device_state(&sms, &wp.error);
    if (st != PKV_OK) return st;
    pkv_kv_write_kernel<<<grid, kWriteThreads, 0, static_cast<cudaStream_t>(stream)>>>(wp);
    return launched("K/V write");
}

pkv_status pkv_kv_write_fp8_block(const void* k, const void* v, void* k_pages, void* v_pages,
                                  float* k_scales, float* v_scales, const int32_t* slots, int T,
                                  int Hkv, int head_dim, long long k_stride,
                                  long long k_head_stride, long long v_stride,
                                  long long v_head_stride, int physical_pages, int page_size,
                                  int block_tokens, pkv_dtype dtype, void* stream) {
    WriteParams wp;
    pkv_status st = write_params(wp, k, v, k_pages, v_pages, slots, T, Hkv, head_dim, k_stride,
                                 k_head_stride, v_stride, v_head_stride, physical_pages,
                                 page_size, dtype);
    if (st != PKV_OK) return st;
    st = block_params(wp, k_scales, v_scales, physical_pages, block_tokens);
    if (st != PKV_OK) return st;
    if (T == 0) return ok();
    int sms = 0;
    st = device_state(&sms, &wp.error);
    if (st != PKV_OK) return st;
    // up to a warp per token while the grid has at most 32 warps an SM (28 of them
    // are resident at a time)
    const long long windows = ((long long)T + kRunRows - 1) / kRunRows;
    wp.split_log2 = 0;
    while ((1 << wp.split_log2) < kRunRows &&
           (windows * 2 * Hkv << (wp.split_log2 + 1)) <= 32ll * sms)
        ++wp.split_log2;
    const long long rows = block_rows(Hkv, wp.split_log2);
    const dim3 grid((unsigned)windows, (unsigned)rows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PKV_DTYPE_F16)
        pkv_kv_write_block_kernel<__half><<<grid, kWriteThreads, 0, s>>>(wp);
    else
        pkv_kv_write_block_kernel<__nv_bfloat16><<<grid, kWriteThreads, 0, s>>>(wp);
    return launched("e4m3 K/V write");
}

pkv_status pkv_prompt_attention(const void* q, const void* k, const void* v,
                                const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                void* output, float* lse, int B, int q_tokens, int k_tokens,
                                int Hq, int Hkv, int head_dim, long long q_stride,
                                long long q_head_stride, long long k_stride,
                                long long k_head_stride, long long v_stride,
                                long long v_head_stride, pkv_dtype dtype, void* stream) {
    PromptParams pp;
    pkv_status st = prompt_params(pp, q, k, v, cu_seqlens_q, cu_seqlens_k, output, lse, B, q_tokens,
                                  k_tokens, Hq, Hkv, head_dim, q_stride, q_head_stride, k_stride,
                                  k_head_stride, v_stride, v_head_stride, dtype);
    if (st != PKV_OK) return st;
    if (B == 0 || q_tokens == 0) return ok();
    int sms = 0;
    st = device_state(&sms, &pp.error);
    if (st != PKV_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == PKV_DTYPE_F16 ? launch_prompt<__half>(pp, dtype, sms, s)
                                  : launch_prompt<__nv_bfloat16>(pp, dtype, sms, s);
}

pkv_status pkv_prefill_check(const void* q, const void* k, const void* v, const void* output,
                             const float* lse, const void* k_pages, const void* v_pages,
                             const float* k_scales, const float* v_scales, int B, int T, int Hq,
                             int Hkv, int head_dim, long long q_stride, long long q_head_stride,
                             long long k_stride, long long k_head_stride, long long v_stride,
                             long long v_head_stride, int physical_pages, int page_size,
                             int block_tokens, pkv_dtype dtype) {
    // (slots and cu_seqlens are the caller's to come: any address stands in)
    const int32_t* some = static_cast<const int32_t*>(k_pages);
    const bool scaled = k_scales != nullptr || v_scales != nullptr;
    WriteParams wp;
    pkv_status st = write_params(wp, k, v, const_cast<void*>(k_pages), const_cast<void*>(v_pages),
                                 some, T, Hkv, head_dim, k_stride, k_head_stride, v_stride,
                                 v_head_stride, physical_pages, page_size, dtype);
    unsigned grid = 0;
    if (st == PKV_OK)
        st = scaled ? block_params(wp, const_cast<float*>(k_scales), const_cast<float*>(v_scales),
                                   physical_pages, block_tokens)
                    : copy_params(wp, physical_pages, &grid);
    PromptParams pp;
    if (st == PKV_OK)
        st = prompt_params(pp, q, k, v, some, some, const_cast<void*>(output),
                           const_cast<float*>(lse), B, T, T, Hq, Hkv, head_dim, q_stride,
                           q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride, dtype);
    if (st != PKV_OK) return st;
    const long long pool = (long long)physical_pages * Hkv * page_size * kHeadDim;
    const long long scale_bytes = scaled ? pool / kHeadDim / block_tokens * 4 : 0;
    const Range cache[4] = {{static_cast<const char*>(k_pages), scaled ? pool : 2 * pool},
                            {static_cast<const char*>(v_pages), scaled ? pool : 2 * pool},
                            {reinterpret_cast<const char*>(k_scales), scale_bytes},
                            {reinterpret_cast<const char*>(v_scales), scale_bytes}};
    const long long rows = (long long)T * Hq;
    for (const Range& c : cache)
        if (overlap(c, {static_cast<const char*>(output), rows * kRowBytes}) ||
            overlap(c, {reinterpret_cast<const char*>(lse), lse != nullptr ? rows * 4 : 0}))
            return fail_fmt(PKV_ERR_INVALID_ARGUMENT, "output and lse must not overlap the cache");
    return ok();
}

}  // extern "C"
