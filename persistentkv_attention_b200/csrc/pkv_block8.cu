// pkv_block8.cu -- launch of the decode over e4m3 pools with block scales.
#include "pkv_block8.cuh"
#include "pkv_launch.cuh"

namespace pkv_internal {
namespace {


// A pool of e4m3 lines, [lines][128 bytes]; one box is `box` lines.
pkv_status line_map(CUtensorMap* map, const void* base, long long lines, int box) {
    const cuuint64_t dims[2] = {(cuuint64_t)pkv::kB8Line, (cuuint64_t)lines};
    const cuuint64_t strides[1] = {(cuuint64_t)pkv::kB8Line};
    const cuuint32_t boxes[2] = {(cuuint32_t)pkv::kB8Line, (cuuint32_t)box};
    const cuuint32_t elem[2] = {1u, 1u};
    const EncodeTiledFn fn = encode_tiled();
    if (fn == nullptr) return fail_fmt(PKV_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims,
                          strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail_fmt(PKV_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return PKV_OK;
}

template <int G, typename T, int BOX>
pkv_status launch_typed8(const LaunchSpec& ls, cudaStream_t stream) {
    using namespace pkv;
    CUtensorMap tk, tv;
    pkv_status st = line_map(&tk, ls.k, ls.rows, BOX);
    if (st == PKV_OK) st = line_map(&tv, ls.v, ls.rows, BOX);
    if (st != PKV_OK) return st;
    auto kern = pkv_block8_kernel<G, T, BOX, kSlots>;
    const size_t smem = block8_smem_bytes<G, kSlots>();
    // the device schedule's grid (2 CTAs per SM) must be resident in one wave
    static_assert(2 * (block8_smem_bytes<G, kSlots>() + 1024) <= 228 * 1024,
                  "decode CTA too large for 2 per SM");
    static std::atomic<unsigned long long> attr_done{0ull};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    cudaError_t e = cudaSuccess;
    if (!(attr_done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return fail_fmt(PKV_ERR_CUDA, "cudaFuncSetAttribute failed: %s",
                            cudaGetErrorString(e));
        }
        attr_done.fetch_or(bit, std::memory_order_acq_rel);
    }
    Block8Params bp;
    bp.d = ls.dp;
    bp.k_scales = ls.k_scales;
    bp.v_scales = ls.v_scales;
    bp.block = ls.scale_block;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ls.dp.auto_groups * ls.dp.Hkv);
    cfg.blockDim = dim3(kB8Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ls.pdl ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, bp, tk, tv);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail_fmt(PKV_ERR_CUDA, "decode launch failed: %s", cudaGetErrorString(e));
    }
    return ok();
}

// Copies of 32 tokens where pages hold whole ones, else of 16.
template <int G, typename T>
pkv_status launch_box8(const LaunchSpec& ls, cudaStream_t stream) {
    return ls.dp.page_size % 32 == 0 ? launch_typed8<G, T, 32>(ls, stream)
                                     : launch_typed8<G, T, 16>(ls, stream);
}

template <typename T>
pkv_status launch_g8(const LaunchSpec& ls, cudaStream_t stream) {
    switch (ls.G) {
        case 1: return launch_box8<1, T>(ls, stream);
        case 2: return launch_box8<2, T>(ls, stream);
        case 4: return launch_box8<4, T>(ls, stream);
        case 8: return launch_box8<8, T>(ls, stream);
        default: return fail_fmt(PKV_ERR_UNSUPPORTED, "unsupported G=%d", ls.G);
    }
}

}  // namespace

pkv_status launch_block8(const LaunchSpec& ls, cudaStream_t stream) {
    return ls.dtype == PKV_DTYPE_F16 ? launch_g8<__half>(ls, stream)
                                     : launch_g8<__nv_bfloat16>(ls, stream);
}

}  // namespace pkv_internal
