// pkv_block8.cu -- launch of the decode over e4m3 pools with block scales.
#include "pkv_block8.cuh"
#include "pkv_launch.cuh"

namespace pkv_internal {
namespace {

template <int G, typename T>
pkv_status launch_typed8(const LaunchSpec& ls, cudaStream_t stream) {
    using namespace pkv;
    auto kern = pkv_block8_kernel<G, T, kSlots>;
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
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ls.pdl ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, bp);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail_fmt(PKV_ERR_CUDA, "decode launch failed: %s", cudaGetErrorString(e));
    }
    return ok();
}

template <typename T>
pkv_status launch_g8(const LaunchSpec& ls, cudaStream_t stream) {
    switch (ls.G) {
        case 1: return launch_typed8<1, T>(ls, stream);
        case 2: return launch_typed8<2, T>(ls, stream);
        case 4: return launch_typed8<4, T>(ls, stream);
        case 8: return launch_typed8<8, T>(ls, stream);
        default: return fail_fmt(PKV_ERR_UNSUPPORTED, "unsupported G=%d", ls.G);
    }
}

}  // namespace

pkv_status launch_block8(const LaunchSpec& ls, cudaStream_t stream) {
    return ls.dtype == PKV_DTYPE_F16 ? launch_g8<__half>(ls, stream)
                                     : launch_g8<__nv_bfloat16>(ls, stream);
}

}  // namespace pkv_internal
