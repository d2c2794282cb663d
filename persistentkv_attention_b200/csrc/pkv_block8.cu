// pkv_block8.cu -- launch of the decode over e4m3 pools with block scales.
#include "pkv_block8.cuh"
#include "pkv_launch.cuh"

namespace pkv_internal {

pkv_status launch_block8(const LaunchSpec& ls, cudaStream_t stream) {
    pkv::Block8Params bp;
    bp.d = ls.dp;
    bp.k_scales = ls.k_scales;
    bp.v_scales = ls.v_scales;
    bp.block = ls.scale_block;
    const dim3 grid(ls.dp.Hq, ls.dp.B);
    if (ls.dtype == PKV_DTYPE_F16)
        pkv::pkv_block8_rows_kernel<__half><<<grid, 32, 0, stream>>>(bp);
    else
        pkv::pkv_block8_rows_kernel<__nv_bfloat16><<<grid, 32, 0, stream>>>(bp);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
        return fail_fmt(PKV_ERR_CUDA, "decode launch failed: %s", cudaGetErrorString(e));
    return ok();
}

}  // namespace pkv_internal
