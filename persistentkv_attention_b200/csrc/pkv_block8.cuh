// pkv_block8.cuh -- decode over an e4m3 cache with one scale per block of
// tokens and head.  Included by pkv_block8.cu only.
#pragma once

#include "pkv_kernels.cuh"

namespace pkv {

struct Block8Params {
    DecodeParams d;
    const float* k_scales;  // [P][Hkv][page / block]
    const float* v_scales;
    int block;  // tokens per scale, a multiple of 16 that divides page_size
};

// One warp per (row, query head), straight from the formula.
template <typename T>
__global__ void __launch_bounds__(32)
    pkv_block8_rows_kernel(const __grid_constant__ Block8Params bp) {
    const DecodeParams& p = bp.d;
    const int lane = threadIdx.x;
    const int h = blockIdx.x, b = blockIdx.y;
    const int kvh = h / (p.Hq / p.Hkv);
    const int qr = p.q_indices != nullptr ? __ldg(p.q_indices + b) : b;
    const int orow = p.out_indices != nullptr ? __ldg(p.out_indices + b) : b;
    if (qr < 0 || qr >= p.q_rows || orow < 0 || orow >= p.out_rows) {
        if (lane == 0) raise_error(p.error, kErrIndex);
        return;
    }
    const int limit = p.max_pages * p.page_size;
    int n = __ldg(p.seq_lens + b);
    if (n > limit) {
        if (lane == 0) raise_error(p.error, kErrLogicalPage);
        n = limit;
    }
    float q[4];
    const T* qrow = reinterpret_cast<const T*>(p.q) + ((size_t)qr * p.Hq + h) * kHeadDim;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = (float)qrow[4 * lane + i];
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int nblk = p.page_size / bp.block;
    for (int t = 0; t < n; ++t) {
        const int page = __ldg(p.block_table + (size_t)b * p.max_pages + t / p.page_size);
        if (page < 0 || page >= p.num_pages) {
            if (lane == 0) raise_error(p.error, kErrPageId);
            continue;
        }
        const int off = t % p.page_size;
        const size_t head = (size_t)page * p.Hkv + kvh;
        const size_t at = (head * p.page_size + off) * kHeadDim + 4 * lane;
        const float ks = __ldg(bp.k_scales + head * nblk + off / bp.block);
        const float vs = __ldg(bp.v_scales + head * nblk + off / bp.block);
        const __nv_fp8_e4m3* k8 = reinterpret_cast<const __nv_fp8_e4m3*>(p.k_pages + at);
        const __nv_fp8_e4m3* v8 = reinterpret_cast<const __nv_fp8_e4m3*>(p.v_pages + at);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fmaf(q[i], (float)k8[i], s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= ks * p.scale_log2;
        const float mn = fmaxf(m, s);
        const float corr = fast_exp2(m - mn), w = fast_exp2(s - mn);
        m = mn;
        l = l * corr + w;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * corr + w * vs * (float)v8[i];
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* o = reinterpret_cast<T*>(p.out) + ((size_t)orow * p.Hq + h) * kHeadDim;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[4 * lane + i] = ElemOps<T>::from_float(acc[i] * inv);
}

}  // namespace pkv
