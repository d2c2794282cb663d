// pkv_prompt_kernels.cuh -- causal attention of packed prompts with grouped
// heads.  Included by pkv_prompt.cu only.
#pragma once

#include "pkv_device.cuh"

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

// One query row by one warp, straight from the formula: scores of 8 keys at a
// time, running maximum and sum in 32 bits, lane l holding dims 4l .. 4l + 3.
// Only the row's n visible keys are read.  A row that sees no key gives
// zeros and a log-sum of -inf.
template <typename T>
__device__ __forceinline__ void prompt_row(const PromptParams& p, const uint8_t* q,
                                           const uint8_t* k, const uint8_t* v, int n, T* out,
                                           float* lse, int lane) {
    auto load4 = [lane](const uint8_t* row) -> float4 {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(row) + lane);
        float2 a, b;
        if constexpr (std::is_same<T, __half>::value) {
            a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
            b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        } else {
            a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
            b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
        }
        return make_float4(a.x, a.y, b.x, b.y);
    };
    const float4 qv = load4(q);
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kKeys = 8;
    for (int j0 = 0; j0 < n; j0 += kKeys) {
        float s[kKeys];
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const int key = min(j0 + j, n - 1);
            const float4 kv = load4(k + (size_t)key * p.k_tok);
            float d = qv.x * kv.x;
            d = fmaf(qv.y, kv.y, d);
            d = fmaf(qv.z, kv.z, d);
            s[j] = fmaf(qv.w, kv.w, d);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
#pragma unroll
            for (int j = 0; j < kKeys; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], off);
        }
        float mx = m;
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            s[j] = j0 + j < n ? s[j] * p.scale_log2 : -INFINITY;
            mx = fmaxf(mx, s[j]);
        }
        // a maximum of -inf leaves every weight exp(-inf - 0) = 0
        const float base = mx == -INFINITY ? 0.f : mx;
        const float corr = fast_exp2(m - base);
        m = mx;
        l *= corr;
        acc.x *= corr;
        acc.y *= corr;
        acc.z *= corr;
        acc.w *= corr;
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            if (j0 + j >= n) break;
            const float pj = fast_exp2(s[j] - base);
            const float4 vv = load4(v + (size_t)(j0 + j) * p.v_tok);
            l += pj;
            acc.x = fmaf(pj, vv.x, acc.x);
            acc.y = fmaf(pj, vv.y, acc.y);
            acc.z = fmaf(pj, vv.z, acc.z);
            acc.w = fmaf(pj, vv.w, acc.w);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint2 o;
    o.x = ElemOps<T>::pack(acc.x * inv, acc.y * inv);
    o.y = ElemOps<T>::pack(acc.z * inv, acc.w * inv);
    reinterpret_cast<uint2*>(out)[lane] = o;
    if (lse != nullptr && lane == 0) *lse = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
}

}  // namespace pkv
