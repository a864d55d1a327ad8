// What the windowed-attention kernels share: value conversions, the ragged batch and the pattern.
#ifndef MCSPARSE_B200_WINDOW_COMMON_H_
#define MCSPARSE_B200_WINDOW_COMMON_H_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"

namespace mcsp_b200 {
namespace window {

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The ragged batch as the kernels read it. Offsets that do not ascend or leave the tensors are cut to them, so that no
// access can leave the tensors whatever the arrays hold.
struct Ragged {
    const int* q_offsets;
    const int* k_offsets;
    int batch, total_q, total_k;
};
struct Sequence {
    int q0, lq, k0, lk;
};
__device__ __forceinline__ int clamp_offset(int v, int total) { return min(max(v, 0), total); }
__device__ __forceinline__ Sequence sequence_of(const Ragged& r, int b) {
    if (r.q_offsets == nullptr) return Sequence{0, r.total_q, 0, r.total_k};
    Sequence s;
    s.q0 = clamp_offset(__ldg(r.q_offsets + b), r.total_q);
    s.lq = max(clamp_offset(__ldg(r.q_offsets + b + 1), r.total_q) - s.q0, 0);
    s.k0 = clamp_offset(__ldg(r.k_offsets + b), r.total_k);
    s.lk = max(clamp_offset(__ldg(r.k_offsets + b + 1), r.total_k) - s.k0, 0);
    return s;
}
// The sequence that holds row t, or -1.
__device__ __forceinline__ int sequence_at(const int* offsets, int batch, int total, int t) {
    if (offsets == nullptr) return 0;
    int lo = 0, hi = batch;  // the last b with offsets[b] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(offsets + mid) <= t)
            lo = mid;
        else
            hi = mid;
    }
    return t >= clamp_offset(__ldg(offsets + lo), total) && t < clamp_offset(__ldg(offsets + lo + 1), total) ? lo : -1;
}

}  // namespace window
}  // namespace mcsp_b200

#endif  // MCSPARSE_B200_WINDOW_COMMON_H_
