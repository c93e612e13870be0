// gdn_ssm_common.cuh -- what the selective scan kernels share.
//
//   dt' = softplus(dt + dt_bias),  a = -exp(A_log) dt'          (per token and head)
//   S_t = exp(a_t) S_{t-1} + dt'_t x_t B_t^T,   y_t = S_t C_t + D x_t,   [y_t <- y_t silu(z_t)]
//
// with S [head_size][128] fp32 per head (k-last), x, z [head_size] per head and B, C [128]
// shared by the heads / groups consecutive heads of a group.
#pragma once

#include "gdn_common.cuh"
#include "gdn_launch.h"

namespace gdn {

constexpr int kSsmState = 128;   // the only state size the kernels are built for

// dt' of one token and head, in fp32.
__device__ __forceinline__ float ssm_step(const SsmArgs &p, int64_t row, int h) {
    float v = load_scalar(p.dt, row * p.dt_stride + h, p.dt_dtype);
    if (p.dt_bias) v += load_scalar(p.dt_bias, h, p.param_dtype);
    return softplus_torch(v);
}

// exp(A_log), NaN if A_log is, and at most the largest finite number: with an infinite rate a
// step of length zero, such as that of a row behind the last token, would be 0 x inf.
__device__ __forceinline__ float ssm_rate(float A_log) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(expf(A_log)), "f"(3.402823466e38f));
    return r;
}

}  // namespace gdn
