// 8-bit integer rows with one FP32 scale each: the launches behind the
// si_hip_*_i8 entry points (si_i8.hip, si_i8_gemm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace si {

// codes[r][i] = rint(y / scale[r]), scale[r] = max_i |y| / 127, of
//   y = u * (1 / sqrt(sum(u^2) / n + eps)) * weight, u = hidden (+ residual)
// and, with a residual, updated = u.
hipError_t launch_rms_norm_i8(const float* hidden, const float* residual, const float* weight, float* updated,
                              int8_t* codes, float* scale, int64_t rows, int64_t n, float eps, hipStream_t s);
// The same codes and scales of rows as they are; fmt SI_HIP_F32, F16 or BF16.
hipError_t launch_quantize_i8(int fmt, const void* x, int8_t* codes, float* scale, int64_t rows, int64_t n,
                              hipStream_t s);
// out[r][i] = codes[r][i] * scale[r]
hipError_t launch_dequant_i8(const int8_t* codes, const float* scale, float* out, int64_t rows, int64_t n,
                             hipStream_t s);

// y[t][o] = float(sum_k x[t][k] * w[o][k]) * x_scale[t] * w_scale[o]
// (+ residual[t][o]), x [m, cols] and w [rows, cols] codes, cols % 16 == 0,
// both 16-byte aligned.
struct GemmI8Args {
    const int8_t* x;
    const float* x_scale;
    const int8_t* w;
    const float* w_scale;
    const float* residual;     // optional, may be y
    float* y;
    int64_t m;
    int64_t rows;
    int64_t cols;
};
hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s);

}  // namespace si
