// Y = X . W^T of 8-bit integer rows with a scale for each token and each
// output channel: exact int32 sums on the matrix cores, the scales (and the
// residual) applied once to each sum.
#include "si_i8.hpp"

namespace si {

namespace {

using i32x4 = __attribute__((__vector_size__(4 * sizeof(int)))) int;
using i32x16 = __attribute__((__vector_size__(16 * sizeof(int)))) int;

// One wave: 32 channels x 32 tokens, operands straight from memory.
__global__ void __launch_bounds__(256)
gemm_i8_kernel(const GemmI8Args a)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t o0 = int64_t(blockIdx.x) * 64 + (wave & 1) * 32;
    const int64_t t0 = int64_t(blockIdx.y) * 64 + (wave >> 1) * 32;
    const int64_t o = o0 + (lane & 31), t = t0 + (lane & 31);
    const int8_t* wp = a.w + (o < a.rows ? o : a.rows - 1) * a.cols;
    const int8_t* xp = a.x + (t < a.m ? t : a.m - 1) * a.cols;
    i32x16 acc{};
    for (int64_t k = 16 * (lane >> 5); k < a.cols + 16 * (lane >> 5); k += 32) {
        i32x4 fw{}, fx{};
        if (k < a.cols) {
            fw = *reinterpret_cast<const i32x4*>(wp + k);
            fx = *reinterpret_cast<const i32x4*>(xp + k);
        }
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw, fx, acc, 0, 0, 0);
    }
    if (t >= a.m)
        return;
    const float sx = a.x_scale[t];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int64_t c = o0 + (i & 3) + 8 * (i >> 2) + 4 * (lane >> 5);
        if (c < a.rows) {
            float v = float(acc[i]) * sx * a.w_scale[c];
            if (a.residual)
                v += a.residual[t * a.rows + c];
            a.y[t * a.rows + c] = v;
        }
    }
}

}  // namespace

hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s)
{
    gemm_i8_kernel<<<dim3(unsigned((a.rows + 63) / 64), unsigned((a.m + 63) / 64)), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace si
