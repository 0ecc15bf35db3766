// Rows in 8 bits with one scale each: RMSNorm (with the residual's addition)
// straight into codes, the codes of rows that are there already, and the
// codes' values.
//
// The codes are decided in FP64: u * weight is exact there, so
//   q = rint(u * weight * c),  c = (1 / sqrt(mean(u^2) + eps)) / scale
// carries one rounding of 2^-53 before its own, and the sum's order, the
// thread count and the row's neighbours change no code.  FP64 runs at half
// the FP32 rate here, and the row's bytes (13 a value with a residual) are
// what bounds the kernel, so the wider type costs nothing.  One pass over
// memory: the row stays in registers between the reduction (sum of squares
// and largest |u * weight|, both in the first pass) and the codes.
#include "si_i8.hpp"
#include "si_internal.hpp"

#include "sharpinference_hip.h"

#include <hip/hip_fp16.h>

namespace si {

namespace {

// Values of a row that a thread keeps in registers; longer rows are read
// again (from L2, mostly) for their codes.
constexpr int KEEP = 32;

enum InKind : int { IN_NORM, IN_NORM_RESIDUAL, IN_F32, IN_F16, IN_BF16 };

struct RowsArgs {
    const void* x;            // hidden, or the rows to quantize
    const float* residual;
    const float* weight;
    float* updated;
    int8_t* codes;
    float* scale;
    int64_t n;
    int64_t rows;
    float eps;
};

template <int VEC>
struct Values {
    float v[VEC];
};

template <int VEC>
__device__ __forceinline__ Values<VEC> load_f32(const float* p)
{
    Values<VEC> r;
    if constexpr (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        r.v[0] = t.x, r.v[1] = t.y, r.v[2] = t.z, r.v[3] = t.w;
    } else {
        r.v[0] = *p;
    }
    return r;
}

// The row's value as the codes are made of it: the input, plus the residual.
template <int IN, int VEC>
__device__ __forceinline__ Values<VEC> load_in(const RowsArgs& a, int64_t at)
{
    if constexpr (IN == IN_F16 || IN == IN_BF16) {
        Values<VEC> r;
        const uint16_t* p = static_cast<const uint16_t*>(a.x) + at;
        uint16_t h[VEC];
        if constexpr (VEC == 4) {
            const uint2 t = *reinterpret_cast<const uint2*>(p);
            h[0] = t.x & 0xFFFFu, h[1] = t.x >> 16, h[2] = t.y & 0xFFFFu, h[3] = t.y >> 16;
        } else {
            h[0] = *p;
        }
#pragma unroll
        for (int i = 0; i < VEC; i++)
            r.v[i] = IN == IN_F16 ? __half2float(__ushort_as_half(h[i])) : __uint_as_float(uint32_t(h[i]) << 16);
        return r;
    } else {
        Values<VEC> r = load_f32<VEC>(static_cast<const float*>(a.x) + at);
        if constexpr (IN == IN_NORM_RESIDUAL) {
            const Values<VEC> b = load_f32<VEC>(a.residual + at);
#pragma unroll
            for (int i = 0; i < VEC; i++)
                r.v[i] += b.v[i];
        }
        return r;
    }
}

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1)
        v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ double wave_max(double v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1)
        v = fmax(v, __shfl_xor(v, m));
    return v;
}

// THREADS threads a row (64: four rows a workgroup of 256).
template <int IN, int THREADS, int VEC>
__global__ void __launch_bounds__(THREADS == 64 ? 256 : THREADS)
rows_i8_kernel(const RowsArgs a)
{
    constexpr bool NORM = IN == IN_NORM || IN == IN_NORM_RESIDUAL;
    constexpr int STEPS = KEEP / VEC;
    const int lane = threadIdx.x % THREADS;
    const int64_t row = THREADS == 64 ? int64_t(blockIdx.x) * 4 + threadIdx.x / 64 : blockIdx.x;
    if (row >= a.rows)
        return;   // whole waves, and no barrier follows where THREADS is 64
    const int64_t base = row * a.n;
    const int64_t stride = int64_t(THREADS) * VEC;

    Values<VEC> kept[STEPS], w[NORM ? STEPS : 1];
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int64_t i = k * stride + lane * VEC;
        if (i < a.n) {
            kept[k] = load_in<IN, VEC>(a, base + i);
            if constexpr (NORM)
                w[k] = load_f32<VEC>(a.weight + i);
        }
    }
    double sum = 0.0, top = 0.0;
    bool bad = false;
    auto take = [&](const Values<VEC>& u, const Values<VEC>& wt, int64_t i) {
        if constexpr (IN == IN_NORM_RESIDUAL) {
            if constexpr (VEC == 4)
                *reinterpret_cast<float4*>(a.updated + base + i) = make_float4(u.v[0], u.v[1], u.v[2], u.v[3]);
            else
                a.updated[base + i] = u.v[0];
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const double x = u.v[j];
            double y = x;
            if constexpr (NORM) {
                sum = fma(x, x, sum);
                y = x * double(wt.v[j]);
            }
            bad |= !(fabs(y) < INFINITY);
            top = fmax(top, fabs(y));
        }
    };
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int64_t i = k * stride + lane * VEC;
        if (i < a.n)
            take(kept[k], w[NORM ? k : 0], i);
    }
    for (int64_t i = STEPS * stride + lane * VEC; i < a.n; i += stride) {
        Values<VEC> wt{};
        if constexpr (NORM)
            wt = load_f32<VEC>(a.weight + i);
        take(load_in<IN, VEC>(a, base + i), wt, i);
    }
    // the reduction: a value that is not finite travels as a NaN sum
    if (bad)
        sum = NAN;
    sum = wave_sum(sum);
    top = wave_max(top);
    if constexpr (THREADS > 64) {
        __shared__ double parts[2][THREADS / 64];
        if ((threadIdx.x & 63) == 0) {
            parts[0][threadIdx.x / 64] = sum;
            parts[1][threadIdx.x / 64] = top;
        }
        __syncthreads();
        sum = parts[0][0];
        top = parts[1][0];
#pragma unroll
        for (int i = 1; i < THREADS / 64; i++) {
            sum += parts[0][i];
            top = fmax(top, parts[1][i]);
        }
    }
    const double inv = NORM ? 1.0 / sqrt(sum / double(a.n) + double(a.eps)) : 1.0;
    float scale = top == 0.0 ? 0.0f : float(top * inv / 127.0);
    if (!(sum == sum) || !(scale < INFINITY))
        scale = NAN;
    if (lane == 0)
        a.scale[row] = scale;
    // no scale, no codes: a row of zeros, or one that holds something infinite or NaN
    const double c = scale > 0.0f ? inv / double(scale) : 0.0;
    auto give = [&](const Values<VEC>& u, const Values<VEC>& wt, int64_t i) {
        int q[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const double y = NORM ? double(u.v[j]) * double(wt.v[j]) : double(u.v[j]);
            // (a scale among the subnormals is coarse enough to pass 127)
            q[j] = scale > 0.0f ? int(fmin(fmax(rint(y * c), -127.0), 127.0)) : 0;
        }
        if constexpr (VEC == 4)
            *reinterpret_cast<uint32_t*>(a.codes + base + i) =
                (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | uint32_t(q[3]) << 24;
        else
            a.codes[base + i] = static_cast<int8_t>(q[0]);
    };
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int64_t i = k * stride + lane * VEC;
        if (i < a.n)
            give(kept[k], w[NORM ? k : 0], i);
    }
    for (int64_t i = STEPS * stride + lane * VEC; i < a.n; i += stride) {
        Values<VEC> wt{};
        if constexpr (NORM)
            wt = load_f32<VEC>(a.weight + i);
        give(load_in<IN, VEC>(a, base + i), wt, i);
    }
}

template <int IN, int VEC>
hipError_t launch_rows(const RowsArgs& a, hipStream_t s)
{
    if (a.n <= 64 * KEEP && a.rows >= 1024)
        rows_i8_kernel<IN, 64, VEC><<<unsigned((a.rows + 3) / 4), 256, 0, s>>>(a);
    else if (a.n <= 256 * KEEP)
        rows_i8_kernel<IN, 256, VEC><<<unsigned(a.rows), 256, 0, s>>>(a);
    else
        rows_i8_kernel<IN, 1024, VEC><<<unsigned(a.rows), 1024, 0, s>>>(a);
    return hipGetLastError();
}

bool on(const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0; }

template <int IN>
hipError_t launch_rows(const RowsArgs& a, hipStream_t s)
{
    const uintptr_t in = IN == IN_F16 || IN == IN_BF16 ? 8 : 16;
    const bool wide = a.n % 4 == 0 && on(a.x, in) && on(a.residual, 16) && on(a.weight, 16) && on(a.updated, 16) &&
                      on(a.codes, 4);
    return wide ? launch_rows<IN, 4>(a, s) : launch_rows<IN, 1>(a, s);
}

template <int VEC>
__global__ void __launch_bounds__(256)
dequant_i8_kernel(const int8_t* codes, const float* scale, float* out, int64_t rows, int64_t n)
{
    // a workgroup takes 256 * VEC columns of one row at a time
    const int64_t per_row = (n + 256 * VEC - 1) / (256 * VEC);
    for (int64_t b = blockIdx.x; b < rows * per_row; b += gridDim.x) {
        const int64_t row = b / per_row;
        const int64_t i = (b - row * per_row) * (256 * VEC) + threadIdx.x * VEC;
        if (i >= n)
            continue;
        const float d = scale[row];
        if constexpr (VEC == 4) {
            const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + row * n + i);
            *reinterpret_cast<float4*>(out + row * n + i) =
                make_float4(float(int8_t(q)) * d, float(int8_t(q >> 8)) * d, float(int8_t(q >> 16)) * d,
                            float(int8_t(q >> 24)) * d);
        } else {
            out[row * n + i] = float(codes[row * n + i]) * d;
        }
    }
}

}  // namespace

hipError_t launch_rms_norm_i8(const float* hidden, const float* residual, const float* weight, float* updated,
                              int8_t* codes, float* scale, int64_t rows, int64_t n, float eps, hipStream_t s)
{
    const RowsArgs a{hidden, residual, weight, updated, codes, scale, n, rows, eps};
    return residual ? launch_rows<IN_NORM_RESIDUAL>(a, s) : launch_rows<IN_NORM>(a, s);
}

hipError_t launch_quantize_i8(int fmt, const void* x, int8_t* codes, float* scale, int64_t rows, int64_t n,
                              hipStream_t s)
{
    const RowsArgs a{x, nullptr, nullptr, nullptr, codes, scale, n, rows, 0.0f};
    return fmt == SI_HIP_F32 ? launch_rows<IN_F32>(a, s)
           : fmt == SI_HIP_F16 ? launch_rows<IN_F16>(a, s) : launch_rows<IN_BF16>(a, s);
}

hipError_t launch_dequant_i8(const int8_t* codes, const float* scale, float* out, int64_t rows, int64_t n,
                             hipStream_t s)
{
    const bool wide = n % 4 == 0 && on(codes, 4) && on(out, 16);
    const int64_t blocks = rows * ((n + (wide ? 1023 : 255)) / (wide ? 1024 : 256));
    const unsigned grid = unsigned(blocks < (1 << 20) ? blocks : 1 << 20);
    if (wide)
        dequant_i8_kernel<4><<<grid, 256, 0, s>>>(codes, scale, out, rows, n);
    else
        dequant_i8_kernel<1><<<grid, 256, 0, s>>>(codes, scale, out, rows, n);
    return hipGetLastError();
}

}  // namespace si
