// Rows in 8 bits with one scale each: RMSNorm (with the residual's addition)
// straight into codes, the codes of rows that are there already, and the
// codes' values.
//
// The codes are decided in FP64: u * weight is exact there, so
//   q = rint(y / scale),  y = u * weight * (1 / sqrt(mean(u^2) + eps))
// carries a few roundings of 2^-53 before its own (rows as they are: none that
// could move a half); the sum's order, which the thread count and so the number of
// rows decide, reaches a code or scale by no more than those.  FP64 runs at half
// the FP32 rate here, and the row's bytes (13 a value with a residual) are
// what bounds the kernel, so the wider type costs nothing.  One pass over
// memory: the row stays in registers between the reduction (sum of squares
// and largest |u * weight|, both in the first pass) and the codes.  4093 rows of
// 4096 values with a residual take 34 us again and again over the same buffers, of
// which the cache before HBM holds a part, and 43 us (5.1 TB/s) over others each
// time; without it 22.  Rows as they are (F32 or 16 bits) take 16 to 19 us.
// One row takes 3.2 us, a launch and two round trips.
#include "si_i8.hpp"
#include "si_internal.hpp"

#include "sharpinference_hip.h"

#include <hip/hip_fp16.h>

namespace si {

namespace {

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

// Four values beside each other; ODD: at any address that one value may have.
// (The instructions are the same, but not their order: 4000 rows of 4096 values
// and their codes read back took 55 us with the aligned types and 64 us with the others;
// 1900 rows of 8001 took 103 us a value at a time, and take 64, 43 without the read-back.)
template <bool ODD>
struct Fours {
    typedef float f32 __attribute__((ext_vector_type(4)));
    typedef uint16_t f16 __attribute__((ext_vector_type(4)));
    typedef uint32_t codes;
};
template <>
struct Fours<true> {
    typedef float f32 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint16_t f16 __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t codes __attribute__((aligned(1)));
};

struct Values {
    float v[4];
};

// The row's four values from i on, 0 behind its end.  Without a branch: all of a
// row's loads are asked for before one is waited for.  ODD: rows of a length that
// four does not divide, or at such addresses; the last four of such a row begin up
// to three values before the ones that are wanted.
template <typename T4, typename T>
__device__ __forceinline__ void load_four(const T* row, int64_t i, int64_t n, bool odd, T* v)
{
    const int past = int(min(max(i - (n - 4), int64_t(0)), int64_t(4)));
    const T4 t = *reinterpret_cast<const T4*>(row + i - (past < 4 ? past : i - (n - 4)));
    const T z = T(0);
    if (odd) {
        v[0] = past < 2 ? (past ? t.y : t.x) : past < 4 ? (past == 2 ? t.z : t.w) : z;
        v[1] = past < 2 ? (past ? t.z : t.y) : past == 2 ? t.w : z;
        v[2] = past < 2 ? (past ? t.w : t.z) : z;
        v[3] = past ? z : t.w;
    } else {
        v[0] = past ? z : t.x, v[1] = past ? z : t.y, v[2] = past ? z : t.z, v[3] = past ? z : t.w;
    }
}
template <typename T4, bool ODD, typename T>
__device__ __forceinline__ void load_row(const T* row, int64_t i, int64_t n, T* v)
{
    if (ODD && n < 4) {                    // (the same for all rows)
#pragma unroll
        for (int j = 0; j < 4; j++)
            v[j] = i + j < n ? row[i + j] : T(0);
    } else {
        load_four<T4, T>(row, i, n, ODD, v);
    }
}

template <bool ODD>
__device__ __forceinline__ Values load_f32(const float* row, int64_t i, int64_t n)
{
    Values r;
    load_row<typename Fours<ODD>::f32, ODD>(row, i, n, r.v);
    return r;
}

// The row's input as FP32.
template <int IN, bool ODD>
__device__ __forceinline__ Values load_in(const RowsArgs& a, int64_t base, int64_t i)
{
    if constexpr (IN == IN_F16 || IN == IN_BF16) {
        Values r;
        uint16_t h[4];
        load_row<typename Fours<ODD>::f16, ODD>(static_cast<const uint16_t*>(a.x) + base, i, a.n, h);
#pragma unroll
        for (int j = 0; j < 4; j++)
            r.v[j] = IN == IN_F16 ? __half2float(__ushort_as_half(h[j])) : __uint_as_float(uint32_t(h[j]) << 16);
        return r;
    } else {
        return load_f32<ODD>(static_cast<const float*>(a.x) + base, i, a.n);
    }
}

// over N neighbouring lanes
template <int N>
__device__ __forceinline__ double lanes_sum(double v)
{
#pragma unroll
    for (int m = N / 2; m; m >>= 1)
        v += __shfl_xor(v, m);
    return v;
}
template <int N>
__device__ __forceinline__ double lanes_max(double v)
{
#pragma unroll
    for (int m = N / 2; m; m >>= 1)
        v = fmax(v, __shfl_xor(v, m));
    return v;
}

// THREADS threads a row (16, 64: 16 or 4 rows a workgroup of 256), STEPS fours of
// it in a thread's registers; longer rows are read again (from L2, mostly) for
// their codes.
template <int IN, int THREADS, int STEPS, bool ODD>
__global__ void __launch_bounds__(THREADS <= 64 ? 256 : THREADS)
rows_i8_kernel(const RowsArgs a)
{
    constexpr bool NORM = IN == IN_NORM || IN == IN_NORM_RESIDUAL;
    constexpr bool RESIDUAL = IN == IN_NORM_RESIDUAL;
    constexpr int LANES = THREADS < 64 ? THREADS : 64;
    const int lane = threadIdx.x % THREADS;
    const int64_t row = THREADS <= 64 ? int64_t(blockIdx.x) * (256 / THREADS) + threadIdx.x / THREADS : blockIdx.x;
    if (row >= a.rows)
        return;   // all lanes of a row, and no barrier follows where THREADS is at most 64
    const int64_t base = row * a.n;
    const int64_t stride = int64_t(THREADS) * 4;

    Values kept[STEPS], add[RESIDUAL ? STEPS : 1], w[NORM ? STEPS : 1];
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int64_t i = k * stride + lane * 4;
        kept[k] = load_in<IN, ODD>(a, base, i);
        if constexpr (RESIDUAL)
            add[k] = load_f32<ODD>(a.residual + base, i, a.n);
        if constexpr (NORM)
            w[k] = load_f32<ODD>(a.weight, i, a.n);
    }
    if constexpr (RESIDUAL) {
#pragma unroll
        for (int k = 0; k < STEPS; k++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                kept[k].v[j] += add[k].v[j];
    }
    double sum = 0.0, top = 0.0;
    bool bad = false;
    auto take = [&](const Values& u, const Values& wt, int64_t i) {
        if constexpr (RESIDUAL) {
            if (ODD && a.n - i < 4) {
#pragma unroll
                for (int j = 0; j < 3; j++)
                    if (j < a.n - i)
                        a.updated[base + i + j] = u.v[j];
            } else if (i < a.n) {
                *reinterpret_cast<typename Fours<ODD>::f32*>(a.updated + base + i) = typename Fours<ODD>::f32{u.v[0], u.v[1], u.v[2], u.v[3]};
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
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
        take(kept[k], w[NORM ? k : 0], k * stride + lane * 4);
    }
    auto again = [&](int64_t i, Values* wt) {
        Values u = load_in<IN, ODD>(a, base, i);
        if constexpr (RESIDUAL) {
            const Values b = load_f32<ODD>(a.residual + base, i, a.n);
#pragma unroll
            for (int j = 0; j < 4; j++)
                u.v[j] += b.v[j];
        }
        *wt = Values{};
        if constexpr (NORM)
            *wt = load_f32<ODD>(a.weight, i, a.n);
        return u;
    };
    for (int64_t i = STEPS * stride + lane * 4; i < a.n; i += stride) {
        Values wt;
        const Values u = again(i, &wt);
        take(u, wt, i);
    }
    // the reduction: a value that is not finite travels as a NaN sum
    if (bad)
        sum = NAN;
    sum = lanes_sum<LANES>(sum);
    top = lanes_max<LANES>(top);
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
    const double c = scale > 0.0f ? 1.0 / double(scale) : 0.0;
    auto give = [&](const Values& u, const Values& wt, int64_t i) {
        int q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const double y = NORM ? double(u.v[j]) * double(wt.v[j]) * inv : double(u.v[j]);
            // The quotient y / scale: y * c may miss a half by its last bit (9487.5 / 75
            // gave 127 and not the even 126); what is left of y, exact for a scale of 24
            // bits, puts it right.
            double t = y * c;
            t = fma(fma(-t, double(scale), y), c, t);
            // (a scale among the subnormals is coarse enough to pass 127)
            q[j] = scale > 0.0f ? int(fmin(fmax(rint(t), -127.0), 127.0)) : 0;
        }
        if (ODD && a.n - i < 4) {
#pragma unroll
            for (int j = 0; j < 3; j++)
                if (j < a.n - i)
                    a.codes[base + i + j] = static_cast<int8_t>(q[j]);
        } else {
            *reinterpret_cast<typename Fours<ODD>::codes*>(a.codes + base + i) =
                (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | uint32_t(q[3]) << 24;
        }
    };
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int64_t i = k * stride + lane * 4;
        if (i < a.n)
            give(kept[k], w[NORM ? k : 0], i);
    }
    for (int64_t i = STEPS * stride + lane * 4; i < a.n; i += stride) {
        Values wt;
        const Values u = again(i, &wt);
        give(u, wt, i);
    }
}

template <int IN, bool ODD>
hipError_t launch_rows(const RowsArgs& a, hipStream_t s)
{
    // the fewest threads a row that keep it in registers, but for few rows, which
    // the whole chip has to share
    if (a.n <= 16 * 16 && a.rows >= 1024)
        rows_i8_kernel<IN, 16, 4, ODD><<<unsigned((a.rows + 15) / 16), 256, 0, s>>>(a);
    else if (a.n <= 64 * 16 && a.rows >= 1024)
        rows_i8_kernel<IN, 64, 4, ODD><<<unsigned((a.rows + 3) / 4), 256, 0, s>>>(a);
    else if (a.n <= 64 * 32 && a.rows >= 1024)
        rows_i8_kernel<IN, 64, 8, ODD><<<unsigned((a.rows + 3) / 4), 256, 0, s>>>(a);
    else if (a.n <= 256 * 16)
        rows_i8_kernel<IN, 256, 4, ODD><<<unsigned(a.rows), 256, 0, s>>>(a);
    else if (a.n <= 256 * 32)
        rows_i8_kernel<IN, 256, 8, ODD><<<unsigned(a.rows), 256, 0, s>>>(a);
    else
        rows_i8_kernel<IN, 1024, 4, ODD><<<unsigned(a.rows), 1024, 0, s>>>(a);
    return hipGetLastError();
}

bool on(const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0; }

template <int IN>
hipError_t launch_rows(const RowsArgs& a, hipStream_t s)
{
    const uintptr_t in = IN == IN_F16 || IN == IN_BF16 ? 8 : 16;
    const bool fours = a.n % 4 == 0 && on(a.x, in) && on(a.residual, 16) && on(a.weight, 16) && on(a.updated, 16) &&
                       on(a.codes, 4);
    return fours ? launch_rows<IN, false>(a, s) : launch_rows<IN, true>(a, s);
}

// a workgroup takes 1024 columns of one row at a time
template <bool ODD>
__global__ void __launch_bounds__(256)
dequant_i8_kernel(const int8_t* codes, const float* scale, float* out, int64_t rows, int64_t n)
{
    const int64_t per_row = (n + 1023) / 1024;
    for (int64_t b = blockIdx.x; b < rows * per_row; b += gridDim.x) {
        const int64_t row = b / per_row;
        const int64_t i = (b - row * per_row) * 1024 + threadIdx.x * 4;
        if (i >= n)
            continue;
        const float d = scale[row];
        const int8_t* const from = codes + row * n + i;
        float* const to = out + row * n + i;
        if (ODD && n - i < 4) {
            for (int j = 0; j < n - i; j++)
                to[j] = float(from[j]) * d;
        } else {
            const uint32_t q = *reinterpret_cast<const typename Fours<ODD>::codes*>(from);
            *reinterpret_cast<typename Fours<ODD>::f32*>(to) = typename Fours<ODD>::f32{
                float(int8_t(q)) * d, float(int8_t(q >> 8)) * d, float(int8_t(q >> 16)) * d, float(int8_t(q >> 24)) * d};
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
    const int64_t blocks = rows * ((n + 1023) / 1024);
    const unsigned grid = unsigned(blocks < (1 << 20) ? blocks : 1 << 20);
    if (n % 4 == 0 && on(codes, 4) && on(out, 16))
        dequant_i8_kernel<false><<<grid, 256, 0, s>>>(codes, scale, out, rows, n);
    else
        dequant_i8_kernel<true><<<grid, 256, 0, s>>>(codes, scale, out, rows, n);
    return hipGetLastError();
}

}  // namespace si
