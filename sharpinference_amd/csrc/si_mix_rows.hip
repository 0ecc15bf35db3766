// LayerNorm of token rows, mixed with the row before of the same sequence
// (PortableRwkv7GraphProvider.cs:163-170, 180-184, 202-210, 280-288).
#include "si_sequences.hpp"
#include "si_lanes.hpp"

#include <type_traits>

namespace si {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

template <typename T>
struct alignas(4 * sizeof(T)) Four {
    T x, y, z, w;
};

// A workgroup takes `run` rows one after another, PER values of a row a
// thread (four neighbours each where FOURS, else every 256th).  The row before
// stays in registers, so only a run's first row is normalised twice; the
// sequence's state is read by the workgroup of its first row, which also
// normalises the last row for the state's slot: the slot has one reader and
// writer, whatever the other workgroups have done by then.
// Bound by HBM: 4 bytes in (8 with a residual, 4 more out) and 2 or 4 out a mix.
template <int PER, bool FOURS, typename OUT>
__global__ __launch_bounds__(THREADS) void mix_rows_kernel(MixRowsArgs a, int run)
{
    __shared__ float s_sum[WAVES], s_squares[WAVES];
    __shared__ int s_at[WAVES];
    const int t = threadIdx.x, wave = t >> 6, n = a.n;
    const RowBatch& b = a.batch;
    auto place = [&](int j) { return FOURS ? 4 * (t + THREADS * (j >> 2)) + (j & 3) : t + THREADS * j; };

    // the sequence of the run's first row: as many as end at or before it
    int row = blockIdx.x * run;
    const int end = min(row + run, b.rows);
    int at = 0;
    for (int i = t; i < b.sequences; i += THREADS)
        at += b.starts[i + 1] <= row;
    at = static_cast<int>(rows_sum(row_sum<16>(static_cast<float>(at))));   // at most 4096: exact
    if ((t & 63) == 0)
        s_at[wave] = at;
    __syncthreads();
    int s = 0;
    for (int w = 0; w < WAVES; w++)
        s += s_at[w];
    s = __builtin_amdgcn_readfirstlane(s);

    auto load = [&](const float* p, float* v) {
        if constexpr (FOURS) {
#pragma unroll
            for (int j = 0; j < PER; j += 4) {
                float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (place(j) < n)
                    f = *reinterpret_cast<const float4*>(p + place(j));
                v[j] = f.x, v[j + 1] = f.y, v[j + 2] = f.z, v[j + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; j++)
                v[j] = place(j) < n ? p[place(j)] : 0.0f;
        }
    };
    auto store = [&](auto* p, const float* v) {
        using T = std::remove_reference_t<decltype(*p)>;
        if constexpr (FOURS) {
#pragma unroll
            for (int j = 0; j < PER; j += 4)
                if (place(j) < n)
                    *reinterpret_cast<Four<T>*>(p + place(j)) =
                        Four<T>{static_cast<T>(v[j]), static_cast<T>(v[j + 1]), static_cast<T>(v[j + 2]), static_cast<T>(v[j + 3])};
        } else {
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (place(j) < n)
                    p[place(j)] = static_cast<T>(v[j]);
        }
    };
    auto block_sum = [&](float v, float* part) {
        v = rows_sum(row_sum<16>(v));
        if ((t & 63) == 0)
            part[wave] = v;
        __syncthreads();
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++)
            sum += part[w];
        return sum;
    };
    float weight[PER], bias[PER];
    load(a.weight, weight);
    load(a.bias, bias);
    // the norm of a row, and (its own workgroup's row) the residual sum's store
    auto norm = [&](int r, float* v, bool keep) {
        load(a.x + static_cast<int64_t>(r) * n, v);
        if (a.residual) {
            float add[PER];
            load(a.residual + static_cast<int64_t>(r) * n, add);
#pragma unroll
            for (int j = 0; j < PER; j++)
                v[j] += add[j];
            if (keep)
                store(a.updated + static_cast<int64_t>(r) * n, v);
        }
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; j++)
            sum += v[j];
        const float mean = block_sum(sum, s_sum) / static_cast<float>(n);
        float squares = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            v[j] = place(j) < n ? v[j] - mean : 0.0f;
            squares = fmaf(v[j], v[j], squares);
        }
        const float inv = 1.0f / sqrtf(block_sum(squares, s_squares) / static_cast<float>(n) + a.eps);
#pragma unroll
        for (int j = 0; j < PER; j++)
            v[j] = fmaf(v[j] * inv, weight[j], bias[j]);
    };

    float before[PER], now[PER];
    bool have = false;   // `before` is the row before
    OUT* const out = static_cast<OUT*>(a.out);
    for (; row < end; row++) {
        while (s < b.sequences && row >= b.starts[s + 1]) {
            s++;
            have = false;
        }
        if (s >= b.sequences)
            break;
        const RowSpan span = rows_of(b, s);
        if (row < span.first || row >= span.last) {
            have = false;
            continue;
        }
        if (a.mixes == 0) {
            norm(row, now, true);
            store(out + static_cast<int64_t>(row) * n, now);
            continue;
        }
        if (row == span.first) {
            const int from = b.from[s];
            if (from >= 0 && from < b.slots) {
                load(a.state + static_cast<int64_t>(from) * n, before);
            } else {
#pragma unroll
                for (int j = 0; j < PER; j++)
                    before[j] = from == -1 ? 0.0f : __builtin_nanf("");
            }
        } else if (!have) {
            norm(row - 1, before, false);
        }
        norm(row, now, true);
        for (int m = 0; m < a.mixes; m++) {
            float mix[PER];
            load(a.mix + static_cast<int64_t>(m) * n, mix);
#pragma unroll
            for (int j = 0; j < PER; j++)
                mix[j] = fmaf(before[j] - now[j], mix[j], now[j]);
            store(out + (static_cast<int64_t>(m) * b.rows + row) * n, mix);
        }
        if (row == span.first) {
            const int to = b.to[s];
            if (to >= 0 && to < b.slots) {
                if (span.last - 1 == row) {
                    store(a.state + static_cast<int64_t>(to) * n, now);
                } else {
                    norm(span.last - 1, before, false);
                    store(a.state + static_cast<int64_t>(to) * n, before);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < PER; j++)
            before[j] = now[j];
        have = true;
    }
}

template <int PER, bool FOURS>
void launch(const MixRowsArgs& a, int run, hipStream_t s)
{
    const dim3 grid((a.batch.rows + run - 1) / run);
    if (a.out_format == ROWS_OUT_F32)
        hipLaunchKernelGGL((mix_rows_kernel<PER, FOURS, float>), grid, dim3(THREADS), 0, s, a, run);
    else if (a.out_format == ROWS_OUT_F16)
        hipLaunchKernelGGL((mix_rows_kernel<PER, FOURS, _Float16>), grid, dim3(THREADS), 0, s, a, run);
    else
        hipLaunchKernelGGL((mix_rows_kernel<PER, FOURS, __bf16>), grid, dim3(THREADS), 0, s, a, run);
}

}  // namespace

hipError_t launch_layernorm_mix_rows(const MixRowsArgs& a, hipStream_t s)
{
    auto aligned16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const bool fours = a.n % 4 == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) && aligned16(a.bias) &&
                       aligned16(a.mix) && aligned16(a.state) && aligned16(a.updated) && aligned16(a.out);
    const int run = a.batch.rows <= 1024 ? 1 : a.batch.rows <= 4096 ? 4 : 8;
    if (a.n <= 8 * THREADS)
        fours ? launch<8, true>(a, run, s) : launch<8, false>(a, run, s);
    else
        fours ? launch<32, true>(a, run, s) : launch<32, false>(a, run, s);
    return hipGetLastError();
}

}  // namespace si
