// LayerNorm of token rows, mixed with the row before of the same sequence
// (PortableRwkv7GraphProvider.cs:163-170, 180-184, 202-210, 280-288).
#include "si_sequences.hpp"
#include "si_lanes.hpp"

#include <type_traits>

namespace si {
namespace {

constexpr int PER = 8;   // values of a row a thread

// How a thread's eight values of a row lie: ALIGNED: neighbours at multiples of 16 bytes.  NEIGHBOURS: at any address; where
// eight does not divide the width, the last thread takes the last eight, of which the thread before has some too: it leaves them out of the
// sums and writes them again (the state's are read two barriers before).  SINGLE: every THREADS-th (widths under eight; 3900 rows of
// 2047 in six mixes so 56 us, as neighbours 41).
enum Lie { ALIGNED, NEIGHBOURS, SINGLE };
typedef float AlignedFour __attribute__((ext_vector_type(4)));
typedef float AnyFour __attribute__((ext_vector_type(4), aligned(4)));

// A workgroup of THREADS, as many as a row has eights, takes `run` rows one after another (4000 rows of 768 in six mixes 15 us,
// with 256 threads 21).  Weights and mixes stay in registers, and so does the row before: only a run's
// first row is normalised twice.  The next row is requested while this one is normalised.  The sequence's
// state is read by the workgroup of its first row, which also normalises the last row for the state's slot:
// the slot has one reader and writer, whatever the other workgroups have done by then.
// Bound by HBM: 4 bytes in (8 with a residual, 4 more out) and 2 or 4 out a mix (4163 rows of 2048 with the residual in six mixes 37.5 us, 5.5
// TB/s); a single row by its round trips (16 rows 4.5 us).
// HELD: mixes that registers hold (0: they are loaded with every row: 1024 threads leave no room for more than one; 976 rows of 8192 in
// six mixes 39 us, 1953 of 4096 34).
// PAST: outputs go past the L2s.
template <int THREADS, Lie LIE, int HELD, bool PAST, typename OUT>
__global__ __launch_bounds__(THREADS) void mix_rows_kernel(MixRowsArgs a, int run)
{
    constexpr int WAVES = THREADS / 64;
    __shared__ float s_sum[WAVES], s_squares[WAVES];
    __shared__ int s_at[WAVES];
    const int t = threadIdx.x, wave = t >> 6, n = a.n;
    const RowBatch& b = a.batch;
    const int base = LIE == NEIGHBOURS ? min(PER * t, n - PER) : PER * t;
    auto place = [&](int j) { return LIE != SINGLE ? base + j : t + THREADS * j; };
    auto counts = [&](int j) { return place(j) < n && (LIE != NEIGHBOURS || place(j) >= PER * t); };
    auto load = [&](const float* p, float* v) {
        if constexpr (LIE != SINGLE) {
            using Four = std::conditional_t<LIE == ALIGNED, AlignedFour, AnyFour>;
            Four f[2] = {};
            if (PER * t < n) {
                f[0] = *reinterpret_cast<const Four*>(p + base);
                f[1] = *reinterpret_cast<const Four*>(p + base + 4);
            }
#pragma unroll
            for (int j = 0; j < PER; j++)
                v[j] = f[j / 4][j % 4];
        } else {
#pragma unroll
            for (int j = 0; j < PER; j++)
                v[j] = place(j) < n ? p[place(j)] : 0.0f;
        }
    };
    auto store = [&](auto* p, const float* v) {
        using T = std::remove_reference_t<decltype(*p)>;
        if constexpr (LIE != SINGLE) {
            typedef T Eight __attribute__((ext_vector_type(PER), aligned(LIE == ALIGNED ? 16 : sizeof(T))));
            const Eight e = {static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3]),
                             static_cast<T>(v[4]), static_cast<T>(v[5]), static_cast<T>(v[6]), static_cast<T>(v[7])};
            if (PER * t < n) {
                if constexpr (PAST)   // (a choice at run time is merged into one ordinary store)
                    __builtin_nontemporal_store(e, reinterpret_cast<Eight*>(p + base));
                else
                    *reinterpret_cast<Eight*>(p + base) = e;
            }
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

    // what the first row needs, requested before its sequence is known
    int row = blockIdx.x * run;
    const int end = min(row + run, b.rows);
    const int64_t width = n;
    float x[PER], add[PER], weight[PER], bias[PER], mix[HELD ? HELD : 1][PER];
    auto request = [&](int r) {
        load(a.x + r * width, x);
        if (a.residual)
            load(a.residual + r * width, add);
    };
    request(row);
    int at = 0;
    for (int i = t; i < b.sequences; i += THREADS)
        at += b.starts[i + 1] <= row;
    load(a.weight, weight);
    load(a.bias, bias);
#pragma unroll
    for (int m = 0; m < HELD; m++)
        if (m < a.mixes)
            load(a.mix + m * width, mix[m]);
    // the sequence of the run's first row: as many as end at or before it
    at = static_cast<int>(rows_sum(row_sum<16>(static_cast<float>(at))));   // at most 4096: exact
    if ((t & 63) == 0)
        s_at[wave] = at;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++)
        s += s_at[w];
    s = __builtin_amdgcn_readfirstlane(s);

    // the norm of the requested row
    auto norm = [&](float* v) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            v[j] = a.residual ? x[j] + add[j] : x[j];
            sum += LIE != NEIGHBOURS || counts(j) ? v[j] : 0.0f;
        }
        return sum;
    };
    auto normalise = [&](float* v, float sum) {
        const float mean = block_sum(sum, s_sum) / static_cast<float>(n);
        float squares = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            v[j] -= mean;
            squares = counts(j) ? fmaf(v[j], v[j], squares) : squares;
        }
        const float inv = 1.0f / sqrtf(block_sum(squares, s_squares) / static_cast<float>(n) + a.eps);
#pragma unroll
        for (int j = 0; j < PER; j++)
            v[j] = fmaf(v[j] * inv, weight[j], bias[j]);
    };
    auto other_row = [&](int r, float* v) {
        request(r);
        normalise(v, norm(v));
    };

    float before[PER], now[PER];
    bool have = false;        // `before` is the row before
    bool requested = true;    // x and add are this row's
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
            have = requested = false;
            continue;
        }
        if (a.mixes > 0 && row == span.first) {
            const int from = b.from[s];
            if (from >= 0 && from < b.slots) {
                load(a.state + from * width, before);
            } else {
#pragma unroll
                for (int j = 0; j < PER; j++)
                    before[j] = from == -1 ? 0.0f : __builtin_nanf("");
            }
        } else if (a.mixes > 0 && !have) {
            other_row(row - 1, before);
            requested = false;
        }
        if (!requested)
            request(row);
        const float sum = norm(now);
        if (a.residual)
            store(a.updated + row * width, now);
        requested = row + 1 < end;
        if (requested)
            request(row + 1);
        normalise(now, sum);
        if (a.mixes == 0) {
            store(out + row * width, now);
            continue;
        }
        auto mixed = [&](int m, const float* held) {
            float v[PER];
#pragma unroll
            for (int j = 0; j < PER; j++)
                v[j] = fmaf(before[j] - now[j], held[j], now[j]);
            store(out + (static_cast<int64_t>(m) * b.rows + row) * width, v);
        };
        if constexpr (HELD > 0) {
#pragma unroll
            for (int m = 0; m < HELD; m++)
                if (m < a.mixes)
                    mixed(m, mix[m]);
        } else {
            for (int m = 0; m < a.mixes; m++) {
                load(a.mix + m * width, mix[0]);
                mixed(m, mix[0]);
            }
        }
        if (row == span.first) {
            const int to = b.to[s];
            if (to >= 0 && to < b.slots) {
                if (span.last - 1 == row) {
                    store(a.state + to * width, now);
                } else {
                    other_row(span.last - 1, before);
                    requested = false;
                    store(a.state + to * width, before);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < PER; j++)
            before[j] = now[j];
        have = true;
    }
}

template <int THREADS, Lie LIE, int HELD, bool PAST>
void launch(const MixRowsArgs& a, int run, hipStream_t s)
{
    const dim3 grid((a.batch.rows + run - 1) / run);
    if (a.out_format == ROWS_OUT_F32)
        hipLaunchKernelGGL((mix_rows_kernel<THREADS, LIE, HELD, PAST, float>), grid, dim3(THREADS), 0, s, a, run);
    else if (a.out_format == ROWS_OUT_F16)
        hipLaunchKernelGGL((mix_rows_kernel<THREADS, LIE, HELD, PAST, _Float16>), grid, dim3(THREADS), 0, s, a, run);
    else
        hipLaunchKernelGGL((mix_rows_kernel<THREADS, LIE, HELD, PAST, __bf16>), grid, dim3(THREADS), 0, s, a, run);
}

template <int THREADS, int HELD>
void launch(const MixRowsArgs& a, bool aligned, bool past, int run, hipStream_t s)
{
    if (aligned && past)
        launch<THREADS, ALIGNED, HELD, true>(a, run, s);
    else if (aligned)
        launch<THREADS, ALIGNED, HELD, false>(a, run, s);
    else if (past)
        launch<THREADS, NEIGHBOURS, HELD, true>(a, run, s);
    else
        launch<THREADS, NEIGHBOURS, HELD, false>(a, run, s);
}

template <int THREADS>
void launch(const MixRowsArgs& a, hipStream_t s)
{
    constexpr int MANY = THREADS == 1024 ? 0 : MIX_MAX;
    auto aligned16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const bool aligned = a.n % 8 == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) && aligned16(a.bias) &&
                        aligned16(a.mix) && aligned16(a.state) && aligned16(a.updated) && aligned16(a.out);
    // Outputs that the L2s (32 MiB) cannot keep for the next kernel go past them: 4000 rows of 2048 values in six mixes
    // take 35 us instead of 47.  Smaller ones stay there for the products that read them.
    const int64_t out = static_cast<int64_t>(a.batch.rows) * a.n *
                        ((a.out_format == ROWS_OUT_F32 ? 4 : 2) * (a.mixes > 0 ? a.mixes : 1) + (a.residual ? 4 : 0));
    const bool past = out > (16 << 20);
    // Runs such that so many waves a compute unit have one each, of wide rows as many whole workgroups (976 rows of 8192 in six mixes 39
    // us, at 0.9 workgroups a compute unit 52); few rows one a workgroup.  4000 rows of 2048 take so, 9 rows a run, 35 us; with runs of 3,
    // 4, 5 and 8 rows 38, 41, 45 and 36 (odd ones keep the workgroups' rows from lying a power of two apart).
    const int waves = a.mixes <= 1 ? 20 : 7, most = waves * 64 / THREADS, rows = a.batch.rows;
    const int resident = THREADS < 512 ? 256 * waves * 64 / THREADS : 256 * (most > 1 ? most : 1);
    const int run = rows <= resident ? 1 : rows < 15 * resident ? ((rows + resident - 1) / resident) | 1 : 15;
    if (a.mixes <= 1)
        launch<THREADS, 1>(a, aligned, past, run, s);
    else
        launch<THREADS, MANY>(a, aligned, past, run, s);
}

}  // namespace

hipError_t launch_layernorm_mix_rows(const MixRowsArgs& a, hipStream_t s)
{
    if (a.n < PER)
        launch<64, SINGLE, MIX_MAX, false>(a, 1, s);
    else if (a.n <= 64 * PER)
        launch<64>(a, s);
    else if (a.n <= 128 * PER)
        launch<128>(a, s);
    else if (a.n <= 256 * PER)
        launch<256>(a, s);
    else if (a.n <= 512 * PER)
        launch<512>(a, s);
    else if (a.n <= 768 * PER)
        launch<768>(a, s);
    else
        launch<1024>(a, s);
    return hipGetLastError();
}

}  // namespace si
