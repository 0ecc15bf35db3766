// Y = X . W^T of 8-bit integer rows with a scale for each token and each
// output channel: exact int32 sums on the matrix cores, the scales (and the
// residual) applied once to each sum.
#include "si_i8.hpp"

#include "si_copies.hpp"

namespace si {

namespace {

using i32x4 = __attribute__((__vector_size__(4 * sizeof(int)))) int;
using i32x16 = __attribute__((__vector_size__(16 * sizeof(int)))) int;

// What a lane reads in place of columns behind the last one.
__device__ __attribute__((aligned(16))) const uint32_t no_columns[4] = {};

// One output value.
__device__ __forceinline__ void store_y(const GemmI8Args& a, int64_t t, int64_t o, float sx, int sum)
{
    float v = float(sum) * sx * a.w_scale[o];
    if (a.residual)
        v += a.residual[t * a.rows + o];
    a.y[t * a.rows + o] = v;
}

// Four neighbouring channels o..o+3 of token t; `wide`: all there, and the
// rows of y, the residual and the scales aligned for it.
__device__ __forceinline__ void store_y4(const GemmI8Args& a, int64_t t, int64_t o, float sx, i32x4 sum, bool wide)
{
    if (wide) {
        const float4 w = *reinterpret_cast<const float4*>(a.w_scale + o);
        float4 v = make_float4(float(sum[0]) * sx * w.x, float(sum[1]) * sx * w.y, float(sum[2]) * sx * w.z,
                               float(sum[3]) * sx * w.w);
        if (a.residual) {
            const float4 r = *reinterpret_cast<const float4*>(a.residual + t * a.rows + o);
            v.x += r.x, v.y += r.y, v.z += r.z, v.w += r.w;
        }
        *reinterpret_cast<float4*>(a.y + t * a.rows + o) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (o + i < a.rows)
                store_y(a, t, o + i, sx, sum[i]);
    }
}

bool on(const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0; }

// ---- many tokens: tiles in LDS ----------------------------------------------------------

// A workgroup of WM x WN waves owns 32 MT WM channels x 32 NT WN tokens; a
// wave MT x NT blocks of v_mfma_i32_32x32x32_i8.  Steps of 128 columns go
// through two LDS buffers: the copies of the next step (16 bytes a lane,
// straight into LDS) are in flight while this one is multiplied.
//
// LDS rows are 128 bytes; piece p (16 bytes) of row r lies at p ^ ((r >> 1) &
// 7), so the 32 rows that a fragment read takes hit every bank evenly.  The
// copies write LDS in lane order; each lane asks for the piece that belongs
// where its bytes land, still 128 whole bytes of a row to eight lanes.
template <int MT, int NT, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN == 8 ? 2 : 2)
gemm_i8_tile_kernel(const GemmI8Args a, int o_tiles, int t_tiles)
{
    constexpr int BM = 32 * MT * WM, BN = 32 * NT * WN, WAVES = WM * WN;
    constexpr int COPIES = (BM + BN) / 8 / WAVES;         // of a wave and step, 8 rows each
    static_assert(COPIES * 8 * WAVES == BM + BN && BM % 8 == 0, "whole copies");
    __shared__ __align__(16) int8_t lds[2][(BM + BN) * 128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Tiles in the order of the dies that run them: workgroup b runs on die b
    // % 8, and each die takes a run of tiles of its own, eight token tiles
    // beside one another, so their operands meet in its L2.
    const int tiles = o_tiles * t_tiles;
    int id = blockIdx.x;
    {
        const int per = tiles / 8, more = tiles % 8, die = id % 8;
        id = die * per + min(die, more) + id / 8;
    }
    constexpr int ROW = 8;
    const int band = id / (ROW * o_tiles), in = id % (ROW * o_tiles), height = min(ROW, t_tiles - band * ROW);
    const int64_t t0 = int64_t(band * ROW + in % height) * BN, o0 = int64_t(in / height) * BM;

    const int8_t* src[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; i++) {
        const int r = (wave * COPIES + i) * 8 + (lane >> 3);
        const int piece = (lane & 7) ^ ((r >> 1) & 7);
        const int64_t row = r < BM ? min(o0 + r, a.rows - 1) : min(t0 + r - BM, a.m - 1);
        src[i] = (r < BM ? a.w : a.x) + row * a.cols + 16 * piece;
    }
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>(&lds[0][0])));
    auto copy = [&](int64_t k, int buffer) {
        const bool whole = k + 128 <= a.cols;
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
            const int8_t* p = src[i] + k;
            if (!whole) {
                const int r = (wave * COPIES + i) * 8 + (lane >> 3);
                if (k + 16 * ((lane & 7) ^ ((r >> 1) & 7)) >= a.cols)
                    p = reinterpret_cast<const int8_t*>(no_columns);
            }
            copy16_to_lds(p, lds_base + uint32_t(buffer * (BM + BN) * 128 + (wave * COPIES + i) * 1024));
        }
    };

    const int wm = wave % WM, wn = wave / WM;
    const int r = lane & 31, h = lane >> 5;
    int at[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
        at[k] = r * 128 + (((2 * k + h) ^ ((r >> 1) & 7)) << 4);
    i32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                acc[i][j][e] = 0;

    const int8_t* const wl = lds[0] + wm * (32 * MT) * 128;
    const int8_t* const xl = lds[0] + (BM + wn * (32 * NT)) * 128;
    i32x4 fw[2][MT], fx[2][NT];
    auto read = [&](int buffer, int k, int set) {
#pragma unroll
        for (int i = 0; i < MT; i++)
            fw[set][i] = *reinterpret_cast<const i32x4*>(wl + buffer * ((BM + BN) * 128) + at[k] + i * 4096);
#pragma unroll
        for (int j = 0; j < NT; j++)
            fx[set][j] = *reinterpret_cast<const i32x4*>(xl + buffer * ((BM + BN) * 128) + at[k] + j * 4096);
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[set][j], fw[set][i], acc[i][j], 0, 0, 0);
    };
    // One of a step's four quarters: the next fragments are read among the products.
    auto interleave = [&] {
#pragma unroll
        for (int i = 0; i < MT + NT; i++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // one LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one MFMA
        }
        __builtin_amdgcn_sched_group_barrier(0x008, MT * NT, 0);
    };
    const int64_t steps = (a.cols + 127) / 128;
    copy(0, 0);
    if (steps > 1)
        copy(128, 1);
    if (steps > 1)
        wait_copies<COPIES>();
    else
        wait_copies<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0, 0);
    for (int64_t s = 0; s < steps; s++) {
        const int buffer = int(s & 1);
#pragma unroll
        for (int k = 0; k < 3; k++) {
            read(buffer, k + 1, (k + 1) & 1);
            multiply(k & 1);
            interleave();
        }
        // All of this step is in registers: when every wave says so, its
        // buffer takes the step after the next one, and the next one's first
        // fragments are read while the last products run.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + 2 < steps)
            copy((s + 2) * 128, buffer);
        if (s + 1 < steps)
            read(buffer ^ 1, 0, 0);
        multiply(1);
    }
    // A lane holds one channel of each block, its registers the tokens: a
    // store instruction writes whole 128-byte lines of two tokens (four
    // channels a lane, 32 tokens an instruction, took three times as long).
    float sw[MT];
#pragma unroll
    for (int i = 0; i < MT; i++)
        sw[i] = a.w_scale[min(o0 + (wm * MT + i) * 32 + r, a.rows - 1)];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int64_t tj = t0 + (wn * NT + j) * 32 + 4 * h;
        float sx[16];
#pragma unroll
        for (int e = 0; e < 16; e++)
            sx[e] = a.x_scale[min(tj + 8 * (e >> 2) + (e & 3), a.m - 1)];
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const int64_t o = o0 + (wm * MT + i) * 32 + r;
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; e++)
                v[e] = float(acc[i][j][e]) * sx[e] * sw[i];
            if (a.residual) {
                float add[16];
#pragma unroll
                for (int e = 0; e < 16; e++)
                    add[e] = a.residual[min(tj + 8 * (e >> 2) + (e & 3), a.m - 1) * a.rows + min(o, a.rows - 1)];
#pragma unroll
                for (int e = 0; e < 16; e++)
                    v[e] += add[e];
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int64_t t = tj + 8 * (e >> 2) + (e & 3);
                if (t < a.m && o < a.rows)
                    a.y[t * a.rows + o] = v[e];
            }
        }
    }
}

template <int MT, int NT, int WM, int WN>
hipError_t launch_tiles(const GemmI8Args& a, hipStream_t s)
{
    constexpr int BM = 32 * MT * WM, BN = 32 * NT * WN;
    const int64_t o_tiles = (a.rows + BM - 1) / BM, t_tiles = (a.m + BN - 1) / BN;
    gemm_i8_tile_kernel<MT, NT, WM, WN>
        <<<unsigned(o_tiles * t_tiles), 64 * WM * WN, 0, s>>>(a, int(o_tiles), int(t_tiles));
    return hipGetLastError();
}

// ---- few tokens: weights straight into registers -------------------------------------------

// A workgroup owns 16 MT channels and all tokens (up to 16 NT); its waves
// share the columns, 64 at a time in turn, and add their int32 sums in LDS (in
// any order: integers).  A wave's fragments come straight from memory: the
// weights are read once, the tokens from L2.
template <int MT, int NT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
gemm_i8_few_kernel(const GemmI8Args a, bool wide)
{
    constexpr int DEPTH = NT <= 2 ? 4 : 2;               // steps of loads in flight
    __shared__ __align__(16) int sums[16 * NT][16 * MT + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int64_t o0 = int64_t(blockIdx.x) * (16 * MT);
    const int8_t* wp[MT];
    const int8_t* xp[NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
        wp[i] = a.w + min(o0 + 16 * i + r, a.rows - 1) * a.cols + 16 * g;
#pragma unroll
    for (int j = 0; j < NT; j++)
        xp[j] = a.x + min(int64_t(16 * j + r), a.m - 1) * a.cols + 16 * g;
    for (int i = threadIdx.x; i < 16 * NT * (16 * MT + 4); i += 64 * WAVES)
        (&sums[0][0])[i] = 0;
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
            acc[i][j] = i32x4{0, 0, 0, 0};
    const int64_t steps = (a.cols + 63) / 64;
    for (int64_t s0 = wave; s0 < steps; s0 += WAVES * DEPTH) {
        i32x4 fw[DEPTH][MT], fx[DEPTH][NT];
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int64_t k = (s0 + d * WAVES) * 64;
            const bool in = k + 16 * g < a.cols;
#pragma unroll
            for (int i = 0; i < MT; i++)
                fw[d][i] = in ? *reinterpret_cast<const i32x4*>(wp[i] + k) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NT; j++)
                fx[d][j] = in ? *reinterpret_cast<const i32x4*>(xp[j] + k) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[d][i], fx[d][j], acc[i][j], 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                atomicAdd(&sums[16 * j + r][16 * i + 4 * g + e], acc[i][j][e]);
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT * (4 * MT); i += 64 * WAVES) {
        const int64_t t = i / (4 * MT), o = o0 + 4 * (i % (4 * MT));
        if (t < a.m && o < a.rows)
            store_y4(a, t, o, a.x_scale[t], *reinterpret_cast<const i32x4*>(&sums[t][4 * (i % (4 * MT))]),
                     wide && o + 4 <= a.rows);
    }
}

template <int MT, int NT, int WAVES>
hipError_t launch_few(const GemmI8Args& a, bool wide, hipStream_t s)
{
    gemm_i8_few_kernel<MT, NT, WAVES><<<unsigned((a.rows + 16 * MT - 1) / (16 * MT)), 64 * WAVES, 0, s>>>(a, wide);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s)
{
    const bool wide = a.rows % 4 == 0 && on(a.y, 16) && on(a.w_scale, 16) && on(a.residual, 16);
    if (a.m <= 16)
        return launch_few<1, 1, 8>(a, wide, s);
    if (a.m <= 32)
        return launch_few<2, 2, 16>(a, wide, s);
    if (a.m <= 64)
        return launch_few<2, 4, 16>(a, wide, s);
    const int64_t big = ((a.rows + 255) / 256) * ((a.m + 255) / 256);
    if (big >= 192)
        return launch_tiles<4, 2, 2, 4>(a, s);
    return launch_tiles<2, 2, 2, 2>(a, s);
}

}  // namespace si
