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

// Tile `id` of the launch.  Tiles go in the order of the dies that run them:
// workgroup b runs on die b % 8, and each die takes a run of tiles of its
// own, eight token tiles beside one another, so their operands meet in its L2.
__device__ __forceinline__ void tile_of(int id, int o_tiles, int t_tiles, int bm, int bn, int64_t* o0, int64_t* t0)
{
    const int tiles = o_tiles * t_tiles, per = tiles / 8, more = tiles % 8, die = id % 8;
    id = die * per + min(die, more) + id / 8;
    constexpr int ROW = 8;
    const int band = id / (ROW * o_tiles), in = id % (ROW * o_tiles), height = min(ROW, t_tiles - band * ROW);
    *t0 = int64_t(band * ROW + in % height) * bn;
    *o0 = int64_t(in / height) * bm;
}

// A pointer that is the same in all lanes, in scalar registers.
__device__ __forceinline__ const int8_t* uniform(const int8_t* p)
{
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const int8_t*>(uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(v)))) |
                                           uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(v >> 32)))) << 32);
}

// A 32 x 32 block of sums: this lane holds channel o, register e token t0 + 8
// (e / 4) + e % 4, whose scales are sx[8 (e / 4) + e % 4] in LDS.  A store
// instruction writes whole 128-byte lines of two tokens (four channels a
// lane, 32 tokens an instruction, took three times as long).  WHOLE: every
// token and channel of the tile is there.  Kept in one piece: spread over
// the blocks before it, its values would need registers that the sums hold.
template <bool WHOLE>
__device__ __forceinline__ void store_block(const GemmI8Args& a, const i32x16& acc, const float* sx, int64_t t0, int64_t o,
                                            float sw)
{
    const int64_t first = WHOLE ? t0 * a.rows + o : min(t0, a.m - 1) * a.rows + min(o, a.rows - 1);
    float* const y = a.y + first;
    const float* const add = a.residual + first;
    const uint32_t rows = uint32_t(a.rows);
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; e++)
        v[e] = float(acc[e]) * sx[8 * (e >> 2) + (e & 3)] * sw;
    if (a.residual) {
        float r[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int t = 8 * (e >> 2) + (e & 3);
            r[e] = WHOLE || (t0 + t < a.m && o < a.rows) ? add[t * rows] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 16; e++)
            v[e] += r[e];
    }
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const int t = 8 * (e >> 2) + (e & 3);
        if (WHOLE || (t0 + t < a.m && o < a.rows))
            y[t * rows] = v[e];
    }
    __builtin_amdgcn_sched_barrier(0);
}

// The blocks of a wave, MT of channels from o0 on and NT of tokens from t0 on.
template <int MT, int NT>
__device__ __forceinline__ void store_blocks(const GemmI8Args& a, const i32x16 (&acc)[MT][NT], const float* sx, int64_t t0,
                                             int64_t o0)
{
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    float sw[MT];
#pragma unroll
    for (int i = 0; i < MT; i++)
        sw[i] = a.w_scale[min(o0 + i * 32 + r, a.rows - 1)];
    if (o0 + 32 * MT <= a.rows && t0 + 32 * NT <= a.m) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++)
                store_block<true>(a, acc[i][j], sx + j * 32 + 4 * h, t0 + j * 32 + 4 * h, o0 + i * 32 + r, sw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++)
                store_block<false>(a, acc[i][j], sx + j * 32 + 4 * h, t0 + j * 32 + 4 * h, o0 + i * 32 + r, sw[i]);
    }
}

// A workgroup owns 32 MT WM channels x 32 NT WN tokens: WM x WN waves with
// MT x NT blocks of v_mfma_i32_32x32x32_i8 each, WK times over with the
// columns of a step shared between them (their sums meet in LDS at the end).
// Steps of 128 PER columns go through a ring of LDS buffers that asynchronous
// copies fill, 16 bytes a lane straight into LDS, RING - 1 steps ahead; a
// copy's address is a scalar base that moves and an offset that does not
// (with 64-bit addresses per lane a step of the 64 x 64 tile took half as
// long again).  PER 2 halves the barriers of the smallest tile, whose step
// is otherwise a barrier, two LDS reads and one MFMA (64 x 4096 x 4096 9.0 ->
// 6.9 us); the larger tiles gain nothing from it.
//
// LDS rows are 128 bytes; piece p (16 bytes) of row r lies at p ^ ((r >> 1) &
// 7), so the 32 rows that a fragment read takes hit every bank evenly
// (no conflicts counted).  The copies write LDS in lane order; each lane asks
// for the piece that belongs where its bytes land, still 128 whole bytes of a
// row to eight lanes.
//
// 4093 x 8192 x 4096 takes 136 us (2.0 POP/s), 4096 x 16384 x 8192 519 us
// (2.12); the vendor's plain product of 8-bit integers, int32 out and no
// scales, reaches 2.18 and 2.10 on such shapes.  In a single workgroup a step
// of the 256 x 256 tile takes 1.2 us, near the LDS traffic of its fragments;
// with all CUs at work 1.6 us, and a form with half that traffic (128 x 128
// a wave, one wave a SIMD, 0.9 us a step alone) gained nothing there.
template <int MT, int NT, int WM, int WN, int WK, int RING, int PER>
__global__ void __launch_bounds__(64 * WM * WN * WK)
gemm_i8_tile_kernel(const GemmI8Args a, int o_tiles, int t_tiles)
{
    constexpr int BM = 32 * MT * WM, BN = 32 * NT * WN, WAVES = WM * WN * WK;
    constexpr int QUARTERS = 4 / WK * PER;                // 32-column pieces of a step, of a wave
    constexpr int ROUNDS = (BM + BN) / 8 / WAVES;         // copies of a wave for 128 columns, 8 rows each
    constexpr int COPIES = ROUNDS * PER;
    constexpr int SLAB = (BM + BN) * 128;
    static_assert(ROUNDS * 8 * WAVES == BM + BN && BM % 8 == 0, "whole copies");
    static_assert((RING & (RING - 1)) == 0 && (RING - 1) * COPIES < 64, "buffers by mask, vmcnt range");
    __shared__ __align__(16) int8_t lds[RING][PER * SLAB];
    __shared__ __align__(16) float sx[BN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    int64_t o0, t0;
    tile_of(blockIdx.x, o_tiles, t_tiles, BM, BN, &o0, &t0);
    for (int i = threadIdx.x; i < BN; i += 64 * WAVES)
        sx[i] = a.x_scale[min(t0 + i, a.m - 1)];

    // copy i of this wave: eight rows of the weights or of the tokens
    uint32_t off[ROUNDS];
    const int8_t* base[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int r0 = (wave * ROUNDS + i) * 8, r = r0 + (lane >> 3), piece = (lane & 7) ^ ((r >> 1) & 7);
        const bool of_w = r0 < BM;
        const int64_t row = of_w ? min(int64_t(r), a.rows - 1 - o0) : min(int64_t(r - BM), a.m - 1 - t0);
        off[i] = uint32_t(row * a.cols) + 16 * piece;
        base[i] = uniform(of_w ? a.w + o0 * a.cols : a.x + t0 * a.cols);
    }
    const uint32_t lds_base =
        __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>(&lds[0][0])) + wave * ROUNDS * 1024);
    const int cols = int(a.cols), steps = (cols + 128 * PER - 1) / (128 * PER), wholes = cols / (128 * PER);
    auto copy = [&](int s) {
        const uint32_t to = lds_base + (s & (RING - 1)) * (PER * SLAB);
#pragma unroll
        for (int p = 0; p < PER; p++) {
            const int k = (s * PER + p) * 128;
            if (s < wholes) {
#pragma unroll
                for (int i = 0; i < ROUNDS; i++)
                    copy16_to_lds(off[i], base[i] + k, to + p * SLAB + i * 1024);
            } else {
#pragma unroll
                for (int i = 0; i < ROUNDS; i++) {
                    const int r = (wave * ROUNDS + i) * 8 + (lane >> 3), piece = (lane & 7) ^ ((r >> 1) & 7);
                    const bool in = k + 16 * piece < cols;
                    copy16_to_lds(in ? base[i] + k + off[i] : reinterpret_cast<const int8_t*>(no_columns),
                                  to + p * SLAB + i * 1024);
                }
            }
        }
    };

    const int wm = wave % WM, wn = wave / WM % WN, wk = wave / (WM * WN);
    const int r = lane & 31, h = lane >> 5;
    int at[QUARTERS];
#pragma unroll
    for (int k = 0; k < QUARTERS; k++)
        at[k] = r * 128 + (((2 * (wk * (4 / WK) + k % (4 / WK)) + h) ^ ((r >> 1) & 7)) << 4) + k / (4 / WK) * SLAB;
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
            fw[set][i] = *reinterpret_cast<const i32x4*>(wl + buffer * (PER * SLAB) + at[k] + i * 4096);
#pragma unroll
        for (int j = 0; j < NT; j++)
            fx[set][j] = *reinterpret_cast<const i32x4*>(xl + buffer * (PER * SLAB) + at[k] + j * 4096);
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
    for (int i = 0; i < RING && i < steps; i++)
        copy(i);
    if (steps >= RING)
        wait_copies<(RING - 1) * COPIES>();
    else
        wait_copies<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0, 0);
    for (int s = 0; s < steps; s++) {
        const int buffer = s & (RING - 1);
#pragma unroll
        for (int k = 0; k + 1 < QUARTERS; k++) {
            read(buffer, k + 1, (k + 1) & 1);
            multiply(k & 1);
            interleave();
        }
        // All of this step is in registers: when every wave says so, its
        // buffer takes the step RING steps on, and the next one's first
        // fragments are read while the last products run.
        if (s + RING <= steps)
            wait_copies<(RING - 2) * COPIES>();
        else
            wait_copies<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + RING < steps)
            copy(s + RING);
        constexpr int LAST = (QUARTERS - 1) & 1;
        if (s + 1 < steps)
            read((buffer + 1) & (RING - 1), 0, LAST ^ 1);
        multiply(LAST);
        if constexpr (LAST == 0) {
#pragma unroll
            for (int i = 0; i < MT; i++)
                fw[0][i] = fw[1][i];
#pragma unroll
            for (int j = 0; j < NT; j++)
                fx[0][j] = fx[1][j];
        }
    }
    if constexpr (WK > 1) {
        // The waves that shared a block's columns add their sums in LDS.
        static_assert(WK * BM * BN * 4 <= sizeof(lds), "the sums fit the ring");
        int* const sums = reinterpret_cast<int*>(&lds[0][0]);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    sums[(wk * BN + (wn * NT + j) * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) * BM + (wm * MT + i) * 32 + r] =
                        acc[i][j][e];
        __syncthreads();
        constexpr int OUTS = BM * BN / (64 * WAVES);      // of a thread
        const int o_in = threadIdx.x % BM;
        const int64_t o = o0 + o_in;
        float v[OUTS], add[OUTS];
        const float sw = a.w_scale[min(o, a.rows - 1)];
#pragma unroll
        for (int e = 0; e < OUTS; e++) {
            const int t_in = int(threadIdx.x) / BM + e * (64 * WAVES / BM);
            const int64_t t = min(t0 + t_in, a.m - 1);
            int sum = 0;
#pragma unroll
            for (int k = 0; k < WK; k++)
                sum += sums[(k * BN + t_in) * BM + o_in];
            v[e] = float(sum) * sx[t_in];
            add[e] = a.residual ? a.residual[t * a.rows + min(o, a.rows - 1)] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < OUTS; e++) {
            const int64_t t = t0 + int(threadIdx.x) / BM + e * (64 * WAVES / BM);
            if (t < a.m && o < a.rows) {
                float y = v[e] * sw;
                if (a.residual)
                    y += add[e];
                a.y[t * a.rows + o] = y;
            }
        }
        return;
    }
    store_blocks<MT, NT>(a, acc, sx + wn * NT * 32, t0 + wn * NT * 32, o0 + wm * MT * 32);
}

template <int MT, int NT, int WM, int WN, int WK, int RING, int PER>
hipError_t launch_tiles(const GemmI8Args& a, hipStream_t s)
{
    constexpr int BM = 32 * MT * WM, BN = 32 * NT * WN;
    const int64_t o_tiles = (a.rows + BM - 1) / BM, t_tiles = (a.m + BN - 1) / BN;
    gemm_i8_tile_kernel<MT, NT, WM, WN, WK, RING, PER>
        <<<unsigned(o_tiles * t_tiles), 64 * WM * WN * WK, 0, s>>>(a, int(o_tiles), int(t_tiles));
    return hipGetLastError();
}

// ---- few tokens: weights straight into registers -------------------------------------------

// Up to 16 tokens on few channels: a workgroup owns 16 channels, its waves share the columns,
// 64 at a time in turn, and add their int32 sums in LDS (in any order:
// integers).  Fragments of v_mfma_i32_16x16x64_i8 come straight from memory,
// four steps of them in flight: the weights are read once, the tokens from
// L2.  2048 channels of 8192 columns take 6.8 us with one token, 2.5 TB/s of
// weights: 128 workgroups, and the launch.
__global__ void __launch_bounds__(512)
gemm_i8_few_kernel(const GemmI8Args a, bool wide)
{
    constexpr int DEPTH = 4, WAVES = 8;
    __shared__ __align__(16) int sums[16][16 + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int64_t o0 = int64_t(blockIdx.x) * 16;
    const int8_t* const wp = a.w + min(o0 + r, a.rows - 1) * a.cols + 16 * g;
    const int8_t* const xp = a.x + min(int64_t(r), a.m - 1) * a.cols + 16 * g;
    for (int i = threadIdx.x; i < 16 * (16 + 4); i += 64 * WAVES)
        (&sums[0][0])[i] = 0;
    i32x4 acc = {0, 0, 0, 0};
    const int cols = int(a.cols), steps = (cols + 63) / 64;
    for (int s0 = wave; s0 < steps; s0 += WAVES * DEPTH) {
        i32x4 fw[DEPTH], fx[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int k = (s0 + d * WAVES) * 64;
            const bool in = k + 16 * g < cols;
            fw[d] = in ? *reinterpret_cast<const i32x4*>(wp + k) : i32x4{0, 0, 0, 0};
            fx[d] = in ? *reinterpret_cast<const i32x4*>(xp + k) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[d], fx[d], acc, 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; e++)
        atomicAdd(&sums[r][4 * g + e], acc[e]);
    __syncthreads();
    if (threadIdx.x < 64) {
        const int64_t t = threadIdx.x / 4, o = o0 + 4 * (threadIdx.x % 4);
        if (t < a.m && o < a.rows)
            store_y4(a, t, o, a.x_scale[t], *reinterpret_cast<const i32x4*>(&sums[t][4 * (threadIdx.x % 4)]),
                     wide && o + 4 <= a.rows);
    }
}

hipError_t launch_few(const GemmI8Args& a, bool wide, hipStream_t s)
{
    gemm_i8_few_kernel<<<unsigned((a.rows + 15) / 16), 512, 0, s>>>(a, wide);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s)
{
    const bool wide = a.rows % 4 == 0 && on(a.y, 16) && on(a.w_scale, 16) && on(a.residual, 16);
    auto tiles = [&](int64_t n) { return ((a.rows + n - 1) / n) * ((a.m + n - 1) / n); };
    // Few tokens and too few channels for a tile of 32 on half the CUs: the
    // form whose workgroups take 16 (one token, 2048 channels of 8192 columns
    // 6.8 / 9.7 us; at 8192 channels of 4096 columns and 16 tokens 9.7 / 7.7).
    if (a.m <= 16 && tiles(32) < 128)
        return launch_few(a, wide, s);
    // The largest tile that still gives the 256 CUs one each: large tiles
    // read less per product, small ones fill the chip.  Both sides measured
    // at 4096 columns (us, tokens x channels): 256 x 256 and 128 x 128 at 2048
    // x 8192 74 / 80, at 2048 x 4096 (128 tiles) 50 / 41; 128 and 64 at 1024 x
    // 4096 27 / 33, at 512 x 4096 (128 tiles) 25 / 18; 64 and 32 at 64 x 16384
    // 16.7 / 23, at 32 x 16384 (512 tiles of 32: two a CU) 15.0 / 14.1, at 64 x
    // 4096 10.4 / 6.9.
    if (tiles(256) >= 224)
        return launch_tiles<4, 2, 2, 4, 1, 2, 1>(a, s);
    if (tiles(128) >= 192)
        return launch_tiles<2, 2, 2, 2, 1, 2, 1>(a, s);
    if (tiles(32) > 512)
        return launch_tiles<1, 1, 2, 2, 2, 4, 1>(a, s);
    return launch_tiles<1, 1, 1, 1, 4, 4, 2>(a, s);
}

}  // namespace si
