// The newest rows of many sequences into a paged cache (rotary embedding on
// the way), and rows of the pages back as FP32.
//
// A workgroup serves one row of the batch: its waves take the row's heads,
// four neighbouring values a lane, so a 4-bit block of 32 values is eight
// lanes of the wave and its largest value a DPP reduction.  The
// rotation runs in FP64 (angle, cosine, sine, products; rounded to FP32
// once): positions of any size keep their angle, and a key's codes do not
// depend on which kernel rotated it.
//
// Bound by bytes: five prompts of up to 1500 rows (24 + 2 x 8 heads of 128, 4-bit
// pages) take 30 us over the same buffers again and again, 4.7 TB/s with the help of
// the cache before HBM, and 40 over others each time, with one row a workgroup (two
// values a lane, loads behind the turns, neighbouring rows on different dies: 46 where
// this takes 30); 64 single rows take
// 4.6 us, five workgroups a row, of which the search for the row's sequence, its
// page and the turns are three round trips.
#include "si_paged.hpp"

#include "si_lanes.hpp"

#include <hip/hip_fp16.h>

namespace si {

namespace {

// Where the batch's row t belongs; page < 0: nowhere (behind the last
// sequence, a position outside the table, a page outside the pool).
struct Place {
    int64_t page;
    int slot;
    int position;
    bool live;                 // the row belongs to a sequence
};

// All threads of the workgroup look for the sequence (the count of
// sequences that end at or before row t) together: one round trip for up to
// 256 sequences.
__device__ __forceinline__ Place find_place(const PagedBatch& b, const PagedCache& c, int t)
{
    __shared__ int counts[4];
    int n = 0;
    for (int s = threadIdx.x; s < b.sequences; s += 256)
        n += b.starts[s + 1] <= t;
    for (int m = 32; m; m >>= 1)
        n += __shfl_xor(n, m);
    if ((threadIdx.x & 63) == 0)
        counts[threadIdx.x >> 6] = n;
    __syncthreads();
    const int s = counts[0] + counts[1] + counts[2] + counts[3];
    Place r{-1, 0, 0, false};
    if (s >= b.sequences)
        return r;
    const int first = b.starts[s], end = b.starts[s + 1];
    if (t < first || t >= end)
        return r;
    r.live = true;
    const int64_t p = int64_t(b.lengths[s]) - end + t;
    if (p < 0 || p >= int64_t(b.max_pages) << c.page_shift)
        return r;
    const int page = b.table[int64_t(s) * b.max_pages + (p >> c.page_shift)];
    if (page < 0 || page >= c.pages)
        return r;
    r.page = page;
    r.slot = int(p) & (c.page_size - 1);
    r.position = int(p);
    return r;
}

// The 4-bit block that eight lanes hold, four values each: scale = the value of
// largest magnitude (the first of them) / -8 in FP16, code = value / scale
// rounded to the nearest (ties to even) + 8.  A value that FP16 could not
// hold makes the whole block NaN.
__device__ __forceinline__ void block_codes(const float* v, int lane, uint16_t* codes, uint16_t* scale)
{
    float mine = v[0];
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        mine = fabsf(v[j]) > fabsf(mine) ? v[j] : mine;        // (the first of equal ones stays)
        odd |= !(fabsf(v[j]) <= 65504.0f);                     // NaN too
    }
    const float top = row_max<8>(fabsf(mine));
    const uint32_t shift = lane & 56;
    const uint32_t holders = uint32_t(__ballot(fabsf(mine) == top) >> shift) & 0xFFu;
    const uint32_t bad = uint32_t(__ballot(odd) >> shift) & 0xFFu;
    const float first = __shfl(mine, int(shift) + (holders ? __ffs(holders) - 1 : 0));
    uint16_t d = __half_as_ushort(__float2half_rn(first / -8.0f));
    const float df = __half2float(__ushort_as_half(d));
    uint32_t q = 0x8888;
    if (bad) {
        d = 0x7E00;
    } else if (df == 0.0f) {
        d = 0;                                                 // a block of zeros, whatever their signs
    } else {
        q = 0;
#pragma unroll
        for (int j = 0; j < 4; j++)
            q |= uint32_t(int(fminf(fmaxf(rintf(v[j] / df) + 8.0f, 0.0f), 15.0f))) << (4 * j);
    }
    *codes = uint16_t(q);
    *scale = d;
}

// Values beside each other (qkv and query are aligned to 4 bytes only).
typedef float float4_4 __attribute__((ext_vector_type(4), aligned(4)));

// The batch's row of workgroup x: the rows of a page on one die (workgroup b
// runs on die b % 8), whose L2 joins their 64-byte rows and 2-byte scales to
// whole lines.
__device__ __forceinline__ int row_of_workgroup() { return int(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8); }

template <int D, bool Q4>
__global__ void __launch_bounds__(256)
paged_append_kernel(const PagedAppendArgs a, int per_group)
{
    constexpr int PER = 256 / D;                   // heads a wave serves at once
    __shared__ double turn[2][64];                 // cos, sin of the row's pairs
    const int t = row_of_workgroup();
    if (t >= a.batch.rows)
        return;
    const Place at = find_place(a.batch, a.cache, t);
    if (at.page < 0)
        return;                                    // the whole workgroup
    const int half = a.rotary >> 1;
    const int lane = threadIdx.x & 63;
    const int kv = a.cache.kv_heads, total = a.heads + 2 * kv;
    const int i0 = 4 * (lane % (D / 4));           // this lane's values i0 .. i0 + 3 of its head
    auto partner = [&](int i) { return i < half ? i + half : i < 2 * half ? i - half : i; };
    const float* row = a.qkv + int64_t(t) * total * D;
    const int64_t head_bytes = paged_head_bytes(Q4, a.cache.page_size, D);
    const int end = min(total, (int(blockIdx.y) + 1) * per_group);
    // A lane's values and their partners; asked for before they are needed.
    float4_4 own, other;
    auto load = [&](int h0) {
        // (a lane without a head works on the last one and stores nothing)
        const int h = min(h0 + lane / (D / 4), end - 1);
        const float* const x = row + int64_t(h) * D;
        own = *reinterpret_cast<const float4_4*>(x + i0);
        other = own;
        if (h < a.heads + kv) {
            if (half & 3) {                        // the four may lie on different sides
#pragma unroll
                for (int j = 0; j < 4; j++)
                    other[j] = x[partner(i0 + j)];
            } else {
                other = *reinterpret_cast<const float4_4*>(x + partner(i0));
            }
        }
    };
    int h0 = int(blockIdx.y) * per_group + int(threadIdx.x >> 6) * PER;
    if (h0 < end)
        load(h0);
    if (int(threadIdx.x) < half) {
        double s, c;
        sincos(double(at.position) * double(a.frequencies[threadIdx.x]), &s, &c);
        turn[0][threadIdx.x] = c * double(a.rope_scale);
        turn[1][threadIdx.x] = s * double(a.rope_scale);
    }
    __syncthreads();
    // the lane's turns: the same for every head
    double c[4] = {}, s[4] = {};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = i0 + j;
        if (i < 2 * half) {
            const int pair = i < half ? i : i - half;
            c[j] = turn[0][pair];
            s[j] = i < half ? -turn[1][pair] : turn[1][pair];
        }
    }
    for (; h0 < end; h0 += 4 * PER) {
        const int h = h0 + lane / (D / 4);
        float4_4 v = own;
        const float4_4 w = other;
        if (h0 + 4 * PER < end)
            load(h0 + 4 * PER);
        if (h < a.heads + kv) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i0 + j < 2 * half)
                    v[j] = float(double(v[j]) * c[j] + double(w[j]) * s[j]);
        }
        if (h >= end)
            v = float4_4{0.0f, 0.0f, 0.0f, 0.0f};
        uint16_t codes = 0, scale = 0;
        if constexpr (Q4)
            if (h0 + PER > a.heads) {              // (some lane has a key or value)
                const float x[4] = {v.x, v.y, v.z, v.w};
                block_codes(x, lane, &codes, &scale);
            }
        if (h >= end)
            continue;
        if (h < a.heads) {
            *reinterpret_cast<float4_4*>(a.query + (int64_t(t) * a.heads + h) * D + i0) = v;
            continue;
        }
        const int kvh = h - a.heads < kv ? h - a.heads : h - a.heads - kv;
        char* page = (h - a.heads < kv ? a.cache.keys : a.cache.values) + (at.page * kv + kvh) * head_bytes;
        if constexpr (Q4) {
            reinterpret_cast<uint16_t*>(page)[at.slot * (D / 4) + i0 / 4] = codes;
            if ((lane & 7) == 0)
                reinterpret_cast<uint16_t*>(page + a.cache.page_size * (D / 2))[(i0 / 32) * a.cache.page_size + at.slot] = scale;
        } else {
            const __half2 lo = __halves2half2(__float2half_rn(v.x), __float2half_rn(v.y));
            const __half2 hi = __halves2half2(__float2half_rn(v.z), __float2half_rn(v.w));
            reinterpret_cast<uint2*>(page)[at.slot * (D / 4) + i0 / 4] =
                make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
        }
    }
}

template <int D, bool Q4>
__global__ void __launch_bounds__(256)
paged_read_kernel(const PagedBatch b, const PagedCache c, float* keys, float* values)
{
    const int t = row_of_workgroup();
    if (t >= b.rows)
        return;
    const Place at = find_place(b, c, t);
    if (!at.live)
        return;
    const int64_t head_bytes = paged_head_bytes(Q4, c.page_size, D);
    const int quads = c.kv_heads * (D / 4);
    for (int i = threadIdx.x; i < 2 * quads; i += 256) {
        const int j = i < quads ? i : i - quads, h = j / (D / 4), e = j % (D / 4);
        float4_4 v = {NAN, NAN, NAN, NAN};
        if (at.page >= 0) {
            const char* page = (i < quads ? c.keys : c.values) + (at.page * c.kv_heads + h) * head_bytes;
            if constexpr (Q4) {
                const uint32_t q = reinterpret_cast<const uint16_t*>(page)[at.slot * (D / 4) + e];
                const float d = __half2float(
                    reinterpret_cast<const __half*>(page + c.page_size * (D / 2))[(e / 8) * c.page_size + at.slot]);
#pragma unroll
                for (int n = 0; n < 4; n++)
                    v[n] = float(int(q >> (4 * n) & 15) - 8) * d;
            } else {
                const uint2 q = reinterpret_cast<const uint2*>(page)[at.slot * (D / 4) + e];
                const float2 lo = __half22float2(__builtin_bit_cast(__half2, q.x)), hi = __half22float2(__builtin_bit_cast(__half2, q.y));
                v = float4_4{lo.x, lo.y, hi.x, hi.y};
            }
        }
        *reinterpret_cast<float4_4*>((i < quads ? keys : values) + (int64_t(t) * quads + j) * 4) = v;
    }
}

// as many rows for each die
unsigned workgroups(int rows) { return (unsigned(rows) + 7) / 8 * 8; }

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s)
{
    // few rows: a row's heads over several workgroups
    const int total = a.heads + 2 * a.cache.kv_heads;
    const int one = 4 * (256 / a.cache.head);
    const int per_group = a.batch.rows < 512 ? one : (total + one - 1) / one * one;
    const dim3 grid(workgroups(a.batch.rows), unsigned((total + per_group - 1) / per_group));
    if (a.cache.head == 128) {
        if (a.cache.q4)
            paged_append_kernel<128, true><<<grid, 256, 0, s>>>(a, per_group);
        else
            paged_append_kernel<128, false><<<grid, 256, 0, s>>>(a, per_group);
    } else {
        if (a.cache.q4)
            paged_append_kernel<64, true><<<grid, 256, 0, s>>>(a, per_group);
        else
            paged_append_kernel<64, false><<<grid, 256, 0, s>>>(a, per_group);
    }
    return hipGetLastError();
}

hipError_t launch_paged_read(const PagedBatch& b, const PagedCache& c, float* keys, float* values, hipStream_t s)
{
    if (c.head == 128) {
        if (c.q4)
            paged_read_kernel<128, true><<<workgroups(b.rows), 256, 0, s>>>(b, c, keys, values);
        else
            paged_read_kernel<128, false><<<workgroups(b.rows), 256, 0, s>>>(b, c, keys, values);
    } else {
        if (c.q4)
            paged_read_kernel<64, true><<<workgroups(b.rows), 256, 0, s>>>(b, c, keys, values);
        else
            paged_read_kernel<64, false><<<workgroups(b.rows), 256, 0, s>>>(b, c, keys, values);
    }
    return hipGetLastError();
}

}  // namespace si
