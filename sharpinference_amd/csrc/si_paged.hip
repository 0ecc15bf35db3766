// The newest rows of many sequences into a paged cache (rotary embedding on
// the way), and rows of the pages back as FP32.
//
// A workgroup serves one row of the batch: its waves take the row's heads,
// two neighbouring values a lane, so a 4-bit block of 32 values is one
// 16-lane row of the wave and its largest value a DPP reduction.  The
// rotation runs in FP64 (angle, cosine, sine, products; rounded to FP32
// once): positions of any size keep their angle, and a key's codes do not
// depend on which kernel rotated it.
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

// The 4-bit block that 16 lanes hold, two values each: scale = the value of
// largest magnitude (the first of them) / -8 in FP16, code = value / scale
// rounded to the nearest (ties to even) + 8.  A value that FP16 could not
// hold makes the whole block NaN.
__device__ __forceinline__ void block_codes(float v0, float v1, int lane, uint32_t* codes, uint16_t* scale)
{
    const float a0 = fabsf(v0), a1 = fabsf(v1);
    const float top = row_max<16>(fmaxf(a0, a1));
    const bool has = a0 == top || a1 == top;
    const bool odd = !(a0 <= 65504.0f) || !(a1 <= 65504.0f);   // NaN too
    const uint32_t shift = lane & 48;
    const uint32_t holders = uint32_t(__ballot(has) >> shift) & 0xFFFFu;
    const uint32_t bad = uint32_t(__ballot(odd) >> shift) & 0xFFFFu;
    const float mine = a0 == top ? v0 : v1;
    const float first = __shfl(mine, int(shift) + (holders ? __ffs(holders) - 1 : 0));
    uint16_t d = __half_as_ushort(__float2half_rn(first / -8.0f));
    const float df = __half2float(__ushort_as_half(d));
    uint32_t q0 = 8, q1 = 8;
    if (bad) {
        d = 0x7E00;
    } else if (df == 0.0f) {
        d = 0;                                                 // a block of zeros, whatever their signs
    } else {
        q0 = uint32_t(int(fminf(fmaxf(rintf(v0 / df) + 8.0f, 0.0f), 15.0f)));
        q1 = uint32_t(int(fminf(fmaxf(rintf(v1 / df) + 8.0f, 0.0f), 15.0f)));
    }
    *codes = q0 | q1 << 4;
    *scale = d;
}

template <int D, bool Q4>
__global__ void __launch_bounds__(256)
paged_append_kernel(const PagedAppendArgs a, int per_group)
{
    constexpr int PER = 128 / D;                   // heads a wave serves at once
    __shared__ double turn[2][64];                 // cos, sin of the row's pairs
    const int t = blockIdx.x;
    const Place at = find_place(a.batch, a.cache, t);
    if (at.page < 0)
        return;                                    // the whole workgroup
    const int half = a.rotary >> 1;
    if (int(threadIdx.x) < half) {
        double s, c;
        sincos(double(at.position) * double(a.frequencies[threadIdx.x]), &s, &c);
        turn[0][threadIdx.x] = c * double(a.rope_scale);
        turn[1][threadIdx.x] = s * double(a.rope_scale);
    }
    __syncthreads();
    const int lane = threadIdx.x & 63;
    const int kv = a.cache.kv_heads, total = a.heads + 2 * kv;
    const int i0 = 2 * (lane % (D / 2));           // this lane's values i0, i0 + 1 of its head
    const float* row = a.qkv + int64_t(t) * total * D;
    const int64_t head_bytes = paged_head_bytes(Q4, a.cache.page_size, D);
    const int end = min(total, (int(blockIdx.y) + 1) * per_group);
    for (int h0 = int(blockIdx.y) * per_group + int(threadIdx.x >> 6) * PER; h0 < end; h0 += 4 * PER) {
        const int h = h0 + lane / (D / 2);
        // (a lane without a head works on the last one and stores nothing)
        const float* x = row + int64_t(min(h, end - 1)) * D;
        float v[2];
        const bool turned = h < a.heads + kv;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int i = i0 + j;
            v[j] = x[i];
            if (turned && i < 2 * half) {
                const bool low = i < half;
                const int pair = low ? i : i - half;
                const double own = v[j], other = x[low ? i + half : pair];
                const double c = turn[0][pair], s = turn[1][pair];
                v[j] = float(low ? own * c - other * s : own * c + other * s);
            }
        }
        if (h >= end)
            v[0] = v[1] = 0.0f;
        uint32_t codes = 0;
        uint16_t scale = 0;
        if constexpr (Q4)
            block_codes(v[0], v[1], lane, &codes, &scale);
        if (h >= end)
            continue;
        if (h < a.heads) {
            float* q = a.query + (int64_t(t) * a.heads + h) * D + i0;
            q[0] = v[0];
            q[1] = v[1];
            continue;
        }
        const int kvh = h - a.heads < kv ? h - a.heads : h - a.heads - kv;
        char* page = (h - a.heads < kv ? a.cache.keys : a.cache.values) + (at.page * kv + kvh) * head_bytes;
        if constexpr (Q4) {
            page[at.slot * (D / 2) + i0 / 2] = char(codes);
            if ((lane & 15) == 0)
                reinterpret_cast<uint16_t*>(page + a.cache.page_size * (D / 2))[(i0 / 32) * a.cache.page_size + at.slot] = scale;
        } else {
            reinterpret_cast<__half2*>(page)[at.slot * (D / 2) + i0 / 2] =
                __halves2half2(__float2half_rn(v[0]), __float2half_rn(v[1]));
        }
    }
}

template <int D, bool Q4>
__global__ void __launch_bounds__(256)
paged_read_kernel(const PagedBatch b, const PagedCache c, float* keys, float* values)
{
    const int t = blockIdx.x;
    const Place at = find_place(b, c, t);
    if (!at.live)
        return;
    const int64_t head_bytes = paged_head_bytes(Q4, c.page_size, D);
    const int pairs = c.kv_heads * (D / 2);
    for (int i = threadIdx.x; i < 2 * pairs; i += 256) {
        const int j = i < pairs ? i : i - pairs, h = j / (D / 2), e = j % (D / 2);
        float2 v = make_float2(NAN, NAN);
        if (at.page >= 0) {
            const char* page = (i < pairs ? c.keys : c.values) + (at.page * c.kv_heads + h) * head_bytes;
            if constexpr (Q4) {
                const uint32_t q = static_cast<uint8_t>(page[at.slot * (D / 2) + e]);
                const float d = __half2float(
                    reinterpret_cast<const __half*>(page + c.page_size * (D / 2))[(e / 16) * c.page_size + at.slot]);
                v = make_float2(float(int(q & 15) - 8) * d, float(int(q >> 4) - 8) * d);
            } else {
                v = __half22float2(reinterpret_cast<const __half2*>(page)[at.slot * (D / 2) + e]);
            }
        }
        float* out = (i < pairs ? keys : values) + (int64_t(t) * pairs + j) * 2;
        out[0] = v.x;
        out[1] = v.y;
    }
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s)
{
    // few rows: a row's heads over several workgroups, two for each wave
    const int total = a.heads + 2 * a.cache.kv_heads;
    const int two = 2 * 4 * (128 / a.cache.head);
    const int per_group = a.batch.rows < 512 ? two : (total + two - 1) / two * two;
    const dim3 grid(unsigned(a.batch.rows), unsigned((total + per_group - 1) / per_group));
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
            paged_read_kernel<128, true><<<unsigned(b.rows), 256, 0, s>>>(b, c, keys, values);
        else
            paged_read_kernel<128, false><<<unsigned(b.rows), 256, 0, s>>>(b, c, keys, values);
    } else {
        if (c.q4)
            paged_read_kernel<64, true><<<unsigned(b.rows), 256, 0, s>>>(b, c, keys, values);
        else
            paged_read_kernel<64, false><<<unsigned(b.rows), 256, 0, s>>>(b, c, keys, values);
    }
    return hipGetLastError();
}

}  // namespace si
