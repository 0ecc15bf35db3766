// Causal attention of the newest rows of many sequences over a paged cache
// (4-bit or FP16 pages), KV heads shared by a group of query heads.
//
// Mathematics: with s_j = q . k_j / sqrt(d) over the positions j that a row
// sees, out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), m the largest
// s_j; in one pass over the positions, m, the sum and the accumulators
// rescaled when m grows.  Everything is kept transposed (positions down,
// rows across): the matrix cores then leave S^T with a row's statistics in
// one lane column, its exponentials are the next product's operand as they
// stand, and no value moves between lanes.
#include "si_paged.hpp"

#include "si_lanes.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace si {

namespace {

using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using f32x4 = float __attribute__((ext_vector_type(4)));

constexpr int TILE_ROWS = 16;            // packed query rows (position, head of the group) of a tile
constexpr int UNIT = 64;                 // positions of a step: four granules of 16
constexpr int GRANULE = 16;              // positions that always lie in one page

__device__ __forceinline__ f16x2 as_f16x2(uint32_t v) { return __builtin_bit_cast(f16x2, v); }
__device__ __forceinline__ uint32_t as_u32(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }

// 4-bit values at bits 0..3 and 16..19 of w as FP16 value - 8 (exact): the
// nibble under the exponent of 1024 is 1024 + nibble.
__device__ __forceinline__ f16x2 nibbles(uint32_t w)
{
    const f16x2 k = {_Float16(1032.0f), _Float16(1032.0f)};
    return as_f16x2((w & 0x000F000Fu) | 0x64006400u) - k;
}

union Frag {
    uint32_t w[4];
    f16x8 v;
};

// The tile that a wave works on.
struct Tile {
    int sequence;
    int first;                 // first batch row of the sequence
    int count;                 // its rows
    int length;                // its positions
    int row0;                  // first packed row
};

__device__ __forceinline__ int wave_scan(int v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(v, m);
        v += lane >= m ? o : 0;
    }
    return v;
}

// Rows of sequence s, as far as the batch's buffers hold them.
__device__ __forceinline__ void sequence_rows(const PagedBatch& b, int s, int* first, int* count)
{
    *first = b.starts[s];
    const int end = b.starts[s + 1];
    *count = *first < 0 || end < *first || end > b.rows ? 0 : end - *first;
}

// Finds tile `index` in the sequences' tiles of TILE_ROWS packed rows; the whole
// wave searches.  False when there are fewer tiles.
__device__ __forceinline__ bool find_tile(const PagedBatch& b, int group, int64_t index, Tile* out)
{
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < b.sequences; base += 64) {
        const int s = base + lane;
        int first = 0, count = 0;
        if (s < b.sequences)
            sequence_rows(b, s, &first, &count);
        const int tiles = (count * group + TILE_ROWS - 1) / TILE_ROWS;
        const int upto = wave_scan(tiles);
        const uint64_t past = __ballot(upto > index);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            out->sequence = base + at;
            out->first = __shfl(first, at);
            out->count = __shfl(count, at);
            out->length = b.lengths[base + at];
            out->row0 = int(index - __shfl(upto - tiles, at)) * TILE_ROWS;
            return true;
        }
        index -= __shfl(upto, 63);
    }
    return false;
}

// Running state of a tile: the lane's packed row is lane & 15.
template <int D>
struct State {
    static constexpr int NV = D / 16;
    f32x4 acc[NV];             // acc[n][i]: column NV * (4 * (lane >> 4) + i) + n
    float top;                 // largest score so far (in units of log 2)
    float sum;                 // of this lane's positions
};

template <int D, bool Q4>
struct Attend {
    static constexpr int NJ = D / 32;    // products of 32 values that a score takes
    static constexpr int NV = D / 16;    // column sets of a row of values
    const PagedAttentionArgs& a;
    int lane, g, c;
    int64_t head_bytes;
    f16x8 q[NJ];

    __device__ __forceinline__ explicit Attend(const PagedAttentionArgs& args)
        : a(args), lane(threadIdx.x & 63), g(lane >> 4), c(lane & 15),
          head_bytes(paged_head_bytes(Q4, args.cache.page_size, D))
    {
    }

    // The lane's query row, times 1 / sqrt(D) and log2(e), in FP16, in the
    // order in which the keys' values come out of their words.
    __device__ __forceinline__ void load_query(const float* row)
    {
        const float f = 1.44269504088896340736f / sqrtf(float(D));
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int at = Q4 ? (D / 4) * g + 8 * j : 32 * j + 8 * g;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                v[i] = row ? row[at + i] * f : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++)
                q[j][i] = _Float16(Q4 ? v[(i >> 1) + 4 * (i & 1)] : v[i]);
        }
    }

    // One unit of 64 positions from `base` on: positions up to `limit` count
    // for this lane's row, `full`: the whole unit for every row.  pages[i]:
    // the page of granule i (-1: none that can be read).
    __device__ __forceinline__ void unit(State<D>& st, int kvh, int base, const int* pages, int limit, bool full)
    {
        const int ps = a.cache.page_size;
        f32x4 s[4];
        Frag vf[2][NV];
        bool odd = false;              // a value of these positions is infinite or NaN
        uint32_t odd_tokens = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int slot = (base + GRANULE * u) & (ps - 1);
            const int64_t off = (int64_t(pages[u] < 0 ? 0 : pages[u]) * a.cache.kv_heads + kvh) * head_bytes;
            const char* kp = a.cache.keys + off;
            const char* vp = a.cache.values + off;
            s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (Q4) {
                uint32_t kw[NJ];
                const char* kr = kp + (slot + c) * (D / 2) + (D / 8) * g;
                if constexpr (D == 128) {
                    const uint4 t = *reinterpret_cast<const uint4*>(kr);
                    kw[0] = t.x, kw[1] = t.y, kw[2] = t.z, kw[3] = t.w;
                } else {
                    const uint2 t = *reinterpret_cast<const uint2*>(kr);
                    kw[0] = t.x, kw[1] = t.y;
                }
                const uint32_t kd = reinterpret_cast<const uint16_t*>(kp + ps * (D / 2))[(D == 128 ? g : g >> 1) * ps + slot + c];
                const f16x2 d = as_f16x2(kd | kd << 16);
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    Frag k;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        k.w[i] = as_u32(nibbles(kw[j] >> (4 * i)) * d);
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.v, q[j], s[u], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const f16x8 k = *reinterpret_cast<const f16x8*>(kp + (slot + c) * (2 * D) + 64 * j + 16 * g);
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[j], s[u], 0, 0, 0);
                }
            }
            // values: this lane's four positions 4 g .. of the granule
            if constexpr (Q4) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const char* vr = vp + (slot + 4 * g + i) * (D / 2);
                    w[i] = D == 128 ? reinterpret_cast<const uint32_t*>(vr)[c] : reinterpret_cast<const uint16_t*>(vr)[c];
                }
                const uint2 scales = *reinterpret_cast<const uint2*>(
                    reinterpret_cast<const uint16_t*>(vp + ps * (D / 2)) + (D == 128 ? c >> 2 : c >> 3) * ps + slot + 4 * g);
                uint32_t d[2] = {scales.x, scales.y};
                if (!full) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // 8192 and up: 8 x it passes FP16's largest value
                        const uint32_t e = 0x7000u << (16 * (i & 1));
                        if ((d[i >> 1] & e) == e) {
                            odd = true;
                            odd_tokens |= 1u << (4 * u + i);
                            d[i >> 1] &= ~(0xFFFFu << (16 * (i & 1)));
                        }
                    }
                }
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const f16x2 dp = as_f16x2(d[p]);
                    const uint32_t lo = __builtin_amdgcn_perm(w[2 * p + 1], w[2 * p], 0x05040100u);
                    const uint32_t hi = __builtin_amdgcn_perm(w[2 * p + 1], w[2 * p], 0x07060302u);
#pragma unroll
                    for (int n = 0; n < NV; n++)
                        vf[u >> 1][n].w[2 * (u & 1) + p] = as_u32(nibbles((n < 4 ? lo : hi) >> (4 * (n & 3))) * dp);
                }
            } else {
                uint32_t w[4][NV / 2];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const char* vr = vp + (slot + 4 * g + i) * (2 * D) + 2 * NV * c;
                    if constexpr (D == 128) {
                        const uint4 t = *reinterpret_cast<const uint4*>(vr);
                        w[i][0] = t.x, w[i][1] = t.y, w[i][2] = t.z, w[i][3] = t.w;
                    } else {
                        const uint2 t = *reinterpret_cast<const uint2*>(vr);
                        w[i][0] = t.x, w[i][1] = t.y;
                    }
                }
                if (!full) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int k = 0; k < NV / 2; k++)
                            if ((w[i][k] & 0x7C00u) == 0x7C00u || (w[i][k] & 0x7C000000u) == 0x7C000000u) {
                                odd = true;
                                odd_tokens |= 1u << (4 * u + i);
                                w[i][k] = 0;
                            }
                }
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int n = 0; n < NV; n++)
                        vf[u >> 1][n].w[2 * (u & 1) + p] =
                            __builtin_amdgcn_perm(w[2 * p + 1][n >> 1], w[2 * p][n >> 1], n & 1 ? 0x07060302u : 0x05040100u);
            }
        }
        // what a row does not see scores -inf, a position without a page NaN
        if (!full) {
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int pos = base + GRANULE * u + 4 * g + i;
                    s[u][i] = pos > limit ? -INFINITY : s[u][i];
                }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (pages[u] < 0)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    s[u][i] = s[u][i] == -INFINITY ? s[u][i] : NAN;
        if (!full && __any(odd)) {
            // An infinite or NaN value in a position that some row does not
            // see: it was taken out of the operand, and a row that does see
            // it becomes NaN by its score.
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint64_t who = __ballot((odd_tokens >> (4 * u + i)) & 1);
                    const bool mine = ((who >> (16 * g)) & 0xFFFFu) != 0;
                    if (mine && base + GRANULE * u + 4 * g + i <= limit)
                        s[u][i] = NAN;
                }
        }
        float top = st.top;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                top = fmaxf(top, s[u][i]);
        top = rows_max(top);
        const float at = fmaxf(top, -3.4028235e38f);      // (a row that has seen nothing yet)
        const float fade = exp2f(st.top - at);
        st.top = top;
        float sum = 0.0f;
        Frag pf[2];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[i] = exp2f(s[u][i] - at);
                sum += p[i];
            }
            pf[u >> 1].w[2 * (u & 1)] = as_u32(f16x2{_Float16(p[0]), _Float16(p[1])});
            pf[u >> 1].w[2 * (u & 1) + 1] = as_u32(f16x2{_Float16(p[2]), _Float16(p[3])});
        }
        st.sum = st.sum * fade + sum;
#pragma unroll
        for (int n = 0; n < NV; n++) {
            st.acc[n] *= fade;
            st.acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[0][n].v, pf[0].v, st.acc[n], 0, 0, 0);
            st.acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[1][n].v, pf[1].v, st.acc[n], 0, 0, 0);
        }
    }
};

__device__ __forceinline__ uint32_t pack_out(float x, float y, bool bf16)
{
    if (bf16) {
        const __hip_bfloat16 a = __float2bfloat16(x), b = __float2bfloat16(y);
        return uint32_t(__builtin_bit_cast(uint16_t, a)) | uint32_t(__builtin_bit_cast(uint16_t, b)) << 16;
    }
    return as_u32(f16x2{_Float16(x), _Float16(y)});
}

template <int D, bool Q4>
__global__ void __launch_bounds__(256)
paged_attention_kernel(const PagedAttentionArgs a)
{
    constexpr int NV = D / 16;
    const int kv = a.cache.kv_heads, group = a.heads / kv;
    const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int kvh = int(item % kv);
    Tile t;
    if (!find_tile(a.batch, group, item / kv, &t))
        return;
    Attend<D, Q4> w(a);
    const int packed = t.row0 + w.c, i = packed / group;
    const bool live = i < t.count;
    const int64_t row = int64_t(t.first) + i;
    const int head = kvh * group + packed % group;
    const bool wrong = t.length < 0 || t.length > int64_t(a.batch.max_pages) << a.cache.page_shift ||
                       t.count > a.batch.max_rows;
    const int limit = live && !wrong ? t.length - t.count + i : -1;
    w.load_query(live ? a.query + (row * a.heads + head) * D : nullptr);
    State<D> st;
#pragma unroll
    for (int n = 0; n < NV; n++)
        st.acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    st.top = -INFINITY;
    st.sum = 0.0f;
    const int last_row = min(t.count - 1, (t.row0 + TILE_ROWS - 1) / group);
    const int most = wrong ? -1 : t.length - t.count + last_row;          // last position that a row of the tile sees
    const int least = t.length - t.count + t.row0 / group;                // that all of them see
    const int32_t* table = a.batch.table + int64_t(t.sequence) * a.batch.max_pages;
    for (int base = 0; base <= most; base += UNIT) {
        int pages[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int pos = base + GRANULE * u;
            int page = pos <= most ? table[pos >> a.cache.page_shift] : 0;
            if (page >= a.cache.pages)
                page = -1;
            pages[u] = __builtin_amdgcn_readfirstlane(page);
        }
        w.unit(st, kvh, base, pages, limit, base + UNIT - 1 <= least);
    }
    const float sum = rows_sum(st.sum);
    const float inv = wrong ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
    if (!live)
        return;
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (row * a.heads + head) * D + NV * 4 * w.g);
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int n = 0; n < NV; n += 2)
            out[(NV * r + n) / 2] = pack_out(st.acc[n][r] * inv, st.acc[n + 1][r] * inv, a.bf16);
}

}  // namespace

int64_t paged_attention_workspace_floats(int, int, int) { return 4; }

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t s)
{
    const int group = a.heads / a.cache.kv_heads;
    const int64_t tiles = int64_t(a.batch.rows) * group / TILE_ROWS + a.batch.sequences;   // at most
    const unsigned grid = unsigned((tiles * a.cache.kv_heads + 3) / 4);
    if (a.cache.head == 128) {
        if (a.cache.q4)
            paged_attention_kernel<128, true><<<grid, 256, 0, s>>>(a);
        else
            paged_attention_kernel<128, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (a.cache.q4)
            paged_attention_kernel<64, true><<<grid, 256, 0, s>>>(a);
        else
            paged_attention_kernel<64, false><<<grid, 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

}  // namespace si
