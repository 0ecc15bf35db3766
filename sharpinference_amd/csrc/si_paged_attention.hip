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

// Rows of sequence s, as far as the batch's buffers hold them.
__device__ __forceinline__ void sequence_rows(const PagedBatch& b, int s, int* first, int* count)
{
    *first = b.starts[s];
    const int end = b.starts[s + 1];
    *count = *first < 0 || end < *first || end > b.rows ? 0 : end - *first;
}

// A sequence as the kernels see it: its rows, the tiles of TILE_ROWS packed
// rows that they make, and the units that a tile goes through.
struct Sequence {
    int index;
    int first;
    int count;
    int length;                // positions; -1: the sequence's rows become NaN
    int tiles;
    int units;
};

__device__ __forceinline__ Sequence take_sequence(const PagedBatch& b, int page_shift, int group, int s)
{
    Sequence q{s, 0, 0, 0, 0, 0};
    if (s >= b.sequences)
        return q;
    sequence_rows(b, s, &q.first, &q.count);
    q.length = b.lengths[s];
    if (q.length < 0 || q.length > int64_t(b.max_pages) << page_shift || q.count > b.max_rows)
        q.length = -1;
    q.tiles = (q.count * group + TILE_ROWS - 1) / TILE_ROWS;
    q.units = max(1, (q.length + UNIT - 1) / UNIT);
    return q;
}

__device__ __forceinline__ int64_t wave_scan(int64_t v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int64_t o = __shfl_up(v, m);
        v += lane >= m ? o : 0;
    }
    return v;
}

__device__ __forceinline__ Sequence from_lane(const Sequence& q, int lane)
{
    return {__shfl(q.index, lane), __shfl(q.first, lane), __shfl(q.count, lane), __shfl(q.length, lane),
            __shfl(q.tiles, lane), __shfl(q.units, lane)};
}

// The work of a launch in one line: sequence after sequence, of each its KV
// heads, of each its tiles, of each its units.  A wave searches together,
// one sequence a lane.
struct Line {
    const PagedBatch& b;
    int page_shift, group, kv;

    __device__ __forceinline__ int64_t units_of(const Sequence& q) const { return int64_t(kv) * q.tiles * q.units; }
    __device__ __forceinline__ int64_t total() const
    {
        int64_t sum = 0;
        for (int base = 0; base < b.sequences; base += 64)
            sum += units_of(take_sequence(b, page_shift, group, base + int(threadIdx.x & 63)));
        return __shfl(wave_scan(sum), 63);
    }
    // The sequence that holds unit x, and the number of its first unit.
    __device__ __forceinline__ bool at_unit(int64_t x, Sequence* q, int64_t* start) const
    {
        int64_t before = 0;
        for (int base = 0; base < b.sequences; base += 64) {
            const Sequence mine = take_sequence(b, page_shift, group, base + int(threadIdx.x & 63));
            const int64_t upto = before + wave_scan(units_of(mine));
            const uint64_t past = __ballot(upto > x);
            if (past) {
                const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
                *q = from_lane(mine, at);
                *start = __shfl(upto - units_of(mine), at);
                return true;
            }
            before = __shfl(upto, 63);
        }
        return false;
    }
    // The sequence that holds tile x of one KV head, the tile's number in it
    // and its first unit (of KV head 0).
    __device__ __forceinline__ bool at_tile(int64_t x, Sequence* q, int64_t* tile, int64_t* start) const
    {
        int64_t before = 0, units = 0;
        for (int base = 0; base < b.sequences; base += 64) {
            const Sequence mine = take_sequence(b, page_shift, group, base + int(threadIdx.x & 63));
            const int64_t upto = before + wave_scan(mine.tiles), units_upto = units + wave_scan(units_of(mine));
            const uint64_t past = __ballot(upto > x);
            if (past) {
                const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
                *q = from_lane(mine, at);
                *tile = x - __shfl(upto - mine.tiles, at);
                *start = __shfl(units_upto - units_of(mine), at);
                return true;
            }
            before = __shfl(upto, 63);
            units = __shfl(units_upto, 63);
        }
        return false;
    }
};

// The waves that share a line of `total` units: wave w of `waves` takes
// units first(w) .. first(w + 1) - 1, at least MIN_UNITS of them.
constexpr int MIN_UNITS = 2;
constexpr int WAVES = 2048;
struct Shares {
    int64_t total, waves;
    __device__ __forceinline__ explicit Shares(int64_t t) : total(t), waves(min(int64_t(WAVES), (t + MIN_UNITS - 1) / MIN_UNITS)) {}
    __device__ __forceinline__ int64_t first(int64_t w) const { return w * total / waves; }
    __device__ __forceinline__ int64_t wave_of(int64_t unit) const { return ((unit + 1) * waves - 1) / total; }
};

// What a wave leaves of a tile whose units it shares with other waves: the
// accumulators [TILE_ROWS][D], largest scores and sums [TILE_ROWS] each.
// Slot 2 w: of the tile that began before wave w's units, slot 2 w + 1: of
// the one that goes on behind them.
constexpr int slot_floats(int d) { return TILE_ROWS * d + 2 * TILE_ROWS; }

// Running state of a tile: the lane's packed row is lane & 15.
template <int D>
struct State {
    static constexpr int NV = D / 16;
    f32x4 acc[NV];             // acc[n][i]: column NV * (4 * (lane >> 4) + i) + n
    float top;                 // largest score so far (in units of log 2)
    float sum;                 // of this lane's positions
};

// The bytes of a unit as they are loaded, for this lane.
template <int D, bool Q4>
struct Raw {
    static constexpr int KW = Q4 ? D / 32 : D / 8;   // words of a granule's keys
    static constexpr int VW = Q4 ? 1 : D / 32;       // words of a position's values
    uint32_t k[4][KW];
    uint32_t kd[4];            // 4-bit: the key scale
    uint32_t v[4][4][VW];
    uint32_t vd[4][2];         // 4-bit: the value scales of the lane's four positions
    uint32_t lost;             // bit u: granule u has no page
};

// FINE: products of two-term FP16 operands (exact 4-bit values, queries and
// exponentials to 22 bits), for outputs that show more than BF16 does.
template <int D, bool Q4, bool FINE>
struct Attend {
    static constexpr int NJ = D / 32;    // products of 32 values that a score takes
    static constexpr int NV = D / 16;    // column sets of a row of values
    const PagedAttentionArgs& a;
    int lane, g, c;
    int64_t head_bytes;
    f16x8 q[NJ], ql[FINE ? NJ : 1];

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
            float4 x = make_float4(0, 0, 0, 0), y = x;
            if (row) {
                x = *reinterpret_cast<const float4*>(row + at);
                y = *reinterpret_cast<const float4*>(row + at + 4);
            }
            v[0] = x.x * f, v[1] = x.y * f, v[2] = x.z * f, v[3] = x.w * f;
            v[4] = y.x * f, v[5] = y.y * f, v[6] = y.z * f, v[7] = y.w * f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float t = Q4 ? v[(i >> 1) + 4 * (i & 1)] : v[i];
                q[j][i] = _Float16(t);
                if constexpr (FINE)
                    ql[j][i] = _Float16(t - float(q[j][i]));
            }
        }
    }

    __device__ __forceinline__ int64_t page_at(int page, int kvh) const
    {
        return (int64_t(page < 0 ? 0 : page) * a.cache.kv_heads + kvh) * head_bytes;
    }

    // Loads the keys of the unit of 64 positions from `base` on; pages[u]: the
    // page of granule u, -1 for one that is not there (page 0 is read in its place).
    __device__ __forceinline__ void load_keys(Raw<D, Q4>& r, int kvh, int base, const int* pages) const
    {
        const int ps = a.cache.page_size;
        r.lost = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int slot = (base + GRANULE * u) & (ps - 1);
            r.lost |= pages[u] < 0 ? 1u << u : 0u;
            const char* kp = a.cache.keys + page_at(pages[u], kvh);
            if constexpr (Q4) {
                const char* kr = kp + slot * (D / 2) + (D / 2 * c + D / 8 * g);
                if constexpr (D == 128) {
                    const uint4 t = *reinterpret_cast<const uint4*>(kr);
                    r.k[u][0] = t.x, r.k[u][1] = t.y, r.k[u][2] = t.z, r.k[u][3] = t.w;
                } else {
                    const uint2 t = *reinterpret_cast<const uint2*>(kr);
                    r.k[u][0] = t.x, r.k[u][1] = t.y;
                }
                r.kd[u] = *reinterpret_cast<const uint16_t*>(kp + ps * (D / 2) + 2 * slot + 2 * ((D == 128 ? g : g >> 1) * ps + c));
            } else {
                const char* kr = kp + slot * (2 * D) + (2 * D * c + 16 * g);
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const uint4 t = *reinterpret_cast<const uint4*>(kr + 64 * j);
                    r.k[u][4 * j] = t.x, r.k[u][4 * j + 1] = t.y, r.k[u][4 * j + 2] = t.z, r.k[u][4 * j + 3] = t.w;
                }
            }
        }
    }

    __device__ __forceinline__ void load_values(Raw<D, Q4>& r, int kvh, int base, const int* pages) const
    {
        const int ps = a.cache.page_size;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int slot = (base + GRANULE * u) & (ps - 1);
            const char* vp = a.cache.values + page_at(pages[u], kvh);
            if constexpr (Q4) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const char* vr = vp + slot * (D / 2) + (4 * g + i) * (D / 2) + NV / 2 * c;
                    r.v[u][i][0] = D == 128 ? *reinterpret_cast<const uint32_t*>(vr) : *reinterpret_cast<const uint16_t*>(vr);
                }
                const uint2 t = *reinterpret_cast<const uint2*>(vp + ps * (D / 2) + 2 * slot +
                                                                2 * ((D == 128 ? c >> 2 : c >> 3) * ps + 4 * g));
                r.vd[u][0] = t.x, r.vd[u][1] = t.y;
            } else {
                const char* vr = vp + slot * (2 * D) + (2 * D * 4 * g + 2 * NV * c);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (D == 128) {
                        const uint4 t = *reinterpret_cast<const uint4*>(vr + 2 * D * i);
                        r.v[u][i][0] = t.x, r.v[u][i][1] = t.y, r.v[u][i][2] = t.z, r.v[u][i][3] = t.w;
                    } else {
                        const uint2 t = *reinterpret_cast<const uint2*>(vr + 2 * D * i);
                        r.v[u][i][0] = t.x, r.v[u][i][1] = t.y;
                    }
                }
            }
        }
    }

    // One product S += K . Q of 32 values (4-bit keys: from their words and scale).
    __device__ __forceinline__ f32x4 score(const Raw<D, Q4>& r, int u, int j, f32x4 s) const
    {
        Frag k, kl;
        if constexpr (Q4) {
            const f16x2 d = as_f16x2(r.kd[u] | r.kd[u] << 16);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f16x2 n = nibbles(r.k[u][j] >> (4 * i)), v = n * d;
                k.w[i] = as_u32(v);
                if constexpr (FINE)
                    kl.w[i] = as_u32(__builtin_elementwise_fma(n, d, -v));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                k.w[i] = r.k[u][4 * j + i];
        }
        if constexpr (FINE && Q4)
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl.v, q[j], s, 0, 0, 0);
        if constexpr (FINE)
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.v, ql[j], s, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(k.v, q[j], s, 0, 0, 0);
    }

    __device__ __forceinline__ void scores(const Raw<D, Q4>& r, f32x4* s) const
    {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NJ; j++)
                s[u] = score(r, u, j, s[u]);
        }
    }

    // One unit of 64 positions from `base` on, its scores in s: positions up
    // to `limit` count for this lane's row, `full`: the whole unit for every
    // row; bit u of `lost`: granule u has no page.
    __device__ __forceinline__ void unit(State<D>& st, Raw<D, Q4>& r, f32x4* s, uint32_t lost, int base, int limit,
                                         bool full) const
    {
        if (!full) {
            // what a row does not see scores -inf
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    s[u][i] = base + GRANULE * u + 4 * g + i > limit ? -INFINITY : s[u][i];
            take_out_odd(r, s, base, limit);
        }
        if (lost) {
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    s[u][i] = (lost >> u & 1) && base + GRANULE * u + 4 * g + i <= limit ? NAN : s[u][i];
        }
        float top = st.top;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                top = fmaxf(top, s[u][i]);
        top = rows_max(top);
        const float at = fmaxf(top, -3.4028235e38f);      // (a row that has seen nothing yet)
        if (__any(top > st.top)) {
            const float fade = __builtin_amdgcn_exp2f(st.top - at);
            st.sum *= fade;
#pragma unroll
            for (int n = 0; n < NV; n++)
                st.acc[n] *= fade;
            st.top = top;
        }
        Frag pf[2], pl[2];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[i] = __builtin_amdgcn_exp2f(s[u][i] - at);
                st.sum += p[i];
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const f16x2 h = {_Float16(p[2 * k]), _Float16(p[2 * k + 1])};
                pf[u >> 1].w[2 * (u & 1) + k] = as_u32(h);
                if constexpr (FINE)
                    pl[u >> 1].w[2 * (u & 1) + k] =
                        as_u32(f16x2{_Float16(p[2 * k] - float(h[0])), _Float16(p[2 * k + 1] - float(h[1]))});
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t lo[4], hi[4];                         // 4-bit: words of two positions by halves
            if constexpr (Q4) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t w0 = r.v[2 * h + (k >> 1)][2 * (k & 1)][0], w1 = r.v[2 * h + (k >> 1)][2 * (k & 1) + 1][0];
                    lo[k] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                    hi[k] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
                }
            }
#pragma unroll
            for (int n = 0; n < NV; n++) {
                Frag v, vl;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int u = 2 * h + (k >> 1), i = 2 * (k & 1);
                    if constexpr (Q4) {
                        const f16x2 d = as_f16x2(r.vd[u][k & 1]);
                        const f16x2 x = nibbles((n < 4 ? lo[k] : hi[k]) >> (4 * (n & 3))), y = x * d;
                        v.w[k] = as_u32(y);
                        if constexpr (FINE)
                            vl.w[k] = as_u32(__builtin_elementwise_fma(x, d, -y));
                    } else {
                        v.w[k] = __builtin_amdgcn_perm(r.v[u][i + 1][n >> 1], r.v[u][i][n >> 1],
                                                       n & 1 ? 0x07060302u : 0x05040100u);
                    }
                }
                if constexpr (FINE && Q4)
                    st.acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl.v, pf[h].v, st.acc[n], 0, 0, 0);
                if constexpr (FINE)
                    st.acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.v, pl[h].v, st.acc[n], 0, 0, 0);
                st.acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.v, pf[h].v, st.acc[n], 0, 0, 0);
            }
        }
    }

    // An infinite or NaN value in a position that some row does not see is
    // taken out of the operand (its weight of 0 would make it NaN there), and
    // a row that does see it becomes NaN by its score.
    __device__ __forceinline__ void take_out_odd(Raw<D, Q4>& r, f32x4* s, int base, int limit) const
    {
        uint32_t odd = 0;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (Q4) {
                    // 8192 and up: 8 x it passes FP16's largest value
                    const uint32_t e = 0x7000u << (16 * (i & 1));
                    if ((r.vd[u][i >> 1] & e) == e) {
                        odd |= 1u << (4 * u + i);
                        r.vd[u][i >> 1] &= ~(0xFFFFu << (16 * (i & 1)));
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < D / 32; k++)
                        if ((r.v[u][i][k] & 0x7C00u) == 0x7C00u || (r.v[u][i][k] & 0x7C000000u) == 0x7C000000u) {
                            odd |= 1u << (4 * u + i);
                            r.v[u][i][k] = 0;
                        }
                }
            }
        if (!__any(odd != 0))
            return;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint64_t who = __ballot((odd >> (4 * u + i)) & 1);
                if (((who >> (16 * g)) & 0xFFFFu) != 0 && base + GRANULE * u + 4 * g + i <= limit)
                    s[u][i] = NAN;
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

// Four neighbouring values of an output row, at value index `at`.
__device__ __forceinline__ void store_out(const PagedAttentionArgs& a, int64_t at, float x, float y, float z, float w)
{
    if (a.out_format == PAGED_OUT_F32)
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x, y, z, w);
    else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
            make_uint2(pack_out(x, y, a.out_format == PAGED_OUT_BF16), pack_out(z, w, a.out_format == PAGED_OUT_BF16));
}

// Every wave takes an equal run of the line's units, whatever sequences they
// lie in; tiles that are wholly its own are written out, the others left in
// its slots for the merge.
template <int D, bool Q4, bool FINE>
__global__ void __launch_bounds__(256, 2)
paged_attention_kernel(const PagedAttentionArgs a)
{
    constexpr int NV = D / 16;
    const int kv = a.cache.kv_heads, group = a.heads / kv;
    const int64_t wave = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const Line line{a.batch, a.cache.page_shift, group, kv};
    const int64_t total = line.total();
    if (total == 0)
        return;
    const Shares share(total);
    if (wave >= share.waves)
        return;
    const int64_t begin = share.first(wave), end = share.first(wave + 1);
    Attend<D, Q4, FINE> w(a);
    Sequence q{};
    int64_t q_start = 0, q_end = 0;
    for (int64_t x = begin; x < end;) {
        if (x >= q_end) {
            if (!line.at_unit(x, &q, &q_start))
                return;
            q_end = q_start + line.units_of(q);
        }
        // unit x: of which KV head, tile and positions
        const int64_t in = x - q_start;
        const int64_t tile_no = in / q.units;
        const int kvh = __builtin_amdgcn_readfirstlane(int(tile_no / q.tiles));
        const int row0 = __builtin_amdgcn_readfirstlane(int(tile_no % q.tiles) * TILE_ROWS);
        const int unit0 = __builtin_amdgcn_readfirstlane(int(in % q.units));
        const int64_t tile_start = x - unit0, tile_end = tile_start + q.units;
        const int unit1 = __builtin_amdgcn_readfirstlane(int(min(tile_end, end) - tile_start));
        x = min(tile_end, end);

        const int packed = row0 + w.c, i = packed / group;
        const bool live = i < q.count;
        const int64_t row = int64_t(q.first) + i;
        const int head = kvh * group + packed % group;
        const bool wrong = q.length < 0;
        const int limit = live && !wrong ? q.length - q.count + i : -1;
        w.load_query(live ? a.query + (row * a.heads + head) * D : nullptr);
        State<D> st;
#pragma unroll
        for (int n = 0; n < NV; n++)
            st.acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        st.top = -INFINITY;
        st.sum = 0.0f;
        // the last position that a row of the tile sees, and that all of them see
        const int last_row = min(q.count - 1, (row0 + TILE_ROWS - 1) / group);
        const int most = __builtin_amdgcn_readfirstlane(wrong ? -1 : q.length - q.count + last_row);
        const int least = __builtin_amdgcn_readfirstlane(q.length - q.count + row0 / group);
        const int stop = min(unit1, (most + UNIT) / UNIT);
        const int32_t* table = a.batch.table + int64_t(q.index) * a.batch.max_pages;
        // the pages of 64 granules (16 units), one a lane
        int held = 0;
        auto pages_of = [&](int u, int* pages) {
            if (u == unit0 || (u & 15) == 0) {
                const int pos = ((u & ~15) * 4 + w.lane) * GRANULE;
                held = pos <= most ? table[pos >> a.cache.page_shift] : 0;
                if (held >= a.cache.pages)
                    held = -1;
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                pages[k] = __builtin_amdgcn_readlane(held, (u & 15) * 4 + k);
        };
        // One set of registers: the next unit's keys are on their way while
        // this one's weights and values are worked on, its values while the
        // next scores are.
        int pages[4];
        Raw<D, Q4> raw;
        if (unit0 < stop) {
            pages_of(unit0, pages);
            w.load_keys(raw, kvh, unit0 * UNIT, pages);
            w.load_values(raw, kvh, unit0 * UNIT, pages);
        }
        for (int u = unit0; u < stop; u++) {
            f32x4 s[4];
            w.scores(raw, s);
            const uint32_t lost = raw.lost;
            if (u + 1 < stop) {
                pages_of(u + 1, pages);
                w.load_keys(raw, kvh, (u + 1) * UNIT, pages);
            }
            w.unit(st, raw, s, lost, u * UNIT, limit, u * UNIT + UNIT - 1 <= least);
            if (u + 1 < stop)
                w.load_values(raw, kvh, (u + 1) * UNIT, pages);
        }
        const float sum = rows_sum(st.sum);
        if (tile_start >= begin && tile_end <= end) {
            const float inv = wrong ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
            if (live) {
                const int64_t at = (row * a.heads + head) * D + NV * 4 * w.g;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int n = 0; n < NV; n += 4)
                        store_out(a, at + NV * r + n, st.acc[n][r] * inv, st.acc[n + 1][r] * inv, st.acc[n + 2][r] * inv,
                                  st.acc[n + 3][r] * inv);
            }
        } else if (live) {
            float* slot = a.workspace + (2 * wave + (tile_start >= begin)) * slot_floats(D);
            float* at = slot + w.c * D + NV * 4 * w.g;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int n = 0; n < NV; n += 4)
                    *reinterpret_cast<f32x4*>(at + NV * r + n) =
                        f32x4{st.acc[n][r], st.acc[n + 1][r], st.acc[n + 2][r], st.acc[n + 3][r]};
            if (w.g == 0) {
                slot[TILE_ROWS * D + w.c] = st.top;
                slot[TILE_ROWS * D + TILE_ROWS + w.c] = sum;
            }
        }
    }
}

// Joins the tiles that several waves share.  A workgroup takes 256 / D rows
// of four values a lane in each of its waves, and the waves take the tile's
// slots in turn.
template <int D>
__global__ void __launch_bounds__(256)
paged_merge_kernel(const PagedAttentionArgs a)
{
    constexpr int ROWS = 256 / D;
    const int kv = a.cache.kv_heads, group = a.heads / kv;
    const Line line{a.batch, a.cache.page_shift, group, kv};
    const int64_t total = line.total();
    Sequence q;
    int64_t tile, q_start;
    if (total == 0 || !line.at_tile(blockIdx.x / kv, &q, &tile, &q_start))
        return;
    const int kvh = blockIdx.x % kv;
    const Shares share(total);
    const int64_t first = q_start + (int64_t(kvh) * q.tiles + tile) * q.units;
    const int64_t w0 = share.wave_of(first), w1 = share.wave_of(first + q.units - 1);
    if (w0 == w1)
        return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int r = int(blockIdx.y) * ROWS + lane / (D / 4), col = 4 * (lane % (D / 4));
    const int packed = int(tile) * TILE_ROWS + r, i = packed / group;
    const bool live = i < q.count;
    float top = -INFINITY, sum = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    bool seen_nan = false;
    if (live) {
        for (int64_t p = w0 + wave; p <= w1; p += 4) {
            const float* slot = a.workspace + (2 * p + (p == w0)) * slot_floats(D);
            const float m = slot[TILE_ROWS * D + r], l = slot[TILE_ROWS * D + TILE_ROWS + r];
            const f32x4 v = *reinterpret_cast<const f32x4*>(slot + r * D + col);
            const float t = fmaxf(top, m), at = fmaxf(t, -3.4028235e38f);
            const float f = __builtin_amdgcn_exp2f(top - at), g = __builtin_amdgcn_exp2f(m - at);
            seen_nan |= !(l == l);
            sum = sum * f + l * g;
            acc = acc * f + v * g;
            top = t;
        }
    }
    __shared__ float parts[3][64][6];
    if (wave) {
        float* t = parts[wave - 1][lane];
        t[0] = top, t[1] = seen_nan ? NAN : sum, t[2] = acc[0], t[3] = acc[1], t[4] = acc[2], t[5] = acc[3];
    }
    __syncthreads();
    if (wave || !live)
        return;
#pragma unroll
    for (int k = 0; k < 3; k++) {
        const float* t = parts[k][lane];
        const float n = fmaxf(top, t[0]), at = fmaxf(n, -3.4028235e38f);
        const float f = __builtin_amdgcn_exp2f(top - at), g = __builtin_amdgcn_exp2f(t[0] - at);
        seen_nan |= !(t[1] == t[1]);
        sum = sum * f + t[1] * g;
        acc = acc * f + f32x4{t[2], t[3], t[4], t[5]} * g;
        top = n;
    }
    const float inv = seen_nan ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
    store_out(a, ((int64_t(q.first) + i) * a.heads + kvh * group + packed % group) * D + col, acc[0] * inv, acc[1] * inv,
              acc[2] * inv, acc[3] * inv);
}

template <int D>
hipError_t launch(const PagedAttentionArgs& a, hipStream_t s)
{
    const bool fine = a.out_format != PAGED_OUT_BF16;
    constexpr unsigned grid = WAVES / 4;
    if (a.cache.q4) {
        if (fine)
            paged_attention_kernel<D, true, true><<<grid, 256, 0, s>>>(a);
        else
            paged_attention_kernel<D, true, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (fine)
            paged_attention_kernel<D, false, true><<<grid, 256, 0, s>>>(a);
        else
            paged_attention_kernel<D, false, false><<<grid, 256, 0, s>>>(a);
    }
    const int group = a.heads / a.cache.kv_heads;
    const int64_t tiles = int64_t(a.batch.rows) * group / TILE_ROWS + min(a.batch.rows, a.batch.sequences);   // at most
    const int tile_rows = min(TILE_ROWS, int(min(int64_t(TILE_ROWS), int64_t(a.batch.max_rows) * group)));
    const dim3 merge(unsigned(tiles * a.cache.kv_heads), unsigned((tile_rows + 256 / D - 1) / (256 / D)));
    paged_merge_kernel<D><<<merge, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

int64_t paged_attention_workspace_floats(int, int, int head) { return int64_t(WAVES) * 2 * slot_floats(head); }

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t s)
{
    return a.cache.head == 128 ? launch<128>(a, s) : launch<64>(a, s);
}

}  // namespace si
