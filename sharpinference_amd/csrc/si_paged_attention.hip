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
// (mask and exponent in registers: one v_and_or_b32, which takes no literals)
__device__ __forceinline__ f16x2 nibbles(uint32_t w)
{
    const f16x2 k = {_Float16(1032.0f), _Float16(1032.0f)};
    uint32_t mask = 0x000F000Fu, magic = 0x64006400u, v;
    asm("" : "+s"(mask));
    asm("" : "+v"(magic));
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(v) : "v"(w), "s"(mask), "v"(magic));
    return as_f16x2(v) - k;
}

// Whether one of the word's two FP16 values is infinite or NaN.
__device__ __forceinline__ bool infinite(uint32_t w)
{
    return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
}

union Frag {
    uint32_t w[4];
    f16x8 v;
};

// The weights 2^(s - at) go into the second product as FP16, whose smallest step is
// 2^-24 (of their second terms too): relative to the largest score itself, a weight
// below 2^-14 of the largest would lose bits and one below 2^-25 be nothing, however
// many there are.  So `at` lies `room` below that score; sums and accumulators carry
// the factor 2^room, and the division takes it out.  Weights stay under 2^15, half of
// FP16's range.
constexpr float WEIGHTS_UNDER = 15.0f;
__device__ __forceinline__ float reference(float top, float room)
{
    const float at = fmaxf(top, -3.4028235e38f), low = at - room;      // (a row that has seen nothing yet)
    return at - low <= WEIGHTS_UNDER ? low : at;   // (beyond 2^27 the difference may round to 16 and more)
}

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

// few: sequences of more packed rows are the prompt kernel's
__device__ __forceinline__ Sequence take_sequence(const PagedBatch& b, int page_shift, int group, int few, int s)
{
    Sequence q{s, 0, 0, 0, 0, 0};
    if (s >= b.sequences)
        return q;
    sequence_rows(b, s, &q.first, &q.count);
    q.length = b.lengths[s];
    if (q.length < 0 || q.length > int64_t(b.max_pages) << page_shift || q.count > b.max_rows)
        q.length = -1;
    // (more rows than the call said: NaN from here, the prompt kernel may not run)
    const bool prompt = q.count * group > few && q.count <= b.max_rows;
    q.tiles = prompt ? 0 : (q.count * group + TILE_ROWS - 1) / TILE_ROWS;
    q.units = max(1, (q.length + UNIT - 1) / UNIT);
    return q;
}

// a / b for 0 <= a < 2^53, b > 0: a fifth of the code of a 64-bit division.
// The kernels run their beginnings once, from a cold instruction cache, so
// what counts there is how many instructions there are.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b)
{
    int64_t q = int64_t(double(a) / double(b));
    const int64_t r = a - q * b;
    q += r >= b ? 1 : r < 0 ? -1 : 0;
    return q;
}

__device__ __forceinline__ int64_t of_lane(int64_t v, int lane)
{
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(v), lane)), hi = uint32_t(__builtin_amdgcn_readlane(int(v >> 32), lane));
    return int64_t(uint64_t(hi) << 32 | lo);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp_or_zero(int64_t v)
{
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xF, false));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(v >> 32), CTRL, ROWS, 0xF, false));
    return int64_t(uint64_t(hi) << 32 | lo);
}
// Sums of the lanes up to each: within rows of 16, then over them.
__device__ __forceinline__ int64_t wave_scan(int64_t v)
{
    v += dpp_or_zero<0x111, 0xF>(v);       // row_shr:1
    v += dpp_or_zero<0x112, 0xF>(v);
    v += dpp_or_zero<0x114, 0xF>(v);
    v += dpp_or_zero<0x118, 0xF>(v);
    v += dpp_or_zero<0x142, 0xA>(v);       // row_bcast:15 into rows 1 and 3
    v += dpp_or_zero<0x143, 0xC>(v);       // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int64_t wave_total(int64_t v) { return of_lane(wave_scan(v), 63); }

__device__ __forceinline__ Sequence from_lane(const Sequence& q, int lane)
{
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, lane); };
    return {of(q.index), of(q.first), of(q.count), of(q.length), of(q.tiles), of(q.units)};
}

constexpr int LONG = 128;                // units: see Shares

// The work of a launch in one line: sequence after sequence, of each its KV
// heads, of each its tiles, of each its units.  A wave searches together,
// one sequence a lane.
struct Line {
    const PagedBatch& b;
    int page_shift, group, kv, few;
    int64_t total;             // units
    bool some_long;            // a tile is more than LONG units
    // up to 64 sequences are looked at once: the lane's, and the units up to it
    Sequence mine;
    int64_t upto;

    __device__ __forceinline__ int64_t units_of(const Sequence& q) const { return int64_t(kv) * q.tiles * q.units; }
    __device__ __forceinline__ void look(int base, int64_t before)
    {
        mine = take_sequence(b, page_shift, group, few, base + int(threadIdx.x & 63));
        upto = before + wave_scan(units_of(mine));
    }
    __device__ __forceinline__ explicit Line(const PagedAttentionArgs& a)
        : b(a.batch), page_shift(a.cache.page_shift), group(a.heads / a.cache.kv_heads), kv(a.cache.kv_heads),
          few(a.few_rows), total(0), some_long(false)
    {
        for (int base = 0; base < b.sequences; base += 64) {
            look(base, total);
            some_long |= __any(mine.tiles && mine.units > LONG);
            total = of_lane(upto, 63);
        }
    }
    // The sequence that holds unit x, and the number of its first unit.
    __device__ __forceinline__ bool at_unit(int64_t x, Sequence* q, int64_t* start)
    {
        if (b.sequences > 64) {
            int64_t before = 0;
            for (int base = 0; base < b.sequences; base += 64) {
                look(base, before);
                before = of_lane(upto, 63);
                if (before > x)
                    break;
            }
        }
        const uint64_t past = __ballot(upto > x);
        if (!past)
            return false;
        const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
        *q = from_lane(mine, at);
        *start = of_lane(upto - units_of(mine), at);
        return true;
    }
};

// The waves that share a line take equal runs of it.  Two units at least where a
// tile is more than LONG units: there its many slots take longer to join than a
// second unit does.  (One unit against two: 4 sequences of up to 500 positions 10.1
// and 12.8 us, one of 8000 14.6 and 14.3, one of 60000 with one KV head 33 and 24.)
constexpr int WAVES = 2048;
struct Shares {
    int64_t share;
    __device__ __forceinline__ explicit Shares(const Line& line)
        : share(max(int64_t(line.some_long ? 2 : 1), (line.total + WAVES - 1) / WAVES))
    {
    }
    __device__ __forceinline__ int64_t wave_of(int64_t unit) const { return quotient(unit, share); }
};

// What the merge has to do behind a wave (or worker): join `parts` slots, from
// the second of this one on, into rows row0 .. of a tile; parts 0: nothing.
struct Record {
    int32_t parts;
    int32_t first;             // the sequence's first batch row
    int32_t count;             // its rows
    int32_t row0;              // the tile's first packed row
    int32_t kvh;
    int32_t unused[3];
};

// What a wave leaves of a tile whose units it shares with other waves: the
// accumulators [TILE_ROWS][D], what they are relative to and sums [TILE_ROWS] each.
// Slot 2 w: of the tile that began before wave w's units, slot 2 w + 1: of
// the one that goes on behind them.
constexpr int slot_floats(int d) { return TILE_ROWS * d + 2 * TILE_ROWS; }
constexpr int PROMPT_WORKERS = 256;      // workgroups of the prompt kernel, one a CU
// A workspace: the waves' and the workers' records, their slots.
constexpr int64_t RECORD_FLOATS = sizeof(Record) / 4 * (WAVES + PROMPT_WORKERS);
constexpr int64_t prompt_workspace(int d) { return RECORD_FLOATS + int64_t(WAVES) * 2 * slot_floats(d); }
__device__ __forceinline__ Record* records(float* workspace) { return reinterpret_cast<Record*>(workspace); }

// Running state of a tile: the lane's packed row is lane & 15.
template <int D>
struct State {
    static constexpr int NV = D / 16;
    f32x4 acc[NV];             // acc[n][i]: column NV * (4 * (lane >> 4) + i) + n
    float top;                 // largest score so far (in units of log 2)
    float at;                  // what the weights are relative to
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
    static constexpr float ROOM = 14.0f; // weights of up to 2^14
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
        if constexpr (!Q4) {
            // An infinite key (FP16 pages hold what they were given; finite ones do not
            // score so) may make a score -inf: not a position of no weight, but NaN.
            float low = INFINITY;
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    low = fminf(low, s[u][i]);
            if (__any(low == -INFINITY)) {
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s[u][i] = s[u][i] == -INFINITY && base + GRANULE * u + 4 * g + i <= limit ? NAN : s[u][i];
            }
        }
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
        if (__any(top > st.top)) {
            const float at = reference(top, ROOM), fade = __builtin_amdgcn_exp2f(st.at - at);
            st.sum *= fade;
#pragma unroll
            for (int n = 0; n < NV; n++)
                st.acc[n] *= fade;
            st.top = top;
            st.at = at;
        }
        // (a unit's weights are summed by themselves: added one by one to a sum that
        // one weight dominates, ten thousand of them would lose 2^-11 of it)
        Frag pf[2], pl[2];
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[i] = __builtin_amdgcn_exp2f(s[u][i] - st.at);
                if constexpr (FINE)
                    sum += p[i];
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const f16x2 h = {_Float16(p[2 * k]), _Float16(p[2 * k + 1])};
                pf[u >> 1].w[2 * (u & 1) + k] = as_u32(h);
                // (the sum of what the product takes: their roundings cancel in the division)
                if constexpr (!FINE)
                    sum = __builtin_amdgcn_fdot2(h, f16x2{_Float16(1.0f), _Float16(1.0f)}, sum, false);
                if constexpr (FINE)
                    pl[u >> 1].w[2 * (u & 1) + k] =
                        as_u32(f16x2{_Float16(p[2 * k] - float(h[0])), _Float16(p[2 * k + 1] - float(h[1]))});
            }
        }
        st.sum += sum;
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
                        if (infinite(r.v[u][i][k])) {
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
__device__ __forceinline__ void store_out(const PagedAttentionArgs& a, int format, int64_t at, float x, float y, float z, float w)
{
    if (format == PAGED_OUT_F32)
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x, y, z, w);
    else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
            make_uint2(pack_out(x, y, format == PAGED_OUT_BF16), pack_out(z, w, format == PAGED_OUT_BF16));
}
// (what is not FINE is BF16)
template <bool FINE>
__device__ __forceinline__ int format_of(const PagedAttentionArgs& a) { return FINE ? a.out_format : PAGED_OUT_BF16; }

// Every wave takes an equal run of the line's units, whatever sequences they
// lie in; tiles that are wholly its own are written out, the others left in
// its slots for the merge.  (A workgroup a tile, with the longest sequence of 64 the
// last to end: 1080 us where this takes 80.)
// FP16 pages are bound by their bytes where there are enough of them; 4-bit ones by
// the 650 vector instructions of a unit, which run for two thirds of the time, and the
// round trips that two waves a SIMD leave open: 64 sequences of 500 to 16000
// positions take 80 us with the merge, 4.4 TB/s, where FP16 pages reach 5.6.  A unit
// takes a wave 2.7 us by itself: short batches are a launch, the search, one unit and the
// merge, 10 us.
// A unit of 128 FP16 values a position is 128 registers a lane: two waves on a
// SIMD would spill them (64 sequences of 500 to 16000 positions: 5.14 TB/s,
// with one wave 5.59).
template <int D, bool Q4, bool FINE>
__global__ void __launch_bounds__(256, !Q4 && D == 128 ? 1 : 2)
paged_attention_kernel(const PagedAttentionArgs a)
{
    constexpr int NV = D / 16;
    const int kv = a.cache.kv_heads, group = a.heads / kv;
    Line line(a);
    const int64_t total = line.total;
    const Shares shares(line);
    // Neighbours in the line on one die (workgroup b runs on die b % 8): the tiles
    // of a sequence's rows go through the same pages, and meet in its L2.
    const int per = int(quotient(total + 32 * shares.share - 1, 32 * shares.share));       // workgroups of a die
    const int block = int(blockIdx.x) / 8 < per ? int(blockIdx.x) % 8 * per + int(blockIdx.x) / 8 : int(blockIdx.x);
    const int64_t wave = int64_t(block) * 4 + (threadIdx.x >> 6);
    const int64_t begin = wave * shares.share, end = min(total, begin + shares.share);
    Record record{};
    Attend<D, Q4, FINE> w(a);
    Sequence q{};
    int64_t q_start = 0, q_end = 0;
    for (int64_t x = begin; x < end;) {
        if (x >= q_end) {
            if (!line.at_unit(x, &q, &q_start))
                break;
            q_end = q_start + line.units_of(q);
        }
        // unit x: of which KV head, tile and positions
        const int64_t in = x - q_start;
        const uint32_t tile_no = uint32_t(quotient(in, q.units));       // at most 2^20 tiles and 256 heads
        const int kvh = __builtin_amdgcn_readfirstlane(int(tile_no / uint32_t(q.tiles)));
        const int row0 = __builtin_amdgcn_readfirstlane(int(tile_no - kvh * q.tiles) * TILE_ROWS);
        const int unit0 = __builtin_amdgcn_readfirstlane(int(in - int64_t(tile_no) * q.units));
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
        st.at = reference(st.top, 0.0f);
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
        // (a row that sees some position here has a weight of 1 and more, but for a query
        // beyond FP16 whose keys all have the other sign: every score is -inf)
        float sum = rows_sum(st.sum);
        sum = sum == 0.0f && limit >= unit0 * UNIT ? NAN : sum;
        if (tile_start >= begin && tile_end <= end) {
            const float inv = wrong ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
            if (live) {
                const int64_t at = (row * a.heads + head) * D + NV * 4 * w.g;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int n = 0; n < NV; n += 4)
                        store_out(a, format_of<FINE>(a), at + NV * r + n, st.acc[n][r] * inv, st.acc[n + 1][r] * inv, st.acc[n + 2][r] * inv,
                                  st.acc[n + 3][r] * inv);
            }
        } else if (live) {
            float* slot = a.workspace + RECORD_FLOATS + (2 * wave + (tile_start >= begin)) * slot_floats(D);
            float* at = slot + w.c * D + NV * 4 * w.g;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int n = 0; n < NV; n += 4)
                    *reinterpret_cast<f32x4*>(at + NV * r + n) =
                        f32x4{st.acc[n][r], st.acc[n + 1][r], st.acc[n + 2][r], st.acc[n + 3][r]};
            if (w.g == 0) {
                slot[TILE_ROWS * D + w.c] = st.at;
                slot[TILE_ROWS * D + TILE_ROWS + w.c] = sum;
            }
        }
        if (tile_start >= begin && tile_end > end)
            record = {int(shares.wave_of(tile_end - 1) - wave) + 1, q.first, q.count, row0, kvh, {}};
    }
    if (w.lane == 0)
        records(a.workspace)[wave] = record;
}

// Joins what `parts` slots, `stride` floats apart, hold of four neighbouring
// values of a row: those of its accumulators at `at`, what it is relative to and
// its sum at `stats` and `stats` + rows.
struct Joined {
    float top = -INFINITY, sum = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    __device__ __forceinline__ void take(float m, float l, f32x4 v)
    {
        const float t = fmaxf(top, m), at = fmaxf(t, -3.4028235e38f);
        const float f = __builtin_amdgcn_exp2f(top - at), g = __builtin_amdgcn_exp2f(m - at);
        sum = sum * f + l * g;             // (NaN stays NaN)
        acc = acc * f + v * g;
        top = t;
    }
};

// What the four waves of a workgroup hold, in its first; true there.
__device__ __forceinline__ bool join_waves(Joined& sum)
{
    __shared__ float parts[3][2][64];
    __shared__ f32x4 parts_acc[3][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (wave) {
        parts[wave - 1][0][lane] = sum.top;
        parts[wave - 1][1][lane] = sum.sum;
        parts_acc[wave - 1][lane] = sum.acc;
    }
    __syncthreads();
    if (wave)
        return false;
#pragma unroll
    for (int k = 0; k < 3; k++)
        sum.take(parts[k][0][lane], parts[k][1][lane], parts_acc[k][lane]);
    return true;
}

// Joins the tile that begins in wave `owner` and ends behind it: rows 256 / D x
// `piece` and on, four values a lane; the workgroup's waves take the slots in turn.
template <int D>
__device__ __forceinline__ void join_tile(const PagedAttentionArgs& a, const Record& todo, int owner, int piece)
{
    constexpr int ROWS = 256 / D;
    const int group = a.heads / a.cache.kv_heads;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int r = piece * ROWS + lane / (D / 4), col = 4 * (lane % (D / 4));
    const int packed = todo.row0 + r, i = packed / group;
    const bool live = i < todo.count;
    Joined sum;
    if (live) {
        // (a tile's own wave has it in its second slot, the others in their first)
        const float* slot = a.workspace + RECORD_FLOATS + 2 * int64_t(owner) * slot_floats(D);
#pragma unroll 8
        for (int p = wave; p < todo.parts; p += 4) {
            const float* const at = slot + (2 * p + (p == 0)) * slot_floats(D);
            sum.take(at[TILE_ROWS * D + r], at[TILE_ROWS * D + TILE_ROWS + r], *reinterpret_cast<const f32x4*>(at + r * D + col));
        }
    }
    if (!join_waves(sum) || !live)
        return;
    const float inv = sum.sum == 0.0f ? 0.0f : 1.0f / sum.sum;
    store_out(a, a.out_format, ((int64_t(todo.first) + i) * a.heads + todo.kvh * group + packed % group) * D + col, sum.acc[0] * inv,
              sum.acc[1] * inv, sum.acc[2] * inv, sum.acc[3] * inv);
}

// Joins the tiles that several waves share: workgroup x the one that begins in wave x.
template <int D>
__global__ void __launch_bounds__(256)
paged_merge_kernel(const PagedAttentionArgs a)
{
    const Record todo = records(a.workspace)[blockIdx.x];
    if (todo.parts)
        join_tile<D>(a, todo, blockIdx.x, blockIdx.y);
}

// ---- many rows of a sequence ------------------------------------------------------------

// A workgroup of eight waves takes 256 packed rows of one sequence and KV
// head, 32 a wave, through units of 64 positions.  The unit's keys and values
// go through LDS as FP16, dequantized once for the eight waves, two buffers: the
// next unit's bytes are loaded while this one is multiplied.  Scores stay
// transposed here too, with v_mfma_f32_32x32x16_f16.
//
// What bounds it: of the 4880 cycles that a unit of 64 positions takes, the two
// waves of a SIMD spend 2050 in matrix instructions and 2100 in vector ones (580
// of them the exponentials), which overlap little.  840 TFLOP/s within the units
// at the 1.95 GHz that the card then runs at, 0.55 of what a large matrix product
// reaches.
// Chunks of up to 2000 rows over up to 6000 positions take 210 us, joins included; when
// this form took 229, one of 128 rows in four waves took 252.
constexpr int PROMPT_ROWS = 256;
constexpr int PROMPT_THREADS = 512;
// What the scores are taken relative to follows their maximum only when the weights
// would pass 2^15 (WEIGHTS_UNDER): the accumulators are rescaled a few times a row
// instead of once a unit (440 vector instructions a unit then, 300 now).  It then lies
// this far below the maximum: a maximum that grows by 8, or (two-term operands,
// whose weights are to keep their bits further down) by 2, moves it again.
constexpr float prompt_room(bool fine) { return fine ? 13.0f : 7.0f; }
constexpr int PROMPT_PIECE = 7;          // what a piece of a tile costs besides its units, in units
constexpr int PROMPT_MIN = 9;            // units that a worker takes at least, with a piece's cost

using f32x16 = float __attribute__((ext_vector_type(16)));

constexpr int prompt_slot_floats(int d) { return PROMPT_ROWS * d + 2 * PROMPT_ROWS; }

struct PromptSequence {
    int index, first, count, length, tiles;
    int64_t a, c;              // weight of the tiles: see PromptLine
};

// The work of a launch in one line: sequence after sequence, of each its KV
// heads, of each its tiles.  Tile i of a sequence goes through about (length
// - count) / 64 + (i + 1/2) 4 / group units (a tile is 256 / group positions
// long, and each sees all before it), and costs PROMPT_PIECE units more, which its
// queries and outputs take.  Its weight is group times that: w_i = a + 2 c i + c
// with c = 2, all of tiles 0 .. t - 1 together a t + c t^2.  Every worker takes an
// equal run of the line; a border inside a tile is at the same share of its units.
//
// Where there are few tiles, a border that every worker meets somewhere in its
// run costs more than parts that are not quite equal: there all tiles of a
// sequence are cut into as many parts as its last one needs (c = 0, a = parts *
// share), and no worker has more than one part.
struct PromptLine {
    const PagedBatch& b;
    int page_shift, group, kv, few;
    int64_t share;             // of a worker
    bool cut;                  // into parts

    static __device__ __forceinline__ int64_t before(const PromptSequence& q, int64_t t) { return (q.a + q.c * t) * t; }
    static __device__ __forceinline__ int64_t tile_weight(const PromptSequence& q, int64_t t) { return q.a + q.c * (2 * t + 1); }
    __device__ __forceinline__ int64_t weight(const PromptSequence& q) const { return kv * before(q, q.tiles); }
    __device__ __forceinline__ PromptSequence take(int s) const
    {
        PromptSequence q{s, 0, 0, 0, 0, 0, 2};
        if (s >= b.sequences)
            return q;
        sequence_rows(b, s, &q.first, &q.count);
        q.length = b.lengths[s];
        if (q.length < 0 || q.length > int64_t(b.max_pages) << page_shift)
            q.length = -1;
        const bool prompt = q.count * group > few && q.count <= b.max_rows;
        q.tiles = prompt ? (q.count * group + PROMPT_ROWS - 1) / PROMPT_ROWS : 0;
        q.a = int64_t(group) * (max(0, q.length - q.count) / UNIT + PROMPT_PIECE);
        if (cut && q.tiles) {
            q.a = (quotient(tile_weight(q, q.tiles - 1) - 1, share) + 1) * share;
            q.c = 0;
        }
        return q;
    }
    __device__ __forceinline__ explicit PromptLine(const PagedAttentionArgs& a)
        : b(a.batch), page_shift(a.cache.page_shift), group(a.heads / a.cache.kv_heads), kv(a.cache.kv_heads),
          few(a.few_rows), share(0), cut(false)
    {
        // all weight, tiles, and the weight if a sequence's tiles were all like its last
        int64_t total = 0, tiles = 0, last = 0;
        for (int base = 0; base < b.sequences; base += 64) {
            const PromptSequence q = take(base + int(threadIdx.x & 63));
            total += weight(q);
            tiles += int64_t(kv) * q.tiles;
            last += q.tiles ? int64_t(kv) * q.tiles * tile_weight(q, q.tiles - 1) : 0;
        }
        total = wave_total(total);
        tiles = wave_total(tiles);
        last = wave_total(last);
        share = max(int64_t(PROMPT_MIN) * group, (total + PROMPT_WORKERS - 1) / PROMPT_WORKERS);
        if (tiles < PROMPT_WORKERS) {
            // at most last / parts + tiles <= PROMPT_WORKERS parts
            const int64_t parts = max(int64_t(PROMPT_MIN) * group, quotient(last, PROMPT_WORKERS - tiles) + 1);
            cut = parts <= share + PROMPT_PIECE * group;
            share = cut ? parts : share;
        }
    }
    __device__ __forceinline__ int64_t worker_of(int64_t place) const { return quotient(place, share); }
    static __device__ __forceinline__ PromptSequence from_lane(const PromptSequence& q, int lane)
    {
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, lane); };
        return {of(q.index), of(q.first), of(q.count), of(q.length), of(q.tiles), of_lane(q.a, lane), of_lane(q.c, lane)};
    }
    // The sequence that holds place x, and the place of its begin.
    __device__ __forceinline__ bool find(int64_t x, PromptSequence* q, int64_t* start) const
    {
        int64_t places = 0;
        for (int base = 0; base < b.sequences; base += 64) {
            const PromptSequence mine = take(base + int(threadIdx.x & 63));
            const int64_t w = weight(mine);
            const int64_t places_upto = places + wave_scan(w);
            const uint64_t past = __ballot(places_upto > x);
            if (past) {
                const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
                *q = from_lane(mine, at);
                *start = of_lane(places_upto - w, at);
                return true;
            }
            places = of_lane(places_upto, 63);
        }
        return false;
    }
    // The tile that holds place y of a KV head.
    static __device__ __forceinline__ int64_t tile_at(const PromptSequence& q, int64_t y)
    {
        const double a = double(q.a);
        int64_t t = q.c ? int64_t((sqrt(a * a + 4.0 * q.c * double(y)) - a) / (2.0 * q.c)) : quotient(y, q.a);
        t = min(int64_t(q.tiles) - 1, t);
        while (t > 0 && before(q, t) > y)
            t--;
        while (before(q, t + 1) <= y)
            t++;
        return t;
    }
};

template <int D>
__device__ __forceinline__ int key_at(int row, int piece)      // bytes of 16-byte piece `piece` of a key
{
    return row * (2 * D) + ((piece ^ (D == 128 ? row & 15 : (row >> 1) & 7)) << 4);
}
__device__ __forceinline__ int value_at(int col, int piece)    // of eight positions of a column
{
    return col * 128 + ((piece ^ (((col >> 1) ^ (col >> 4)) & 7)) << 4);
}

// What a lane loads of a unit.  Wave w takes eight positions' keys, an eighth of
// a row a lane, and piece w of the values' columns, two columns a lane: positions
// 16 (w / 2) + 4 (w % 2) + {0..3, 8..11}.  Both lie in one page, so everything
// that changes from unit to unit is in scalar registers; the lane keeps its
// places in the page and in LDS.  (Waves that took keys or values only: the
// registers of both then met behind the branch, which waited for the loads
// there and then.)
template <int D, bool Q4, bool FINE>
struct PromptLoad {
    static constexpr int ROW = Q4 ? D / 2 : 2 * D;             // bytes of a row in a page
    static constexpr int PIECES = D / 64;                      // of the lane's keys: words (4-bit) or 16 bytes, 128 apart
    static constexpr bool ALL = D == 128;                      // lanes that have values
    uint32_t k[Q4 ? PIECES : 4 * PIECES], kd;
    uint32_t v[Q4 ? 2 : 8], vd[Q4 ? 4 : 1];
    uint32_t byte;                         // of the words of a quad of lanes: this lane's
    int key_from, key_scale, key_to, value_from, value_scale, value_to;
    int key_first, value_first;            // first positions in the unit
    bool has_values;

    __device__ __forceinline__ PromptLoad(int wave, int lane, int page_size, int values_at)
    {
        const int half = wave & 1, row = 8 * half + (lane >> 3), piece = lane & 7;
        key_first = GRANULE * (wave >> 1) + row;
        key_from = row * ROW + (Q4 ? 4 * PIECES : 16) * piece;
        key_scale = 2 * ((PIECES * piece >> 2) * page_size + row);
        key_to = key_at<D>(key_first, Q4 ? PIECES * piece : piece);
        has_values = ALL || lane < D / 2;
        const int c = lane % (D / 2);
        value_first = GRANULE * (wave >> 1) + 4 * half;
        value_from = Q4 ? (4 * half + (c & 3)) * ROW + (c & ~3) : 4 * half * ROW + 4 * c;
        byte = 0x0C040C00u + 0x00010001u * (c & 3);
        value_scale = 2 * ((c >> 4) * page_size + 4 * half);
        value_to = values_at + value_at(2 * c, wave);
    }

    // keys, values: the granule's page of this KV head, slot: the granule's place in it
    __device__ __forceinline__ void load(const char* keys, const char* values, int slot, int page_size)
    {
        const char* const kr = keys + slot * ROW;
        const char* const vr = values + slot * ROW;
        const int scales = page_size * (D / 2) + 2 * slot;
        if constexpr (Q4) {
            if constexpr (PIECES == 2) {
                const uint2 x = *reinterpret_cast<const uint2*>(kr + key_from);
                k[0] = x.x, k[1] = x.y;
            } else {
                k[0] = *reinterpret_cast<const uint32_t*>(kr + key_from);
            }
            kd = *reinterpret_cast<const uint16_t*>(keys + scales + key_scale);
        } else {
#pragma unroll
            for (int j = 0; j < PIECES; j++) {
                const uint4 x = *reinterpret_cast<const uint4*>(kr + key_from + 128 * j);
                k[4 * j] = x.x, k[4 * j + 1] = x.y, k[4 * j + 2] = x.z, k[4 * j + 3] = x.w;
            }
        }
        // (a lane without values reads those of another)
        if constexpr (!Q4) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                v[i] = *reinterpret_cast<const uint32_t*>(vr + value_from + ((i & 3) + 8 * (i >> 2)) * ROW);
        } else {
            // four lanes read the words of four positions each, and share them below
            v[0] = *reinterpret_cast<const uint32_t*>(vr + value_from);
            v[1] = *reinterpret_cast<const uint32_t*>(vr + value_from + 8 * ROW);
            const char* const d = values + scales + value_scale;
            const uint2 x = *reinterpret_cast<const uint2*>(d), y = *reinterpret_cast<const uint2*>(d + 16);
            vd[0] = x.x, vd[1] = x.y, vd[2] = y.x, vd[3] = y.y;
        }
    }

    // Into LDS as FP16 (FINE 4-bit: and what is left of the products `lo` bytes
    // on).  `partial`: some row does not see all of the unit; keys and values
    // that are not finite are then taken out and their positions marked in `odd`.
    __device__ __forceinline__ void store(char* lds, int lo, bool partial, uint32_t* odd)
    {
        if (partial)
            take_out_odd(odd);
        if constexpr (Q4) {
            const f16x2 d = as_f16x2(kd | kd << 16);
#pragma unroll
            for (int j = 0; j < PIECES; j++) {
                Frag x, y;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const f16x2 n = nibbles(k[j] >> (4 * e)), p = n * d;
                    x.w[e] = as_u32(p);
                    if constexpr (FINE)
                        y.w[e] = as_u32(__builtin_elementwise_fma(n, d, -p));
                }
                *reinterpret_cast<f16x8*>(lds + (key_to ^ j << 4)) = x.v;
                if constexpr (FINE)
                    *reinterpret_cast<f16x8*>(lds + lo + (key_to ^ j << 4)) = y.v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PIECES; j++)
                *reinterpret_cast<uint4*>(lds + (key_to ^ j << 7)) = make_uint4(k[4 * j], k[4 * j + 1], k[4 * j + 2], k[4 * j + 3]);
        }
        if (!has_values)
            return;
        uint32_t both[4];                                  // 4-bit: two positions' two columns
        if constexpr (Q4) {
#pragma unroll
            for (int p = 0; p < 2; p++) {
                both[2 * p] = __builtin_amdgcn_perm(of_quad<1>(v[p]), of_quad<0>(v[p]), byte);
                both[2 * p + 1] = __builtin_amdgcn_perm(of_quad<3>(v[p]), of_quad<2>(v[p]), byte);
            }
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            Frag x, y;
#pragma unroll
            for (int p = 0; p < 4; p++) {
                if constexpr (Q4) {
                    const f16x2 d = as_f16x2(vd[p]);
                    const f16x2 m = nibbles(both[p] >> (4 * n)), z = m * d;
                    x.w[p] = as_u32(z);
                    if constexpr (FINE)
                        y.w[p] = as_u32(__builtin_elementwise_fma(m, d, -z));
                } else {
                    x.w[p] = __builtin_amdgcn_perm(v[2 * p + 1], v[2 * p], n & 1 ? 0x07060302u : 0x05040100u);
                }
            }
            *reinterpret_cast<f16x8*>(lds + value_to + n * 128) = x.v;
            if constexpr (FINE && Q4)
                *reinterpret_cast<f16x8*>(lds + lo + value_to + n * 128) = y.v;
        }
    }

    // v of lane I of the quad
    template <int I>
    static __device__ __forceinline__ uint32_t of_quad(uint32_t v)
    {
        return uint32_t(__builtin_amdgcn_mov_dpp(int(v), 0x55 * I, 0xF, 0xF, true));
    }

    __device__ __forceinline__ void take_out_odd(uint32_t* odd)
    {
        bool bad = false;
        if constexpr (Q4) {
            bad = (kd & 0x7000u) == 0x7000u;               // 8192 and up: 8 x it passes FP16's largest value
            kd = bad ? 0 : kd;
        } else {
#pragma unroll
            for (int j = 0; j < 4 * PIECES; j++) {
                const bool b = infinite(k[j]);
                bad |= b;
                k[j] = b ? 0 : k[j];
            }
        }
        if (bad)
            atomicOr(&odd[key_first >> 5], 1u << (key_first & 31));
        uint32_t mask = 0;                                 // positions from value_first on
#pragma unroll
        for (int i = 0; i < 8; i++) {
            bool b;
            if constexpr (Q4) {
                const uint32_t e = 0x7000u << (16 * (i & 1));
                b = (vd[i >> 1] & e) == e;
                vd[i >> 1] = b ? vd[i >> 1] & ~(0xFFFFu << (16 * (i & 1))) : vd[i >> 1];
            } else {
                b = infinite(v[i]);
                v[i] = b ? 0 : v[i];
            }
            mask |= b ? 1u << ((i & 3) + 8 * (i >> 2)) : 0u;
        }
        // (a granule lies in one of the two words)
        if (mask)
            atomicOr(&odd[value_first >> 5], mask << (value_first & 31));
    }
};

template <int D, bool Q4, bool FINE>
__global__ void __launch_bounds__(PROMPT_THREADS, 2)
paged_prompt_kernel(const PagedAttentionArgs a)
{
    constexpr int NK = D / 16, NC = D / 32;
    constexpr int PLANE = UNIT * D * 2;                   // bytes of a unit's keys, and of its values
    constexpr int PLANES = FINE && Q4 ? 4 : 2;
    __shared__ __align__(16) char lds[2][PLANES * PLANE];
    __shared__ uint32_t odd[3][2];
    const int kv = a.cache.kv_heads, group = a.heads / kv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
    const int64_t head_bytes = paged_head_bytes(Q4, a.cache.page_size, D);
    const PromptLine line(a);
    // neighbours in the line on one die (workgroup b runs on die b % 8): they
    // go through the same keys and values, and meet in its L2
    const int64_t worker = int64_t(blockIdx.x % 8) * (PROMPT_WORKERS / 8) + blockIdx.x / 8;
    const int64_t begin = worker * line.share, end = begin + line.share;
    PromptLoad<D, Q4, FINE> raw(wave, lane, a.cache.page_size, PLANE);
    Record record{};
    PromptSequence q{};
    int64_t q_start = 0, q_end = 0;
    for (int64_t x = begin; x < end;) {
        if (x >= q_end) {
            if (!line.find(x, &q, &q_start))
                break;
            q_end = q_start + line.weight(q);
        }
        const int64_t head_weight = PromptLine::before(q, q.tiles);
        const int kvh = __builtin_amdgcn_readfirstlane(int(quotient(x - q_start, head_weight)));
        const int64_t y = x - q_start - kvh * head_weight;
        const int tile = __builtin_amdgcn_readfirstlane(int(PromptLine::tile_at(q, y)));
        const int64_t weight = PromptLine::tile_weight(q, tile), lo = y - PromptLine::before(q, tile);
        const int64_t hi = min(weight, lo + (end - x));
        x += hi - lo;
        if (lo == 0 && hi < weight)
            record = {int(line.worker_of(x + weight - hi - 1) - worker) + 1, q.first, q.count, tile * PROMPT_ROWS, kvh, {}};
        const bool wrong = q.length < 0;
        const int row0 = tile * PROMPT_ROWS;
        const int packed = row0 + 32 * wave + r, i = packed / group;
        const bool live = i < q.count;
        const int64_t row = int64_t(q.first) + i;
        const int head = kvh * group + packed % group;
        const int limit = live && !wrong ? q.length - q.count + i : -1;
        const int last_row = min(q.count - 1, (row0 + PROMPT_ROWS - 1) / group);
        const int most = __builtin_amdgcn_readfirstlane(wrong ? -1 : q.length - q.count + last_row);
        const int least = __builtin_amdgcn_readfirstlane(q.length - q.count + row0 / group);
        // of this tile; 0 where no row sees anything, however far before position 0 its rows lie
        const int units = max(0, (most + UNIT) / UNIT);
        const int unit0 = __builtin_amdgcn_readfirstlane(int(quotient(units * lo, weight)));
        const int unit1 = __builtin_amdgcn_readfirstlane(int(quotient(units * hi, weight)));
        const int32_t* const table = a.batch.table + int64_t(q.index) * a.batch.max_pages;

        // queries of this lane's row: piece 2 k + h of its values for product k
        f16x8 qf[NK], ql[FINE ? NK : 1];
        {
            const float f = 1.44269504088896340736f / sqrtf(float(D));
            const float* const p = live ? a.query + (row * a.heads + head) * D : nullptr;
#pragma unroll
            for (int k = 0; k < NK; k++) {
                float4 x = make_float4(0, 0, 0, 0), y = x;
                if (p) {
                    x = *reinterpret_cast<const float4*>(p + 16 * k + 8 * h);
                    y = *reinterpret_cast<const float4*>(p + 16 * k + 8 * h + 4);
                }
                const float v[8] = {x.x * f, x.y * f, x.z * f, x.w * f, y.x * f, y.y * f, y.z * f, y.w * f};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float t = Q4 ? v[(e >> 1) + 4 * (e & 1)] : v[e];
                    qf[k][e] = _Float16(t);
                    if constexpr (FINE)
                        ql[k][e] = _Float16(t - float(qf[k][e]));
                }
            }
        }
        f32x16 acc[NC];
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                acc[n][e] = 0.0f;
        float ref = 0.0f, gate = -INFINITY, sum = 0.0f;
        // Places of the lane's fragments: rows 32 apart share their swizzle,
        // columns 32 apart differ in it by 2 n, so eight and four offsets do.
        int key_of[NK], value_of[4];
#pragma unroll
        for (int k = 0; k < NK; k++)
            key_of[k] = key_at<D>(r, 2 * k + h);
#pragma unroll
        for (int k = 0; k < 4; k++)
            value_of[k] = PLANE + value_at(r, 2 * k + h);

        // Pages of the 64 granules around a unit, one a lane of every wave; those
        // that are not there: page 0 is read in their place.
        int held = 0, held_at = -1;
        uint64_t held_lost = 0;
        const char* const keys = a.cache.keys + kvh * head_bytes;
        const char* const values = a.cache.values + kvh * head_bytes;
        const uint32_t page_bytes = uint32_t(a.cache.kv_heads * head_bytes);       // at most 16 MiB
        auto load = [&](int u) -> uint32_t {
            if (u >> 4 != held_at) {
                held_at = u >> 4;
                const int pos = (held_at * 64 + lane) * GRANULE;
                held = pos <= most ? table[pos >> a.cache.page_shift] : 0;
                if (held >= a.cache.pages)
                    held = -1;
                held_lost = __ballot(held < 0);
            }
            const int granule = (u & 15) * 4 + (wave >> 1);
            const int page = max(0, __builtin_amdgcn_readlane(held, granule));
            const uint64_t at = uint64_t(uint32_t(page)) * page_bytes;
            raw.load(keys + at, values + at, (u * UNIT + (wave >> 1) * GRANULE) & (a.cache.page_size - 1), a.cache.page_size);
            return uint32_t(held_lost >> (u & 15) * 4) & 15;
        };
        auto partial = [&](int u) { return u * UNIT + UNIT - 1 > least; };
        uint32_t lost = 0, lost_next = 0;
        __syncthreads();                                  // the item before is done with LDS
        if (threadIdx.x < 6)
            (&odd[0][0])[threadIdx.x] = 0;
        // The loop begins with a unit before the first one, whose scores are
        // -inf and whose values are zeros: what it does for the next units
        // (storing, loading, the scores) need not stand here once more.
#pragma unroll 1
        for (int p = 1; p < PLANES; p += 2)
            for (int at = 16 * threadIdx.x; at < PLANE; at += 16 * PROMPT_THREADS)
                *reinterpret_cast<uint4*>(lds[(unit0 + 1) & 1] + p * PLANE + at) = make_uint4(0, 0, 0, 0);
        if (unit0 < unit1)
            lost_next = load(unit0);
        __syncthreads();

        // Fragments are read ahead of their products (FINE: by a smaller step, for
        // want of registers); the order is pinned, or the compiler reads each right
        // before it is used.
        constexpr int GROUP = FINE ? 1 : 2, SETS = FINE ? 2 : 3;
        f16x8 f[SETS][GROUP], fl[SETS][FINE && Q4 ? GROUP : 1];
        f32x16 s[2];
        Frag pf[2][2], pl[2][2];
        auto read = [&](const char* at, int set, int i) {
            f[set][i] = *reinterpret_cast<const f16x8*>(at);
            if constexpr (FINE && Q4)
                fl[set][i] = *reinterpret_cast<const f16x8*>(at + 2 * PLANE);
        };
        auto column = [](int p) { return 2 * (p >> 3) + (p & 1); };
        auto read_keys = [&](int u, int g, int set) {
#pragma unroll
            for (int i = 0; i < GROUP; i++) {
                const int p = g * GROUP + i;
                read(lds[u & 1] + key_of[p >> 1] + 32 * (p & 1) * 2 * D, set, i);
            }
        };
        auto read_values = [&](int u, int g, int set) {
#pragma unroll
            for (int i = 0; i < GROUP; i++) {
                const int p = g * GROUP + i, n = column(p);
                read(lds[u & 1] + value_of[(p >> 1 & 3) ^ (n & 3)] + 32 * n * 128, set, i);
            }
        };
        // Two accumulators take turns, so a product does not wait for the one
        // before it: product p of the scores is of block p % 2 and values p / 2,
        // of the sums of columns column(p) and positions p / 2 % 4.
        constexpr int AHEAD = SETS - 1;
        constexpr int SCORES = 2 * NK / GROUP, SUMS = 4 * NC / GROUP;      // groups of a unit
        // The scores of unit u, whose first fragments are in sets `set` and on.  They
        // start from what is taken off them, and are -inf where a row does not see the position.
        // Element e of block b: position base + 32 b + 8 (e / 4) + 4 h + e % 4.
        auto scores = [&](int u, int set) {
#pragma unroll
            for (int e = 0; e < 16; e++)
                s[0][e] = s[1][e] = -ref;
#pragma unroll
            for (int g = 0; g < SCORES; g++) {
                if (g + AHEAD < SCORES)
                    read_keys(u, g + AHEAD, (set + g + AHEAD) % SETS);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < GROUP; i++) {
                    const int k = (g * GROUP + i) >> 1, b = (g * GROUP + i) & 1, at = (set + g) % SETS;
                    if constexpr (FINE && Q4)
                        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl[at][i], qf[k], s[b], 0, 0, 0);
                    if constexpr (FINE)
                        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[at][i], ql[k], s[b], 0, 0, 0);
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[at][i], qf[k], s[b], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (!Q4) {
                // an infinite key's -inf is NaN to those that see it (all of them, or the
                // key was taken out)
                float low = INFINITY;
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        low = fminf(low, s[b][e]);
                if (__any(low == -INFINITY)) {
#pragma unroll
                    for (int b = 0; b < 2; b++)
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            s[b][e] = s[b][e] == -INFINITY ? NAN : s[b][e];
                }
            }
            if (partial(u)) {
                // (a new value each time, or 32 positions live through the loop)
                int first = 4 * h;
                asm volatile("" : "+v"(first));
                const int seen = limit - u * UNIT - first;
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        s[b][e] = 32 * b + 8 * (e >> 2) + (e & 3) > seen ? -INFINITY : s[b][e];
            }
        };
        // One barrier a unit: between two of them a wave takes the scores of a
        // unit, its exponentials and sums, and stores its part of the next one.
        // The two waves of a SIMD come to each step after each other, so one is at
        // its products while the other is at its exponentials.  (Halves of the
        // workgroup that take turns behind two barriers a unit were no faster, with
        // the conversions among the exponentials or among the products: 198 to 219
        // against 197 us for 137216 positions.)
#pragma unroll
        for (int e = 0; e < 16; e++)
            s[0][e] = s[1][e] = -INFINITY;
        for (int u = unit0 - 1; u < unit1; u++) {
            const int base = u * UNIT;
            if (u >= unit0 && (partial(u) || lost)) {
                // a row that sees a position without a page, or with a key or
                // value that is not finite (0 in LDS), is NaN
                const uint32_t bad0 = odd[u % 3][0] | (lost & 1 ? 0xFFFFu : 0u) | (lost & 2 ? 0xFFFF0000u : 0u);
                const uint32_t bad1 = odd[u % 3][1] | (lost & 4 ? 0xFFFFu : 0u) | (lost & 8 ? 0xFFFF0000u : 0u);
                const int seen = limit - base;
                const uint32_t see0 = seen >= 31 ? ~0u : seen < 0 ? 0u : (2u << seen) - 1;
                const uint32_t see1 = seen >= 63 ? ~0u : seen < 32 ? 0u : (2u << (seen - 32)) - 1;
                sum = (bad0 & see0) | (bad1 & see1) ? NAN : sum;
            }
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    top = fmaxf(top, s[b][e]);
            {
                auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
            }
            if (__any(top > gate)) {
                // (a row that has seen nothing yet has nothing to rescale, and its
                // first score may be far below 0)
                const float by = top > gate ? reference(top, prompt_room(FINE)) : 0.0f;
                const float fade = top > gate && gate < 0.0f ? 0.0f : __builtin_amdgcn_exp2f(-by);
                gate = top > gate ? WEIGHTS_UNDER : gate;
                ref += by;
                sum *= fade;
#pragma unroll
                for (int n = 0; n < NC; n++)
                    acc[n] *= fade;
#pragma unroll
                for (int b = 0; b < 2; b++)
                    s[b] -= by;
            }
            float more = 0.0f;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float x = __builtin_amdgcn_exp2f(s[b][e]), y = __builtin_amdgcn_exp2f(s[b][e + 1]);
                    const f16x2 p = {_Float16(x), _Float16(y)};
                    pf[b][e >> 3].w[(e & 7) >> 1] = as_u32(p);
                    more = FINE ? more + (x + y) : __builtin_amdgcn_fdot2(p, f16x2{_Float16(1.0f), _Float16(1.0f)}, more, false);
                    if constexpr (FINE)
                        pl[b][e >> 3].w[(e & 7) >> 1] = as_u32(f16x2{_Float16(x - float(p[0])), _Float16(y - float(p[1]))});
                }
            sum += more;
            // (last read for unit u - 1, next marked for unit u + 2; marked for
            // partial units alone, which are the last ones)
            if (partial(u + 2) && threadIdx.x < 2)
                odd[(u + 2) % 3][threadIdx.x] = 0;
            read_values(u, 0, 0);
            if constexpr (AHEAD > 1)
                read_values(u, 1, 1);
#pragma unroll
            for (int g = 0; g < SUMS; g++) {
                if (g + AHEAD < SUMS)
                    read_values(u, g + AHEAD, (g + AHEAD) % SETS);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < GROUP; i++) {
                    const int p = g * GROUP + i, n2 = column(p), b = (p >> 2) & 1, k = (p >> 1) & 1;
                    if constexpr (FINE && Q4)
                        acc[n2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl[g % SETS][i], pf[b][k].v, acc[n2], 0, 0, 0);
                    if constexpr (FINE)
                        acc[n2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[g % SETS][i], pl[b][k].v, acc[n2], 0, 0, 0);
                    acc[n2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[g % SETS][i], pf[b][k].v, acc[n2], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            lost = lost_next;
            if (u + 1 < unit1) {
                raw.store(lds[(u + 1) & 1], 2 * PLANE, partial(u + 1), odd[(u + 1) % 3]);
                if (u + 2 < unit1)
                    lost_next = load(u + 2);
            }
            __syncthreads();
            read_keys(u + 1, 0, 0);
            if constexpr (AHEAD > 1)
                read_keys(u + 1, 1, 1);
            scores(u + 1, 0);
        }
        {
            auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
            sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            // (scores that are all -inf: a query beyond FP16)
            sum = sum == 0.0f && unit0 < unit1 && limit >= unit0 * UNIT ? NAN : sum;
        }
        // element e of acc[n]: column 32 n + 8 (e / 4) + 4 h + e % 4
        if (lo == 0 && hi == weight) {
            if (!live)
                continue;
            const float inv = wrong ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
            const int64_t out = (row * a.heads + head) * D + 4 * h;
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    store_out(a, format_of<FINE>(a), out + 32 * n + 2 * e, acc[n][e] * inv, acc[n][e + 1] * inv, acc[n][e + 2] * inv,
                              acc[n][e + 3] * inv);
        } else if (row0 + 32 * wave < q.count * group) {
            float* const slot = a.workspace + prompt_workspace(D) + (2 * worker + (lo == 0)) * prompt_slot_floats(D);
            f32x4* const out = reinterpret_cast<f32x4*>(slot) + wave * (4 * NC * 64) + lane;
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    out[(4 * n + e / 4) * 64] = f32x4{acc[n][e], acc[n][e + 1], acc[n][e + 2], acc[n][e + 3]};
            if (h == 0) {
                slot[PROMPT_ROWS * D + 32 * wave + r] = sum == 0.0f ? -INFINITY : ref;
                slot[PROMPT_ROWS * D + PROMPT_ROWS + 32 * wave + r] = wrong ? NAN : sum;
            }
        }
    }
    if (threadIdx.x == 0)
        records(a.workspace)[WAVES + worker] = record;
}

// Joins the tiles that several workers share, the one that begins in worker y and
// ends behind it by as many workgroups as x has, each four pieces of 64 lanes'
// values; and, in two workgroups each before those, the tiles that several waves of
// the other kernel share (one launch less: 3 to 5 us).
constexpr int prompt_merge_parts(int d) { return PROMPT_ROWS * d / 1024; }
template <int D>
__global__ void __launch_bounds__(256)
paged_prompt_merge_kernel(const PagedAttentionArgs a)
{
    if (blockIdx.x < WAVES * 2) {
        const int wave = int(blockIdx.x) % WAVES, half = int(blockIdx.x) / WAVES;
        const Record todo = records(a.workspace)[wave];
        if (todo.parts)
            for (int k = 0; k < TILE_ROWS * D / 512; k++) {
                join_tile<D>(a, todo, wave, half * (TILE_ROWS * D / 512) + k);
                __syncthreads();
            }
        return;
    }
    const int block = int(blockIdx.x) - WAVES * 2, worker = block / prompt_merge_parts(D), part = block % prompt_merge_parts(D);
    const Record todo = records(a.workspace)[WAVES + worker];
    if (todo.parts == 0)
        return;
    constexpr int PIECES = D / 8;                         // of 32 rows
    const int group = a.heads / a.cache.kv_heads;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float* const slot = a.workspace + prompt_workspace(D) + 2 * int64_t(worker) * prompt_slot_floats(D);
    auto take = [&](Joined& sum, int piece, int r, int p) {
        // (a tile's own worker has it in its second slot, the others in their first)
        const float* const at = slot + (2 * p + (p == 0)) * int64_t(prompt_slot_floats(D));
        sum.take(at[PROMPT_ROWS * D + r], at[PROMPT_ROWS * D + PROMPT_ROWS + r], reinterpret_cast<const f32x4*>(at)[piece * 64 + lane]);
    };
    auto finish = [&](const Joined& sum, int piece, int r) {
        const int packed = todo.row0 + r, i = packed / group;
        if (i >= todo.count)
            return;
        const int col = 8 * (piece % PIECES) + 4 * (lane >> 5);
        const float inv = sum.sum == 0.0f ? 0.0f : 1.0f / sum.sum;
        store_out(a, a.out_format, ((int64_t(todo.first) + i) * a.heads + todo.kvh * group + packed % group) * D + col, sum.acc[0] * inv,
                  sum.acc[1] * inv, sum.acc[2] * inv, sum.acc[3] * inv);
    };
    // Few slots: a piece a wave.  Many: its waves take them in turn.
    const bool turns = todo.parts > 4;
#pragma unroll 1
    for (int k = 0; k < (turns ? 4 : 1); k++) {
        const int piece = 4 * part + (turns ? k : wave), r = 32 * (piece / PIECES) + (lane & 31);
        // (rows that are not in the sequence were not stored)
        if (todo.row0 + 32 * (piece / PIECES) >= todo.count * group)
            return;
        Joined sum;
#pragma unroll 4
        for (int p = turns ? wave : 0; p < todo.parts; p += turns ? 4 : 1)
            take(sum, piece, r, p);
        if (!turns || join_waves(sum))
            finish(sum, piece, r);
        if (turns)
            __syncthreads();
    }
}

template <int D, bool Q4, bool FINE>
hipError_t launch(const PagedAttentionArgs& a, hipStream_t s)
{
    const int group = a.heads / a.cache.kv_heads;
    const int64_t most = int64_t(a.batch.max_rows) * group;       // packed rows of a sequence
    const unsigned tile_rows = unsigned(min(int64_t(TILE_ROWS), most));
    paged_attention_kernel<D, Q4, FINE><<<WAVES / 4, 256, 0, s>>>(a);
    if (most > a.few_rows) {
        paged_prompt_kernel<D, Q4, FINE><<<PROMPT_WORKERS, PROMPT_THREADS, 0, s>>>(a);
        paged_prompt_merge_kernel<D><<<2 * WAVES + PROMPT_WORKERS * prompt_merge_parts(D), 256, 0, s>>>(a);
    } else {
        paged_merge_kernel<D><<<dim3(WAVES, (tile_rows + 256 / D - 1) / (256 / D)), 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <int D>
hipError_t launch(const PagedAttentionArgs& a, hipStream_t s)
{
    const bool fine = a.out_format != PAGED_OUT_BF16;
    if (a.cache.q4)
        return fine ? launch<D, true, true>(a, s) : launch<D, true, false>(a, s);
    return fine ? launch<D, false, true>(a, s) : launch<D, false, false>(a, s);
}

}  // namespace

int64_t paged_attention_workspace_floats(int, int, int head)
{
    return prompt_workspace(head) + int64_t(2 * PROMPT_WORKERS) * prompt_slot_floats(head);
}

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t s)
{
    // Sequences of how many packed rows go to the prompt kernel.  It turns a unit
    // into FP16 once for 256 rows and the other does for 16, but a launch of both
    // costs 10 us more, and few tiles do not fill its workgroups.  Rows a sequence,
    // us with 128 and 64 here (4-bit pages, heads of 128): 4 sequences of 126 rows and
    // up to 300 positions 19 and 28, one of 126 and 9000 37 and 46, 8 of 72 to 126 and
    // 2000 to 6000 64 and 68, 40 of 66 to 96 and 300 to 2000 71 and 84; but 16 of 126
    // and 3000 to 9000 175 and 131.  Lengths, which the host does not know, would move
    // the border: 16 of 96 and 3000 to 9000 135 and 124 (of 72: 116 and 124), 4 of 96
    // and 2000 47 and 40, 3 of 126 and 30000 159 and 117.
    const int64_t group = a.heads / a.cache.kv_heads, most = a.batch.max_rows * group, all = a.batch.rows * group;
    PagedAttentionArgs b = a;
    b.few_rows = most <= 96 || (most <= 128 && all <= 1024) ? 128 : 64;
    return a.cache.head == 128 ? launch<128>(b, s) : launch<64>(b, s);
}

}  // namespace si
