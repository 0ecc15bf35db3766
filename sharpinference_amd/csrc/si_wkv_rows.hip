// The RWKV-7 time-mix core over packed sequences, row after row
// (PortableRwkv7GraphProvider.cs:224-276).  Per head, with S [64 values][64 keys]:
//   S = S diag(w) - (S kn)(kn * a)^T + value key^T,  y = S r,
//   out = (GroupNorm(y) * lnx_w + lnx_b + value * sum(key r r_k)) * gate
#include "si_sequences.hpp"
#include "si_lanes.hpp"

namespace si {
namespace {

constexpr int N = WKV_HEAD;
constexpr float LOG2E = 1.44269504088896f;
constexpr float GROUP_EPS = 64e-5f;

// 1 / (1 + exp(-v)) with the hardware's exponential and reciprocal (1 ulp
// each, and |v| * 2^-24 of the exponent)
__device__ __forceinline__ float sigmoid_fast(float v)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * v));
}

__device__ __forceinline__ float wave_sum(float v) { return rows_sum(row_sum<16>(v)); }

// What one element of a row brings, as loaded.
struct RowIn {
    float r, k, v, wl, al, gate, vl, vf;
};

struct Plan;
__device__ void make_plan(const WkvRowsArgs& a, int over, int from, int room, Plan* plan);   // by 256 threads

// Sequences of few rows: a workgroup takes one head of one sequence, the state
// in registers (a thread holds 8 columns of one or two state rows: 8 lanes a state
// row, whose sums take three DPP steps, and half the LDS reads of 16 columns
// of one row).  As many rows at a time as there are waves: wave w prepares row w (one element a
// lane), all waves take the rows through the state, wave w normalises row w.
// Bound by reading and writing the state (32 KiB a head) where a sequence
// brings one row (64 of them, 32 heads, 13.1 us, 5.5 TB/s); by vector instructions (92 a row and wave of four) and LDS reads
// (10 b128 a lane and row) where it brings many (64 of 8 rows 25 us).
template <int WAVES>
struct FewLds {
    float4 vec[WAVES][5][N / 4];   // decay, key, kn, kn * a, r of the rows
    float value[WAVES][N], y[WAVES][N];
};

template <int WAVES>
__device__ __forceinline__ void few_rows(const WkvRowsArgs& a, FewLds<WAVES>& lds, int s, int h, RowSpan span)
{
    constexpr int OWN = 8 / WAVES, APART = 8 * WAVES;   // state rows of a thread, and how far apart they lie
    const int from = a.batch.from[s], to = a.batch.to[s];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int64_t width = static_cast<int64_t>(a.heads) * N;
    const int e = h * N + lane;

    const int c = t & 7, i0 = t >> 3;
    float4 sv[OWN][2];
    if (from >= 0 && from < a.batch.slots) {
        const float* S = a.state + (static_cast<int64_t>(from) * a.heads + h) * N * N;
#pragma unroll
        for (int p = 0; p < OWN; p++)
#pragma unroll
            for (int q = 0; q < 2; q++)
                sv[p][q] = *reinterpret_cast<const float4*>(S + (i0 + APART * p) * N + 32 * q + 4 * c);
    } else {
        const float z = from == -1 ? 0.0f : __builtin_nanf("");
#pragma unroll
        for (int p = 0; p < OWN; p++)
            sv[p][0] = sv[p][1] = make_float4(z, z, z, z);
    }
    const bool first = a.first_layer != 0;
    const float w0 = a.w0[e], a0 = a.a0[e], kkk = a.k_k[e], kka = a.k_a[e], rk = a.r_k[e], lw = a.lnx_weight[e],
                lb = a.lnx_bias[e], v0 = first ? 0.0f : a.v0[e];
    auto load = [&](int row) {
        RowIn x{};
        if (row < span.last) {
            const int64_t at = row * width + e;
            x.r = a.r[at];
            x.k = a.k[at];
            x.v = a.v[at];
            x.wl = a.w_lora[at];
            x.al = a.a_lora[at];
            x.gate = a.gate[at];
            x.vl = first ? 0.0f : a.v_lora[at];
            x.vf = first ? 0.0f : a.v_first[at];
        }
        return x;
    };
    RowIn next = load(span.first + wave);
    for (int base = span.first; base < span.last; base += WAVES) {
        const RowIn x = next;
        const int row = base + wave;
        float value = 0.0f, bonus = 0.0f;
        if (row < span.last) {
            const float decay = __builtin_amdgcn_exp2f(-0.606531f * LOG2E * sigmoid_fast(x.wl + w0));
            const float ad = sigmoid_fast(x.al + a0);
            const float sk = x.k * kkk;
            const float squares = wave_sum(sk * sk);
            const float kn = sk * (1.0f / sqrtf(squares > 1e-24f ? squares : 1e-24f));
            const float ka = x.k * kka;
            const float key = (x.k + ad * ka) - ka;
            value = first ? x.v : fmaf(x.vf - x.v, sigmoid_fast(x.vl + v0), x.v);
            if (first)
                a.v_first[row * width + e] = x.v;
            bonus = wave_sum(key * x.r * rk);
            float* vec = reinterpret_cast<float*>(lds.vec[wave]);
            vec[lane] = decay;
            vec[N + lane] = key;
            vec[2 * N + lane] = kn;
            vec[3 * N + lane] = kn * ad;
            vec[4 * N + lane] = x.r;
            lds.value[wave][lane] = value;
        }
        next = load(row + WAVES);
        __syncthreads();
        const int live = min(WAVES, span.last - base);
        for (int j = 0; j < live; j++) {
            float kept[OWN], y[OWN], value_of[OWN];   // -S kn, S r, the row's value
            auto dot = [](float4 x, float4 y, float acc) {
                return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, acc))));
            };
#pragma unroll
            for (int p = 0; p < OWN; p++) {
                kept[p] = y[p] = 0.0f;
                value_of[p] = lds.value[j][i0 + APART * p];
            }
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const float4 kn = lds.vec[j][2][8 * q + c];
#pragma unroll
                for (int p = 0; p < OWN; p++)
                    kept[p] = dot(sv[p][q], kn, kept[p]);
            }
#pragma unroll
            for (int p = 0; p < OWN; p++)
                kept[p] = -row_sum<8>(kept[p]);
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const float4 d = lds.vec[j][0][8 * q + c], k = lds.vec[j][1][8 * q + c], ak = lds.vec[j][3][8 * q + c],
                             r = lds.vec[j][4][8 * q + c];
                auto step = [&](float4& S, float p, float v) {
                    S.x = fmaf(p, ak.x, fmaf(v, k.x, S.x * d.x));
                    S.y = fmaf(p, ak.y, fmaf(v, k.y, S.y * d.y));
                    S.z = fmaf(p, ak.z, fmaf(v, k.z, S.z * d.z));
                    S.w = fmaf(p, ak.w, fmaf(v, k.w, S.w * d.w));
                };
#pragma unroll
                for (int p = 0; p < OWN; p++) {
                    step(sv[p][q], kept[p], value_of[p]);
                    y[p] = dot(sv[p][q], r, y[p]);
                }
            }
#pragma unroll
            for (int p = 0; p < OWN; p++) {
                y[p] = row_sum<8>(y[p]);
                if (c == 0)
                    lds.y[j][i0 + APART * p] = y[p];
            }
        }
        __syncthreads();
        if (row < span.last) {
            const float y = lds.y[wave][lane];
            const float d = y - wave_sum(y) * (1.0f / N);
            const float var = wave_sum(d * d) * (1.0f / N);
            const float ln = d * (1.0f / sqrtf(var + GROUP_EPS)) * lw + lb;
            store_row_value(a.out, a.out_format, row * width + e, (ln + value * bonus) * x.gate);
        }
    }
    if (to >= 0 && to < a.batch.slots) {
        float* S = a.state + (static_cast<int64_t>(to) * a.heads + h) * N * N;
#pragma unroll
        for (int p = 0; p < OWN; p++)
#pragma unroll
            for (int q = 0; q < 2; q++)
                *reinterpret_cast<float4*>(S + (i0 + APART * p) * N + 32 * q + 4 * c) = sv[p][q];
    }
}

// With a plan to make, the last workgroup makes it.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void wkv_few_kernel(WkvRowsArgs a, int most, int cut, int room, Plan* plan)
{
    __shared__ FewLds<WAVES> lds;
    const int s = blockIdx.x / a.heads, h = blockIdx.x - s * a.heads;
    if (WAVES == 4 && s == a.batch.sequences)
        return make_plan(a, most, cut, room, plan);
    const RowSpan span = rows_of(a.batch, s);
    if (span.last - span.first >= 1 && span.last - span.first <= most)
        few_rows<WAVES>(a, lds, s, h, span);
}

// ---- blocks of 16 rows on the matrix cores ----------------------------------------------------
//
// Within a block of C = 16 rows let L_t be the decays' product up to row t, and
//   alpha_t = L_(t-1) * kn_t,  beta_t = kn_t a_t / L_t,  khat_t = key_t / L_t,  rho_t = L_t * r_t.
// Then with u_t = -(S_(t-1) kn_t) the block's state is S_0 + sum_s (u_s beta_s^T + v_s khat_s^T), times L_C, and
//   (I + A) U = -(alpha S_0^T + B V),   A_ts = alpha_t . beta_s, B_ts = alpha_t . khat_s  (s < t)
//   Y = rho S_0^T + D U + E V,          D_ts = rho_t . beta_s,   E_ts = rho_t . khat_s    (s <= t).
// What does not need S_0 is formed beforehand, alpha' = (I + A)^-1 alpha and V' = (I + A)^-1 B V, so that a
// block costs the state U = -(alpha' S_0^T + V'), Y as above, S = (S_0 + U^T beta + V^T khat) diag(L_C).
// (I + A) is solved row by row: rows of like keys make A all ones, where a product of powers of A
// loses every digit.  The decays are at least exp(-0.606531), so 1 / L grows to 2^14 at most and the
// factors stay far from FP32's ends; all products are FP32 (v_mfma_f32_16x16x4_f32).
//
// kn_t = sk_t / |sk_t| needs a sum over the head: alpha and beta are formed from sk, and n_t = 1 / |sk_t|
// enters where the rows are solved: z_t = n_t (r_t - sum_s A_ts n_s z_s) for the columns r of alpha and
// of B, and alpha', W = n z (the second n is beta's).
//
// Operands: a matrix instruction takes A[row l % 16][k], B[k][column l % 16] with k = l / 16 and gives
// rows 4 (l / 16) + v.  Taking k = 4 (l / 16) + v in instruction v of four, a result is the next
// product's B (or, transposed, A) operand as it stands: the state is kept as S^T tiles
// [16 keys][16 values], four of them a wave, and never moves.

constexpr int C = 16;                    // rows of a block
constexpr int LD = 68;                   // floats of an LDS row of 64: four rows lie 16 banks apart
constexpr int CHUNK_THREADS = 512;       // waves 0..3: the state, 16 values each; waves 4..7: the next block

typedef float f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f4 mfma4(f4 a, f4 b, f4 c)
{
#pragma unroll
    for (int v = 0; v < 4; v++)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[v], b[v], c, 0, 0, 0);
    return c;
}

// The value that lane I of the row of 16 holds.
template <int I>
__device__ __forceinline__ float row_lane(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + I, 0xF, 0xF, true));
}

// Sum of the values in this lane's column of the rows of 16 lanes before its own.
__device__ __forceinline__ float rows_before(float v)
{
    const int g = (threadIdx.x >> 4) & 3;
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float even = __uint_as_float(a[0]), pair = even + __uint_as_float(a[1]);   // rows 0 0 2 2; 0+1 0+1 2+3 2+3
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(pair), __float_as_uint(pair), false, false);
    return (g & 1 ? even : 0.0f) + (g & 2 ? __uint_as_float(b[0]) : 0.0f);
}

// max(top, |x|, |y|), NaN if any is
__device__ __forceinline__ float largest(float top, float x, float y)
{
    asm("v_maximum3_f32 %0, %1, |%2|, |%3|" : "=v"(top) : "v"(top), "v"(x), "v"(y));
    return top;
}

// The solution z_i = n_i (z_i + sum over s < i of l_i[s] z_s) of 16 rows, column by column: l_i[s] lies in lane s
// of each row of 16 lanes, n_i in lane i.  One instruction a term reads its lane and multiplies (the compiler forms
// two); as soon as a z_s is known it goes into all later rows, so that the terms are independent.  A first
// half of 8 rows, its terms in the second half, the second half.  The wait in front keeps the distance that a
// lane-crossing read needs from what wrote the register; nothing inside writes l or n.
#define SI_TERM(i, l, s, x) "v_fmac_f32_dpp %" #i ", %" #l ", %" #x " row_newbcast:" #s " row_mask:0xf bank_mask:0xf\n\t"
#define SI_LENGTH(i, s) "v_mul_f32_dpp %" #i ", %15, %" #i " row_newbcast:" #s " row_mask:0xf bank_mask:0xf\n\t"
// operands: z_0 .. z_7 = %0 .. %7, l_1 .. l_7 = %8 .. %14, n = %15; B: the half's first lane
#define SI_HALF(B0, B1, B2, B3, B4, B5, B6, B7)                                                                            \
    "s_nop 1\n\t" SI_LENGTH(0, B0)                                                                                         \
    SI_TERM(1, 8, B0, 0) SI_TERM(2, 9, B0, 0) SI_TERM(3, 10, B0, 0) SI_LENGTH(1, B1)                                        \
    SI_TERM(4, 11, B0, 0) SI_TERM(5, 12, B0, 0) SI_TERM(6, 13, B0, 0) SI_TERM(7, 14, B0, 0)                                 \
    SI_TERM(2, 9, B1, 1) SI_TERM(3, 10, B1, 1) SI_TERM(4, 11, B1, 1) SI_LENGTH(2, B2)                                       \
    SI_TERM(5, 12, B1, 1) SI_TERM(6, 13, B1, 1) SI_TERM(7, 14, B1, 1)                                                       \
    SI_TERM(3, 10, B2, 2) SI_TERM(4, 11, B2, 2) SI_TERM(5, 12, B2, 2) SI_LENGTH(3, B3)                                      \
    SI_TERM(6, 13, B2, 2) SI_TERM(7, 14, B2, 2)                                                                             \
    SI_TERM(4, 11, B3, 3) SI_TERM(5, 12, B3, 3) SI_TERM(6, 13, B3, 3) SI_LENGTH(4, B4) SI_TERM(7, 14, B3, 3)                \
    SI_TERM(5, 12, B4, 4) SI_TERM(6, 13, B4, 4) SI_TERM(7, 14, B4, 4) SI_LENGTH(5, B5)                                      \
    SI_TERM(6, 13, B5, 5) SI_TERM(7, 14, B5, 5) SI_LENGTH(6, B6)                                                            \
    SI_TERM(7, 14, B6, 6) SI_LENGTH(7, B7)
// operands: z_8 .. z_15 = %0 .. %7, l_8 .. l_15 = %8 .. %15, z_0 .. z_7 = %16 .. %23
#define SI_ACROSS(s, x)                                                                                                     \
    SI_TERM(0, 8, s, x) SI_TERM(1, 9, s, x) SI_TERM(2, 10, s, x) SI_TERM(3, 11, s, x) SI_TERM(4, 12, s, x)                  \
    SI_TERM(5, 13, s, x) SI_TERM(6, 14, s, x) SI_TERM(7, 15, s, x)
__device__ __forceinline__ void solve_rows(float (&z)[C], const float (&l)[C], float n)
{
    asm(SI_HALF(0, 1, 2, 3, 4, 5, 6, 7)
        : "+&v"(z[0]), "+&v"(z[1]), "+&v"(z[2]), "+&v"(z[3]), "+&v"(z[4]), "+&v"(z[5]), "+&v"(z[6]), "+&v"(z[7])
        : "v"(l[1]), "v"(l[2]), "v"(l[3]), "v"(l[4]), "v"(l[5]), "v"(l[6]), "v"(l[7]), "v"(n));
    asm("s_nop 1\n\t" SI_ACROSS(0, 16) SI_ACROSS(1, 17) SI_ACROSS(2, 18) SI_ACROSS(3, 19) SI_ACROSS(4, 20) SI_ACROSS(5, 21)
            SI_ACROSS(6, 22) SI_ACROSS(7, 23)
        : "+&v"(z[8]), "+&v"(z[9]), "+&v"(z[10]), "+&v"(z[11]), "+&v"(z[12]), "+&v"(z[13]), "+&v"(z[14]), "+&v"(z[15])
        : "v"(l[8]), "v"(l[9]), "v"(l[10]), "v"(l[11]), "v"(l[12]), "v"(l[13]), "v"(l[14]), "v"(l[15]), "v"(z[0]), "v"(z[1]),
          "v"(z[2]), "v"(z[3]), "v"(z[4]), "v"(z[5]), "v"(z[6]), "v"(z[7]));
    asm(SI_HALF(8, 9, 10, 11, 12, 13, 14, 15)
        : "+&v"(z[8]), "+&v"(z[9]), "+&v"(z[10]), "+&v"(z[11]), "+&v"(z[12]), "+&v"(z[13]), "+&v"(z[14]), "+&v"(z[15])
        : "v"(l[9]), "v"(l[10]), "v"(l[11]), "v"(l[12]), "v"(l[13]), "v"(l[14]), "v"(l[15]), "v"(n));
}
#undef SI_TERM
#undef SI_LENGTH
#undef SI_HALF
#undef SI_ACROSS
template <int I>
__device__ __forceinline__ void scale_rows(float* to, const float (&z)[C], float n)
{
    if constexpr (I < C) {
        to[I * LD] = z[I] * row_lane<I>(n);
        scale_rows<I + 1>(to, z, n);
    }
}

// What the preparing waves hand to the state's waves for one block.
struct BlockLds {
    float alpha[C][LD], rho[C][LD], beta[C][LD], khat[C][LD], value[C][LD];
    f4 v_part[4][64];                  // V' tiles as the matrix instructions hold them
    float m[C][LD];                    // A, B, D, E beside one another
    float decay[N];                    // L_C
    float bonus[4][C];                 // parts of sum(key r r_k)
    float squares[4][C];
    int odd;                           // a value is not finite or very large
};

struct ChunkLds {
    BlockLds block[2];
    float w[C][LD];                    // (I + A)^-1 B in the columns that A has in m
    float y[C][LD];
};

__device__ __forceinline__ f4 row4(const float (&m)[C][LD], int row, int col) { return *reinterpret_cast<const f4*>(&m[row][col]); }
__device__ __forceinline__ f4 column4(const float (&m)[C][LD], int row, int col)
{
    return f4{m[row][col], m[row + 1][col], m[row + 2][col], m[row + 3][col]};
}

// The rows of the next block: up to 16, or one by one through a block where a value is not finite or so
// large that a product could overflow (a product of a zero that masks a later row with such a value is NaN).  Both roles
// follow it from the flag of the block before.
struct Blocks {
    int at, end, single;   // next row, last row + 1, rows below this one go one by one
    __device__ int last() const { return at < single ? at + 1 : min(at + C, end); }
    // whether the block [at, last()) counts; moves on
    __device__ bool next(bool odd)
    {
        const int to = last();
        if (odd && to - at > 1) {
            single = to;
            return false;
        }
        at = to;
        return true;
    }
};

__device__ __forceinline__ void put_column4(float (&m)[C][LD], int row, int col, f4 v)
{
#pragma unroll
    for (int i = 0; i < 4; i++)
        m[row + i][col] = v[i];
}

__device__ __forceinline__ f4 load4(const float* p)   // at a multiple of 4 bytes
{
    f4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

__device__ __forceinline__ float load_at(const float* uniform, uint32_t bytes)
{
    return *reinterpret_cast<const float*>(reinterpret_cast<const char*>(uniform) + bytes);
}

// 1 / (1 + exp(-(x + bias))), shift = -LOG2E * bias
__device__ __forceinline__ float sigmoid_shifted(float x, float shift)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(fmaf(x, -LOG2E, shift)));
}

// TRANSFER: only what a stretch's transfer needs (no readout).
template <bool TRANSFER>
__device__ void chunk_prepare(const WkvRowsArgs& a, ChunkLds& lds, int h, Blocks blocks)
{
    const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int q = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const int64_t width = static_cast<int64_t>(a.heads) * N;
    const int ch = 16 * q + t;
    const bool first = a.first_layer != 0;
    const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int e = h * N + ch;
    const float w0 = -LOG2E * a.w0[e], a0 = -LOG2E * a.a0[e], v0 = first ? 0.0f : -LOG2E * a.v0[e], kkk = a.k_k[e], kka = a.k_a[e],
                rk = a.r_k[e];
    struct {
        f4 r, k, v, wl, al, vl, vf;
    } x;
    uint32_t full[4];   // bytes from a block's first value of the head to this lane's
#pragma unroll
    for (int v = 0; v < 4; v++)
        full[v] = 4u * ((4 * g + v) * static_cast<uint32_t>(width) + ch);
    auto load = [&](int first_row, int last) {
        const int64_t from = first_row * width + h * N;
        uint32_t at[4];
#pragma unroll
        for (int v = 0; v < 4; v++)   // (a row behind the block's last reads the last again, and is masked where it counts)
            at[v] = last - first_row == C ? full[v] : 4u * (min(4 * g + v, last - first_row - 1) * static_cast<uint32_t>(width) + ch);
        auto rows = [&](const float* p) {
            p += from;
            return f4{load_at(p, at[0]), load_at(p, at[1]), load_at(p, at[2]), load_at(p, at[3])};
        };
        if (!TRANSFER)
            x.r = rows(a.r);
        x.k = rows(a.k);
        x.v = rows(a.v);
        x.wl = rows(a.w_lora);
        x.al = rows(a.a_lora);
        if (!first) {
            x.vl = rows(a.v_lora);
            x.vf = rows(a.v_first);
        }
    };
    x.r = x.vl = x.vf = zero;
    load(blocks.at, blocks.last());
    for (int stage = 0; blocks.at < blocks.end; stage++) {
        BlockLds& b = lds.block[stage & 1];
        const int at = blocks.at, rows = blocks.last() - at;
        // 1: the rows' factors
        constexpr float FASTEST = -0.606531f * LOG2E;   // a row's decay at most, as an exponent
        f4 fastest = {FASTEST, FASTEST, FASTEST, FASTEST};
        if (rows < C) {   // a decay of 1 (whatever w0 is: by the factor, since no w_lora gives it where w0 is infinite), the rest 0
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const bool in = 4 * g + v < rows;
                x.wl[v] = in ? x.wl[v] : 0.0f;
                fastest[v] = in ? FASTEST : 0.0f;
                x.al[v] = in ? x.al[v] : 0.0f;
                x.vl[v] = in ? x.vl[v] : 0.0f;
                x.vf[v] = in ? x.vf[v] : 0.0f;
                x.k[v] = in ? x.k[v] : 0.0f;
                x.v[v] = in ? x.v[v] : 0.0f;
                x.r[v] = in ? x.r[v] : 0.0f;
            }
        }
        f4 al, rh, be, kh, va, cum, squares, bonus;
#pragma unroll
        for (int v = 0; v < 4; v++)
            cum[v] = fastest[v] * sigmoid_shifted(x.wl[v], w0);
        cum[1] += cum[0];
        cum[2] += cum[1];
        cum[3] += cum[2];
        const float earlier = rows_before(cum[3]);
        float decay = __builtin_amdgcn_exp2f(earlier), top = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const float c = earlier + cum[v];
            const float ad = sigmoid_shifted(x.al[v], a0);
            const float sk = x.k[v] * kkk;
            const float key = fmaf(x.k[v] * kka, ad - 1.0f, x.k[v]);
            va[v] = first ? x.v[v] : fmaf(x.vf[v] - x.v[v], sigmoid_shifted(x.vl[v], v0), x.v[v]);
            al[v] = sk * decay;
            decay = __builtin_amdgcn_exp2f(c);
            const float shrink = __builtin_amdgcn_exp2f(-c);
            be[v] = (sk * ad) * shrink;
            kh[v] = key * shrink;
            rh[v] = x.r[v] * decay;
            squares[v] = sk * sk;
            bonus[v] = key * x.r[v] * rk;
            // sk in alpha's and beta's place: alpha is at most that, beta 2^14 times that (one over the block's decays), so that
            // under 2^50 a product of two rows is at most 64 * 2^(50 + 64).  (beta / alpha is up to 2^27, and khat may be 0.)
            top = largest(largest(top, sk, kh[v]), rh[v], va[v]);
        }
        put_column4(b.alpha, 4 * g, ch, al);
        if (!TRANSFER)
            put_column4(b.rho, 4 * g, ch, rh);
        put_column4(b.beta, 4 * g, ch, be);
        put_column4(b.khat, 4 * g, ch, kh);
        put_column4(b.value, 4 * g, ch, va);
#pragma unroll
        for (int v = 0; v < 4; v++) {
            squares[v] = row_sum<16>(squares[v]);
            if (!TRANSFER)
                bonus[v] = row_sum<16>(bonus[v]);
        }
        if (t == 0) {
            *reinterpret_cast<f4*>(&b.squares[q][4 * g]) = squares;
            if (!TRANSFER)
                *reinterpret_cast<f4*>(&b.bonus[q][4 * g]) = bonus;
        }
        if (g == 3)
            b.decay[ch] = decay;
        if (first && !TRANSFER) {
#pragma unroll
            for (int v = 0; v < 4; v++)
                if (4 * g + v < rows)
                    a.v_first[(at + 4 * g + v) * width + e] = x.v[v];
        }
        if (!(top < 0x1p50f))
            b.odd = 1;
        __syncthreads();
        // 2: the four products of rows with rows, one a wave
        const bool counts = blocks.next(b.odd != 0);
        if (blocks.at < blocks.end)
            load(blocks.at, blocks.last());
        float length = b.squares[0][t] + b.squares[1][t] + b.squares[2][t] + b.squares[3][t];
        length = __builtin_amdgcn_rsqf(length > 1e-24f ? length : 1e-24f);   // 1 / |sk| of row t
        if (!TRANSFER || q < 2) {
            const auto& left = q < 2 ? b.alpha : b.rho;
            const auto& right = q & 1 ? b.khat : b.beta;
            f4 l[4], r[4], m0 = zero, m1 = zero;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                l[j] = row4(left, t, 16 * j + 4 * g);
                r[j] = row4(right, t, 16 * j + 4 * g);
            }
            __builtin_amdgcn_sched_barrier(0);   // all reads before the first product
            m0 = mfma4(l[0], r[0], m0);
            m1 = mfma4(l[1], r[1], m1);
            m0 = mfma4(l[2], r[2], m0);
            m1 = mfma4(l[3], r[3], m1);
            // row i, column t; A with its columns' lengths and its sign turned
            const float f = q == 0 ? -length : 1.0f;
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int i = 4 * g + v;
                const int keep = -static_cast<int>(i < rows && t < (q < 2 ? i : i + 1));   // (as bits: a choice branches)
                b.m[i][ch] = __int_as_float(__float_as_int((m0[v] + m1[v]) * f) & keep);
            }
        }
        __syncthreads();
        // 3: the block's solution and what follows from it (16 channels or values a wave)
        if (counts) {
            // column t of alpha (lanes 0..15 of a half) or of B (16..31), solved row by row:
            // z_i = n_i (r_i + sum_s -A_is n_s z_s), every lane with row i's sums from the row of 16 lanes that holds it
            const bool of_b = (lane & 16) != 0;
            const float* const column = of_b ? &b.m[0][16 + t] : &b.alpha[0][16 * q + t];
            float z[C], l[C];
#pragma unroll
            for (int i = 0; i < C; i++) {
                l[i] = b.m[i][t];
                z[i] = column[i * LD];
            }
            solve_rows(z, l, length);
            float* const solved = of_b ? &lds.w[0][t] : &b.alpha[0][16 * q + t];   // (w: the same from all four waves)
            if (lane < 32)
                scale_rows<0>(solved, z, length);
            wave_sync();
            const f4 v_tile = column4(b.value, 4 * g, 16 * q + t);
            b.v_part[q][lane] = mfma4(row4(lds.w, t, 4 * g), v_tile, zero);
        }
        if (threadIdx.x == CHUNK_THREADS - 1)
            lds.block[(stage & 1) ^ 1].odd = 0;
        __syncthreads();
    }
    // the state's waves take the last block
    __syncthreads();
    __syncthreads();
    __syncthreads();
}

// Where a workgroup's state comes from and goes to.
struct StateEnds {
    const f4* start;   // S^T tiles as the matrix instructions hold them, or null: from `from`
    const float* from; // [64][64], or null: all `fill`
    float fill;
    float* to;         // [64][64], or null
    f4* end;           // tiles as in start, or null
};

__device__ __forceinline__ void load_state(const StateEnds& ends, int w, f4 (&S)[4])
{
    const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < 4; j++)
        S[j] = ends.start ? ends.start[(4 * w + j) * 64 + lane]
               : ends.from ? *reinterpret_cast<const f4*>(ends.from + (16 * w + t) * N + 16 * j + 4 * g)
                           : f4{ends.fill, ends.fill, ends.fill, ends.fill};
}

__device__ void chunk_advance(const WkvRowsArgs& a, ChunkLds& lds, int h, const StateEnds& ends, Blocks blocks)
{
    const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t width = static_cast<int64_t>(a.heads) * N;
    const int tn = 4 * w + g, cn = 4 * t;   // row and four channels in the normalisation
    const f4 lw = load4(a.lnx_weight + h * N + cn), lb = load4(a.lnx_bias + h * N + cn);
    f4 S[4];   // S^T tiles: keys 16 j + 4 g + v, value 16 w + t
    load_state(ends, w, S);
    // while the first block is prepared
    int at = blocks.at, rows = blocks.last() - at;
    __syncthreads();
    bool counts = blocks.next(lds.block[0].odd != 0);
    __syncthreads();
    __syncthreads();
    for (int stage = 1;; stage++) {
        const BlockLds& b = lds.block[(stage & 1) ^ 1];
        const bool have = counts, more = blocks.at < blocks.end;
        const int next_at = blocks.at, next_rows = more ? blocks.last() - next_at : 0;
        f4 gate, xa, xr, v_tile;
        auto part = [&](int j) {
            xa = mfma4(row4(b.alpha, t, 16 * j + 4 * g), S[j], xa);
            xr = mfma4(row4(b.rho, t, 16 * j + 4 * g), S[j], xr);
        };
        if (have) {
            gate = load4(a.gate + (at + min(tn, rows - 1)) * width + h * N + cn);
            xa = b.v_part[w][lane];
            xr = mfma4(row4(b.m, t, 48 + 4 * g), v_tile = column4(b.value, 4 * g, 16 * w + t), f4{0.0f, 0.0f, 0.0f, 0.0f});
            part(0);
            part(1);
        }
        __syncthreads();
        counts = more && blocks.next(lds.block[stage & 1].odd != 0);
        if (have) {
            part(2);
            part(3);
            xa = -xa;   // U
            xr = mfma4(row4(b.m, t, 32 + 4 * g), xa, xr);
#pragma unroll
            for (int v = 0; v < 4; v++)
                lds.y[4 * g + v][16 * w + t] = xr[v];
        }
        __syncthreads();
        if (have) {
            const f4 y = row4(lds.y, tn, cn), value = row4(b.value, tn, cn);
            const float bonus = b.bonus[0][tn] + b.bonus[1][tn] + b.bonus[2][tn] + b.bonus[3][tn];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                S[j] = mfma4(column4(b.beta, 4 * g, 16 * j + t), xa, S[j]);
                S[j] = mfma4(column4(b.khat, 4 * g, 16 * j + t), v_tile, S[j]);
            }
            const float mean = row_sum<16>(y[0] + y[1] + y[2] + y[3]) * (1.0f / N);
            const f4 d = y - mean;
            const float var = row_sum<16>(fmaf(d[3], d[3], fmaf(d[2], d[2], fmaf(d[1], d[1], d[0] * d[0])))) * (1.0f / N);
            const float inv = __builtin_amdgcn_rsqf(var + GROUP_EPS);
            if (tn < rows) {
                f4 o;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[j] = fmaf(value[j], bonus, fmaf(d[j] * inv, lw[j], lb[j])) * gate[j];
                store_row4(a.out, a.out_format, (at + tn) * width + h * N + cn, o);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                S[j] *= *reinterpret_cast<const f4*>(&b.decay[16 * j + 4 * g]);
        }
        at = next_at;
        rows = next_rows;
        __syncthreads();
        if (!more)
            break;
    }
    if (ends.to) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            *reinterpret_cast<f4*>(ends.to + (16 * w + t) * N + 16 * j + 4 * g) = S[j];
    }
    if (ends.end) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            ends.end[(4 * w + j) * 64 + lane] = S[j];
    }
}

// A stretch's transfer: the state behind it is S M + (S's start at zero), and M's rows are 64 more states that start as
// the unit matrix and take no values.
__device__ void chunk_transfer(ChunkLds& lds, float* record, Blocks blocks)
{
    const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f4 S[4], M[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            S[j][v] = 0.0f;
            M[j][v] = 16 * j + 4 * g + v == 16 * w + t ? 1.0f : 0.0f;
        }
    __syncthreads();
    bool counts = blocks.next(lds.block[0].odd != 0);
    __syncthreads();
    __syncthreads();
    for (int stage = 1;; stage++) {
        const BlockLds& b = lds.block[(stage & 1) ^ 1];
        const bool have = counts, more = blocks.at < blocks.end;
        f4 xs, xm;
        auto part = [&](int j) {
            const f4 al = row4(b.alpha, t, 16 * j + 4 * g);
            xs = mfma4(al, S[j], xs);
            xm = mfma4(al, M[j], xm);
        };
        if (have) {
            xs = b.v_part[w][lane];
            xm = f4{0.0f, 0.0f, 0.0f, 0.0f};
            part(0);
            part(1);
        }
        __syncthreads();
        counts = more && blocks.next(lds.block[stage & 1].odd != 0);
        if (have) {
            part(2);
            part(3);
        }
        __syncthreads();
        if (have) {
            const f4 us = -xs, um = -xm, v_tile = column4(b.value, 4 * g, 16 * w + t);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f4 beta = column4(b.beta, 4 * g, 16 * j + t), decay = *reinterpret_cast<const f4*>(&b.decay[16 * j + 4 * g]);
                M[j] = mfma4(beta, um, M[j]) * decay;
                S[j] = mfma4(beta, us, S[j]);
                S[j] = mfma4(column4(b.khat, 4 * g, 16 * j + t), v_tile, S[j]) * decay;
            }
        }
        __syncthreads();
        if (!more)
            break;
    }
    f4* const start = reinterpret_cast<f4*>(record + N * N);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        start[(4 * w + j) * 64 + lane] = S[j];
#pragma unroll
        for (int v = 0; v < 4; v++)   // M^T, row after row
            record[(16 * j + 4 * g + v) * N + 16 * w + t] = M[j][v];
    }
}

// ---- long sequences in stretches ---------------------------------------------------------------
//
// Where the heads of all sequences are too few for the card, long sequences are cut: (1) each first stretch as a
// sequence of its own, beside the transfers (M, N) of the others but the last; (2) the states between them,
// S_(i+1) = S_i M_i + N_i; (3) every other stretch, from its state on, beside the sequences that are whole.  A transfer costs
// 0.95 of its stretch.

constexpr int RECORD = 2 * N * N;        // floats of a stretch and head: M^T; N (the first's: its state), then the next stretch's start
constexpr int CARD = 512;                // workgroups of wkv_chunk_kernel that the card holds: two a compute unit
constexpr int HEAD_STRETCHES = 2 * CARD; // stretches (but each sequence's last) times heads, at most
constexpr int LONG_STRETCH = 256;
constexpr int LEAST_STRETCH = 48, LEAST_CUT = 176;   // rows of a stretch, and of a sequence that is cut, at least (one of 250 rows, 32 heads,
                                                     // 41 us, in stretches of 64 53, whole 59; of 150, cut 40, whole 38)

struct Stretch {
    int sequence, first, last;   // rows
    int record;                  // of the sequence's first stretch, or -1: the sequence is whole
    int index, count;            // of the sequence's stretches
};
struct Plan {
    int stretches, cut;          // in list, and sequences that are cut
    int pad[2];
    Stretch list[1];             // every stretch of the sequences that go by blocks; cut sequences' first ones again behind `room`
};

__device__ __forceinline__ StateEnds state_ends(const WkvRowsArgs& a, int s, int h)
{
    const int from = a.batch.from[s], to = a.batch.to[s];
    auto at = [&](int slot) { return a.state + (static_cast<int64_t>(slot) * a.heads + h) * N * N; };
    return {nullptr, from >= 0 && from < a.batch.slots ? at(from) : nullptr, from == -1 ? 0.0f : __builtin_nanf(""),
            to >= 0 && to < a.batch.slots ? at(to) : nullptr, nullptr};
}

// Rows of a stretch where so many rows of so many sequences are cut: the card's workgroups share them with their heads; where that
// gives each more than LONG_STRETCH, twice as many workgroups do, which even out better beside whole sequences (32 heads; eight
// prompts of 500 to 3000 rows 518 us, by CARD 590, three of 1000 to 6000 rows 530 and 702; one of 4001 rows, by CARD, 195, by
// twice as many 225).
__host__ __device__ inline int stretch_rows(int64_t rows, int heads, int cut)
{
    const int64_t work = rows * heads, more = static_cast<int64_t>(cut) * heads;   // (of each sequence one stretch is idle in every pass)
    const int64_t each = (work + CARD + more - 1) / (CARD + more), half = (work + HEAD_STRETCHES + more - 1) / (HEAD_STRETCHES + more);
    const int64_t least = each < LONG_STRETCH ? each : half > LONG_STRETCH ? half : LONG_STRETCH;
    return static_cast<int>((least > LEAST_STRETCH ? least + C - 1 : LEAST_STRETCH) / C * C);
}

// How a sequence of so many rows lies in its stretches: rows of each but the last, and their number (none of them empty).
struct Parts {
    int each, count;
};
__device__ __forceinline__ Parts parts_of(int rows, bool cut, int stretch)
{
    const int most = cut ? rows / stretch : 1;
    const int each = ((rows + most - 1) / most + C - 1) / C * C;
    return {each, cut ? (rows + each - 1) / each : 1};
}
__device__ __forceinline__ Stretch stretch_of(int sequence, RowSpan span, Parts parts, int record, int index)
{
    return {sequence, span.first + index * parts.each,
            index + 1 < parts.count ? span.first + (index + 1) * parts.each : span.last, record, index, parts.count};
}

// Stretch `index` of a batch's only sequence; false where it has none.  (One sequence needs no plan, and its launch: 4 us.)
__device__ __forceinline__ bool sole_stretch(const WkvRowsArgs& a, int from, int index, Stretch* part)
{
    const RowSpan span = rows_of(a.batch, 0);
    const int rows = span.last - span.first;
    const bool cut = rows >= from;
    const Parts parts = parts_of(rows, cut, cut ? stretch_rows(rows, a.heads, 1) : 1);
    *part = stretch_of(0, span, parts, cut ? 0 : -1, index);
    return index < parts.count;
}

// One head of one sequence or stretch, block after block.  While the state's waves take block i
// (72 matrix instructions each), the others prepare block i + 1 (20 each, and the
// exponentials), in three phases between barriers.  Bound by the SIMDs: FP32 matrix instructions take 32 cycles each in the vector
// units' place, so that a block costs a SIMD 92 * 32 = 2944 cycles of them and about 800 vector instructions, 5100 to 5500 cycles
// in all; two workgroups a compute unit fill one another's barriers (three groups of waves in one, or two that prepare, were
// faster alone, 7000 and 7700 cycles a block for 8900, and slower together, 1560 and 1580 us for 1024 heads of equal length, 1370).
// Eight sequences of 1000 rows, 32 heads, one workgroup a compute unit: 220 us.
enum ChunkPass { CHUNK_SEQUENCES, CHUNK_STRETCHES, CHUNK_TRANSFERS };

template <int PASS>
__global__ __launch_bounds__(CHUNK_THREADS, 4) void wkv_chunk_kernel(WkvRowsArgs a, int over, int from, const Plan* plan, float* records)
{
    __shared__ union {
        ChunkLds blocks;
        FewLds<CHUNK_THREADS / 64> few;
    } shared;
    ChunkLds& lds = shared.blocks;
    const int s = blockIdx.x / a.heads, h = blockIdx.x - s * a.heads;
    RowSpan span;
    StateEnds ends;
    float* record = nullptr;
    bool transfer = false;
    if constexpr (PASS == CHUNK_SEQUENCES) {
        span = rows_of(a.batch, s);
        if (span.last - span.first <= over) {
            if (span.last > span.first)
                few_rows<CHUNK_THREADS / 64>(a, shared.few, s, h, span);
            return;
        }
        ends = state_ends(a, s, h);
    } else {
        Stretch part;
        if (plan == nullptr) {
            if (!sole_stretch(a, from, s, &part))
                return;
            if (part.count == 1 && part.last - part.first <= over) {
                if (PASS == CHUNK_TRANSFERS && part.last > part.first)
                    few_rows<CHUNK_THREADS / 64>(a, shared.few, 0, h, {part.first, part.last});
                return;
            }
        } else {
            if (s >= plan->stretches)
                return;
            part = plan->list[s];
        }
        span = {part.first, part.last};
        auto record_of = [&](int i) { return records + (static_cast<int64_t>(part.record + i) * a.heads + h) * RECORD; };
        if constexpr (PASS == CHUNK_TRANSFERS) {
            if (part.record < 0 || part.index == part.count - 1)
                return;
            record = record_of(part.index);
            transfer = part.index > 0;
        } else if (part.record >= 0 && part.index == 0) {
            return;
        }
        ends = state_ends(a, part.sequence, h);
        if (part.record >= 0 && part.index > 0)
            ends.start = reinterpret_cast<const f4*>(record_of(part.index - 1) + N * N);
        if (part.index < part.count - 1)
            ends.to = nullptr;
        if (PASS == CHUNK_TRANSFERS)
            ends.end = reinterpret_cast<f4*>(record + N * N);
    }
    span.first = __builtin_amdgcn_readfirstlane(span.first);
    span.last = __builtin_amdgcn_readfirstlane(span.last);
    if (threadIdx.x < 2)
        lds.block[threadIdx.x].odd = 0;
    __syncthreads();
    const Blocks blocks{span.first, span.last, span.first};
    const bool prepares = threadIdx.x >= CHUNK_THREADS / 2;
    if constexpr (PASS == CHUNK_TRANSFERS) {
        if (transfer) {
            if (prepares)
                chunk_prepare<true>(a, lds, h, blocks);
            else
                chunk_transfer(lds, record, blocks);
            return;
        }
    }
    if (prepares)
        chunk_prepare<false>(a, lds, h, blocks);
    else
        chunk_advance(a, lds, h, ends, blocks);
}

// The states between a cut sequence's stretches.  A workgroup takes 16 values of one head, each of its waves 16 keys:
// a stretch costs it 16 matrix instructions a wave, an exchange of the state's tiles through LDS, and 4 KiB of M a wave,
// requested AHEAD stretches before (their round trip takes longer than the products: one ahead 1.2 us a stretch).  Bound by the chain of
// stretches: 0.46 us each, of which the matrix instructions are 0.25 (17 stretches of 32 heads 11 us, 43 of 12 heads 22).
__global__ __launch_bounds__(256) void wkv_join_kernel(WkvRowsArgs a, int from, const Plan* plan, int room, float* records)
{
    constexpr int AHEAD = 4;
    __shared__ f4 s_tile[2][4][64];
    const int c = blockIdx.x / (4 * a.heads), rest = blockIdx.x - c * 4 * a.heads, h = rest >> 2, i = rest & 3;
    Stretch part;
    if (plan == nullptr) {
        if (c > 0 || !sole_stretch(a, from, 0, &part) || part.record < 0)
            return;
    } else {
        if (c >= plan->cut)
            return;
        part = plan->list[room + c];
    }
    const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto record_of = [&](int k) { return records + (static_cast<int64_t>(part.record + k) * a.heads + h) * RECORD; };
    auto tile_of = [&](int k) { return reinterpret_cast<f4*>(record_of(k) + N * N) + (4 * i + w) * 64 + lane; };
    f4 S[4], m[AHEAD][4], add[AHEAD];
    const int last = part.count - 2;   // the last one with a record
    auto load = [&](int k, f4(&rows)[4], f4& n) {
        const int at = min(k, last);   // (behind it: read again, not used)
#pragma unroll
        for (int j = 0; j < 4; j++)
            rows[j] = *reinterpret_cast<const f4*>(record_of(at) + (16 * w + t) * N + 16 * j + 4 * g);
        n = *tile_of(at);
    };
    load_state({reinterpret_cast<const f4*>(record_of(0) + N * N)}, i, S);
#pragma unroll
    for (int k = 0; k < AHEAD; k++)
        load(1 + k, m[k], add[k]);
    auto step = [&](int at, int k, bool more) {
        f4 other = {0.0f, 0.0f, 0.0f, 0.0f}, sum = add[k];
        sum = mfma4(m[k][0], S[0], sum);
        other = mfma4(m[k][1], S[1], other);
        sum = mfma4(m[k][2], S[2], sum);
        other = mfma4(m[k][3], S[3], other);
        sum += other;
        if (more)
            load(at + AHEAD, m[k], add[k]);
        *tile_of(at) = sum;   // the next stretch's start, in N's place
        s_tile[k & 1][w][lane] = sum;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++)
            S[j] = s_tile[k & 1][j][lane];
    };
    // (no way out of the loop's middle: it would lead past its head, which then waits for every load)
    int base = 1;
    for (; base + AHEAD <= last + 1; base += AHEAD)
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            step(base + k, k, true);
#pragma unroll
    for (int k = 0; k < AHEAD - 1; k++)
        if (base + k <= last)
            step(base + k, k, false);
}

// From how many rows on a launch cuts its sequences, or 0: none.  Cutting costs the transfers and the join, and pays where the
// longest sequence has 2.5 times the rows that all, shared out evenly, give a workgroup (32 heads; eight of 1000 rows, at 2:
// 220 us whole, 259 cut; sixteen of 100 to 3000, at 3.2: 856 and 595) and becomes three stretches or more.  Where stretches are not
// long, shorter ones that become two, without transfers, then need not wait whole for the last pass (five of 300 to 1500 212 us,
// from three on 249; the sixteen, whose stretches are long, 644 and 595).
int cut_from(const WkvRowsArgs& a)
{
    const int64_t each = (static_cast<int64_t>(a.batch.rows) * a.heads + CARD - 1) / CARD;
    const int stretch = stretch_rows(a.batch.rows, a.heads, 0);
    const int longest = a.batch.max_rows;
    return longest >= LEAST_CUT && longest >= 3 * stretch && 2ll * longest >= 5 * each ? (stretch > LONG_STRETCH ? 3 : 2) * stretch : 0;
}

// The list of stretches of all sequences over `over` rows, by one workgroup: 4096 sequences in turns of 256.
// Whole sequences come first in it: the longest pieces of the last pass.
__device__ void make_plan(const WkvRowsArgs& a, int over, int from, int room, Plan* plan)
{
    __shared__ int64_t s_count[256];
    const int t = threadIdx.x;
    // Rows in all, rows in sequences that are cut, sequences that are not and that are.  Where starts fall, sequences may share rows, and the
    // list's room is for rows that are one sequence's.
    float sums[4] = {};   // (exact to 2^24; whether the first passes 2^20: a sum that does cannot round below it)
    for (int i = t; i < a.batch.sequences; i += 256) {
        const RowSpan span = rows_of(a.batch, i);
        const int rows = span.last - span.first;
        sums[0] += static_cast<float>(rows);
        sums[1] += rows >= from ? static_cast<float>(rows) : 0.0f;
        sums[2] += rows > over && rows < from ? 1.0f : 0.0f;
        sums[3] += rows >= from ? 1.0f : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        sums[i] = wave_sum(sums[i]);
        if ((t & 63) == 0)
            s_count[4 * i + (t >> 6)] = static_cast<int64_t>(sums[i]);
    }
    __syncthreads();
    auto sum_of = [&](int i) { return s_count[4 * i] + s_count[4 * i + 1] + s_count[4 * i + 2] + s_count[4 * i + 3]; };
    const int64_t rows_in_all = sum_of(0), rows_in_cut = sum_of(1);
    const int whole = static_cast<int>(sum_of(2)), cuts = static_cast<int>(sum_of(3));
    __syncthreads();
    if (rows_in_all > a.batch.rows) {
        if (t == 0)
            plan->stretches = plan->cut = 0;
        return;
    }
    const int stretch = stretch_rows(rows_in_cut, a.heads, cuts);   // at most half of `from`
    // whole sequences, cut ones and their stretches in one number, 20 bits each
    int64_t total = 0;
    for (int base = 0; base < a.batch.sequences; base += 256) {
        RowSpan span{0, 0};
        if (base + t < a.batch.sequences)
            span = rows_of(a.batch, base + t);
        const int rows = span.last - span.first;
        const bool cut = rows >= from;
        const Parts lie = parts_of(rows, cut, stretch);
        const int parts = rows <= over ? 0 : lie.count;
        const int64_t own = cut ? 1ll << 20 | static_cast<int64_t>(parts) << 40 : parts;
        s_count[t] = own;
        __syncthreads();
        for (int step = 1; step < min(256, a.batch.sequences - base); step *= 2) {
            const int64_t before = t >= step ? s_count[t - step] : 0;
            __syncthreads();
            s_count[t] += before;
            __syncthreads();
        }
        const int64_t before = total + s_count[t] - own;
        const int cut_before = before >> 20 & 0xfffff, parts_before = static_cast<int>(before >> 40);
        const int record = parts_before - cut_before, at = cut ? whole + parts_before : static_cast<int>(before & 0xfffff);
        for (int k = 0; k < parts; k++) {
            const Stretch part = stretch_of(base + t, span, lie, cut ? record : -1, k);
            plan->list[at + k] = part;
            if (cut && k == 0)
                plan->list[room + cut_before] = part;
        }
        total += s_count[min(255, a.batch.sequences - base - 1)];
        __syncthreads();
    }
    if (t == 0) {
        plan->stretches = static_cast<int>((total & 0xfffff) + (total >> 40));
        plan->cut = total >> 20 & 0xfffff;
    }
}

}  // namespace

// Sequences of up to this many rows go row by row (32 heads; one sequence of 12 rows 7.2 us, of 14 rows 7.9, by blocks 7.2 both; eight of
// 9 rows 7.1, by blocks 8.1, of 14 9.0 and 8.5), and of up to this many where workgroups wait for one another (64 of 17 rows 44,
// by blocks 61, of 24 57 and 63; beside twice the card's workgroups, 32 of 1 to 24 rows, it is 23 and 20).
constexpr int FEW_ROWS = 12, MANY_FEW_ROWS = 24;

// The list: every sequence that goes by blocks, at most, the stretches, and the cut sequences again (at most as many as
// stretches with a record: each has two stretches or more).
constexpr int64_t PLAN_BYTES = (sizeof(Plan) + (ROW_SEQUENCES_MAX + HEAD_STRETCHES * 3) * sizeof(Stretch) + 255) / 256 * 256;

int64_t wkv_rows_workspace_bytes(int) { return PLAN_BYTES + static_cast<int64_t>(HEAD_STRETCHES) * RECORD * 4; }

hipError_t launch_wkv_rows(const WkvRowsArgs& a, hipStream_t s)
{
    const unsigned heads = static_cast<unsigned>(a.heads), grid = static_cast<unsigned>(a.batch.sequences) * heads;
    const int over = grid <= 2 * CARD ? FEW_ROWS : MANY_FEW_ROWS;
    if (a.batch.max_rows <= over) {
        // Eight waves a head where that leaves no workgroup waiting for another (seven sequences of 3 to 6 rows, 32 heads, 5.4 us, of four
        // 6.6; 64 of one row 14.2 and 13.1).
        if (grid <= CARD)
            hipLaunchKernelGGL(wkv_few_kernel<8>, dim3(grid), dim3(512), 0, s, a, INT32_MAX, 0, 0, nullptr);
        else
            hipLaunchKernelGGL(wkv_few_kernel<4>, dim3(grid), dim3(256), 0, s, a, INT32_MAX, 0, 0, nullptr);
        return hipGetLastError();
    }
    const int from = cut_from(a);
    if (from == 0) {
        hipLaunchKernelGGL(wkv_chunk_kernel<CHUNK_SEQUENCES>, dim3(grid), dim3(CHUNK_THREADS), 0, s, a, over, 0, nullptr, nullptr);
        return hipGetLastError();
    }
    Plan* const plan = a.batch.sequences > 1 ? reinterpret_cast<Plan*>(a.workspace) : nullptr;
    float* const records = a.workspace + PLAN_BYTES / 4;
    // What the host knows of the list's length.  Stretches have at least LEAST_STRETCH rows, and
    // as many as share all cut rows and heads out to HEAD_STRETCHES workgroups and one more for each sequence and head.
    auto least = [](int x, int y) { return x < y ? x : y; };
    const int whole = least(a.batch.rows / (FEW_ROWS + 1), a.batch.sequences);
    const int records_most = HEAD_STRETCHES / a.heads, cut = least(a.batch.rows / from, records_most);
    const int room = whole + least(a.batch.rows / LEAST_STRETCH, records_most + cut);
    if (plan)
        hipLaunchKernelGGL(wkv_few_kernel<4>, dim3(grid + 1), dim3(256), 0, s, a, FEW_ROWS, from, room, plan);
    hipLaunchKernelGGL(wkv_chunk_kernel<CHUNK_TRANSFERS>, dim3(room * heads), dim3(CHUNK_THREADS), 0, s, a, FEW_ROWS, from, plan, records);
    hipLaunchKernelGGL(wkv_join_kernel, dim3(cut * heads * 4), dim3(256), 0, s, a, from, plan, room, records);
    hipLaunchKernelGGL(wkv_chunk_kernel<CHUNK_STRETCHES>, dim3(room * heads), dim3(CHUNK_THREADS), 0, s, a, FEW_ROWS, from, plan, records);
    return hipGetLastError();
}

}  // namespace si
