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

// Sequences of few rows: a workgroup takes one head of one sequence, the state
// in registers (a thread holds 8 columns of two state rows: 8 lanes a state
// row, whose sums take three DPP steps, and half the LDS reads of 16 columns
// of one row).  Four rows at a time: wave w prepares row w (one element a
// lane), all waves take the four rows through the state, wave w normalises row w.
// Bound by reading and writing the state (32 KiB a head) where a sequence
// brings one row; by vector instructions (92 a row and wave) and LDS reads
// (10 b128 a lane and row) where it brings many.
__global__ __launch_bounds__(256) void wkv_few_kernel(WkvRowsArgs a, int most)
{
    __shared__ float4 s_vec[4][5][N / 4];   // decay, key, kn, kn * a, r of the four rows
    __shared__ float s_value[4][N], s_y[4][N];
    const int s = blockIdx.x / a.heads, h = blockIdx.x - s * a.heads;
    const RowSpan span = rows_of(a.batch, s);
    const int from = a.batch.from[s], to = a.batch.to[s];
    if (span.last - span.first < 1 || span.last - span.first > most)
        return;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int64_t width = static_cast<int64_t>(a.heads) * N;
    const int e = h * N + lane;

    const int c = t & 7, i0 = t >> 3;
    float4 sv[2][2];
    if (from >= 0 && from < a.batch.slots) {
        const float* S = a.state + (static_cast<int64_t>(from) * a.heads + h) * N * N;
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int q = 0; q < 2; q++)
                sv[p][q] = *reinterpret_cast<const float4*>(S + (i0 + 32 * p) * N + 32 * q + 4 * c);
    } else {
        const float z = from == -1 ? 0.0f : __builtin_nanf("");
#pragma unroll
        for (int p = 0; p < 2; p++)
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
    for (int base = span.first; base < span.last; base += 4) {
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
            float* vec = reinterpret_cast<float*>(s_vec[wave]);
            vec[lane] = decay;
            vec[N + lane] = key;
            vec[2 * N + lane] = kn;
            vec[3 * N + lane] = kn * ad;
            vec[4 * N + lane] = x.r;
            s_value[wave][lane] = value;
        }
        next = load(row + 4);
        __syncthreads();
        const int live = min(4, span.last - base);
        for (int j = 0; j < live; j++) {
            float p0 = 0.0f, p1 = 0.0f, y0 = 0.0f, y1 = 0.0f;
            const float v0i = s_value[j][i0], v1i = s_value[j][i0 + 32];
            auto dot = [](float4 x, float4 y, float acc) {
                return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, acc))));
            };
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const float4 kn = s_vec[j][2][8 * q + c];
                p0 = dot(sv[0][q], kn, p0);
                p1 = dot(sv[1][q], kn, p1);
            }
            p0 = -row_sum<8>(p0);
            p1 = -row_sum<8>(p1);
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const float4 d = s_vec[j][0][8 * q + c], k = s_vec[j][1][8 * q + c], ak = s_vec[j][3][8 * q + c],
                             r = s_vec[j][4][8 * q + c];
                auto step = [&](float4& S, float p, float v) {
                    S.x = fmaf(p, ak.x, fmaf(v, k.x, S.x * d.x));
                    S.y = fmaf(p, ak.y, fmaf(v, k.y, S.y * d.y));
                    S.z = fmaf(p, ak.z, fmaf(v, k.z, S.z * d.z));
                    S.w = fmaf(p, ak.w, fmaf(v, k.w, S.w * d.w));
                };
                step(sv[0][q], p0, v0i);
                step(sv[1][q], p1, v1i);
                y0 = dot(sv[0][q], r, y0);
                y1 = dot(sv[1][q], r, y1);
            }
            y0 = row_sum<8>(y0);
            y1 = row_sum<8>(y1);
            if (c == 0) {
                s_y[j][i0] = y0;
                s_y[j][i0 + 32] = y1;
            }
        }
        __syncthreads();
        if (row < span.last) {
            const float y = s_y[wave][lane];
            const float d = y - wave_sum(y) * (1.0f / N);
            const float var = wave_sum(d * d) * (1.0f / N);
            const float ln = d * (1.0f / sqrtf(var + GROUP_EPS)) * lw + lb;
            store_row_value(a.out, a.out_format, row * width + e, (ln + value * bonus) * x.gate);
        }
    }
    if (to >= 0 && to < a.batch.slots) {
        float* S = a.state + (static_cast<int64_t>(to) * a.heads + h) * N * N;
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int q = 0; q < 2; q++)
                *reinterpret_cast<float4*>(S + (i0 + 32 * p) * N + 32 * q + 4 * c) = sv[p][q];
    }
}

// ---- blocks of 16 rows on the matrix cores ----------------------------------------------------
//
// Within a block of C = 16 rows let L_t be the decays' product up to row t, and
//   alpha_t = L_(t-1) * kn_t,  beta_t = kn_t a_t / L_t,  khat_t = key_t / L_t,  rho_t = L_t * r_t.
// Then with u_t = -(S_(t-1) kn_t) the block's state is S_0 + sum_s (u_s beta_s^T + v_s khat_s^T), times L_C, and
//   (I + A) U = -(alpha S_0^T + B V),   A_ts = alpha_t . beta_s, B_ts = alpha_t . khat_s  (s < t)
//   Y = rho S_0^T + D U + E V,          D_ts = rho_t . beta_s,   E_ts = rho_t . khat_s    (s <= t).
// What does not need S_0 is formed beforehand: alpha' = (I + A)^-1 alpha, W = (I + A)^-1 B,
// rho' = rho - D alpha', Z = E - D W, V' = W V, Y' = Z V, so that a block costs the state
//   U = -(alpha' S_0^T + V'),  Y = rho' S_0^T + Y',  S = (S_0 + U^T beta + V^T khat) diag(L_C).
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

template <int SHIFT>
__device__ __forceinline__ float row_shr(float v)   // the value SHIFT lanes before in the row of 16, or 0
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x110 + SHIFT, 0xF, 0xF, true));
}

// The value of the lane before in the row of 16; 1 in the first.
__device__ __forceinline__ float row_shr_or_one(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0x3f800000, __float_as_int(v), 0x111, 0xF, 0xF, false));
}

// The value that lane I of the row of 16 holds.
template <int I>
__device__ __forceinline__ float row_lane(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + I, 0xF, 0xF, true));
}

// max(top, |x|, |y|), NaN if any is
__device__ __forceinline__ float largest(float top, float x, float y)
{
    asm("v_maximum3_f32 %0, %1, |%2|, |%3|" : "=v"(top) : "v"(top), "v"(x), "v"(y));
    return top;
}

// z + sum of the values that lanes S .. S + TERMS - 1 of the row of 16 hold in l, times x[S] ..: one instruction a term (the
// compiler forms two).  The wait in front keeps the two instructions' distance that a lane-crossing read of a register just
// written needs; nothing here writes l.
template <int S, int TERMS>
__device__ __forceinline__ float add_terms(float z, float l, const float* x)
{
    if constexpr (TERMS == 4)
        asm("s_nop 1\n\t"
            "v_fmac_f32_dpp %0, %1, %2 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n\t"
            "v_fmac_f32_dpp %0, %1, %3 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n\t"
            "v_fmac_f32_dpp %0, %1, %4 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n\t"
            "v_fmac_f32_dpp %0, %1, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf"
            : "+&v"(z)
            : "v"(l), "v"(x[S]), "v"(x[S + 1]), "v"(x[S + 2]), "v"(x[S + 3]), "n"(S), "n"(S + 1), "n"(S + 2), "n"(S + 3));
    else
        asm("s_nop 1\n\t"
            "v_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf"
            : "+&v"(z)
            : "v"(l), "v"(x[S]), "n"(S));
    return z;
}
// z_i = n_i (z_i + sum over s < i of l_i[s] z_s) row after row; l_i[s] lies in lane s of each row of 16, as n does.
template <int I, int S>
__device__ __forceinline__ void add_rows(float (&z)[C], const float (&l)[C])
{
    if constexpr (S < I) {
        constexpr int TERMS = I - S >= 4 ? 4 : 1;
        z[I] = add_terms<S, TERMS>(z[I], l[I], z);
        add_rows<I, S + TERMS>(z, l);
    }
}
template <int I>
__device__ __forceinline__ void solve_rows(float (&z)[C], const float (&l)[C], float n)
{
    if constexpr (I < C) {
        add_rows<I, 0>(z, l);
        z[I] *= row_lane<I>(n);
        solve_rows<I + 1>(z, l, n);
    }
}
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
    f4 v_part[4][64], y_part[4][64];   // V', Y' tiles as the matrix instructions hold them
    float decay[N];                    // L_C
    float bonus[4][C];                 // parts of sum(key r r_k)
    float squares[4][C];
    int odd;                           // a value is not finite or very large
};

struct ChunkLds {
    BlockLds block[2];
    float m[C][LD];                    // A, B, D, E beside one another
    float w[C][LD];                    // W in the columns that A has in m
    float y[C][LD];
    float params[6][N];                // of the head: w0, a0, v0 (times -log2(e)), k_k, k_a, r_k
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

__device__ __forceinline__ f4 load4(const float* p)   // at a multiple of 4 bytes
{
    f4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

__device__ __forceinline__ f4 load_at(const float* uniform, uint32_t bytes)
{
    return *reinterpret_cast<const f4*>(reinterpret_cast<const char*>(uniform) + bytes);
}

// 1 / (1 + exp(-(x + bias))), shift = -LOG2E * bias
__device__ __forceinline__ float sigmoid_shifted(float x, float shift)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(fmaf(x, -LOG2E, shift)));
}

__device__ void chunk_prepare(const WkvRowsArgs& a, ChunkLds& lds, int h, Blocks blocks)
{
    const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int q = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const int64_t width = static_cast<int64_t>(a.heads) * N;
    const int ch = 16 * q + 4 * g;                       // this lane's four channels, of row t
    const bool first = a.first_layer != 0;
    const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    struct {
        f4 r, k, v, wl, al, vl, vf;
    } x;
    // (a row behind the block's last reads the last again, and is masked where it counts)
    auto load = [&](int at, int last) {
        const int64_t from = at * width + h * N;
        const uint32_t lane_at = 4u * (min(t, last - 1 - at) * static_cast<uint32_t>(width) + ch);
        x.r = load_at(a.r + from, lane_at);
        x.k = load_at(a.k + from, lane_at);
        x.v = load_at(a.v + from, lane_at);
        x.wl = load_at(a.w_lora + from, lane_at);
        x.al = load_at(a.a_lora + from, lane_at);
        if (!first) {
            x.vl = load_at(a.v_lora + from, lane_at);
            x.vf = load_at(a.v_first + from, lane_at);
        }
    };
    x.vl = x.vf = zero;
    load(blocks.at, blocks.last());
    for (int stage = 0; blocks.at < blocks.end; stage++) {
        BlockLds& b = lds.block[stage & 1];
        const int at = blocks.at, rows = blocks.last() - at;
        // 1: the rows' factors
        if (rows < C) {   // a decay of 1, the rest 0
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool in = t < rows;
                x.wl[j] = in ? x.wl[j] : -3e38f;
                x.al[j] = in ? x.al[j] : 0.0f;
                x.vl[j] = in ? x.vl[j] : 0.0f;
                x.vf[j] = in ? x.vf[j] : 0.0f;
                x.k[j] = in ? x.k[j] : 0.0f;
                x.v[j] = in ? x.v[j] : 0.0f;
                x.r[j] = in ? x.r[j] : 0.0f;
            }
        }
        f4 al, rh, be, kh, va, decay;
        auto par = [&](int i) { return *reinterpret_cast<const f4*>(&lds.params[i][ch]); };
        const f4 w0 = par(0), a0 = par(1), v0 = par(2), kkk = par(3), kka = par(4), rk = par(5);
        float squares = 0.0f, bonus = 0.0f, top = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float c = -0.606531f * LOG2E * sigmoid_shifted(x.wl[j], w0[j]);
            c += row_shr<1>(c);
            c += row_shr<2>(c);
            c += row_shr<4>(c);
            c += row_shr<8>(c);
            decay[j] = __builtin_amdgcn_exp2f(c);
            const float shrink = __builtin_amdgcn_exp2f(-c);
            const float ad = sigmoid_shifted(x.al[j], a0[j]);
            const float sk = x.k[j] * kkk[j];
            const float key = fmaf(x.k[j] * kka[j], ad - 1.0f, x.k[j]);
            va[j] = first ? x.v[j] : fmaf(x.vf[j] - x.v[j], sigmoid_shifted(x.vl[j], v0[j]), x.v[j]);
            al[j] = sk * row_shr_or_one(decay[j]);
            be[j] = (sk * ad) * shrink;
            kh[j] = key * shrink;
            rh[j] = x.r[j] * decay[j];
            squares = fmaf(sk, sk, squares);
            bonus = fmaf(key * x.r[j], rk[j], bonus);
            top = largest(largest(top, al[j], kh[j]), rh[j], va[j]);   // (beta is at most alpha / decay)
        }
        *reinterpret_cast<f4*>(&b.alpha[t][ch]) = al;
        *reinterpret_cast<f4*>(&b.rho[t][ch]) = rh;
        *reinterpret_cast<f4*>(&b.beta[t][ch]) = be;
        *reinterpret_cast<f4*>(&b.khat[t][ch]) = kh;
        *reinterpret_cast<f4*>(&b.value[t][ch]) = va;
        squares = rows_sum(squares);
        bonus = rows_sum(bonus);
        if (g == 0) {
            b.squares[q][t] = squares;
            b.bonus[q][t] = bonus;
        }
        if (t == C - 1)
            *reinterpret_cast<f4*>(&b.decay[ch]) = decay;
        if (first && t < rows)
            *reinterpret_cast<f4*>(a.v_first + (at + t) * width + h * N + ch) = x.v;
        if (!(top < 0x1p50f))
            b.odd = 1;
        __syncthreads();
        // 2: the four products of rows with rows, one a wave
        const bool counts = blocks.next(b.odd != 0);
        if (blocks.at < blocks.end)
            load(blocks.at, blocks.last());
        float length = b.squares[0][t] + b.squares[1][t] + b.squares[2][t] + b.squares[3][t];
        length = __builtin_amdgcn_rsqf(length > 1e-24f ? length : 1e-24f);   // 1 / |sk| of row t
        {
            const auto& left = q < 2 ? b.alpha : b.rho;
            const auto& right = q & 1 ? b.khat : b.beta;
            f4 l[4], r[4], m0 = zero, m1 = zero;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                l[j] = row4(left, t, 16 * j + 4 * g);
                r[j] = row4(right, t, 16 * j + 4 * g);
            }
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
                lds.m[i][16 * q + t] = __int_as_float(__float_as_int((m0[v] + m1[v]) * f) & keep);
            }
        }
        __syncthreads();
        // 3: the block's solution and what follows from it (16 channels or values a wave)
        if (counts) {
            // column t of alpha (lanes 0..15 of a half) or of B (16..31), solved row by row:
            // z_i = n_i (r_i + sum_s -A_is n_s z_s), every lane with row i's sums from the row of 16 lanes that holds it
            const bool of_b = (lane & 16) != 0;
            const float* const column = of_b ? &lds.m[0][16 + t] : &b.alpha[0][16 * q + t];
            float z[C], l[C];
#pragma unroll
            for (int i = 0; i < C; i++) {
                l[i] = lds.m[i][t];
                z[i] = column[i * LD];
            }
            solve_rows<0>(z, l, length);
            float* const solved = of_b ? &lds.w[0][t] : &b.alpha[0][16 * q + t];   // (w: the same from all four waves)
            if (lane < 32)
                scale_rows<0>(solved, z, length);
            wave_sync();
            const f4 v_tile = column4(b.value, 4 * g, 16 * q + t);
            b.v_part[q][lane] = mfma4(row4(lds.w, t, 4 * g), v_tile, zero);
            const f4 d = -row4(lds.m, t, 32 + 4 * g);
            const f4 rho = mfma4(d, column4(b.alpha, 4 * g, 16 * q + t), column4(b.rho, 4 * g, 16 * q + t));
            const f4 zt = mfma4(column4(lds.w, 4 * g, t), d, row4(lds.m, t, 48 + 4 * g));   // Z^T
#pragma unroll
            for (int v = 0; v < 4; v++)
                b.rho[4 * g + v][16 * q + t] = rho[v];
            b.y_part[q][lane] = mfma4(zt, v_tile, zero);
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

__device__ void chunk_advance(const WkvRowsArgs& a, ChunkLds& lds, int h, int from, int to, Blocks blocks)
{
    const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t width = static_cast<int64_t>(a.heads) * N;
    const int tn = 4 * w + g, cn = 4 * t;   // row and four channels in the normalisation
    const f4 lw = load4(a.lnx_weight + h * N + cn), lb = load4(a.lnx_bias + h * N + cn);
    // S^T tiles: keys 16 j + 4 g + v, value 16 w + t
    f4 S[4];
    if (from >= 0 && from < a.batch.slots) {
        const float* p = a.state + ((static_cast<int64_t>(from) * a.heads + h) * N + 16 * w + t) * N + 4 * g;
#pragma unroll
        for (int j = 0; j < 4; j++)
            S[j] = *reinterpret_cast<const f4*>(p + 16 * j);
    } else {
        const float z = from == -1 ? 0.0f : __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < 4; j++)
            S[j] = f4{z, z, z, z};
    }
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
        f4 gate, xa, xr;
        auto part = [&](int j) {
            xa = mfma4(row4(b.alpha, t, 16 * j + 4 * g), S[j], xa);
            xr = mfma4(row4(b.rho, t, 16 * j + 4 * g), S[j], xr);
        };
        if (have) {
            gate = load_at(a.gate + at * width + h * N, 4u * (min(tn, rows - 1) * static_cast<uint32_t>(width) + cn));
            xa = b.v_part[w][lane];
            xr = b.y_part[w][lane];
            part(0);
            part(1);
        }
        __syncthreads();
        counts = more && blocks.next(lds.block[stage & 1].odd != 0);
        if (have) {
            part(2);
            part(3);
#pragma unroll
            for (int v = 0; v < 4; v++)
                lds.y[4 * g + v][16 * w + t] = xr[v];
        }
        __syncthreads();
        if (have) {
            const f4 y = row4(lds.y, tn, cn), value = row4(b.value, tn, cn);
            const float bonus = b.bonus[0][tn] + b.bonus[1][tn] + b.bonus[2][tn] + b.bonus[3][tn];
            const f4 u = -xa, v_tile = column4(b.value, 4 * g, 16 * w + t);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                S[j] = mfma4(column4(b.beta, 4 * g, 16 * j + t), u, S[j]);
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
    if (to >= 0 && to < a.batch.slots) {
        float* p = a.state + ((static_cast<int64_t>(to) * a.heads + h) * N + 16 * w + t) * N + 4 * g;
#pragma unroll
        for (int j = 0; j < 4; j++)
            *reinterpret_cast<f4*>(p + 16 * j) = S[j];
    }
}

// One head of one sequence, block after block.  While the state's waves take block i
// (64 matrix instructions each), the others prepare block i + 1 (32 each, and the
// exponentials), in three phases between barriers.
__global__ __launch_bounds__(CHUNK_THREADS, 4) void wkv_chunk_kernel(WkvRowsArgs a, int over)
{
    __shared__ ChunkLds lds;
    const int s = blockIdx.x / a.heads, h = blockIdx.x - s * a.heads;
    RowSpan span = rows_of(a.batch, s);
    span.first = __builtin_amdgcn_readfirstlane(span.first);
    span.last = __builtin_amdgcn_readfirstlane(span.last);
    if (span.last - span.first <= over)
        return;
    if (threadIdx.x < 2)
        lds.block[threadIdx.x].odd = 0;
    if (threadIdx.x < N) {
        const int t = threadIdx.x, e = h * N + t;
        lds.params[0][t] = -LOG2E * a.w0[e];
        lds.params[1][t] = -LOG2E * a.a0[e];
        lds.params[2][t] = a.first_layer ? 0.0f : -LOG2E * a.v0[e];
        lds.params[3][t] = a.k_k[e];
        lds.params[4][t] = a.k_a[e];
        lds.params[5][t] = a.r_k[e];
    }
    __syncthreads();
    const Blocks blocks{span.first, span.last, span.first};
    if (threadIdx.x < CHUNK_THREADS / 2)
        chunk_advance(a, lds, h, a.batch.from[s], a.batch.to[s], blocks);
    else
        chunk_prepare(a, lds, h, blocks);
}

}  // namespace

int64_t wkv_rows_workspace_bytes(int) { return 16; }

// Sequences of up to this many rows go row by row.
constexpr int FEW_ROWS = 8;

hipError_t launch_wkv_rows(const WkvRowsArgs& a, hipStream_t s)
{
    const unsigned grid = static_cast<unsigned>(a.batch.sequences) * a.heads;
    const bool long_ones = a.batch.max_rows > FEW_ROWS;
    hipLaunchKernelGGL(wkv_few_kernel, dim3(grid), dim3(256), 0, s, a, long_ones ? FEW_ROWS : INT32_MAX);
    if (long_ones)
        hipLaunchKernelGGL(wkv_chunk_kernel, dim3(grid), dim3(CHUNK_THREADS), 0, s, a, FEW_ROWS);
    return hipGetLastError();
}

}  // namespace si
