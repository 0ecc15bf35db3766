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

}  // namespace

int64_t wkv_rows_workspace_bytes(int) { return 16; }

hipError_t launch_wkv_rows(const WkvRowsArgs& a, hipStream_t s)
{
    hipLaunchKernelGGL(wkv_few_kernel, dim3(static_cast<unsigned>(a.batch.sequences) * a.heads), dim3(256), 0, s, a,
                       INT32_MAX);
    return hipGetLastError();
}

}  // namespace si
