// A recurrent model's step over many sequences and the search over beams: the
// launches behind si_hip_layernorm_mix_rows, si_hip_rwkv7_wkv_rows,
// si_hip_beam_select and si_hip_copy_slots.
#pragma once

#include "sharpinference_hip.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace si {

constexpr int ROW_SEQUENCES_MAX = 4096;
constexpr int MIX_MAX = 8;               // mixes of one call
constexpr int MIX_WIDTH_MAX = 8192;
constexpr int WKV_HEAD = 64;
constexpr int BEAMS_MAX = 16;
constexpr int CANDIDATES_MAX = 32;

enum RowsOut : int { ROWS_OUT_F32, ROWS_OUT_F16, ROWS_OUT_BF16 };

struct RowBatch {
    const int32_t* starts;     // [sequences + 1]
    const int32_t* from;       // [sequences]
    const int32_t* to;         // [sequences]
    int sequences;
    int slots;
    int rows;
    int max_rows;
};

struct MixRowsArgs {
    RowBatch batch;
    const float* x;            // [rows][n]
    const float* residual;     // or null
    const float* weight;
    const float* bias;
    const float* mix;          // [mixes][n]
    float* state;              // [slots][n]
    float* updated;            // [rows][n], with residual
    void* out;                 // [max(mixes, 1)][rows][n]
    int n;
    int mixes;
    int out_format;            // RowsOut
    float eps;
};

hipError_t launch_layernorm_mix_rows(const MixRowsArgs& a, hipStream_t s);

struct WkvRowsArgs {
    RowBatch batch;
    int heads;
    int first_layer;
    const float *r, *k, *v, *w_lora, *a_lora, *gate, *v_lora;                   // [rows][heads * 64]
    const float *w0, *a0, *v0, *k_k, *k_a, *r_k, *lnx_weight, *lnx_bias;        // [heads * 64]
    float* v_first;            // [rows][heads * 64]
    float* state;              // [slots][heads][64][64]
    void* out;                 // [rows][heads * 64]
    float* workspace;
    int out_format;            // RowsOut
};

int64_t wkv_rows_workspace_bytes(int heads);
hipError_t launch_wkv_rows(const WkvRowsArgs& a, hipStream_t s);

struct BeamArgs {
    const void* logits;        // [sequences * beams] rows, stride values apart
    const float* scores;
    const int32_t* done;       // or null
    const int32_t* slots;      // or null
    int32_t* parents;
    int32_t* tokens;
    float* new_scores;
    int32_t* new_done;         // or null
    int32_t* from;             // with slots
    int32_t* to;
    void* workspace;
    int64_t stride;
    int vocab;
    int sequences;
    int beams;
    int candidates;
    int format;                // RowsOut: the logits' type
    int end_token;
};

int64_t beam_workspace_bytes(int sequences, int beams, int candidates, int vocab);
hipError_t launch_beam_select(const BeamArgs& a, hipStream_t s);

constexpr int SLOT_ARRAYS_PER_LAUNCH = 64;
hipError_t launch_copy_slots(const si_hip_slot_array* arrays, int count, int64_t slots, const int32_t* from, const int32_t* to,
                             int moves, hipStream_t s);

#ifdef __HIPCC__
// Rows of sequence s: first .. last - 1 inside the batch's rows, none where the starts fall or leave them.
struct RowSpan {
    int first, last;
};
__device__ __forceinline__ RowSpan rows_of(const RowBatch& b, int s)
{
    const int first = b.starts[s], last = b.starts[s + 1];
    return first < 0 || last < first || last > b.rows ? RowSpan{0, 0} : RowSpan{first, last};
}

__device__ __forceinline__ void store_row_value(void* out, int format, int64_t at, float v)
{
    if (format == ROWS_OUT_F32)
        static_cast<float*>(out)[at] = v;
    else if (format == ROWS_OUT_F16)
        static_cast<_Float16*>(out)[at] = static_cast<_Float16>(v);
    else
        static_cast<__bf16*>(out)[at] = static_cast<__bf16>(v);
}

// LDS written by other lanes of the wave is read behind this.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Four neighbours at a multiple of four.
template <typename V>
__device__ __forceinline__ void store_row4(void* out, int format, int64_t at, V v)
{
    if (format == ROWS_OUT_F32) {
        typedef float W __attribute__((ext_vector_type(4)));
        *reinterpret_cast<W*>(static_cast<float*>(out) + at) = W{v[0], v[1], v[2], v[3]};
    } else if (format == ROWS_OUT_F16) {
        typedef _Float16 W __attribute__((ext_vector_type(4)));
        *reinterpret_cast<W*>(static_cast<_Float16*>(out) + at) =
            W{static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]), static_cast<_Float16>(v[2]), static_cast<_Float16>(v[3])};
    } else {
        typedef __bf16 W __attribute__((ext_vector_type(4)));
        *reinterpret_cast<W*>(static_cast<__bf16*>(out) + at) =
            W{static_cast<__bf16>(v[0]), static_cast<__bf16>(v[1]), static_cast<__bf16>(v[2]), static_cast<__bf16>(v[3])};
    }
}
#endif

}  // namespace si
