// A cache in pages shared by many sequences, and the batch of their newest
// rows: the launches behind the si_hip_paged_* entry points.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace si {

constexpr int PAGED_GROUP_MAX = 16;      // query heads per KV head
constexpr int PAGED_SEQUENCES_MAX = 4096;

struct PagedBatch {
    const int32_t* table;      // [sequences][max_pages]
    const int32_t* starts;     // [sequences + 1]: the sequence's rows of the batch
    const int32_t* lengths;    // [sequences]: positions, the batch's rows included
    int sequences;
    int max_pages;
    int rows;                  // rows of the batch's buffers
    int max_rows;              // most rows of one sequence
};

struct PagedCache {
    char* keys;
    char* values;
    int64_t pages;
    int page_size;             // a power of two, 16..256
    int page_shift;
    int kv_heads;
    int head;                  // 64 or 128
    bool q4;                   // 4-bit pages, else FP16
};

// Bytes of one page of one KV head: FP16 rows, or (4-bit) all positions'
// nibbles and then the FP16 scales [head / 32][page_size].
constexpr int64_t paged_head_bytes(bool q4, int page_size, int head)
{
    return static_cast<int64_t>(page_size) * (q4 ? head / 2 + head / 16 : 2 * head);
}

struct PagedAppendArgs {
    PagedBatch batch;
    PagedCache cache;
    const float* qkv;          // [rows][(heads + 2 * kv_heads) * head]
    const float* frequencies;  // [rotary / 2]
    float* query;              // [rows][heads * head]
    int heads;
    int rotary;
    float rope_scale;
};

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s);
// keys, values: FP32 [rows][kv_heads * head], what the pages hold for the batch's rows
hipError_t launch_paged_read(const PagedBatch& batch, const PagedCache& cache, float* keys, float* values,
                             hipStream_t s);

enum PagedOut : int { PAGED_OUT_F32, PAGED_OUT_F16, PAGED_OUT_BF16 };

struct PagedAttentionArgs {
    PagedBatch batch;
    PagedCache cache;
    const float* query;        // [rows][heads * head], 16-byte aligned
    void* out;                 // [rows][heads * head], 16-byte aligned
    float* workspace;
    int heads;
    int out_format;            // PagedOut
    int few_rows;              // set by the launch
};

int64_t paged_attention_workspace_floats(int heads, int kv_heads, int head);
hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t s);

}  // namespace si
