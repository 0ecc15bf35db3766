// Beam search over the rows of a step: the best candidates over beams and
// vocabulary, and the moves of states that follow.
//
// score(b, t) = s_b + (x_bt - m_b) - log(sum_t exp(x_bt - m_b)), m_b the row's
// largest logit.  Within a row the order is that of the logits, so each part of a
// row needs its sum and its own best `candidates` logits, and scores (in FP64) are
// formed for the rows' best alone.
#include "si_sequences.hpp"
#include "si_lanes.hpp"

#include <hip/hip_bf16.h>

namespace si {
namespace {

constexpr float LOG2E = 1.44269504088896f;
constexpr int TILE = 2048, PER = TILE / 64;   // values of a wave's tile, and of a lane's
constexpr int KEPT = 256;                     // values over a tile's bound that are ranked together
constexpr int SCAN_WAVES = 4, MERGE_WAVES = 8;

typedef unsigned long long Key;   // order of a logit (high word: 0 for none) and of its token, lowest last

// Order of a logit: larger for larger values, 0 for -infinity and NaN; -0 as 0.
__device__ __forceinline__ uint32_t order_of(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    return v > -__builtin_inff() ? u ^ (static_cast<int32_t>(u) < 0 ? 0xffffffffu : 0x80000000u) : 0u;
}
__device__ __forceinline__ float logit_of(uint32_t order)
{
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

__device__ __forceinline__ uint32_t row_max_u32(uint32_t v, int width)
{
    auto max_of = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = max_of(v, dpp_row<0xB1>(static_cast<int>(v)));
    if (width >= 4) v = max_of(v, dpp_row<0x4E>(static_cast<int>(v)));
    if (width >= 8) v = max_of(v, dpp_row<0x141>(static_cast<int>(v)));
    if (width >= 16) v = max_of(v, dpp_row<0x140>(static_cast<int>(v)));
    return v;
}
template <typename F>
__device__ __forceinline__ uint32_t wave_reduce_u32(uint32_t v, F f)
{
    v = f(v, static_cast<uint32_t>(dpp_row<0xB1>(static_cast<int>(v))));
    v = f(v, static_cast<uint32_t>(dpp_row<0x4E>(static_cast<int>(v))));
    v = f(v, static_cast<uint32_t>(dpp_row<0x141>(static_cast<int>(v))));
    v = f(v, static_cast<uint32_t>(dpp_row<0x140>(static_cast<int>(v))));
    auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = f(a[0], a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return f(b[0], b[1]);
}

// Merges a tile's values (PERL a lane: value(j) gives order and token's key) into
// the sorted list of the best k so far.  A bound first: the lanes fall into at least k
// groups, and the smallest of the groups' largest values has k values at or over it, so only
// values at or over the bound (and over the list's last) can be among the best k: some
// dozens of 2048 of spread values, which are ranked by counting.  Where more than
// KEPT remain (long runs of equal or masked logits), the k best are taken out one by one.
template <int PERL, typename F>
__device__ __forceinline__ void merge_tile(const uint32_t (&order)[PERL], F key_of, int k, Key* kept, Key* list)
{
    const int lane = threadIdx.x & 63;
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < PERL; j++)
        best = best > order[j] ? best : order[j];
    const int width = k <= 4 ? 16 : k <= 8 ? 8 : k <= 16 ? 4 : 2;
    const uint32_t low = wave_reduce_u32(row_max_u32(best, width), [](uint32_t a, uint32_t b) { return a < b ? a : b; });
    const uint32_t last = static_cast<uint32_t>(list[k - 1] >> 32);
    // (a value equal to the list's last has a higher token: tiles come in order)
    const uint32_t bound = low > last + 1 ? low : last + 1;
    int count = 0;
#pragma unroll
    for (int j = 0; j < PERL; j++) {
        const uint64_t mask = __ballot(order[j] >= bound);
        if (mask) {
            const int at = count + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                             __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
            if (order[j] >= bound && at < KEPT)
                kept[at] = key_of(j);
            count += __popcll(mask);
        }
    }
    if (count == 0)
        return;
    if (count > KEPT) {
        uint32_t out[(PERL + 31) / 32] = {};   // bit j: value j is taken out already
        count = 0;
        for (; count < k; count++) {
            Key mine = 0;
#pragma unroll
            for (int j = 0; j < PERL; j++) {
                const Key x = order[j] >= bound && !(out[j / 32] >> (j % 32) & 1) ? key_of(j) : 0;
                mine = x > mine ? x : mine;
            }
            const uint32_t high = wave_reduce_u32(static_cast<uint32_t>(mine >> 32), [](uint32_t a, uint32_t b) { return a > b ? a : b; });
            const uint32_t token = wave_reduce_u32(static_cast<uint32_t>(mine >> 32) == high ? static_cast<uint32_t>(mine) : 0u,
                                                   [](uint32_t a, uint32_t b) { return a > b ? a : b; });
            if (high == 0)
                break;
            const Key top = static_cast<Key>(high) << 32 | token;
#pragma unroll
            for (int j = 0; j < PERL; j++)
                out[j / 32] |= static_cast<uint32_t>(order[j] >= bound && key_of(j) == top) << (j % 32);
            if (lane == 0)
                kept[count] = top;
        }
    }
    // the list's own values behind the kept ones, and each one's place by counting
    if (lane < k && list[lane] != 0)
        kept[count + lane] = list[lane];
    const uint64_t held = __ballot(lane < k && list[lane] != 0);   // a prefix of the lanes: the list is sorted
    count += __popcll(held);
    wave_sync();
    for (int i = lane; i < count; i += 64) {
        const Key mine = kept[i];
        int rank = 0;
        for (int j = 0; j < count; j++)
            rank += kept[j] > mine;
        if (rank < k)
            list[rank] = mine;
    }
    wave_sync();
}

// How a row is cut: tiles a part, parts a row.  A wave takes a part; where there are
// more tiles than some waves for every SIMD, it takes several one after another.
struct Cut {
    int tiles, parts;
};
Cut cut_of(int rows, int vocab)
{
    const int all = (vocab + TILE - 1) / TILE;
    const int64_t waves = static_cast<int64_t>(rows) * all;
    const int tiles = static_cast<int>(waves <= 4096 ? 1 : (waves + 4095) / 4096);
    return {tiles, (all + tiles - 1) / tiles};
}

struct Part {
    float most, sum;   // largest logit, sum of exp(x - most) (NaN: the row has no candidates)
};

template <int FMT>
__device__ __forceinline__ float value_at(const void* p, int64_t i)
{
    if constexpr (FMT == ROWS_OUT_F32)
        return static_cast<const float*>(p)[i];
    else if constexpr (FMT == ROWS_OUT_F16)
        return static_cast<float>(static_cast<const _Float16*>(p)[i]);
    else
        return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
}

// One wave a part of a row.  Bound by HBM (the logits, read once); in small calls by
// the launch and one tile's latency.
template <int FMT>
__global__ __launch_bounds__(64 * SCAN_WAVES) void beam_scan_kernel(BeamArgs a, int rows, int tiles, int parts, Part* part, Key* keys)
{
    __shared__ Key s_kept[SCAN_WAVES][KEPT + CANDIDATES_MAX], s_list[SCAN_WAVES][CANDIDATES_MAX];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * SCAN_WAVES + wave;
    if (unit >= static_cast<int64_t>(rows) * parts)
        return;
    const int row = static_cast<int>(unit / parts), p = static_cast<int>(unit - static_cast<int64_t>(row) * parts);
    if (a.done && a.done[row] != 0)
        return;   // its logits are not looked at
    const int k = a.candidates;
    Key* const list = s_list[wave];
    if (lane < CANDIDATES_MAX)
        list[lane] = 0;
    wave_sync();
    constexpr int SIZE = FMT == ROWS_OUT_F32 ? 4 : 2;
    const char* const x = static_cast<const char*>(a.logits) + row * a.stride * SIZE;
    float most = -__builtin_inff(), sum = 0.0f;
    const int64_t first = static_cast<int64_t>(p) * tiles * TILE;
    for (int i = 0; i < tiles; i++) {
        const int64_t base = first + static_cast<int64_t>(i) * TILE;
        if (base >= a.vocab)
            break;
        constexpr int VEC = 16 / SIZE;
        float v[PER];
        const bool full = base + TILE <= a.vocab;
        // token of value j: neighbours in a 16-byte load, or (a row's last tile) every 64th
        auto token = [&](int j) {
            return static_cast<uint32_t>(base) + (full ? VEC * (lane + 64 * (j / VEC)) + j % VEC : lane + 64 * j);
        };
        if (full) {
            uint4 w[PER / VEC];
#pragma unroll
            for (int j = 0; j < PER / VEC; j++)
                __builtin_memcpy(&w[j], x + (base + VEC * (lane + 64 * j)) * SIZE, 16);
#pragma unroll
            for (int j = 0; j < PER; j++)
                v[j] = value_at<FMT>(&w[j / VEC], j % VEC);
        } else {
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int64_t at = base + lane + 64 * j;
                v[j] = value_at<FMT>(x, at < a.vocab ? at : a.vocab - 1);
                v[j] = at < a.vocab ? v[j] : -__builtin_inff();
            }
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < PER; j++)
            top = fmaxf(top, v[j]);
        top = fmaxf(rows_max(row_max<16>(top)), most);
        const float shift = top == -__builtin_inff() ? 0.0f : top;
        float add = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; j++)
            add += __builtin_amdgcn_exp2f((v[j] - shift) * LOG2E);
        sum = sum * (most == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((most - top) * LOG2E)) + add;
        most = top;
        uint32_t order[PER];
#pragma unroll
        for (int j = 0; j < PER; j++)
            order[j] = order_of(v[j]);
        merge_tile<PER>(order, [&](int j) { return static_cast<Key>(order[j]) << 32 | (0xffffffffu - token(j)); }, k,
                        s_kept[wave], list);
    }
    sum = rows_sum(row_sum<16>(sum));
    if (lane == 0)
        part[unit] = {most, sum};
    if (lane < k)
        keys[unit * k + lane] = list[lane];
}

// One workgroup a sequence: each wave joins rows' parts, then all candidates of the rows are
// ranked by score.
__global__ __launch_bounds__(64 * MERGE_WAVES) void beam_merge_kernel(BeamArgs a, int parts, const Part* part, const Key* keys)
{
    constexpr int LANE_KEYS = 8;
    __shared__ Key s_kept[MERGE_WAVES][KEPT + CANDIDATES_MAX];
    __shared__ Key s_list[BEAMS_MAX][CANDIDATES_MAX];
    __shared__ double s_score[BEAMS_MAX * CANDIDATES_MAX];
    __shared__ int s_parent[CANDIDATES_MAX], s_slot[BEAMS_MAX], s_count;
    const int s = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int k = a.candidates, beams = a.beams;
    if (t == 0)
        s_count = 0;
    if (t < beams)
        s_slot[t] = a.slots ? a.slots[static_cast<int64_t>(s) * beams + t] : 0;
    for (int b = wave; b < beams; b += MERGE_WAVES) {
        const int64_t row = static_cast<int64_t>(s) * beams + b;
        const double given = a.scores[row];
        Key* const list = s_list[b];
        if (lane < CANDIDATES_MAX)
            list[lane] = 0;
        wave_sync();
        if (a.done && a.done[row] != 0) {
            if (lane < k)
                s_score[b * k + lane] = lane == 0 ? given : -__builtin_inf();
            if (lane == 0)
                list[0] = 0xffffffffu - static_cast<uint32_t>(a.end_token);
            continue;
        }
        const Part* const mine = part + row * parts;
        float most = -__builtin_inff();
        for (int i = lane; i < parts; i += 64)
            most = fmaxf(most, mine[i].most);
        most = rows_max(row_max<16>(most));
        double sum = 0.0;
        for (int i = lane; i < parts; i += 64) {
            const Part q = mine[i];
            // (a part without a finite logit has the sum 0, or NaN)
            sum += q.most == -__builtin_inff() ? static_cast<double>(q.sum)
                                               : static_cast<double>(q.sum) * exp(static_cast<double>(q.most) - static_cast<double>(most));
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1)
            sum += __shfl_xor(sum, m);
        const double log_sum = log(sum);
        const Key* const from = keys + row * parts * k;
        const int64_t total = static_cast<int64_t>(parts) * k;
        for (int64_t base = 0; base < total; base += 64 * LANE_KEYS) {
            Key key[LANE_KEYS];
            uint32_t order[LANE_KEYS];
#pragma unroll
            for (int j = 0; j < LANE_KEYS; j++) {
                const int64_t at = base + 64 * j + lane;
                key[j] = at < total ? from[at] : 0;
                order[j] = static_cast<uint32_t>(key[j] >> 32);
            }
            merge_tile<LANE_KEYS>(order, [&](int j) { return key[j]; }, k, s_kept[wave], list);
        }
        if (lane < k) {
            const Key key = list[lane];
            const double x = static_cast<double>(logit_of(static_cast<uint32_t>(key >> 32)));
            const double score = given + ((x - static_cast<double>(most)) - log_sum);
            s_score[b * k + lane] = key != 0 && fabs(score) < __builtin_inf() ? score : -__builtin_inf();
        }
    }
    __syncthreads();
    const int64_t out = static_cast<int64_t>(s) * k;
    const int i = t;   // at most 16 * 32 candidates
    if (i < beams * k) {
        const double mine = s_score[i];
        if (fabs(mine) < __builtin_inf()) {
            int rank = 0;
            for (int j = 0; j < beams * k; j++) {
                const double other = s_score[j];
                rank += other > mine || (other == mine && j < i);
            }
            atomicAdd(&s_count, 1);
            if (rank < k) {
                const int b = i / k;
                const int token = static_cast<int>(0xffffffffu - static_cast<uint32_t>(s_list[b][i - b * k]));
                a.parents[out + rank] = b;
                a.tokens[out + rank] = token;
                a.new_scores[out + rank] = static_cast<float>(mine);
                if (a.new_done)
                    a.new_done[out + rank] = token == a.end_token;
                s_parent[rank] = b;
            }
        }
    }
    __syncthreads();
    const int count = min(s_count, k);
    if (t >= count && t < k) {
        a.parents[out + t] = -1;
        a.tokens[out + t] = -1;
        a.new_scores[out + t] = -__builtin_inff();
        if (a.new_done)
            a.new_done[out + t] = 0;
        s_parent[t] = -1;
    }
    if (!a.slots)
        return;
    __syncthreads();
    if (t < beams) {   // candidates = beams
        const int parent = s_parent[t];
        auto keeps = [&](int c) {
            const int p = s_parent[c];
            bool first = p >= 0;
            for (int d = 0; d < c; d++)
                first = first && s_parent[d] != p;
            return first;
        };
        int slot = parent >= 0 ? s_slot[parent] : -1;
        a.from[out + t] = slot;
        if (!keeps(t)) {
            int turn = 0;   // candidates before this one that take over a slot
            for (int c = 0; c < t; c++)
                turn += !keeps(c);
            for (int b = 0; b < beams; b++) {
                bool childless = true;
                for (int c = 0; c < beams; c++)
                    childless = childless && s_parent[c] != b;
                if (childless && turn-- == 0)
                    slot = s_slot[b];
            }
        }
        a.to[out + t] = slot;
    }
}

struct SlotArrays {
    si_hip_slot_array at[SLOT_ARRAYS_PER_LAUNCH];
};

constexpr int COPY_THREADS = 256, COPY_BYTES = COPY_THREADS * 16 * 4;   // of a workgroup

// A workgroup copies 16 KiB of one slot of one array.  Bound by HBM.
__global__ __launch_bounds__(COPY_THREADS) void copy_slots_kernel(SlotArrays arrays, int64_t slots, const int32_t* from, const int32_t* to,
                                                                  int moves)
{
    const si_hip_slot_array a = arrays.at[blockIdx.z];
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * COPY_BYTES;
    if (first >= a.slot_bytes)
        return;
    const uint64_t last = min(first + COPY_BYTES, a.slot_bytes);
    for (int i = blockIdx.y; i < moves; i += gridDim.y) {
        const int64_t source = from[i], target = to[i];
        if (source < 0 || target < 0 || source >= slots || target >= slots || source == target)
            continue;
        const char* const src = static_cast<char*>(a.base) + source * a.slot_bytes;
        char* const dst = static_cast<char*>(a.base) + target * a.slot_bytes;
        if (last - first == COPY_BYTES) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                __builtin_memcpy(&v[j], src + first + (threadIdx.x + COPY_THREADS * j) * 16, 16);
#pragma unroll
            for (int j = 0; j < 4; j++)
                __builtin_memcpy(dst + first + (threadIdx.x + COPY_THREADS * j) * 16, &v[j], 16);
        } else {
            const uint64_t whole = first + (last - first) / 16 * 16;
            for (uint64_t at = first + threadIdx.x * 16; at < whole; at += COPY_THREADS * 16) {
                uint4 v;
                __builtin_memcpy(&v, src + at, 16);
                __builtin_memcpy(dst + at, &v, 16);
            }
            if (whole + threadIdx.x < last)
                dst[whole + threadIdx.x] = src[whole + threadIdx.x];
        }
    }
}

int64_t parts_bytes(int64_t units) { return (units * static_cast<int64_t>(sizeof(Part)) + 15) / 16 * 16; }

}  // namespace

int64_t beam_workspace_bytes(int sequences, int beams, int candidates, int vocab)
{
    const int rows = sequences * beams;
    const int64_t units = static_cast<int64_t>(rows) * cut_of(rows, vocab).parts;
    return parts_bytes(units) + units * candidates * static_cast<int64_t>(sizeof(Key));
}

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t s)
{
    const int rows = a.sequences * a.beams;
    const Cut cut = cut_of(rows, a.vocab);
    const int64_t units = static_cast<int64_t>(rows) * cut.parts;
    Part* const part = static_cast<Part*>(a.workspace);
    Key* const keys = reinterpret_cast<Key*>(static_cast<char*>(a.workspace) + parts_bytes(units));
    const dim3 grid(static_cast<unsigned>((units + SCAN_WAVES - 1) / SCAN_WAVES)), block(64 * SCAN_WAVES);
    if (a.format == ROWS_OUT_F32)
        hipLaunchKernelGGL(beam_scan_kernel<ROWS_OUT_F32>, grid, block, 0, s, a, rows, cut.tiles, cut.parts, part, keys);
    else if (a.format == ROWS_OUT_F16)
        hipLaunchKernelGGL(beam_scan_kernel<ROWS_OUT_F16>, grid, block, 0, s, a, rows, cut.tiles, cut.parts, part, keys);
    else
        hipLaunchKernelGGL(beam_scan_kernel<ROWS_OUT_BF16>, grid, block, 0, s, a, rows, cut.tiles, cut.parts, part, keys);
    hipLaunchKernelGGL(beam_merge_kernel, dim3(a.sequences), dim3(64 * MERGE_WAVES), 0, s, a, cut.parts, part, keys);
    return hipGetLastError();
}

hipError_t launch_copy_slots(const si_hip_slot_array* arrays, int count, int64_t slots, const int32_t* from, const int32_t* to,
                             int moves, hipStream_t s)
{
    for (int first = 0; first < count; first += SLOT_ARRAYS_PER_LAUNCH) {
        const int n = count - first < SLOT_ARRAYS_PER_LAUNCH ? count - first : SLOT_ARRAYS_PER_LAUNCH;
        SlotArrays some{};
        uint64_t most = 0;
        for (int i = 0; i < n; i++) {
            some.at[i] = arrays[first + i];
            most = most > some.at[i].slot_bytes ? most : some.at[i].slot_bytes;
        }
        const dim3 grid(static_cast<unsigned>((most + COPY_BYTES - 1) / COPY_BYTES), moves < 65535 ? moves : 65535, n);
        hipLaunchKernelGGL(copy_slots_kernel, grid, dim3(COPY_THREADS), 0, s, some, slots, from, to, moves);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
            return e;
    }
    return hipSuccess;
}

}  // namespace si
