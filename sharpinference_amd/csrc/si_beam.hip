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
constexpr int KEPT = 256;                     // values that are ranked together
constexpr int ROOM = KEPT + CANDIDATES_MAX + 8;
constexpr int HALVES = 5;                     // of the way from a bound to the largest value
constexpr int LARGEST = 24;                   // a lane's 16-byte words of a group of tiles, whose largest values are held
constexpr int SCAN_WAVES = 4, MERGE_WAVES = BEAMS_MAX;
constexpr float INF = __builtin_inff(), LOWEST = -3.402823466e38f;   // of the finite values

typedef uint32_t Sixteen __attribute__((ext_vector_type(4), aligned(1)));   // bytes at any address, in one load or store

typedef unsigned long long Key;   // order of a logit (high word: 0 for none) and of its token, lowest last
typedef Key KeyPair __attribute__((ext_vector_type(2)));

// Order of a logit: larger for larger values, 0 for -infinity and NaN; -0 as 0.
__device__ __forceinline__ uint32_t order_of(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    return v > -INF ? u ^ (static_cast<int32_t>(u) < 0 ? 0xffffffffu : 0x80000000u) : 0u;
}
__device__ __forceinline__ float logit_of(uint32_t order)
{
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

// The smallest over groups of lanes of the groups' largest values: with k groups or more, so many values lie at or over it.
__device__ __forceinline__ float group_bound(float best, int k)
{
    best = fmaxf(best, dpp_row<0xB1>(best));
    if (k <= 16) best = fmaxf(best, dpp_row<0x4E>(best));
    if (k <= 8) best = fmaxf(best, dpp_row<0x141>(best));
    if (k <= 4) best = fmaxf(best, dpp_row<0x140>(best));
    return -rows_max(row_max<16>(-best));
}

// A value that k lanes' largest ones or more reach, near the k-th of them: the groups' bound, raised by halves of what lies
// between it and the largest.  The groups' alone lets k H_k values through (54 of 2048 spread ones for k = 16), this one few more
// than k: 8 sequences of 16 beams over 151936 values 29 us where that one takes 62, 2 of 9 beams and 18 candidates 14 and 40.
__device__ __forceinline__ float near_kth(float best, int k)
{
    float low = group_bound(best, k), high = rows_max(row_max<16>(best));
    if (low == -INF && __popcll(__ballot(best > -INF)) >= k)   // (a group without a value, but lanes enough)
        low = -rows_max(row_max<16>(best > -INF ? -best : -INF));
#pragma unroll
    for (int i = 0; i < HALVES; i++) {
        const float middle = 0.5f * low + 0.5f * high;
        const bool reached = __popcll(__ballot(best >= middle)) >= k;
        low = reached ? middle : low;
        high = reached ? high : middle;
    }
    return low;
}

// Puts `count` kept keys and the list's own (k of them, sorted, 0 for none) in order: a key's place is the number of larger ones.
__device__ __forceinline__ void rank_kept(int count, int k, Key* kept, Key* list)
{
    const int lane = threadIdx.x & 63;
    const Key own = lane < k ? list[lane] : 0;
    if (own != 0)
        kept[count + lane] = own;
    count += __popcll(__ballot(own != 0));   // (a prefix of the lanes)
    if (lane < 8)
        kept[count + lane] = 0;
    wave_sync();
    for (int i = lane; i < count; i += 64) {
        const Key mine = kept[i];
        int rank = 0;
        for (int j = 0; j < count; j += 8) {   // eight at a time: a chain of LDS reads else
            KeyPair other[4];
#pragma unroll
            for (int m = 0; m < 4; m++)
                other[m] = *reinterpret_cast<const KeyPair*>(kept + j + 2 * m);
#pragma unroll
            for (int m = 0; m < 4; m++)
                rank += (other[m][0] > mine) + (other[m][1] > mine);
        }
        if (rank < k)
            list[rank] = mine;
    }
    wave_sync();
}

// The smallest value that may enter a sorted list of k.
__device__ __forceinline__ float least_of(const Key* list, int k)
{
    const uint32_t last = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(list[k - 1] >> 32));
    return last == 0 ? -INF : logit_of(last);
}

// Appends what `in` marks behind the `count` kept ones (as many as there is room for); returns how many there would be.
template <typename F>
__device__ __forceinline__ int append(bool in, F key, int count, Key* kept)
{
    const uint64_t mask = __ballot(in);
    if (mask == 0)
        return count;
    const int at = count + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
    if (in && at < KEPT)
        kept[at] = key();
    return count + __popcll(mask);
}

// Merges a tile's values (PERL a lane) into the sorted list of the best k so far, a few a lane at a time.  Only values over
// the groups' bound, and over the list's last, can be among the best k.  (One equal to the last may have a lower token
// where it is of the same tile.)
template <int PERL, typename F>
__device__ __forceinline__ void merge_tile(const float (&v)[PERL], float bound, F key_of, int k, Key* kept, Key* list)
{
    constexpr int STEP = KEPT / 64;
    float over = least_of(list, k);
#pragma unroll
    for (int j = 0; j < PERL; j += STEP) {
        int count = 0;
#pragma unroll
        for (int i = j; i < j + STEP; i++)
            count = append(v[i] >= bound && v[i] >= over && v[i] > -INF, [&] { return key_of(i); }, count, kept);
        if (count > 0) {
            rank_kept(count, k, kept, list);
            over = least_of(list, k);
        }
    }
}

// Sum over the wave, in every lane, with moves inside rows of lanes and swaps between them.
template <int CTRL>
__device__ __forceinline__ double moved(double v)
{
    return __hiloint2double(dpp_row<CTRL>(__double2hiint(v)), dpp_row<CTRL>(__double2loint(v)));
}
__device__ __forceinline__ double wave_sum(double v)
{
    v += moved<0xB1>(v);
    v += moved<0x4E>(v);
    v += moved<0x141>(v);
    v += moved<0x140>(v);
    auto swapped = [&](auto swap) {
        const auto high = swap(static_cast<uint32_t>(__double2hiint(v))), low = swap(static_cast<uint32_t>(__double2loint(v)));
        v = __hiloint2double(static_cast<int>(high[0]), static_cast<int>(low[0])) +
            __hiloint2double(static_cast<int>(high[1]), static_cast<int>(low[1]));
    };
    swapped([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
    swapped([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
    return v;
}

// How a row is cut: tiles a part, parts a row.  A wave takes a part; where there are
// more tiles than the card holds waves of this kernel, it takes several one after another (192 rows of 98 tiles, with the merge:
// five a wave 23.1 us, ten 23.3, three 24.0, one 30).  Larger parts for fewer keys to merge pay a little in some shapes and cost more in others
// (a sequence of 16 beams and 32 candidates: 98 parts 28 to 31 us, 49 26, 25 43).
struct Cut {
    int tiles, parts;
};
Cut cut_of(int rows, int vocab)
{
    constexpr int WAVES = 4096;
    const int all = (vocab + TILE - 1) / TILE;
    const int64_t waves = static_cast<int64_t>(rows) * all;
    const int tiles = static_cast<int>(waves <= WAVES ? 1 : (waves + WAVES - 1) / WAVES);
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

// One wave a part of a row.  Over a group of tiles it takes the sum and each 16-byte word's largest value; then it reads the
// words again that may hold one of the best (few more than those), and ranks those values together: ranked tile by tile
// out of registers, that part took as long as the rest.  Bound by HBM, then by the tail of ranking and launch: 24 sequences of 8 beams over
// 200064 16-bit logits, 65 MB of them read, 18.2 us, 3.6 TB/s (tile by tile 28).  One sequence of 4 beams over
// 65536 FP32 logits: 5.1 us, the launch and one chain of round trips.
template <int FMT>
__global__ __launch_bounds__(64 * SCAN_WAVES, 4) void beam_scan_kernel(BeamArgs a, int rows, int tiles, int parts, Part* part, Key* keys)
{
    alignas(16) __shared__ Key s_kept[SCAN_WAVES][ROOM];
    __shared__ Key s_list[SCAN_WAVES][CANDIDATES_MAX];
    __shared__ float4 s_largest[SCAN_WAVES][LARGEST / 4][64];
    constexpr int SIZE = FMT == ROWS_OUT_F32 ? 4 : 2, VEC = 16 / SIZE, LOADS = PER / VEC, GROUP = LARGEST / LOADS;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * SCAN_WAVES + wave;
    if (unit >= static_cast<int64_t>(rows) * parts)
        return;
    const int row = static_cast<int>(unit / parts), p = static_cast<int>(unit - static_cast<int64_t>(row) * parts);
    const int first = p * tiles * TILE, last = min(first + tiles * TILE, a.vocab);
    const char* const x = static_cast<const char*>(a.logits) + row * a.stride * SIZE;
    // Word `at` of the row (tokens at and the following), or, behind the row's last whole word, that one: what lies before `at` in it
    // does not count.  A row of less than a word is put together value by value.
    const int last_word = a.vocab - VEC;
    auto word = [&](int at) {
        if (last_word >= 0)
            return *reinterpret_cast<const Sixteen*>(x + static_cast<int64_t>(min(at, last_word)) * SIZE);
        Sixteen got = {0, 0, 0, 0};
        for (int j = 0; j < a.vocab; j++) {
            const uint32_t bits = SIZE == 4 ? reinterpret_cast<const uint32_t*>(x)[j] : reinterpret_cast<const uint16_t*>(x)[j];
            const int to = VEC - a.vocab + j;   // the row ends where the word does
            got[to * SIZE / 4] |= bits << (SIZE == 4 ? 0 : to % 2 * 16);
        }
        return got;
    };
    Sixteen raw[LOADS];
    auto request = [&](int base) {
#pragma unroll
        for (int j = 0; j < LOADS; j++)
            raw[j] = word(base + VEC * (lane + 64 * j));
    };
    request(first);
    if (a.done && a.done[row] != 0)
        return;   // its logits do not count
    const int k = a.candidates;
    Key* const list = s_list[wave];
    if (lane < CANDIDATES_MAX)
        list[lane] = 0;
    wave_sync();
    Key* const kept = s_kept[wave];
    float4(*const largest)[64] = s_largest[wave];
    uint16_t* const found = reinterpret_cast<uint16_t*>(largest);   // (after `largest` is used)
    float most = -INF, sum = 0.0f;
    Key least = 0;   // the list's last
    for (int group = first; group < last; group += GROUP * TILE) {
        const int end = min(group + GROUP * TILE, last);
        float lane_best = -INF;
        int count = 0;   // of tiles
        for (int base = group; base < end; base += TILE, count++) {
            float v[PER];
#pragma unroll
            for (int j = 0; j < PER; j++)
                v[j] = value_at<FMT>(&raw[j / VEC], j % VEC);
            if (base + TILE < last)
                request(base + TILE);
            if (base + TILE > a.vocab) {
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    const int at = base + VEC * (lane + 64 * (j / VEC));
                    v[j] = min(at, last_word) + j % VEC >= at ? v[j] : -INF;
                }
            }
            float best[LOADS];
#pragma unroll
            for (int j = 0; j < LOADS; j++) {
                best[j] = v[j * VEC];
#pragma unroll
                for (int i = 1; i < VEC; i++)
                    best[j] = fmaxf(best[j], v[j * VEC + i]);
                best[j] = fmaxf(best[j], -INF);   // (a word of NaN)
            }
            float tile_best = best[0];
#pragma unroll
            for (int j = 0; j < LOADS; j += 4)
                largest[count * (LOADS / 4) + j / 4][lane] = make_float4(best[j], best[j + 1], best[j + 2], best[j + 3]);
#pragma unroll
            for (int j = 1; j < LOADS; j++)
                tile_best = fmaxf(tile_best, best[j]);
            lane_best = fmaxf(lane_best, tile_best);
            const float top = fmaxf(rows_max(row_max<16>(tile_best)), most);
            const float shift = top == -INF ? 0.0f : top;
            float add = 0.0f, more = 0.0f;
#pragma unroll
            for (int j = 0; j < PER; j += 2) {
                add += __builtin_amdgcn_exp2f((v[j] - shift) * LOG2E);
                more += __builtin_amdgcn_exp2f((v[j + 1] - shift) * LOG2E);
            }
            sum = sum * (most == -INF ? 0.0f : __builtin_amdgcn_exp2f((most - top) * LOG2E)) + (add + more);
            most = top;
        }
        // The words that hold a value over the list's last so far (one equal to it has a higher token: groups come in order)
        // and over the groups' bound.
        const float over = least_of(list, k);
        if (__ballot(lane_best > over) == 0)
            continue;
        const float bound = fmaxf(fmaxf(near_kth(lane_best, k), over), LOWEST);
        uint32_t mine = 0;
        for (int i = 0; i < count * (LOADS / 4); i++) {
            const float4 m = largest[i][lane];
            mine |= ((m.x >= bound ? 1u : 0u) | (m.y >= bound ? 2u : 0u) | (m.z >= bound ? 4u : 0u) | (m.w >= bound ? 8u : 0u)) << 4 * i;
        }
        wave_sync();
        int at = 0, words = 0;   // found in lanes before, and in all
        const int own = __popc(mine);
#pragma unroll
        for (int bit = 0; bit < 5; bit++) {   // (at most LARGEST)
            const uint64_t lanes = __ballot(own >> bit & 1);
            at += __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(lanes >> 32),
                                            __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(lanes), 0)) << bit;
            words += __popcll(lanes) << bit;
        }
        while (mine != 0) {
            found[at++] = static_cast<uint16_t>(__builtin_ctz(mine) << 6 | lane);
            mine &= mine - 1;
        }
        wave_sync();
        int held = 0;
        auto key_of = [&](float v, int token) { return static_cast<Key>(order_of(v)) << 32 | (0xffffffffu - static_cast<uint32_t>(token)); };
        for (int base = 0; base < words; base += 64) {
            const int which = found[min(base + lane, words - 1)], i = which >> 6;
            const int from = group + i / LOADS * TILE + VEC * ((which & 63) + 64 * (i % LOADS)), start = min(from, last_word);
            const Sixteen got = word(from);
            const bool in = base + lane < words;
            int more = held;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float v = value_at<FMT>(&got, j);
                more = append(in && v >= bound && start + j >= from, [&] { return key_of(v, start + j); }, more, kept);
            }
            if (more <= KEPT) {
                held = more;
                continue;
            }
            // more than there is room for: what was kept before these words is in place, these go a value a lane at a time
            for (int j = 0; j < VEC; j++) {
                if (held > KEPT - 64) {
                    rank_kept(held, k, kept, list);
                    held = 0;
                    least = list[k - 1];
                }
                const float v = value_at<FMT>(x, max(start + j, 0));
                const Key key = key_of(v, start + j);
                held = append(in && v >= bound && start + j >= from && key > least, [&] { return key; }, held, kept);
            }
        }
        if (held > 0)
            rank_kept(held, k, kept, list);
        least = list[k - 1];
    }
    sum = rows_sum(row_sum<16>(sum));
    if (lane == 0)
        part[unit] = {most, sum};
    if (lane < k)
        keys[unit * k + lane] = list[lane];
}

// One workgroup a sequence.  Wave b merges the lists of row b's parts, wave 15 - b sums the row; then all candidates
// of the rows are ranked by score.  A chain of round trips, bound by their latency, with many beams by the 16 waves' instructions
// on one compute unit: what does not hang on another load is requested first, and only keys and candidates that near_kth lets through
// are ranked (24 sequences of 8 beams 6.0 us, one of 4 beams 4.5, 3 of 16 beams over one part a row 6.5; 16 beams' 98 parts of 32
// candidates 22).
__global__ __launch_bounds__(64 * MERGE_WAVES) void beam_merge_kernel(BeamArgs a, int parts, const Part* part, const Key* keys)
{
    constexpr int LANE_KEYS = 8;
    alignas(16) __shared__ Key s_kept[MERGE_WAVES][ROOM];
    __shared__ Key s_list[BEAMS_MAX][CANDIDATES_MAX];
    __shared__ double s_log[BEAMS_MAX], s_score[BEAMS_MAX * CANDIDATES_MAX], s_top_score[BEAMS_MAX * CANDIDATES_MAX];
    __shared__ float s_most[BEAMS_MAX];
    __shared__ int s_top[BEAMS_MAX * CANDIDATES_MAX], s_parent[CANDIDATES_MAX], s_slot[BEAMS_MAX], s_child[BEAMS_MAX], s_free[BEAMS_MAX];
    const int s = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int k = a.candidates, beams = a.beams, all = beams * k;
    const int64_t first_row = static_cast<int64_t>(s) * beams;
    // thread t's candidate: t - b k of beam b
    const int beam = t < all ? t / k : 0;
    const double given = a.scores[first_row + beam];
    const bool ended = a.done && a.done[first_row + beam] != 0;
    const int slot = a.slots && t < beams ? a.slots[first_row + t] : 0;
    // a beam's keys, requested; the sum of another's row; the keys' list
    auto ended_at = [&](int b) { return a.done && a.done[first_row + b] != 0; };
    const int own = wave < beams ? wave : 0, total = parts * k;
    const Key* const from = keys + (first_row + own) * total;
    const bool own_ended = ended_at(own);
    Key key[LANE_KEYS];
    auto request = [&](int base) {
#pragma unroll
        for (int j = 0; j < LANE_KEYS; j++)
            key[j] = from[min(base + 64 * j + lane, total - 1)];
    };
    if (wave < beams)
        request(0);
    const int summed = MERGE_WAVES - 1 - wave;
    if (summed < beams && !ended_at(summed)) {
        const Part* const mine = part + (first_row + summed) * parts;
        Part held = mine[min(lane, parts - 1)];
        if (lane >= parts)
            held = {-INF, 0.0f};
        float most = held.most;
        for (int i = lane + 64; i < parts; i += 64)
            most = fmaxf(most, mine[i].most);
        most = rows_max(row_max<16>(most));
        // (a part without a finite logit has the sum 0, or NaN)
        auto scaled = [&](Part q) {
            return static_cast<double>(q.sum) * (q.most == -INF ? 1.0f : __builtin_amdgcn_exp2f((q.most - most) * LOG2E));
        };
        double sum = scaled(held);
        for (int i = lane + 64; i < parts; i += 64)
            sum += scaled(mine[i]);
        const double log_sum = log(wave_sum(sum));
        if (lane == 0) {
            s_most[summed] = most;
            s_log[summed] = log_sum;
        }
    }
    if (wave < beams) {
        Key* const list = s_list[wave];
        if (lane < CANDIDATES_MAX)
            list[lane] = own_ended && lane == 0 ? 0xffffffffu - static_cast<uint32_t>(a.end_token) : 0;
        wave_sync();
        // In several turns: a value that k parts' largest ones reach, with which few keys are left.
        float reached = -INF, over = -INF;
        if (total > 64 * LANE_KEYS && !own_ended) {
            float top = -INF;
            for (int i = lane; i < parts; i += 64)
                top = fmaxf(top, part[(first_row + own) * parts + i].most);
            reached = near_kth(top, k);
        }
        int held = 0;   // kept ones that are not in the list yet
        const bool joined = own_ended || parts == 1;   // (one part's list is the row's)
        if (!own_ended && parts == 1 && lane < k)
            list[lane] = key[0];
        for (int base = 0; base < total && !joined; base += 64 * LANE_KEYS) {
            if (base > 0)
                request(base);
            float v[LANE_KEYS], best = -INF;
#pragma unroll
            for (int j = 0; j < LANE_KEYS; j++) {
                const uint32_t order = base + 64 * j + lane < total ? static_cast<uint32_t>(key[j] >> 32) : 0u;
                v[j] = order == 0 ? -INF : logit_of(order);
                best = fmaxf(best, v[j]);
            }
            const float bound = fmaxf(reached == -INF ? near_kth(best, k) : reached, over);
            int count = held;
#pragma unroll
            for (int j = 0; j < LANE_KEYS; j++)
                if (base + 64 * j < total)
                    count = append(v[j] >= bound && v[j] > -INF, [&] { return key[j]; }, count, s_kept[wave]);
            if (count <= KEPT) {
                held = count;
                continue;
            }
            rank_kept(held, k, s_kept[wave], list);
            merge_tile<LANE_KEYS>(v, bound, [&](int j) { return key[j]; }, k, s_kept[wave], list);
            over = least_of(list, k);
            held = 0;
        }
        if (held > 0)
            rank_kept(held, k, s_kept[wave], list);
    }
    __syncthreads();
    const Key got = t < all ? s_list[beam][t - beam * k] : 0;
    const double x = static_cast<double>(logit_of(static_cast<uint32_t>(got >> 32)));
    double score = given + ((x - static_cast<double>(s_most[beam])) - s_log[beam]);
    if (ended)
        score = t == beam * k ? given : -__builtin_inf();
    if (t < all)
        s_score[t] = got != 0 && fabs(score) < __builtin_inf() ? score : -__builtin_inf();
    __syncthreads();
    if (wave > 0)
        return;
    if (t < beams) {
        s_slot[t] = slot;
        s_child[t] = BEAMS_MAX;   // a beam's first candidate
    }
    // The candidates among which the best k are (their scores rounded to FP32: the order stays), put in order by the number of
    // larger ones (of equal ones the first).
    constexpr int PERL = BEAMS_MAX * CANDIDATES_MAX / 64;
    float v[PERL], best = -INF;
#pragma unroll
    for (int j = 0; j < PERL; j++) {
        v[j] = 64 * j < all && lane + 64 * j < all ? static_cast<float>(s_score[lane + 64 * j]) : -INF;
        best = fmaxf(best, v[j]);
    }
    const float bound = all <= 32 ? -INF : near_kth(best, k);   // (so few are ranked as soon as a bound is found)
    int count = 0;
#pragma unroll
    for (int j = 0; j < PERL; j++) {
        if (64 * j >= all)
            break;
        const bool in = v[j] >= bound && v[j] > -INF;
        const uint64_t lanes = __ballot(in);
        if (in) {
            const int at = count + __popcll(lanes & ((1ull << lane) - 1));
            s_top[at] = lane + 64 * j;
            s_top_score[at] = s_score[lane + 64 * j];
        }
        count += __popcll(lanes);
    }
    wave_sync();
    const int64_t out = static_cast<int64_t>(s) * k;
    const float per_beam = 1.0f / static_cast<float>(k);
    for (int i = lane; i < count; i += 64) {
        const int c = s_top[i];
        const double mine = s_top_score[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; j++) {   // (of equal ones the lower candidate first: they lie in their order)
            const double other = s_top_score[j];
            rank += other > mine || (other == mine && j < i);
        }
        if (rank < k) {
            const int parent = static_cast<int>((static_cast<float>(c) + 0.5f) * per_beam);   // c / k: exact for so few
            const int token = static_cast<int>(0xffffffffu - static_cast<uint32_t>(s_list[parent][c - parent * k]));
            a.parents[out + rank] = parent;
            a.tokens[out + rank] = token;
            a.new_scores[out + rank] = static_cast<float>(mine);
            if (a.new_done)
                a.new_done[out + rank] = token == a.end_token;
            s_parent[rank] = parent;
        }
    }
    if (t >= count && t < k) {
        a.parents[out + t] = -1;
        a.tokens[out + t] = -1;
        a.new_scores[out + t] = -INF;
        if (a.new_done)
            a.new_done[out + t] = 0;
        s_parent[t] = -1;
    }
    if (!a.slots)
        return;
    // candidates = beams, one a lane: a parent's first child keeps its slot, the others take those of beams without children in turn
    wave_sync();
    const int parent = t < beams ? s_parent[t] : -1;
    if (parent >= 0)
        atomicMin(&s_child[parent], t);
    wave_sync();
    const uint64_t keepers = __ballot(parent >= 0 && s_child[max(parent, 0)] == t);
    const uint64_t childless = __ballot(t < beams && s_child[min(t, BEAMS_MAX - 1)] == BEAMS_MAX);
    const uint64_t before = (1ull << t) - 1;
    if (childless >> t & 1)
        s_free[__popcll(childless & before)] = slot;
    wave_sync();
    if (t < beams) {
        const int source = parent >= 0 ? s_slot[parent] : -1;
        const bool keeps = keepers >> t & 1;
        a.from[out + t] = source;
        a.to[out + t] = keeps ? source : s_free[__popcll(~keepers & before)];
    }
}

struct SlotArrays {
    si_hip_slot_array at[SLOT_ARRAYS_PER_LAUNCH];
};

constexpr int COPY_THREADS = 256, COPY_BYTES = COPY_THREADS * 16 * 2;   // of a workgroup

// A workgroup copies 8 KiB of one slot of one array, past the L2s (24 arrays, 12 slots of 540 KB each moved: 43 us;
// through them 47; 4 or 16 KiB a workgroup 56 and 45; a plain copy of the bytes 65).  Bound by HBM, small moves
// by the launch.
__global__ __launch_bounds__(COPY_THREADS) void copy_slots_kernel(SlotArrays arrays, int64_t slots, const int32_t* from, const int32_t* to,
                                                                  int moves, int lanes)
{
    const int t = threadIdx.x & (lanes - 1), turn = blockIdx.y * (COPY_THREADS / lanes) + threadIdx.x / lanes;
    const si_hip_slot_array a = arrays.at[blockIdx.z];
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * COPY_BYTES;
    if (first >= a.slot_bytes)
        return;
    const uint64_t last = min(first + COPY_BYTES, a.slot_bytes);
    for (int i = turn; i < moves; i += gridDim.y * (COPY_THREADS / lanes)) {
        const int64_t source = from[i], target = to[i];
        if (source < 0 || target < 0 || source >= slots || target >= slots || source == target)
            continue;
        const char* const src = static_cast<char*>(a.base) + source * a.slot_bytes;
        char* const dst = static_cast<char*>(a.base) + target * a.slot_bytes;
        if (last - first == COPY_BYTES) {   // (of such slots a workgroup takes one)
            Sixteen v[2];
#pragma unroll
            for (int j = 0; j < 2; j++)
                v[j] = *reinterpret_cast<const Sixteen*>(src + first + (threadIdx.x + COPY_THREADS * j) * 16);
#pragma unroll
            for (int j = 0; j < 2; j++)
                __builtin_nontemporal_store(v[j], reinterpret_cast<Sixteen*>(dst + first + (threadIdx.x + COPY_THREADS * j) * 16));
        } else {
            const uint64_t whole = first + (last - first) / 16 * 16;
            for (uint64_t at = first + t * 16; at < whole; at += lanes * 16)
                *reinterpret_cast<Sixteen*>(dst + at) = *reinterpret_cast<const Sixteen*>(src + at);
            if (whole + t < last)
                dst[whole + t] = src[whole + t];
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
        // Small slots several a workgroup (500 moves in 64 arrays of 364 bytes 6.3 us, one a workgroup 22).
        const int lanes = most <= 1024 ? 16 : most <= 4096 ? 64 : COPY_THREADS, turns = (moves + COPY_THREADS / lanes - 1) / (COPY_THREADS / lanes);
        const dim3 grid(static_cast<unsigned>((most + COPY_BYTES - 1) / COPY_BYTES), turns < 65535 ? turns : 65535, n);
        hipLaunchKernelGGL(copy_slots_kernel, grid, dim3(COPY_THREADS), 0, s, some, slots, from, to, moves, lanes);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
            return e;
    }
    return hipSuccess;
}

}  // namespace si
