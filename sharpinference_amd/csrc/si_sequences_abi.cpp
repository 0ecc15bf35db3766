// C ABI of a recurrent model's step over many sequences and of the beam search
// (si_mix_rows.hip, si_wkv_rows.hip, si_beam.hip): argument checks, then the launches on the
// context stream.
#include "si_context.hpp"
#include "si_internal.hpp"
#include "si_sequences.hpp"

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

using namespace si_abi;

namespace {

constexpr int MAX_ROWS = 1 << 20, MAX_HEADS = 1024, MAX_BEAM_ROWS = 65536, MAX_VOCAB = 1 << 21, MAX_ARRAYS = 4096;
constexpr uint64_t MAX_SLOT_BYTES = 1ull << 36;

int check_ptr(si_hip_context* ctx, const char* op, const void* p, const char* name, uintptr_t align)
{
    if (!p || !aligned(p, align))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %s must be a non-null %u-byte aligned device pointer", op, name,
                    static_cast<unsigned>(align));
    return SI_HIP_OK;
}

struct Span {
    const void* p;
    uint64_t n;
};

// The memory that a call reads or writes: a list on the stack, long enough for every call here.
struct Spans {
    Span at[24];
    int count = 0;
    void add(const void* p, uint64_t n) { at[count++] = {p, n}; }
};

int check_apart(si_hip_context* ctx, const char* op, const Spans& writes, const Spans& reads)
{
    for (int i = 0; i < writes.count; i++) {
        for (int j = 0; j < reads.count; j++)
            if (overlaps(writes.at[i].p, writes.at[i].n, reads.at[j].p, reads.at[j].n))
                return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: an output overlaps an input", op);
        for (int j = i + 1; j < writes.count; j++)
            if (overlaps(writes.at[i].p, writes.at[i].n, writes.at[j].p, writes.at[j].n))
                return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: outputs overlap", op);
    }
    return SI_HIP_OK;
}

int check_batch(si_hip_context* ctx, const char* op, const si_hip_row_batch& b, Spans* reads)
{
    if (b.sequences < 1 || b.sequences > si::ROW_SEQUENCES_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d sequences outside 1..%d", op, b.sequences, si::ROW_SEQUENCES_MAX);
    if (b.slots < 1)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d slots", op, b.slots);
    if (b.rows < 1 || b.rows > MAX_ROWS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d rows outside 1..%d", op, b.rows, MAX_ROWS);
    if (b.max_rows < 1 || b.max_rows > b.rows)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d rows of a sequence outside 1..%d", op, b.max_rows, b.rows);
    if (check_ptr(ctx, op, b.row_starts, "row starts", 4) || check_ptr(ctx, op, b.from, "from", 4) ||
        check_ptr(ctx, op, b.to, "to", 4))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t bytes = static_cast<uint64_t>(b.sequences) * 4;
    reads->add(b.row_starts, bytes + 4);
    reads->add(b.from, bytes);
    reads->add(b.to, bytes);
    return SI_HIP_OK;
}

si::RowBatch batch_of(const si_hip_row_batch& b)
{
    return {b.row_starts, b.from, b.to, b.sequences, b.slots, b.rows, b.max_rows};
}

int check_format(si_hip_context* ctx, const char* op, const char* what, int fmt, int* out)
{
    if (fmt != SI_HIP_F32 && fmt != SI_HIP_F16 && fmt != SI_HIP_BF16)
        return fail(ctx, SI_HIP_ERR_UNSUPPORTED, "%s: %s of %s (%d) are not F32, F16 or BF16", op, what, fmt_name(fmt), fmt);
    *out = fmt == SI_HIP_F32 ? si::ROWS_OUT_F32 : fmt == SI_HIP_F16 ? si::ROWS_OUT_F16 : si::ROWS_OUT_BF16;
    return SI_HIP_OK;
}

uint64_t out_size(int out) { return out == si::ROWS_OUT_F32 ? 4 : 2; }

int launched(si_hip_context* ctx, hipError_t e, const char* op)
{
    return e == hipSuccess ? SI_HIP_OK : hip_fail(ctx, e, op);
}

int check_beams(si_hip_context* ctx, const char* op, int sequences, int beams, int candidates, int64_t vocab)
{
    if (beams < 1 || beams > si::BEAMS_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d beams outside 1..%d", op, beams, si::BEAMS_MAX);
    if (sequences < 1 || static_cast<int64_t>(sequences) * beams > MAX_BEAM_ROWS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d sequences of %d beams outside 1..%d rows", op, sequences, beams,
                    MAX_BEAM_ROWS);
    if (candidates < 1 || candidates > si::CANDIDATES_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d candidates outside 1..%d", op, candidates, si::CANDIDATES_MAX);
    if (vocab < 1 || vocab > MAX_VOCAB)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: vocabulary of %lld outside 1..%d", op, static_cast<long long>(vocab),
                    MAX_VOCAB);
    return SI_HIP_OK;
}

}  // namespace

extern "C" {

int si_hip_layernorm_mix_rows(si_hip_context* ctx, const si_hip_layernorm_mix_rows_args* args)
{
    const char* op = "layernorm_mix_rows";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (!args)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: null arguments", op);
    Spans reads, writes;
    if (const int rc = check_batch(ctx, op, args->batch, &reads))
        return rc;
    if (args->n < 1 || args->n > si::MIX_WIDTH_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: width %d outside 1..%d", op, args->n, si::MIX_WIDTH_MAX);
    if (args->mixes < 0 || args->mixes > si::MIX_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d mixes outside 0..%d", op, args->mixes, si::MIX_MAX);
    if (!std::isfinite(args->eps) || args->eps < 0.0f)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: eps must be finite and not negative", op);
    int out = 0;
    if (const int rc = check_format(ctx, op, "outputs", args->output_format, &out))
        return rc;
    if (check_ptr(ctx, op, args->x, "x", 4) || check_ptr(ctx, op, args->weight, "weight", 4) ||
        check_ptr(ctx, op, args->bias, "bias", 4) || check_ptr(ctx, op, args->output, "output", out_size(out)) ||
        (args->mixes && (check_ptr(ctx, op, args->mix, "mix", 4) || check_ptr(ctx, op, args->state, "state", 4))) ||
        (args->residual && (check_ptr(ctx, op, args->residual, "residual", 4) || check_ptr(ctx, op, args->updated, "updated", 4))))
        return SI_HIP_ERR_ARGUMENT;
    if (!args->residual && args->updated)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: updated goes with a residual", op);
    const uint64_t n = static_cast<uint64_t>(args->n), rows = static_cast<uint64_t>(args->batch.rows);
    writes.add(args->output, rows * n * out_size(out) * (args->mixes ? args->mixes : 1));
    reads.add(args->x, rows * n * 4);
    reads.add(args->weight, n * 4);
    reads.add(args->bias, n * 4);
    if (args->mixes) {
        writes.add(args->state, static_cast<uint64_t>(args->batch.slots) * n * 4);
        reads.add(args->mix, static_cast<uint64_t>(args->mixes) * n * 4);
    }
    if (args->residual) {
        writes.add(args->updated, rows * n * 4);
        reads.add(args->residual, rows * n * 4);
    }
    if (check_apart(ctx, op, writes, reads))
        return SI_HIP_ERR_ARGUMENT;
    const si::MixRowsArgs a{batch_of(args->batch), args->x, args->residual, args->weight, args->bias, args->mix, args->state,
                            args->updated, args->output, args->n, args->mixes, out, args->eps};
    return launched(ctx, si::launch_layernorm_mix_rows(a, ctx->stream), op);
}

int si_hip_rwkv7_wkv_rows_workspace_bytes(int heads, uint64_t* bytes)
{
    const char* op = "rwkv7_wkv_rows_workspace_bytes";
    if (!bytes)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null output", op);
    if (heads < 1 || heads > MAX_HEADS)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: %d heads outside 1..%d", op, heads, MAX_HEADS);
    *bytes = static_cast<uint64_t>(si::wkv_rows_workspace_bytes(heads));
    return SI_HIP_OK;
}

int si_hip_rwkv7_wkv_rows(si_hip_context* ctx, const si_hip_rwkv7_wkv_rows_args* args)
{
    const char* op = "rwkv7_wkv_rows";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (!args)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: null arguments", op);
    Spans reads, writes;
    if (const int rc = check_batch(ctx, op, args->batch, &reads))
        return rc;
    if (args->heads < 1 || args->heads > MAX_HEADS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d heads outside 1..%d", op, args->heads, MAX_HEADS);
    int out = 0;
    if (const int rc = check_format(ctx, op, "outputs", args->output_format, &out))
        return rc;
    const bool first = args->first_layer != 0;
    const uint64_t width = static_cast<uint64_t>(args->heads) * si::WKV_HEAD, rows = static_cast<uint64_t>(args->batch.rows);
    const struct {
        const float* p;
        const char* name;
        bool in_rows, needed;
    } in[] = {{args->r, "r", true, true},
              {args->k, "k", true, true},
              {args->v, "v", true, true},
              {args->w_lora, "w_lora", true, true},
              {args->a_lora, "a_lora", true, true},
              {args->gate, "gate", true, true},
              {args->v_lora, "v_lora", true, !first},
              {args->w0, "w0", false, true},
              {args->a0, "a0", false, true},
              {args->v0, "v0", false, !first},
              {args->k_k, "k_k", false, true},
              {args->k_a, "k_a", false, true},
              {args->r_k, "r_k", false, true},
              {args->lnx_weight, "lnx_weight", false, true},
              {args->lnx_bias, "lnx_bias", false, true}};
    for (const auto& i : in) {
        if (!i.needed)
            continue;
        if (check_ptr(ctx, op, i.p, i.name, i.in_rows ? 16 : 4))
            return SI_HIP_ERR_ARGUMENT;
        reads.add(i.p, width * 4 * (i.in_rows ? rows : 1));
    }
    if (check_ptr(ctx, op, args->v_first, "v_first", 16) || check_ptr(ctx, op, args->state, "state", 16) ||
        check_ptr(ctx, op, args->output, "output", 16) || check_ptr(ctx, op, args->workspace, "workspace", 16))
        return SI_HIP_ERR_ARGUMENT;
    writes.add(args->state, static_cast<uint64_t>(args->batch.slots) * width * si::WKV_HEAD * 4);
    writes.add(args->output, rows * width * out_size(out));
    writes.add(args->workspace, static_cast<uint64_t>(si::wkv_rows_workspace_bytes(args->heads)));
    (first ? writes : reads).add(args->v_first, rows * width * 4);
    if (check_apart(ctx, op, writes, reads))
        return SI_HIP_ERR_ARGUMENT;
    const si::WkvRowsArgs a{batch_of(args->batch), args->heads, first, args->r, args->k, args->v, args->w_lora, args->a_lora,
                            args->gate, args->v_lora, args->w0, args->a0, args->v0, args->k_k, args->k_a, args->r_k,
                            args->lnx_weight, args->lnx_bias, args->v_first, args->state, args->output,
                            static_cast<float*>(args->workspace), out};
    return launched(ctx, si::launch_wkv_rows(a, ctx->stream), op);
}

int si_hip_beam_select_workspace_bytes(int sequences, int beams, int candidates, int64_t vocab, uint64_t* bytes)
{
    const char* op = "beam_select_workspace_bytes";
    if (!bytes)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null output", op);
    if (const int rc = check_beams(nullptr, op, sequences, beams, candidates, vocab))
        return rc;
    *bytes = static_cast<uint64_t>(si::beam_workspace_bytes(sequences, beams, candidates, static_cast<int>(vocab)));
    return SI_HIP_OK;
}

int si_hip_beam_select(si_hip_context* ctx, const si_hip_beam_select_args* args)
{
    const char* op = "beam_select";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (!args)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: null arguments", op);
    if (const int rc = check_beams(ctx, op, args->sequences, args->beams, args->candidates, args->vocab))
        return rc;
    if (args->stride < args->vocab || args->stride > (1ll << 32))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: rows %lld values apart for a vocabulary of %lld (at most 2^32)", op,
                    static_cast<long long>(args->stride), static_cast<long long>(args->vocab));
    int format = 0;
    if (const int rc = check_format(ctx, op, "logits", args->logits_format, &format))
        return rc;
    if (args->end_token < -1 || args->end_token >= args->vocab)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: end token %d outside -1..%lld", op, args->end_token,
                    static_cast<long long>(args->vocab) - 1);
    if (args->end_token < 0 && (args->done || args->new_done))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: done and new_done need an end token", op);
    const bool slots = args->slots != nullptr;
    if (slots && args->candidates != args->beams)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: slots are handed on from %d beams to as many candidates, not %d", op,
                    args->beams, args->candidates);
    if (!slots && (args->from || args->to))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: from and to go with slots", op);
    if (check_ptr(ctx, op, args->logits, "logits", out_size(format)) || check_ptr(ctx, op, args->scores, "scores", 4) ||
        (args->done && check_ptr(ctx, op, args->done, "done", 4)) || (slots && check_ptr(ctx, op, args->slots, "slots", 4)) ||
        check_ptr(ctx, op, args->parents, "parents", 4) || check_ptr(ctx, op, args->tokens, "tokens", 4) ||
        check_ptr(ctx, op, args->new_scores, "new scores", 4) ||
        (args->new_done && check_ptr(ctx, op, args->new_done, "new done", 4)) ||
        (slots && (check_ptr(ctx, op, args->from, "from", 4) || check_ptr(ctx, op, args->to, "to", 4))) ||
        check_ptr(ctx, op, args->workspace, "workspace", 16))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t rows = static_cast<uint64_t>(args->sequences) * args->beams;
    const uint64_t in = rows * 4, count = static_cast<uint64_t>(args->sequences) * args->candidates * 4;
    Spans reads, writes;
    writes.add(args->parents, count);
    writes.add(args->tokens, count);
    writes.add(args->new_scores, count);
    writes.add(args->workspace, static_cast<uint64_t>(si::beam_workspace_bytes(args->sequences, args->beams, args->candidates,
                                                                               static_cast<int>(args->vocab))));
    reads.add(args->logits,
              ((rows - 1) * static_cast<uint64_t>(args->stride) + static_cast<uint64_t>(args->vocab)) * out_size(format));
    // in place where a sequence's workgroup reads its own part before it writes it
    const bool same = args->candidates == args->beams;
    if (!(same && args->new_scores == args->scores))
        reads.add(args->scores, in);
    if (args->new_done)
        writes.add(args->new_done, count);
    if (args->done && !(same && args->new_done == args->done))
        reads.add(args->done, in);
    if (slots) {
        writes.add(args->from, count);
        writes.add(args->to, count);
        if (args->to != args->slots)
            reads.add(args->slots, in);
    }
    if (check_apart(ctx, op, writes, reads))
        return SI_HIP_ERR_ARGUMENT;
    const si::BeamArgs a{args->logits, args->scores, args->done, args->slots, args->parents, args->tokens, args->new_scores,
                         args->new_done, args->from, args->to, args->workspace, args->stride, static_cast<int>(args->vocab),
                         args->sequences, args->beams, args->candidates, format, args->end_token};
    return launched(ctx, si::launch_beam_select(a, ctx->stream), op);
}

int si_hip_copy_slots(si_hip_context* ctx, const si_hip_slot_array* arrays, int count, int64_t slots, const int32_t* from,
                      const int32_t* to, int moves)
{
    const char* op = "copy_slots";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (!arrays || count < 1 || count > MAX_ARRAYS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: null arrays or %d of them outside 1..%d", op, count, MAX_ARRAYS);
    if (slots < 1 || slots > INT32_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %lld slots outside 1..%d", op, static_cast<long long>(slots), INT32_MAX);
    if (moves < 1 || moves > MAX_ROWS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d moves outside 1..%d", op, moves, MAX_ROWS);
    if (check_ptr(ctx, op, from, "from", 4) || check_ptr(ctx, op, to, "to", 4))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t bytes = static_cast<uint64_t>(moves) * 4;
    for (int i = 0; i < count; i++) {
        if (!arrays[i].base || arrays[i].slot_bytes < 1 || arrays[i].slot_bytes > MAX_SLOT_BYTES)
            return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: array %d is null or its slots of %llu bytes lie outside 1..2^36", op, i,
                        static_cast<unsigned long long>(arrays[i].slot_bytes));
        if (static_cast<uint64_t>(slots) > (UINT64_MAX - reinterpret_cast<uintptr_t>(arrays[i].base)) / arrays[i].slot_bytes)
            return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: array %d, %lld slots of %llu bytes, passes the address space", op, i,
                        static_cast<long long>(slots), static_cast<unsigned long long>(arrays[i].slot_bytes));
        const uint64_t size = arrays[i].slot_bytes * static_cast<uint64_t>(slots);
        if (overlaps(arrays[i].base, size, from, bytes) || overlaps(arrays[i].base, size, to, bytes))
            return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: array %d overlaps from or to", op, i);
    }
    // neighbours by address must not overlap
    const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[count]);
    if (!spans)
        return fail(ctx, SI_HIP_ERR_OUT_OF_MEMORY, "%s: no memory to check %d arrays", op, count);
    for (int i = 0; i < count; i++)
        spans[i] = {arrays[i].base, arrays[i].slot_bytes * static_cast<uint64_t>(slots)};
    std::sort(spans.get(), spans.get() + count, [](const Span& a, const Span& b) { return a.p < b.p; });
    for (int i = 1; i < count; i++)
        if (overlaps(spans[i - 1].p, spans[i - 1].n, spans[i].p, spans[i].n))
            return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: arrays overlap", op);
    return launched(ctx, si::launch_copy_slots(arrays, count, slots, from, to, moves, ctx->stream), op);
}

}  // extern "C"
