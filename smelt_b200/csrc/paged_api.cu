// Entry points of the paged cache, its attention and the check of drafted tokens.
#include <cmath>

#include "paged.h"
#include "runtime.h"

using namespace smelt;

namespace {

smelt_status enter(smelt_cuda_ctx* ctx, Launch* l) {
    if (!ctx) return SMELT_ERR_BAD_ARGUMENT;
    if (cudaSetDevice(ctx->device) != cudaSuccess) return fail(ctx, SMELT_ERR_CUDA, "cudaSetDevice");
    l->stream = ctx->stream;
    l->pdl = ctx->pdl;  // every kernel here waits for the one in front before it reads or writes
    return SMELT_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Arrays of `size`-byte values, null among them, where their type wants them: what is not would end the context on the device.
template <class... P> bool aligned(size_t size, const P*... p) { return ((reinterpret_cast<uintptr_t>(p) % size == 0) && ...); }
// Rows of `width` 16-bit values, `stride` apart, that 16-byte loads can take.
bool rows_ok(const void* p, int64_t stride, int64_t width, int64_t rows) {
    return p && aligned16(p) && stride % 8 == 0 && (rows <= 1 || stride >= width) && stride >= 0 && stride < ((int64_t)1 << 38);
}

smelt_status cache_args(smelt_cuda_ctx* ctx, const smelt_paged_cache* k, const smelt_paged_batch* b, PagedArgs* c) {
    if (!k || !b) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged cache: null description");
    if (k->precision != SMELT_PAGED_F16 && k->precision != SMELT_PAGED_BF16) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged cache: unknown precision");
    if (k->n_q <= 0 || k->n_kv <= 0 || k->n_q % k->n_kv || k->page_size <= 0 || k->n_pages <= 0) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged cache: bad geometry");
    if (k->head_dim != 64 && k->head_dim != 128 && k->head_dim != 256) return fail(ctx, SMELT_ERR_UNSUPPORTED, "paged cache: heads of 64, 128 or 256 values");
    const int64_t strides[3] = {k->page_stride, k->head_stride, k->token_stride}, counts[3] = {k->n_pages, k->n_kv, k->page_size};
    double reach = 0;
    for (int i = 0; i < 3; ++i) {
        if (strides[i] < 0 || strides[i] % 8 || (counts[i] > 1 && strides[i] < k->head_dim)) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged cache: strides are multiples of 8 values, of a row at least");
        reach += (double)strides[i] * (double)(counts[i] - 1);
    }
    if (reach > 1e15) return fail(ctx, SMELT_ERR_OUT_OF_RANGE, "paged cache: strides past any memory");
    if (!k->k || !k->v || !aligned16(k->k) || !aligned16(k->v)) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged cache: pools are 16-byte aligned");
    if (b->n_seqs < 0 || b->rows < 0 || b->max_rows < 0 || b->table_stride < 0 || b->prefix_length < 0) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged batch: negative size");
    if ((int64_t)b->rows * k->n_q > 0x3fffffff || (int64_t)b->prefix_length > 0x3fffffff) return fail(ctx, SMELT_ERR_OUT_OF_RANGE, "paged batch: too many rows or tokens");
    if (b->n_seqs > 0 && b->rows > 0 && (!b->row_start || !b->length || (b->table_stride > 0 && !b->table) || (b->prefix_length > 0 && !b->prefix_table)))
        return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged batch: null pointer");
    if (!aligned(4, b->row_start, b->length, b->table, b->prefix_table)) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged batch: misaligned pointer");
    *c = {};
    c->k = k->k; c->v = k->v;
    c->page_stride = k->page_stride; c->head_stride = k->head_stride; c->token_stride = k->token_stride;
    c->page_size = k->page_size; c->n_pages = k->n_pages; c->page_div = Divisor::of((uint32_t)k->page_size);
    c->n_q = k->n_q; c->n_kv = k->n_kv; c->ratio = k->n_q / k->n_kv; c->ratio_div = Divisor::of((uint32_t)c->ratio);
    c->n_seqs = b->n_seqs; c->rows = b->rows; c->table_stride = b->table_stride; c->prefix_length = b->prefix_length;
    const int64_t tokens = (int64_t)b->table_stride * k->page_size;
    c->table_tokens = (int)(tokens < 0x3fffffff ? tokens : 0x3fffffff);
    c->row_start = (const int32_t*)b->row_start; c->length = (const int32_t*)b->length;
    c->table = (const int32_t*)b->table; c->prefix_table = (const int32_t*)b->prefix_table;
    c->err = ctx->err_dev;
    return SMELT_OK;
}

// How a call's work is cut, and where its parts lie in a workspace (null: sizes only).
size_t attention_plan(const smelt_cuda_ctx* ctx, const smelt_paged_cache* k, const smelt_paged_batch* b, PagedAttentionArgs* a, void* workspace) {
    const int D = k->head_dim;
    size_t at = 0;
    auto room = [&](size_t bytes) {
        void* p = workspace ? static_cast<char*>(workspace) + at : nullptr;
        at += (bytes + 31) & ~(size_t)31;
        return p;
    };
    // Columns of a source: up to 16 on the streaming kernel (8 with heads of 256), more on the tensor core.  us with 16 | 32 columns, 16 sequences of
    // 2000 tokens and 8 key heads of 128: streaming 42 | 67, tensor core 46 | 46; heads of 64: 34 | 51 and 35 | 35; heads of 256 and 8 | 16
    // columns: 70 | 122 and 70 | 71.  A launch takes sequences and prefix together where they go to the same kernel, and a prefix that is no
    // more than four tiles a warp goes with the sequences on the streaming kernel (64 sequences of 300 tokens behind a prefix of 1000 | 2000 | 4000,
    // 32 query and 8 key heads of 128: together 53 | 60 | 83 us, a launch each 55 | 60 | 62).
    const int64_t own = (int64_t)(b->max_rows > 0 ? b->max_rows : 1) * a->c.ratio, prefix = b->prefix_length > 0 ? (int64_t)b->rows * a->c.ratio : 0;
    const bool can = paged_wide_takes(D, b->n_seqs);
    const int64_t most = D == 256 ? 8 : 16, prefix_tiles = (prefix + most - 1) / most * k->n_kv * ((b->prefix_length >> paged_narrow_keys()) + 2);
    const bool own_wide = can && own > most, prefix_wide = can && prefix > most && (own_wide || prefix_tiles > (int64_t)4 * ctx->sm_count * paged_narrow_workers(D));
    a->lines = 0;
    a->prefix_line = a->own_line = -1;
    auto add = [&](bool wide, bool with_own, bool with_prefix) {
        if (with_prefix) a->prefix_line = a->lines;
        if (with_own) a->own_line = a->lines;
        PagedLine& line = a->line[a->lines++];
        line.wide = wide;
        line.with_own = with_own;
        line.with_prefix = with_prefix;
        const int64_t columns = with_own && with_prefix ? (own > prefix ? own : prefix) : with_own ? own : prefix;
        line.columns = wide ? paged_wide_columns(D, a->c.ratio) : paged_narrow_columns(D, columns);
        line.column_div = Divisor::of((uint32_t)line.columns);
        line.keys = wide ? paged_wide_keys(D) : paged_narrow_keys();
        // What an item costs beside its steps: 11 us of 2.2 us a step on the tensor core (the first scores, a masked step, the end; three | five | eight
        // places: two ragged prompts of up to 1500 rows behind 4100 tokens 177 | 167 | 170 us, 16 sequences of up to six rows 28.6 | 29.2 | 32.9), 1 us of 1 us a tile on the streaming kernel.
        line.extra = wide ? 5 : 1;
        line.ctas = ctx->sm_count < kPagedCtas ? ctx->sm_count : kPagedCtas;
        line.workers = wide ? 1 : paged_narrow_workers(D);
        line.cum = (int32_t*)room((size_t)(b->n_seqs + 3) * sizeof(int32_t));
        line.slot_o = (float*)room((size_t)2 * line.ctas * line.columns * D * sizeof(float));
        line.slot_ml = (float2*)room((size_t)2 * line.ctas * line.columns * sizeof(float2));
        line.shared = (PagedShared*)room((size_t)line.ctas * sizeof(PagedShared));
    };
    if (prefix == 0) {
        add(own_wide, true, false);
        if (!own_wide) a->counters = (int*)room((size_t)a->line[0].ctas * sizeof(int));  // few sums: the kernel joins them itself
    } else if (own_wide == prefix_wide) {
        add(own_wide, true, true);
    } else {
        add(prefix_wide, false, true);
        add(own_wide, true, false);
    }
    if (b->prefix_length > 0) {
        a->whole_o = (float*)room((size_t)2 * b->rows * k->n_q * D * sizeof(float));
        a->whole_ml = (float2*)room((size_t)2 * b->rows * k->n_q * sizeof(float2));
    }
    return at;
}

smelt_status verify_args(smelt_cuda_ctx* ctx, const smelt_verify_args* v) {
    if (!v) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: null description");
    if (v->precision < SMELT_LOGITS_F16 || v->precision > SMELT_LOGITS_F32) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: unknown precision");
    if (v->n_seqs < 0 || v->rows < 0 || v->vocab <= 0) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: bad sizes");
    if (v->vocab > (1 << 24) || v->n_seqs > (1 << 20) || v->rows > (1 << 20) || (int64_t)v->rows * v->vocab > ((int64_t)1 << 41)) return fail(ctx, SMELT_ERR_OUT_OF_RANGE, "verify drafts: too many rows or tokens");
    return SMELT_OK;
}

}  // namespace

extern "C" {

smelt_status smelt_cuda_rope_frequencies(const smelt_rope_scaling* s, double* out_freq, float* out_factor) {
    if (!s || !out_freq || s->rope_dim <= 0 || s->rope_dim % 2 || s->rope_dim > 1024 || !(s->theta > 1.0) || s->kind < SMELT_ROPE_PLAIN || s->kind > SMELT_ROPE_BANDS) return SMELT_ERR_BAD_ARGUMENT;
    if (s->kind != SMELT_ROPE_PLAIN && !(s->factor >= 1.0)) return SMELT_ERR_BAD_ARGUMENT;
    const bool bands = s->kind == SMELT_ROPE_RAMP || s->kind == SMELT_ROPE_BANDS;
    if (bands && (!(s->known_positions > 0.0) || !(s->slow_turns > 0.0) || !(s->fast_turns > s->slow_turns))) return SMELT_ERR_BAD_ARGUMENT;
    const int n = s->rope_dim;
    const double two_pi = 6.283185307179586476925;
    const double theta = s->kind == SMELT_ROPE_BASE && n > 2 ? s->theta * std::pow(s->factor, (double)n / (n - 2)) : s->theta;
    double from = 0, to = 0;  // RAMP: pairs in front of `from` stay, those behind `to` are stretched
    if (s->kind == SMELT_ROPE_RAMP) {
        auto pair_of = [&](double turns) { return n * std::log(s->known_positions / (turns * two_pi)) / (2 * std::log(s->theta)); };
        from = std::fmax(std::floor(pair_of(s->fast_turns)), 0.0);
        to = std::fmin(std::ceil(pair_of(s->slow_turns)), n - 1.0);
        if (to <= from) to = from + 1e-3;
    }
    for (int i = 0; i < n / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / n), keep = 1.0;
        if (s->kind == SMELT_ROPE_LINEAR) keep = 0.0;
        if (s->kind == SMELT_ROPE_RAMP) keep = 1.0 - std::fmin(std::fmax((i - from) / (to - from), 0.0), 1.0);
        if (s->kind == SMELT_ROPE_BANDS) keep = std::fmin(std::fmax((s->known_positions * f / two_pi - s->slow_turns) / (s->fast_turns - s->slow_turns), 0.0), 1.0);
        if (s->kind == SMELT_ROPE_LINEAR || bands) f = f * keep + f / s->factor * (1.0 - keep);
        out_freq[i] = f;
    }
    if (out_factor) *out_factor = s->kind == SMELT_ROPE_RAMP ? (float)(0.1 * std::log(s->factor) + 1.0) : 1.0f;
    return SMELT_OK;
}

smelt_status smelt_cuda_paged_append(smelt_cuda_ctx* ctx, const smelt_paged_cache* cache, const smelt_paged_batch* batch, const smelt_rope_desc* rope, const void* q, int64_t q_stride,
                                     const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out, int64_t q_out_stride) {
    Launch l;
    PagedAppendArgs a = {};
    smelt_status s = enter(ctx, &l);
    if (!s) s = cache_args(ctx, cache, batch, &a.c);
    if (s) return s;
    if (rope) {
        if (rope->rope_dim < 0 || rope->rope_dim % 2 || rope->rope_dim > cache->head_dim || (rope->layout != SMELT_ROPE_ADJACENT && rope->layout != SMELT_ROPE_HALVES) ||
            (rope->rope_dim > 0 && !rope->freq) || !aligned(8, rope->freq) || !aligned(4, rope->position))
            return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged append: bad rotation");
        a.rope_dim = rope->rope_dim; a.layout = rope->layout; a.factor = rope->factor; a.freq = (const double*)rope->freq; a.position = (const int32_t*)rope->position;
    }
    if (batch->n_seqs == 0 || batch->rows == 0) return SMELT_OK;
    const int64_t D = cache->head_dim, rows = batch->rows;
    if (!rows_ok(k, k_stride, cache->n_kv * D, rows) || !rows_ok(v, v_stride, cache->n_kv * D, rows)) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged append: rows of keys and values are 16-byte aligned, strides multiples of 8");
    if (q && (!rows_ok(q, q_stride, cache->n_q * D, rows) || !rows_ok(q_out, q_out_stride, cache->n_q * D, rows)))
        return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged append: rows of queries are 16-byte aligned, strides multiples of 8");
    if (q && q == q_out && q_stride != q_out_stride) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged append: queries rotated in place keep their stride");
    a.q = q; a.k_new = k; a.v_new = v; a.q_out = q_out;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.q_out_stride = q_out_stride;
    return check_cuda(ctx, launch_paged_append(l, (PagedType)cache->precision, cache->head_dim, a), "paged append");
}

smelt_status smelt_cuda_paged_attention_workspace(smelt_cuda_ctx* ctx, const smelt_paged_cache* cache, const smelt_paged_batch* batch, size_t* out_bytes) {
    Launch l;
    PagedAttentionArgs a = {};
    smelt_status s = enter(ctx, &l);
    if (!s) s = cache_args(ctx, cache, batch, &a.c);
    if (s) return s;
    if (!out_bytes) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged attention: null size");
    *out_bytes = attention_plan(ctx, cache, batch, &a, nullptr);
    return SMELT_OK;
}

smelt_status smelt_cuda_paged_attention(smelt_cuda_ctx* ctx, const smelt_paged_cache* cache, const smelt_paged_batch* batch, const void* q, int64_t q_stride, void* out, int64_t out_stride,
                                        float scale, uint32_t window, void* workspace, size_t workspace_bytes) {
    Launch l;
    PagedAttentionArgs a = {};
    smelt_status s = enter(ctx, &l);
    if (!s) s = cache_args(ctx, cache, batch, &a.c);
    if (s) return s;
    if (batch->n_seqs == 0 || batch->rows == 0) return SMELT_OK;
    if (batch->n_seqs > kPagedSeqs) return fail(ctx, SMELT_ERR_UNSUPPORTED, "paged attention: at most 1024 sequences a call");
    const int64_t D = cache->head_dim, rows = batch->rows;
    if (!rows_ok(q, q_stride, cache->n_q * D, rows) || !rows_ok(out, out_stride, cache->n_q * D, rows)) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged attention: rows are 16-byte aligned, strides multiples of 8");
    if (q == out && q_stride != out_stride) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged attention: an output in the place of the queries keeps their stride");
    if (!(scale == scale) || std::isinf(scale)) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged attention: scale is not finite");
    {  // the line of work is counted in 32 bits
        attention_plan(ctx, cache, batch, &a, nullptr);
        double steps = 0;
        for (int i = 0; i < a.lines; ++i) {
            const PagedLine& line = a.line[i];
            const double blocks = (double)(rows * a.c.ratio / line.columns) + 1;
            if (line.with_own) steps += (blocks + batch->n_seqs) * cache->n_kv * ((a.c.table_tokens >> line.keys) + 2.0 + line.extra);
            if (line.with_prefix) steps += blocks * cache->n_kv * ((batch->prefix_length >> line.keys) + 2.0 + line.extra);
        }
        if (steps > 1e9) return fail(ctx, SMELT_ERR_OUT_OF_RANGE, "paged attention: more rows times pages than a call takes");
    }
    if (!workspace || !aligned16(workspace) || workspace_bytes < attention_plan(ctx, cache, batch, &a, nullptr))
        return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "paged attention: workspace missing, misaligned or smaller than smelt_cuda_paged_attention_workspace says");
    attention_plan(ctx, cache, batch, &a, workspace);
    a.q = q; a.out = out; a.q_stride = q_stride; a.out_stride = out_stride;
    a.scale2 = scale * 1.4426950408889634f;
    a.window = window < 0x7fffffffu ? window : 0;  // positions are below that
    cudaError_t e = cudaSuccess;
    if (a.counters) {
        // Calls on the context's stream follow one another, and so do replays of its own capture: they share its counters, which every call
        // leaves at zero.  A graph that the caller captures from the stream may run beside them: it counts in its workspace.
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (!ctx->capturing) e = cudaStreamIsCapturing(l.stream, &capture);
        if (e == cudaSuccess && capture == cudaStreamCaptureStatusActive) {
            e = cudaMemsetAsync(a.counters, 0, (size_t)a.line[0].ctas * sizeof(int), l.stream);
            l.pdl = false;  // the kernel follows the memset
        } else {
            a.counters = ctx->paged_counters;
        }
    }
    for (int i = 0; i < a.lines && e == cudaSuccess; ++i) e = (a.line[i].wide ? launch_paged_wide : launch_paged_narrow)(l, (PagedType)cache->precision, cache->head_dim, a, i);
    if (e == cudaSuccess && !a.counters) e = (a.whole_o ? launch_paged_merge : launch_paged_join)(l, (PagedType)cache->precision, cache->head_dim, a);
    return check_cuda(ctx, e, "paged attention");
}

smelt_status smelt_cuda_verify_drafts_workspace(smelt_cuda_ctx* ctx, const smelt_verify_args* args, size_t* out_bytes) {
    if (!ctx) return SMELT_ERR_BAD_ARGUMENT;
    const smelt_status s = verify_args(ctx, args);
    if (s) return s;
    if (!out_bytes) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: null size");
    *out_bytes = verify_workspace((LogitsType)args->precision, args->n_seqs, args->rows, args->vocab, args->draft != nullptr);
    return SMELT_OK;
}

smelt_status smelt_cuda_verify_drafts(smelt_cuda_ctx* ctx, const smelt_verify_args* v) {
    Launch l;
    smelt_status s = enter(ctx, &l);
    if (!s) s = verify_args(ctx, v);
    if (s) return s;
    if (v->n_seqs == 0) return SMELT_OK;
    if (!aligned(4, v->row_start, v->tokens, v->temperature, v->random, v->out_tokens, v->accepted)) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: misaligned pointer");
    if (v->rows == 0) {  // nobody has a draft
        if (!v->accepted) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: null pointer");
        return check_cuda(ctx, cudaMemsetAsync(v->accepted, 0, (size_t)v->n_seqs * sizeof(int32_t), l.stream), "verify drafts");
    }
    if (!v->row_start || !v->target || !v->tokens || !v->random || !v->out_tokens || !v->accepted) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: null pointer");
    const uintptr_t width = v->precision == SMELT_LOGITS_F32 ? 4 : 2;
    if ((uintptr_t)v->target % width || (uintptr_t)v->draft % width) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: misaligned logits");
    if ((v->rows > 1 && v->target_stride < v->vocab) || (v->draft && (v->draft_step_stride < 0 || v->draft_seq_stride < 0))) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: bad strides");
    if (v->out_tokens == v->tokens) return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: the answer needs a place of its own");
    const LogitsType type = (LogitsType)v->precision;
    if (!v->workspace || !aligned16(v->workspace) || v->workspace_bytes < verify_workspace(type, v->n_seqs, v->rows, v->vocab, v->draft != nullptr))
        return fail(ctx, SMELT_ERR_BAD_ARGUMENT, "verify drafts: workspace missing, misaligned or smaller than smelt_cuda_verify_drafts_workspace says");
    VerifyArgs a = {};
    a.n_seqs = v->n_seqs; a.rows = v->rows; a.vocab = v->vocab;
    a.steps = v->draft && v->draft_steps ? v->draft_steps : v->rows;
    a.target = v->target; a.draft = v->draft;
    a.target_stride = v->target_stride; a.draft_step_stride = v->draft_step_stride; a.draft_seq_stride = v->draft_seq_stride;
    a.row_start = (const int32_t*)v->row_start; a.tokens = (const int32_t*)v->tokens;
    a.temperature = (const float*)v->temperature; a.random = (const float*)v->random;
    a.out_tokens = (int32_t*)v->out_tokens; a.accepted = (int32_t*)v->accepted;
    a.stats = v->workspace;
    return check_cuda(ctx, launch_verify(l, type, a), "verify drafts");
}

}  // extern "C"
