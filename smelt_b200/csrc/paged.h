// A cache in pages, the packed batch that decodes over it, and the line of work its attention kernels share.
#pragma once
#include "common.cuh"

namespace smelt {

enum PagedType : int { kPagedF16 = 0, kPagedBf16 = 1 };
enum : uint32_t { KERR_BAD_PAGE = 0x10000u };  // a page id outside the pool, a row without a token of its own, or row starts that go down
constexpr int kPagedSeqs = 1024;               // sequences of one call: their rows and lengths are held in shared memory

constexpr int kPagedCtas = 256;                // of a line's kernel at most: the join has a thread for each

// n / d for 0 <= n < 2^31 as a multiplication: with 2^l >= d > 2^(l-1), n / d = (umulhi(m, n) + n) >> l for m = 2^32 (2^l - d) / d + 1.
struct Divisor {
    uint32_t mul, shift;
    static Divisor of(uint32_t d) {
        uint32_t l = 0;
        while ((1ull << l) < d) ++l;
        return {(uint32_t)((((1ull << l) - d) << 32) / d + 1), l};
    }
};
__device__ __forceinline__ int divide(int n, const Divisor& d) { return (int)((__umulhi(d.mul, (uint32_t)n) + (uint32_t)n) >> d.shift); }

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 values side by side, and an operation on both of them in one instruction.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void split(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}

// The last sequence that starts at or before packed row r, -1: none; every lane of a warp calls it.  *start: its first row.
__device__ __forceinline__ int warp_find_seq(const int32_t* row_start, int n_seqs, int rows, int r, int* start) {
    const int lane = threadIdx.x & 31;
    int s = -1;
    for (int base = 0; base < n_seqs; base += 32) {
        const int at = base + lane < n_seqs ? min(max(row_start[base + lane], 0), rows) : 0x7fffffff;
        const uint32_t hit = __ballot_sync(0xffffffffu, at <= r);
        if (hit) {
            s = base + 31 - __clz(hit);
            *start = __shfl_sync(0xffffffffu, at, 31 - __clz(hit));
        }
    }
    return s;
}

struct PagedArgs {
    void *k, *v;
    int64_t page_stride, head_stride, token_stride;  // elements
    int page_size, n_pages;
    Divisor page_div, ratio_div;
    int n_q, n_kv, ratio;
    int n_seqs, rows, table_stride, prefix_length;
    int table_tokens;  // what a row of the table can hold; lengths are cut to it
    const int32_t *row_start, *length, *table, *prefix_table;
    uint32_t* err;
};

// A sequence's tokens on its own pages, cut at both ends to what the table can hold.
__device__ __forceinline__ int tokens_of(const PagedArgs& c, int s) { return min(max(c.length[s], 0), c.table_tokens); }

struct PagedAppendArgs {
    PagedArgs c;
    int rope_dim, layout;  // layout: 0 adjacent pairs, 1 halves
    float factor;
    const double* freq;
    const int32_t* position;  // null: by the sequence
    const void *q, *k_new, *v_new;
    void* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
};
cudaError_t launch_paged_append(const Launch& l, PagedType type, int head_dim, const PagedAppendArgs& a);

// Work of an attention kernel as one line of steps.  A step is 2^keys keys of an item; an item is one key head of one block of
// `columns` (row, query head of the group) pairs of a source; sources are the shared prefix, whose rows are those of the whole batch, and
// the sequences.  Items follow one another source by source, block by block, key head by key head, and every worker (a CTA, or a warp of
// it) takes as many steps in a row: as many keys, however uneven the lengths are, and no CTA has more than two items that it
// shares with others, one at each end.  In front of an item's steps lie `extra` places that stand for what its beginning and end cost; nobody does
// anything there.  Lengths are read on the device, so that a captured call follows them.  The line is at most 2^30
// steps (paged_api.cu).
struct PagedShared { int parts, row, f0, width, head; };  // an item of so many CTAs (0: none): first row of its sequence, first column and how many, key head
struct PagedLine {
    int columns, keys, extra;  // keys as a power of two
    Divisor column_div;
    int ctas, workers;  // workers of a CTA
    int with_prefix, with_own, wide;
    int32_t* cum;     // [n_seqs + 3] written by CTA 0: steps before each source, and the first prefix key that any row sees (kDisordered: see paged_line.cuh)
    float* slot_o;    // [2 ctas][columns][D] weighted sums of items shared by several CTAs
    float2* slot_ml;  // [2 ctas][columns] their running maxima and sums
    PagedShared* shared;  // [ctas] the item that begins in a CTA and goes on behind it, for the join (tensor-core kernel without a prefix)
};
struct PagedAttentionArgs {
    PagedArgs c;
    PagedLine line[2];  // one or two launches' work
    int lines, prefix_line, own_line;  // which of them has the prefix (-1: none), and which the sequences
    int* counters;      // [ctas], zero at a launch's beginning and end: the last CTA of a shared item joins its parts; null: a launch of the join does
    float *whole_o;     // [2][rows n_q][D] items that one CTA finishes, beside a prefix: 0 of the sequences, 1 of the prefix
    float2* whole_ml;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    float scale2;  // scale log2(e)
    uint32_t window;
};
int paged_narrow_columns(int head_dim, int64_t columns);  // columns of a block of the streaming kernel for so many of a source; keys of a step, as a power of two
int paged_narrow_keys();
int paged_narrow_workers(int head_dim);
cudaError_t launch_paged_narrow(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a, int line);
// The tensor-core kernel (paged_wide.cu) and whether its shared memory holds a batch of n_seqs.
int paged_wide_columns(int head_dim, int ratio);
int paged_wide_keys(int head_dim);
bool paged_wide_takes(int head_dim, int n_seqs);
cudaError_t launch_paged_wide(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a, int line);
// What joins the parts of items: with a prefix every row's (merge), without one the shared items' (join).
cudaError_t launch_paged_merge(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a);
cudaError_t launch_paged_join(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a);

// Drafted tokens against the target (verify.cu).
struct VerifyArgs {
    int n_seqs, rows, vocab;
    int steps;  // that the draft holds: a sequence's drafts behind them are not judged
    const void *target, *draft;  // draft may be null
    int64_t target_stride, draft_step_stride, draft_seq_stride;  // elements
    const int32_t *row_start, *tokens;
    const float *temperature, *random;  // temperature may be null
    int32_t *out_tokens, *accepted;
    void* stats;  // verify_workspace bytes
};
enum LogitsType : int { kLogitsF16 = 0, kLogitsBf16 = 1, kLogitsF32 = 2 };
size_t verify_workspace(LogitsType type, int n_seqs, int rows, int vocab, bool draft);
cudaError_t launch_verify(const Launch& l, LogitsType type, const VerifyArgs& a);

}  // namespace smelt
