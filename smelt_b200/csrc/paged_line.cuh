// Device side of the line of work of the paged attention kernels (PagedLine in paged.h).
#pragma once
#include <type_traits>

#include "paged.h"

namespace smelt {
namespace paged {

constexpr float kLowest = -3.402823466e38f;
constexpr int kDisordered = -1;  // in the place of the first prefix key that any row sees: row starts that go down, nothing is computed

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}

struct Range { int lo, hi; };  // keys [lo, hi)

// A sequence's rows of the batch and its tokens, cut to what the arrays hold.
struct Seq { int row, n, length; };

__device__ __forceinline__ int first_row(const PagedArgs& c, int s) { return min(max(c.row_start[s], 0), c.rows); }
// Keys of its own pages that row i of a sequence sees.  (Tokens and rows are below 2^30; a window beyond that is none.)
__device__ __forceinline__ Range own_keys(const Seq& s, int i, uint32_t window) {
    const int hi = max(s.length - s.n + i + 1, 0);
    return {window ? max(0, hi - (int)window) : 0, hi};
}
// Keys of a prefix of P tokens that row i sees; a row without a token of its own sees nothing.
__device__ __forceinline__ Range prefix_keys(const Seq& s, int i, int P, uint32_t window) {
    const int token = s.length - s.n + i;
    if (token < 0) return {0, 0};
    return {window ? min(P, max(0, P - (int)window + token + 1)) : 0, P};
}
// Keys that some row of a block of a sequence sees.
__device__ __forceinline__ Range block_keys(const PagedArgs& c, const PagedLine& line, const Seq& s, int block, uint32_t window) {
    const int f0 = block * line.columns, f1 = min(s.n * c.ratio, f0 + line.columns) - 1;
    return {own_keys(s, divide(f0, c.ratio_div), window).lo, own_keys(s, divide(f1, c.ratio_div), window).hi};
}
__device__ __forceinline__ int blocks_of(const PagedArgs& c, const PagedLine& line, int rows) { return divide(rows * c.ratio + line.columns - 1, line.column_div); }
__device__ __forceinline__ int steps_of(const Range& r, int keys) { return r.hi > r.lo ? ((r.hi - 1) >> keys) - (r.lo >> keys) + 1 : 0; }
// Places on the line of an item of so many steps, and of all blocks of a sequence and one key head.
__device__ __forceinline__ int places_of(const PagedLine& line, int steps) { return steps ? steps + line.extra : 0; }
__device__ __forceinline__ int places_of_seq(const PagedArgs& c, const PagedLine& line, const Seq& s, int blocks, uint32_t window) {
    int sum = 0;
    for (int k = 0; k < blocks; ++k) sum += places_of(line, steps_of(block_keys(c, line, s, k, window), line.keys));
    return sum;
}

// What a CTA holds of the batch in shared memory.
struct Batch {
    int* cum;     // [n_seqs + 2]: places in front of source 0 (the prefix), 1 (sequence 0), ..., and all of them
    int* row;     // [n_seqs + 1]
    int* length;  // [n_seqs]
    int prefix_lo;
    __device__ __forceinline__ Seq seq(int s) const { return {row[s], max(row[s + 1] - row[s], 0), length[s]}; }
};
__host__ __device__ constexpr size_t batch_bytes(int n_seqs) { return ((size_t)(3 * n_seqs + 3) * 4 + 15) & ~(size_t)15; }

// Fills `b` (every thread of the CTA calls it; the sums end behind a barrier).
template <int THREADS>
__device__ __forceinline__ void scan_line(const PagedArgs& c, const PagedLine& line, uint32_t window, Batch& b, unsigned char* memory) {
    __shared__ int warp_sums[THREADS / 32];
    __shared__ int lowest;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = c.n_seqs;
    b.cum = reinterpret_cast<int*>(memory);
    b.row = b.cum + n + 2;
    b.length = b.row + n + 1;
    if (tid == 0) lowest = c.prefix_length;
    for (int s = tid; s <= n; s += THREADS) {
        b.row[s] = first_row(c, s);
        if (s < n) b.length[s] = tokens_of(c, s);
    }
    __syncthreads();
    const int per = (n + THREADS - 1) / THREADS, s0 = min(n, tid * per), s1 = min(n, s0 + per);
    int mine = 0;
    bool down = false;
    for (int s = s0; s < s1; ++s) {
        const Seq q = b.seq(s);
        down |= b.row[s + 1] < b.row[s];
        if (line.with_own) mine += c.n_kv * places_of_seq(c, line, q, blocks_of(c, line, q.n), window);
        if (line.with_prefix && window && q.n) atomicMin(&lowest, prefix_keys(q, 0, c.prefix_length, window).lo);
    }
    int run = mine;
    if (n > 1) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
    }
    if (lane == 31) warp_sums[warp] = run;
    const int disordered = __syncthreads_or(down);
    b.prefix_lo = window ? lowest : 0;
    int before = run - mine;
    if (n > 32 * per)
        for (int w = 0; w < warp; ++w) before += warp_sums[w];
    if (line.with_prefix) before += c.n_kv * blocks_of(c, line, b.row[n]) * places_of(line, steps_of({b.prefix_lo, c.prefix_length}, line.keys));
    if (tid == 0) { b.cum[0] = 0; b.cum[1] = before; }
    if (per == 1) {
        if (s0 < s1) b.cum[s0 + 2] = before + mine;
    } else {
        for (int s = s0; s < s1; ++s) {
            const Seq q = b.seq(s);
            if (line.with_own) before += c.n_kv * places_of_seq(c, line, q, blocks_of(c, line, q.n), window);
            b.cum[s + 2] = before;
        }
    }
    __syncthreads();
    if (disordered) {  // Starts that go down give rows to several sequences, and their places may be more than are counted in 32 bits: nobody has rows.
        for (int s = tid; s < n + 2; s += THREADS) b.cum[s] = 0;
        for (int s = tid; s <= n; s += THREADS) b.row[s] = 0;
        if (tid == 0 && blockIdx.x == 0 && c.err) atomicOr(c.err, KERR_BAD_PAGE);
        __syncthreads();
    }
    if (blockIdx.x == 0) {
        for (int s = tid; s < n + 2; s += THREADS) line.cum[s] = b.cum[s];
        if (tid == 0) line.cum[n + 2] = disordered ? kDisordered : b.prefix_lo;
    }
}

// Who has which places of the line: the first `more` workers have each + 1, the others `each`; workers from `used` on have none, so that none
// between two owners of an item is without.
struct Share {
    int workers, used, each, more;
    __device__ __forceinline__ Share(int total, const PagedLine& line)
        : workers(line.workers), used(min(total, line.ctas * line.workers)), each(used ? total / used : 0), more(total - each * used) {}
    __device__ __forceinline__ int begin(int worker) const { const int w = min(worker, used); return each * w + min(w, more); }
    __device__ __forceinline__ int cta_begin(int cta) const { return begin(cta * workers); }
    __device__ __forceinline__ int cta_of(int at) const {  // the CTA that has a step
        const int first = more * (each + 1), w = at < first ? at / (each + 1) : more + (at - first) / each;
        return w / workers;
    }
};

// A step of an item, at place `at` of the line.
struct Cursor {
    int source, block, head, step, steps, first;  // source 0: the prefix, s + 1: sequence s; first: step of the item's first key
    int at;
    Range keys;
    int n_blocks;

    __device__ __forceinline__ void load_block(const PagedArgs& c, const PagedLine& line, uint32_t window, const Batch& b) {
        keys = source == 0 ? Range{b.prefix_lo, c.prefix_length} : block_keys(c, line, b.seq(source - 1), block, window);
        steps = steps_of(keys, line.keys);
        first = keys.lo >> line.keys;
    }
    __device__ __forceinline__ void load_source(const PagedArgs& c, const PagedLine& line, const Batch& b) {
        n_blocks = blocks_of(c, line, source == 0 ? b.row[c.n_seqs] : b.seq(source - 1).n);
    }
    // The first step at place `from` or behind it, from < cum[n_seqs + 1].
    __device__ __forceinline__ void seek(const PagedArgs& c, const PagedLine& line, uint32_t window, const Batch& b, int from) {
        int lo = 0, hi = c.n_seqs;  // the last source with cum <= from
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (b.cum[mid] <= from) lo = mid;
            else hi = mid - 1;
        }
        source = lo;
        load_source(c, line, b);
        int rest = from - b.cum[source], places;
        for (block = 0;; ++block) {
            load_block(c, line, window, b);
            places = places_of(line, steps);
            if (rest < c.n_kv * places || block + 1 >= n_blocks) break;
            rest -= c.n_kv * places;
        }
        head = rest / places;
        const int in = rest - head * places;
        step = max(in - line.extra, 0);
        at = from + max(line.extra - in, 0);
    }
    // To the next step; where there is none, `at` is behind the line.
    __device__ __forceinline__ void advance(const PagedArgs& c, const PagedLine& line, uint32_t window, const Batch& b) {
        ++at;
        if (++step < steps) return;
        step = 0;
        at += line.extra;
        if (++head < c.n_kv) return;
        head = 0;
        if (at >= b.cum[c.n_seqs + 1]) return;
        do {
            if (++block >= n_blocks) {
                block = 0;
                do ++source; while (b.cum[source + 1] == b.cum[source] && source < c.n_seqs);
                load_source(c, line, b);
            }
            load_block(c, line, window, b);
        } while (steps == 0);
    }
    // To the next item's first step.
    __device__ __forceinline__ void next_item(const PagedArgs& c, const PagedLine& line, uint32_t window, const Batch& b) {
        at += steps - 1 - step;
        step = steps - 1;
        advance(c, line, window, b);
    }
};

// The sequence of a packed row, from row starts in shared memory.
__device__ __forceinline__ int seq_of_row(const Batch& b, int n_seqs, int row) {
    int lo = 0, hi = n_seqs - 1;  // the last sequence that starts at or before the row
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.row[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Infinite values.  A weight times an infinite value is infinite, but weights reach the products in 16 bits, in parts or rounded, and a part that is
// zero makes NaN of it.  Where an item's sums are not finite its values are looked through again (a whole warp calls it): the 32 values from
// `values` on (in the pool's first token of the key head) of the keys [from, to), a key a lane.  pos and neg: bit e where value e of a key that the lane's column
// i sees is +infinity or -infinity, both where it is NaN.
template <int COLS> struct Infinite {
    Range seen[COLS];
    uint32_t pos[COLS], neg[COLS];
    // What the sum over the keys is: as it is, where all values are finite.
    __device__ __forceinline__ float sum(int col, int e, float finite) const {
        const bool p = pos[col] >> e & 1u, n = neg[col] >> e & 1u;
        return p ? (n ? __uint_as_float(0x7FC00000u) : INFINITY) : n ? -INFINITY : finite;
    }
};
template <class E, int COLS>
__device__ __forceinline__ void look_for_infinities(const PagedArgs& c, const int32_t* table, const E* values, int from, int to, Infinite<COLS>& found) {
    constexpr uint32_t kInf = std::is_same<E, __half>::value ? 0x7C00u : 0x7F80u;
    const int lane = threadIdx.x & 31;
    for (int i = 0; i < COLS; ++i) found.pos[i] = found.neg[i] = 0;
    for (int base = from; base < to; base += 32) {
        const int key = base + lane;
        uint32_t p = 0, n = 0;
        if (key < to) {
            const int at = divide(key, c.page_div), page = table[at];
            if ((uint32_t)page < (uint32_t)c.n_pages) {
                const uint4* row = reinterpret_cast<const uint4*>(values + (long long)page * c.page_stride + (long long)(key - at * c.page_size) * c.token_stride);
                for (int i = 0; i < 4; ++i) {
                    const uint4 w = row[i];
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t v = u[e >> 1] >> (16 * (e & 1)) & 0xffffu;
                        if ((v & kInf) != kInf) continue;
                        const bool nan = v & (0x7fffu & ~kInf);
                        if (nan || !(v & 0x8000u)) p |= 1u << (8 * i + e);
                        if (nan || (v & 0x8000u)) n |= 1u << (8 * i + e);
                    }
                }
            }
        }
        for (uint32_t some = __ballot_sync(0xffffffffu, p | n); some; some &= some - 1u) {
            const int from_lane = __ffs(some) - 1, k = base + from_lane;
            const uint32_t pk = __shfl_sync(0xffffffffu, p, from_lane), nk = __shfl_sync(0xffffffffu, n, from_lane);
            for (int i = 0; i < COLS; ++i)
                if (k >= found.seen[i].lo && k < found.seen[i].hi) { found.pos[i] |= pk; found.neg[i] |= nk; }
        }
    }
}

}  // namespace paged
}  // namespace smelt
