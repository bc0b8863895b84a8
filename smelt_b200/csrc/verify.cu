// Drafted tokens against the target's probabilities, from given random numbers.
//
// With p = softmax(target / T) and q = softmax(draft / T): draft x_j stands while u_j q_j(x_j) < p_j(x_j); at the first that does
// not the next token is drawn from max(p - q, 0), behind the last draft from p, as the first index whose running sum passes u times
// the whole.
//
// verify_stats_kernel reads every row of logits once (the bytes that bound the operator): a CTA takes a stretch of one row
// and leaves its maximum, the sum of exp((x - max) / T) and the lowest index of the maximum, in fp32 (a chance's
// error of 1e-7 turns a draw that lies as near to it).  Then one row of a sequence is read again, and with a draft's probabilities one
// of those: there a running sum over the vocabulary is compared with a number, and every index is a border, so probabilities and sums are
// fp64, and all sums are added in the order of the vocabulary.  A piece of such a row is a CTA's: verify_sums_kernel
// (with a draft's probabilities) finds the first draft that falls and adds up the weights of p and q, verify_pick_kernel what the next token is
// drawn by, and its last CTA of a sequence finds the index.  (A cluster of eight CTAs a sequence, which did all of that in one
// launch, took 45 us for one sequence and 70 for 48 of them, its fp64 pipe busy for an eighth of the time.)
//
// us with 152k tokens and a draft's probabilities, logits from memory: 1 sequence of up to six rows 28, 16 46, 48 87, 192 of three 175 (the same logits again, 94 MB
// of 48 sequences in L2: 82).  Memory bounds none of it: the statistics of 48 sequences take 35 of the 87 (11 operations an element, and four
// microseconds of a CTA's beginning and end), the fp64 weights, two to an element and twice over, the rest.
#include <cuda_bf16.h>

#include "paged.h"

namespace smelt {
namespace {

constexpr int kStatThreads = 256, kStatWords = 4;  // words of 16 bytes a thread has on their way at a time
// CTAs of a launch of the draw, and their threads: 80 registers let eight fp64 chains of a thread run side by side (us of the whole, 16 | 48 | 192
// sequences: 256 threads and three CTAs an SM 46 | 87 | 174, 512 and two, of 64 registers, 53 | 91 | 170, 512 and one, of 108, 64 | 108 | 191).
constexpr int kDrawCtas = 1184, kDrawThreads = 256, kDrawWarps = kDrawThreads / 32;
constexpr float kNone = -INFINITY;

// What the kernels behind the statistics leave one another: rows that are drawn from are cut into pieces, a CTA each.
struct Choice;
struct Draws {
    int pieces;
    Choice* choice;   // [n_seqs]
    int* arrived;     // [n_seqs] CTAs that have written their part of `chances`
    double* sums;     // [n_seqs][pieces][2] of the weights of p and of q
    double* chances;  // [n_seqs][pieces][warps]
};

struct Stat { float top, sum; int index, pad; };  // of a chunk or a row: largest logit, sum of exp((x - top) / T), lowest index of the largest

template <class E> struct Logit;
template <> struct Logit<__half> {
    static constexpr int kPerWord = 8;
    static constexpr uint32_t kMasked = 0xFC00FC00u;
    static __device__ __forceinline__ float at(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ void word(const uint4& w, float (&v)[8]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(u32_as_h2(u[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
};
template <> struct Logit<__nv_bfloat16> {
    static constexpr int kPerWord = 8;
    static constexpr uint32_t kMasked = 0xFF80FF80u;
    static __device__ __forceinline__ float at(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void word(const uint4& w, float (&v)[8]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
    }
};
template <> struct Logit<float> {
    static constexpr int kPerWord = 4;
    static constexpr uint32_t kMasked = 0xFF800000u;
    static __device__ __forceinline__ float at(const float* p) { return *p; }
    static __device__ __forceinline__ void word(const uint4& w, float (&v)[4]) {
        v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    }
};
__device__ __forceinline__ float known(float v) { return v == v ? v : kNone; }  // a logit that is not a number counts as masked

// A row of logits as words of 16 aligned bytes: word w holds the elements [w N - skew, (w + 1) N - skew) that lie in [0, vocab).
template <class E>
struct Row {
    static constexpr int N = Logit<E>::kPerWord;
    const E* row;
    int skew, vocab;
    __device__ __forceinline__ Row(const E* p, int v) : row(p), skew((int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(E))), vocab(v) {}
    __device__ __forceinline__ int words() const { return (skew + vocab + N - 1) / N; }
    __device__ __forceinline__ int index(int w) const { return w * N - skew; }
    // Elements of word w; outside the row: masked.
    __device__ __forceinline__ void load(int w, float (&v)[N]) const {
        const int i0 = index(w);
        if (i0 >= 0 && i0 + N <= vocab) {
            Logit<E>::word(__ldg(reinterpret_cast<const uint4*>(row + i0)), v);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i0 + i >= 0 && i0 + i < vocab ? Logit<E>::at(row + i0 + i) : kNone;
        }
    }
};

// Stretches of a row: as many as give every SM four CTAs (us of the whole with four | eight, 152k tokens: 8 sequences 36 | 37.5, 16 43 | 47,
// 48 87 | 89), of 1024 words at least and 16384 at most.
struct Stretches { int count, words; };
Stretches stretches_of(int rows, int vocab, int per_word) {
    const int words = (vocab + 2 * per_word - 2) / per_word, least = (words + 16383) / 16384, most = (words + 1023) / 1024;
    const int wanted = 592 / (rows > 0 ? rows : 1), count = wanted < least ? least : wanted > most ? most : wanted;
    return {count, (words + count - 1) / count};
}

// a and b joined: x = (difference of the maxima) log2(e) / T
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float scale) {
    if (b.top == kNone) return a;
    if (a.top == kNone) return b;
    Stat r;
    r.top = fmaxf(a.top, b.top);
    const float ka = a.top == r.top ? 1.f : exp2f((a.top - r.top) * scale), kb = b.top == r.top ? 1.f : exp2f((b.top - r.top) * scale);
    r.sum = a.sum * ka + b.sum * kb;
    r.index = a.top == r.top ? (b.top == r.top ? min(a.index, b.index) : a.index) : b.index;
    r.pad = 0;
    return r;
}
__device__ __forceinline__ Stat warp_join(Stat v, float scale) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stat w;
        w.top = __shfl_xor_sync(0xffffffffu, v.top, o);
        w.sum = __shfl_xor_sync(0xffffffffu, v.sum, o);
        w.index = __shfl_xor_sync(0xffffffffu, v.index, o);
        w.pad = 0;
        const bool low = (threadIdx.x & o) == 0;  // both lanes add the same two numbers in the same order
        v = low ? join(v, w, scale) : join(w, v, scale);
    }
    return v;
}
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int s) { return a.temperature ? a.temperature[s] : 1.f; }

template <class E>
__device__ __forceinline__ const E* logits_row(const VerifyArgs& a, bool draft, int s, int r, int j) {
    return draft ? static_cast<const E*>(a.draft) + (int64_t)j * a.draft_step_stride + (int64_t)s * a.draft_seq_stride : static_cast<const E*>(a.target) + (int64_t)r * a.target_stride;
}

template <class E>
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyArgs a, const Stretches stretches, const Draws draws) {
    constexpr int N = Logit<E>::kPerWord;
    __shared__ Stat warps[kStatThreads / 32];
    const int tid = threadIdx.x, y = blockIdx.x / stretches.count, stretch = blockIdx.x - y * stretches.count;
    const bool draft = y >= a.rows;
    const int r = draft ? y - a.rows : y;
    pdl_trigger();
    pdl_wait();
    int first = 0, end = 0, whole0 = 0, whole1 = 0;  // words of the stretch, and those of them that lie inside the row
    const uint4* words = nullptr;
    uint4 next[kStatWords];
    auto ask = [&](int w0) {
#pragma unroll
        for (int i = 0; i < kStatWords; ++i) {
            next[i] = make_uint4(Logit<E>::kMasked, Logit<E>::kMasked, Logit<E>::kMasked, Logit<E>::kMasked);
            if (w0 + i * kStatThreads < whole1) next[i] = __ldg(words + w0 + i * kStatThreads);
        }
    };
    auto open = [&](const E* p) {
        const Row<E> row(p, a.vocab);
        first = stretch * stretches.words;
        end = min(row.words(), first + stretches.words);
        whole0 = max(first, row.skew ? 1 : 0);
        whole1 = min(end, (row.skew + a.vocab) / N);
        words = reinterpret_cast<const uint4*>(row.row - row.skew);
        ask(whole0 + tid);
        return row;
    };
    // (a row of the target is on its way before it is known whose it is)
    Row<E> row(static_cast<const E*>(a.target), a.vocab);
    if (!draft) row = open(logits_row<E>(a, false, 0, r, 0));
    for (int i = blockIdx.x * kStatThreads + tid; i < a.n_seqs; i += gridDim.x * kStatThreads) draws.arrived[i] = 0;
    int start = 0;
    const int s = warp_find_seq(a.row_start, a.n_seqs, a.rows, r, &start);
    if (s < 0) return;
    const int n = min(max(a.row_start[s + 1], 0), a.rows) - start, j = r - start;
    if (j >= (draft ? min(n - 1, a.steps) : n)) return;
    const float T = temperature_of(a, s), scale = T > 0.f ? 1.4426950408889634f / T : 0.f;  // 0 with T = inf, too: all tokens alike
    if (draft) row = open(logits_row<E>(a, true, s, r, j));
    Stat mine = {kNone, 0.f, 0x7fffffff, 0};
    auto add = [&](auto& v, auto&& index) {  // v[i][e]: the logit at index(i) + e
        constexpr int K = sizeof(v) / sizeof(v[0]);
        float top = kNone;
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) top = fmaxf(top, v[i][e]);
        if (top == kNone) return;
        if (!(T > 0.f)) {  // only the largest counts
            if (top > mine.top) {
                mine.top = top;
                mine.index = 0x7fffffff;
#pragma unroll
                for (int i = 0; i < K; ++i)
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (v[i][e] == top) mine.index = min(mine.index, index(i) + e);
            } else if (top == mine.top) {  // (words at the ends of a row come out of order)
#pragma unroll
                for (int i = 0; i < K; ++i)
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (v[i][e] == top) mine.index = min(mine.index, index(i) + e);
            }
            return;
        }
        if (top > mine.top) {
            if (mine.top != kNone) mine.sum *= exp2_approx((mine.top - top) * scale);
            mine.top = top;
        }
        // (the difference first: the logits' products with 1 / T would be rounded by as much as the whole argument at a small T)
        const uint64_t scales = pair_of(scale, scale), minus = pair_of(-mine.top, -mine.top);
        uint64_t sums = 0ull;
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                float y0, y1;
                split(mul2(add2(pair_of(v[i][e], v[i][e + 1]), minus), scales), y0, y1);
                sums = add2(sums, pair_of(exp2_approx(y0), exp2_approx(y1)));
            }
        float sum[2];
        split(sums, sum[0], sum[1]);
        sum[0] += sum[1];
        if (sum[0] != sum[0]) {  // NaN counts as masked; infinities that are the largest share what there is
            sum[0] = 0.f;
#pragma unroll
            for (int i = 0; i < K; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[0] += v[i][e] == mine.top ? 1.f : known(v[i][e]) == kNone || mine.top == INFINITY ? 0.f : exp2_approx((v[i][e] - mine.top) * scale);
        }
        mine.sum += sum[0];
    };
    if (tid == 0 && first == 0 && whole0 > 0) {
        float v[1][N];
        row.load(0, v[0]);
        add(v, [&](int) { return row.index(0); });
    }
    if (tid == 0 && end == row.words() && whole1 < end && (end > 1 || whole0 == 0)) {
        float v[1][N];
        row.load(end - 1, v[0]);
        add(v, [&](int) { return row.index(end - 1); });
    }
#pragma unroll 1
    for (int w0 = whole0 + tid; w0 < whole1; w0 += kStatThreads * kStatWords) {
        float v[kStatWords][N];
#pragma unroll
        for (int i = 0; i < kStatWords; ++i) Logit<E>::word(next[i], v[i]);
        ask(w0 + kStatThreads * kStatWords);
        add(v, [&](int i) { return row.index(w0 + i * kStatThreads); });
    }
    mine = warp_join(mine, scale);
    if ((tid & 31) == 0) warps[tid >> 5] = mine;
    __syncthreads();
    if (tid < 32) {
        Stat w = tid < kStatThreads / 32 ? warps[tid] : Stat{kNone, 0.f, 0x7fffffff, 0};
        w = warp_join(w, scale);
        if (tid == 0) static_cast<Stat*>(a.stats)[(size_t)y * stretches.count + stretch] = w;
    }
}

// exp((x - top) / T) in fp64 to about 1e-13; rate = 1 / T.  With y = (top - x) / T >= 0 and k the whole number next to -256 y / ln 2, it is
// 2^(k / 256), from a table and an exponent, times exp(z), z = -y - k ln 2 / 256, |z| < 0.00136, of which the series' fourth power is below 2e-13.
constexpr int kTable = 256;
__device__ __forceinline__ double weight(float x, float top, double rate, const double* table) {
    constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: a sum's mantissa ends in whole numbers
    const double y = ((double)top - (double)x) * rate, t = fma(y, -369.32994629211595, kRound), z = fma(kRound - t, 0.0027076061740622863, -y);  // 256 / ln 2, ln 2 / 256
    const int k = __double2loint(t);
    const double p = table[k & (kTable - 1)], e = fma(p, fma(z * z, fma(z, 1.0 / 6.0, 0.5), z), p);
    const double scaled = __hiloint2double(__double2hiint(e) + ((k >> 8) << 20), __double2loint(e));
    // above 690 (as a pattern of bits; infinity and NaN too): under 1e-299, or one of the infinities that are the largest.  No branch: eight of these run side by side.
    return (uint32_t)__double2hiint(y) < 0x40859000u ? scaled : x == top ? 1.0 : 0.0;
}
__device__ __forceinline__ double not_below_zero(double v) { return __double2hiint(v) < 0 ? 0.0 : v; }

// What a sequence draws its token from: max(p - q, 0), or p.
template <class E>
struct Law {
    Row<E> p, q;
    float p_top, q_top;
    double scale, p_rate, q_rate;  // 1 / T; 1 / sum of the weights
    int without;                   // index that has no weight (a draft without probabilities), -1: none
    bool less;                     // q is taken off
    // What the elements of word w of p's row are drawn by (outside the row: 0).
    __device__ __forceinline__ void chances(int w, bool drop, const double* table, double (&c)[Row<E>::N]) const {
        constexpr int N = Row<E>::N;
        const int i0 = p.index(w);
        float v[N];
        p.load(w, v);
#pragma unroll
        for (int e = 0; e < N; ++e) c[e] = weight(v[e], p_top, scale, table) * p_rate;
        if (!drop) return;
        if (less) {
            if (q.skew == p.skew) {
                q.load(w, v);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = i0 + e >= 0 && i0 + e < p.vocab ? Logit<E>::at(q.row + i0 + e) : kNone;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) c[e] = not_below_zero(fma(-q_rate, weight(v[e], q_top, scale, table), c[e]));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (i0 + e == without) c[e] = 0.0;
        }
    }
};

// How far a sequence's drafts stand, and what the next token is drawn from.
struct Choice {
    int kept;
    float p_top, q_top;
    int token;  // kDraw, or what is known already: the largest logit's index, -1 where every token is masked
};
constexpr int kDraw = -2;
constexpr double kNothing = 1e-12;  // a whole of max(p - q, 0) that is only what equal chances differ by in fp64

__device__ __forceinline__ Stat row_stat(const VerifyArgs& a, const Stretches& stretches, bool draft, int r, float scale) {  // a warp's
    Stat v = {kNone, 0.f, 0x7fffffff, 0};
    const Stat* from = static_cast<const Stat*>(a.stats) + ((size_t)(draft ? a.rows : 0) + r) * stretches.count;
    for (int i = threadIdx.x & 31; i < stretches.count; i += 32) {
        const float4 w = __ldcg(reinterpret_cast<const float4*>(from) + i);
        v = join(v, Stat{w.x, w.y, __float_as_int(w.z), 0}, scale);
    }
    return warp_join(v, scale);
}
// Every thread of the CTA calls it: a warp a draft, `judged` of them, and then all of them the row that is drawn from.
template <class E>
__device__ __forceinline__ Choice choose(const VerifyArgs& a, const Stretches& stretches, int s, int start, int judged, const double* table) {
    __shared__ int fallen;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float T = temperature_of(a, s);
    const bool greedy = !(T > 0.f);
    const float scale_f = greedy ? 0.f : 1.4426950408889634f / T;
    const double scale = greedy ? 0.0 : 1.0 / (double)T;
    if (tid == 0) fallen = judged;
    __syncthreads();
    for (int j = warp; j < judged; j += kDrawWarps) {
        const int r = start + j, x = a.tokens[r + 1];
        const Stat p = row_stat(a, stretches, false, r, scale_f);
        bool stands = false;
        if (x >= 0 && x < a.vocab) {
            if (greedy) {
                stands = p.index == x;
            } else {
                const double px = p.sum > 0.f ? weight(Logit<E>::at(logits_row<E>(a, false, s, r, j) + x), p.top, scale, table) / (double)p.sum : 0.0;
                double qx = 1.0;
                if (a.draft) {
                    const Stat q = row_stat(a, stretches, true, r, scale_f);
                    qx = q.sum > 0.f ? weight(Logit<E>::at(logits_row<E>(a, true, s, r, j) + x), q.top, scale, table) / (double)q.sum : 0.0;
                }
                stands = (double)a.random[r] * qx < px;
            }
        }
        if (!stands && lane == 0) atomicMin(&fallen, j);
    }
    __syncthreads();
    Choice c;
    c.kept = fallen;
    const Stat p = row_stat(a, stretches, false, start + c.kept, scale_f);
    c.p_top = p.top;
    c.q_top = kNone;
    c.token = p.top == kNone ? -1 : greedy ? p.index : kDraw;
    if (c.token == kDraw && a.draft && c.kept < judged) c.q_top = row_stat(a, stretches, true, start + c.kept, scale_f).top;
    return c;
}

// A row's words in the order of (piece of the row, warp of the CTA that has it).
template <class E>
__device__ __forceinline__ int words_of(const Row<E>& row, int pieces, int piece, int warp, int& w1) {
    const int words = row.words(), each = (words + 32 * pieces * kDrawWarps - 1) / (32 * pieces * kDrawWarps) * 32, w0 = min(words, (piece * kDrawWarps + warp) * each);
    w1 = min(words, w0 + each);
    return w0;
}
__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ void fill_table(double* table) {
    for (int i = threadIdx.x; i < kTable; i += kDrawThreads) table[i] = exp2((double)i / kTable);
}
__device__ __forceinline__ int rows_of(const VerifyArgs& a, int s, int& start) {
    start = min(max(a.row_start[s], 0), a.rows);
    return min(max(a.row_start[s + 1], 0), a.rows) - start;
}
__device__ __forceinline__ int judged_of(const VerifyArgs& a, int n) { return min(n - 1, a.steps); }  // drafts of a sequence of n rows

// With a draft's probabilities: which drafts stand, and a piece's sums of the weights of p and q, where they are to be subtracted.
template <class E>
__global__ void __launch_bounds__(kDrawThreads, 3) verify_sums_kernel(const VerifyArgs a, const Stretches stretches, const Draws draws) {
    constexpr int N = Logit<E>::kPerWord;
    __shared__ double table[kTable], sums[2][kDrawWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, s = blockIdx.x / draws.pieces, piece = blockIdx.x - s * draws.pieces;
    fill_table(table);
    pdl_trigger();
    pdl_wait();
    int start;
    const int n = rows_of(a, s, start);
    if (n <= 0) return;
    const int judged = judged_of(a, n);
    const Choice c = choose<E>(a, stretches, s, start, judged, table);
    if (piece == 0 && tid == 0) draws.choice[s] = c;
    if (c.token != kDraw || c.kept == judged) return;
    const double scale = 1.0 / (double)temperature_of(a, s);
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
        const Row<E> row(logits_row<E>(a, side, s, start + c.kept, c.kept), a.vocab);
        const float top = side ? c.q_top : c.p_top;
        double sum = 0.0;
        int w1;
        const int w0 = words_of(row, draws.pieces, piece, warp, w1);
        if (top != kNone)
#pragma unroll 2
            for (int w = w0 + lane; w < w1; w += 32) {
                float v[N];
                row.load(w, v);
#pragma unroll
                for (int e = 0; e < N; ++e) sum += weight(v[e], top, scale, table);
            }
        sum = warp_total(sum);
        if (lane == 0) sums[side][warp] = sum;
    }
    __syncthreads();
    if (tid < 2) {
        double v = 0.0;
#pragma unroll
        for (int w = 0; w < kDrawWarps; ++w) v += sums[tid][w];
        draws.sums[((size_t)s * draws.pieces + piece) * 2 + tid] = v;
    }
}

// The next token.  Every warp leaves what its words of the row are drawn by; the last CTA of a sequence finds the warp in whose words the running
// sum passes u times the whole, and there the index.
template <class E>
__global__ void __launch_bounds__(kDrawThreads, 3) verify_pick_kernel(const VerifyArgs a, const Stretches stretches, const Draws draws) {
    constexpr int N = Logit<E>::kPerWord;
    __shared__ double table[kTable], upto_warp[kDrawWarps], part_at;
    __shared__ int last, first, with, part;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, s = blockIdx.x / draws.pieces, piece = blockIdx.x - s * draws.pieces;
    fill_table(table);
    pdl_trigger();
    pdl_wait();
    int start;
    const int n = rows_of(a, s, start);
    if (n <= 0) {
        if (piece == 0 && tid == 0) a.accepted[s] = 0;
        return;
    }
    const int judged = judged_of(a, n);
    Choice c;
    if (a.draft) {
        const float4 w = __ldcg(reinterpret_cast<const float4*>(draws.choice + s));
        c = {__float_as_int(w.x), w.y, w.z, __float_as_int(w.w)};
        __syncthreads();  // the table
    } else {
        c = choose<E>(a, stretches, s, start, judged, table);
    }
    const int r = start + c.kept;
    auto answer = [&](int token) {  // a warp's
        for (int i = lane; i < n; i += 32) a.out_tokens[start + i] = i < c.kept ? a.tokens[start + 1 + i] : i == c.kept ? token : -1;
        if (lane == 0) a.accepted[s] = c.kept;
    };
    if (c.token != kDraw) {
        if (piece == 0 && warp == 0) answer(c.token);
        return;
    }
    const bool less = c.kept < judged && a.draft;
    Law<E> law = {Row<E>(logits_row<E>(a, false, s, r, c.kept), a.vocab), Row<E>(logits_row<E>(a, less, s, r, c.kept), a.vocab), c.p_top, c.q_top,
                  1.0 / (double)temperature_of(a, s), 1.0, 0.0, c.kept < judged && !a.draft ? a.tokens[r + 1] : -1, less};
    if (less) {  // (without a draft's chances to take off, weights need no common measure)
        double x = 0.0, y = 0.0;
        for (int i = lane; i < draws.pieces; i += 32) {
            const double2 v = __ldcg(reinterpret_cast<const double2*>(draws.sums) + (size_t)s * draws.pieces + i);
            x += v.x;
            y += v.y;
        }
        x = warp_total(x);
        y = warp_total(y);
        law.p_rate = 1.0 / x;
        law.q_rate = y > 0.0 ? 1.0 / y : 0.0;
    }
    double* const by_warp = draws.chances + (size_t)s * draws.pieces * kDrawWarps;
    auto weigh = [&](int of, bool drop) {  // a piece's
        double sum = 0.0;
        int w1;
        const int w0 = words_of(law.p, draws.pieces, of, warp, w1);
#pragma unroll 1
        for (int w = w0 + lane; w < w1; w += 32) {
            double v[N];
            law.chances(w, drop, table, v);
#pragma unroll
            for (int e = 0; e < N; ++e) sum += v[e];
        }
        sum = warp_total(sum);
        if (lane == 0) __stcg(by_warp + of * kDrawWarps + warp, sum);
    };
    bool drop = less || law.without >= 0;
    weigh(piece, drop);
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(draws.arrived + s, 1) == draws.pieces - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    // ── the warp whose words have the border: a thread some of them in a row ──
    const int all = draws.pieces * kDrawWarps, each = (all + kDrawThreads - 1) / kDrawThreads, m0 = min(all, tid * each), m1 = min(all, m0 + each);
    double mine, before, total;
    for (;; drop = false) {
        mine = 0.0;
        for (int m = m0; m < m1; ++m) mine += __ldcg(by_warp + m);
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        before = __shfl_up_sync(0xffffffffu, incl, 1);
        if (lane == 0) before = 0.0;
        if (lane == 31) upto_warp[warp] = incl;
        if (tid == 0) { first = kDrawThreads; with = 0; }
        __syncthreads();
        total = 0.0;
#pragma unroll
        for (int w = 0; w < kDrawWarps; ++w) {
            if (w == warp) before += total;
            total += upto_warp[w];
        }
        if (total > (drop && less ? kNothing : 0.0) || !drop) break;
        for (int of = 0; of < draws.pieces; ++of) weigh(of, false);  // p - q leaves nothing: p, and this CTA alone
        __threadfence();
        __syncthreads();
    }
    const double chance = (double)a.random[start + n - 1] * total, none = INFINITY;
    if (mine > 0.0) {
        atomicMax(&with, tid);
        if (before + mine > chance) atomicMin(&first, tid);
    }
    __syncthreads();
    const bool past = first < kDrawThreads;
    if (tid == (past ? first : with)) {
        int part_with = m0;
        part = -1;
        part_at = none;  // behind every border: the last index with a weight
        for (int m = m0; m < m1; ++m) {
            const double v = __ldcg(by_warp + m);
            if (v > 0.0) part_with = m;
            if (part < 0 && past && v > 0.0 && before + v > chance) { part = m; part_at = before; }
            before += v;
        }
        if (part < 0) part = part_with;
    }
    __syncthreads();
    if (warp) return;
    if (!(total > 0.0)) {
        answer(-1);
        return;
    }
    double base = part_at;
    const bool behind = base == none;
    // ── the index, 32 words at a time ──
    int w1, found = -1, best = -1;
    for (int w = words_of(law.p, draws.pieces, part / kDrawWarps, part % kDrawWarps, w1); w < w1 && found < 0; w += 32) {
        double v[N], lane_sum = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = 0.0;
        if (w + lane < w1) law.chances(w + lane, drop, table, v);
        int lane_best = -1;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            lane_sum += v[e];
            if (v[e] > 0.0) lane_best = law.p.index(w + lane) + e;
        }
        double upto = lane_sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        double run = base + (upto - lane_sum);
        int hit = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            run += v[e];
            if (hit == 0x7fffffff && v[e] > 0.0 && run > chance && !behind) hit = law.p.index(w + lane) + e;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            hit = min(hit, __shfl_xor_sync(0xffffffffu, hit, o));
            lane_best = max(lane_best, __shfl_xor_sync(0xffffffffu, lane_best, o));
        }
        if (hit != 0x7fffffff) found = hit;
        if (lane_best >= 0) best = lane_best;
        base += __shfl_sync(0xffffffffu, upto, 31);
    }
    answer(found >= 0 ? found : best);
}

size_t padded(size_t bytes) { return (bytes + 15) & ~(size_t)15; }
size_t stats_bytes(int rows, const Stretches& stretches) { return (size_t)rows * stretches.count * sizeof(Stat); }
// Where the pieces of the rows that are drawn from leave their sums (memory null: the bytes only).
size_t draws_of(unsigned char* memory, int n_seqs, int vocab, int per_word, Draws* d) {
    const int words = (vocab + 2 * per_word - 2) / per_word, most = (words + kDrawThreads - 1) / kDrawThreads;
    const int wanted = n_seqs < kDrawCtas ? kDrawCtas / (n_seqs > 0 ? n_seqs : 1) : 1, turns = (most + wanted - 1) / wanted;  // of a warp over 32 words
    d->pieces = (most + turns - 1) / turns;
    size_t at = 0;
    auto room = [&](size_t bytes) {
        unsigned char* p = memory ? memory + at : nullptr;
        at += padded(bytes);
        return p;
    };
    d->choice = (Choice*)room((size_t)n_seqs * sizeof(Choice));
    d->arrived = (int*)room((size_t)n_seqs * sizeof(int));
    d->sums = (double*)room((size_t)n_seqs * d->pieces * 2 * sizeof(double));
    d->chances = (double*)room((size_t)n_seqs * d->pieces * kDrawWarps * sizeof(double));
    return at;
}

template <class Kernel, class... Args>
cudaError_t launch(const Launch& l, Kernel kernel, unsigned grid, int threads, Args... args) {
    const cudaError_t e = prefer_max_shared(kernel);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = l.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class E>
cudaError_t go(const Launch& l, const VerifyArgs& a) {
    const int rows = (a.draft ? 2 : 1) * a.rows;
    const Stretches stretches = stretches_of(rows, a.vocab, Logit<E>::kPerWord);
    Draws draws;
    draws_of(static_cast<unsigned char*>(a.stats) + stats_bytes(rows, stretches), a.n_seqs, a.vocab, Logit<E>::kPerWord, &draws);
    const unsigned pieces = (unsigned)a.n_seqs * (unsigned)draws.pieces;
    cudaError_t e = launch(l, verify_stats_kernel<E>, (unsigned)rows * (unsigned)stretches.count, kStatThreads, a, stretches, draws);
    if (e == cudaSuccess && a.draft) e = launch(l, verify_sums_kernel<E>, pieces, kDrawThreads, a, stretches, draws);
    if (e == cudaSuccess) e = launch(l, verify_pick_kernel<E>, pieces, kDrawThreads, a, stretches, draws);
    return e;
}

}  // namespace

size_t verify_workspace(LogitsType type, int n_seqs, int rows, int vocab, bool draft) {
    const int all = (draft ? 2 : 1) * rows, per_word = type == kLogitsF32 ? 4 : 8;
    Draws draws;
    return stats_bytes(all, stretches_of(all, vocab, per_word)) + draws_of(nullptr, n_seqs, vocab, per_word, &draws);
}

cudaError_t launch_verify(const Launch& l, LogitsType type, const VerifyArgs& a) {
    if (type == kLogitsF16) return go<__half>(l, a);
    if (type == kLogitsBf16) return go<__nv_bfloat16>(l, a);
    return go<float>(l, a);
}

}  // namespace smelt
