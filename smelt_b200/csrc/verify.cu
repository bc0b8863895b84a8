// Drafted tokens against the target's probabilities, from given random numbers.
//
// With p = softmax(target / T) and q = softmax(draft / T): draft x_j stands while u_j q_j(x_j) < p_j(x_j); at the first that does
// not the next token is drawn from max(p - q, 0), behind the last draft from p, as the first index whose running sum passes u times
// the whole.
//
// Two kernels.  verify_stats_kernel reads every row of logits once (the bytes that bound the operator): a CTA takes a stretch of one row
// and leaves its maximum, the sum of exp((x - max) / T) and the lowest index of the maximum, in fp32 (a chance's
// error of 1e-7 turns a draw that lies as near to it).  verify_draw_kernel: a cluster of eight CTAs a sequence joins
// the parts, finds the first draft that falls and reads that one row (of the target, and of the draft) again.  There a running
// sum over the vocabulary is compared with a number, and every index is a border: probabilities and sums are fp64, and all sums are added in
// the order of the vocabulary.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "paged.h"

namespace smelt {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatThreads = 256, kStatWords = 4;  // words of 16 bytes a thread has on their way at a time
constexpr int kCluster = 8, kDrawThreads = 512, kDrawWarps = kDrawThreads / 32;
constexpr float kNone = -INFINITY;

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
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = known(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i0 + i >= 0 && i0 + i < vocab ? known(Logit<E>::at(row + i0 + i)) : kNone;
        }
    }
};

// Stretches of a row: as many as give every SM eight CTAs, of 1024 words at least and 8192 at most.
struct Stretches { int count, words; };
Stretches stretches_of(int rows, int vocab, int per_word) {
    const int words = (vocab + 2 * per_word - 2) / per_word, least = (words + 8191) / 8192, most = (words + 1023) / 1024;
    const int wanted = 1184 / (rows > 0 ? rows : 1), count = wanted < least ? least : wanted > most ? most : wanted;
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

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <class E>
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyArgs a, const Stretches stretches) {
    constexpr int N = Logit<E>::kPerWord;
    __shared__ Stat warps[kStatThreads / 32];
    const int tid = threadIdx.x, y = blockIdx.x / stretches.count, stretch = blockIdx.x - y * stretches.count;
    const bool draft = y >= a.rows;
    const int r = draft ? y - a.rows : y;
    pdl_trigger();
    pdl_wait();
    int start = 0;
    const int s = warp_find_seq(a.row_start, a.n_seqs, a.rows, r, &start);
    if (s < 0) return;
    const int n = min(max(a.row_start[s + 1], 0), a.rows) - start, j = r - start;
    if (j >= n - (draft ? 1 : 0)) return;
    const float T = temperature_of(a, s), scale = T > 0.f ? 1.4426950408889634f / T : 0.f;
    const Row<E> row(logits_row<E>(a, draft, s, r, j), a.vocab);
    const int first = stretch * stretches.words, end = min(row.words(), first + stretches.words);
    const int whole0 = max(first, row.skew ? 1 : 0), whole1 = min(end, (row.skew + a.vocab) / N);  // words that lie inside the row
    Stat mine = {kNone, 0.f, 0x7fffffff, 0};
    auto add = [&](auto& v, auto&& index) {  // v[i][e]: the logit at index(i) + e
        constexpr int K = sizeof(v) / sizeof(v[0]);
        float top = kNone;
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) top = fmaxf(top, v[i][e]);
        if (top == kNone) return;
        if (scale == 0.f) {  // only the largest counts
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
            mine.sum *= exp2_approx((mine.top - top) * scale);
            mine.top = top;
        }
        const float minus = -mine.top * scale;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e & 1] += exp2_approx(fmaf(v[i][e], scale, minus));
        sum[0] += sum[1];
        sum[0] = fmaf(-0.69314718f * fmaf(mine.top, scale, minus), sum[0], sum[0]);  // what `minus` was rounded by, which every term has
        if (sum[0] != sum[0]) {  // NaN counts as masked; infinities that are the largest share what there is
            sum[0] = 0.f;
#pragma unroll
            for (int i = 0; i < K; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[0] += v[i][e] == mine.top ? 1.f : known(v[i][e]) == kNone ? 0.f : exp2_approx((v[i][e] - mine.top) * scale);
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
    const uint4* words = reinterpret_cast<const uint4*>(row.row - row.skew);
    uint4 next[kStatWords];
    auto ask = [&](int w0) {
#pragma unroll
        for (int i = 0; i < kStatWords; ++i) {
            next[i] = make_uint4(Logit<E>::kMasked, Logit<E>::kMasked, Logit<E>::kMasked, Logit<E>::kMasked);
            if (w0 + i * kStatThreads < whole1) next[i] = __ldg(words + w0 + i * kStatThreads);
        }
    };
    ask(whole0 + tid);
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

// exp((x - top) / T) in fp64 to about 1e-13; rate = 1 / T.  With y = (x - top) / T <= 0 and k the whole number next to 256 y / ln 2, it is
// 2^(k / 256), from a table and an exponent, times exp(z), z = y - k ln 2 / 256, |z| < 0.00136, of which the series' fourth power is below 2e-13.
constexpr int kTable = 256;
__device__ __forceinline__ double weight(float x, float top, double rate, const double* table) {
    if (top == INFINITY) return x == top ? 1.0 : 0.0;
    constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: a sum's mantissa ends in whole numbers
    const double y = ((double)x - (double)top) * rate, t = fma(y, 369.32994629211595, kRound), z = fma(t - kRound, -0.0027076061740622863, y);  // 256 / ln 2, ln 2 / 256
    if ((uint32_t)__double2hiint(y) >= 0xC0859000u) return 0.0;  // below -690 (as a pattern of bits; -inf and NaN too): under 1e-299
    const int k = __double2loint(t);
    const double p = table[k & (kTable - 1)], e = fma(p, fma(z * z, fma(z, 1.0 / 6.0, 0.5), z), p);
    return __hiloint2double(__double2hiint(e) + ((k >> 8) << 20), __double2loint(e));
}
__device__ __forceinline__ double not_below_zero(double v) { return __double2hiint(v) < 0 ? 0.0 : v; }

// What a sequence draws its token from: max(p - q, 0), or p.
template <class E>
struct Law {
    Row<E> p, q;
    float p_top, q_top;
    double p_rate, q_rate;         // 1 / sum of the weights
    int without;                   // index that has no weight (a draft without probabilities), -1: none
    bool less;                     // q is taken off
};

template <class E>
__global__ void __launch_bounds__(kDrawThreads, 2) __cluster_dims__(kCluster, 1, 1) verify_draw_kernel(const VerifyArgs a, const Stretches stretches) {
    constexpr int N = Logit<E>::kPerWord;
    __shared__ int fallen;
    __shared__ double table[kTable], warp_p[kDrawWarps], warp_q[kDrawWarps], cta_p, cta_q, warp_sums[kDrawWarps], cta_sum;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster.block_rank(), s = blockIdx.x / kCluster;
    for (int i = tid; i < kTable; i += kDrawThreads) table[i] = exp2((double)i / kTable);
    pdl_trigger();
    pdl_wait();
    const int start = min(max(a.row_start[s], 0), a.rows), n = min(max(a.row_start[s + 1], 0), a.rows) - start;
    if (n <= 0) {
        if (rank == 0 && tid == 0) a.accepted[s] = 0;
        return;  // the whole cluster does
    }
    const float T = temperature_of(a, s);
    const bool greedy = !(T > 0.f);
    const float scale_f = greedy ? 0.f : 1.4426950408889634f / T;
    const double scale = greedy ? 0.0 : 1.0 / (double)T;
    const Stat* stats = static_cast<const Stat*>(a.stats);
    auto row_stat = [&](bool draft, int r) {  // a warp's
        Stat v = {kNone, 0.f, 0x7fffffff, 0};
        const Stat* from = stats + ((size_t)(draft ? a.rows : 0) + r) * stretches.count;
        for (int i = lane; i < stretches.count; i += 32) {
            const float4 w = __ldcg(reinterpret_cast<const float4*>(from) + i);
            v = join(v, Stat{w.x, w.y, __float_as_int(w.z), 0}, scale_f);
        }
        return warp_join(v, scale_f);
    };
    if (tid == 0) fallen = n - 1;
    __syncthreads();
    // ── which drafts stand: a warp a draft, the same in every CTA of the cluster ──
    for (int j = warp; j < n - 1; j += kDrawWarps) {
        const int r = start + j, x = a.tokens[r + 1];
        const Stat p = row_stat(false, r);
        bool stands = false;
        if (x >= 0 && x < a.vocab) {
            if (greedy) {
                stands = p.index == x;
            } else {
                const double px = p.sum > 0.f ? weight(known(Logit<E>::at(logits_row<E>(a, false, s, r, j) + x)), p.top, scale, table) / (double)p.sum : 0.0;
                double qx = 1.0;
                if (a.draft) {
                    const Stat q = row_stat(true, r);
                    qx = q.sum > 0.f ? weight(known(Logit<E>::at(logits_row<E>(a, true, s, r, j) + x)), q.top, scale, table) / (double)q.sum : 0.0;
                }
                stands = (double)a.random[r] * qx < px;
            }
        }
        if (!stands && lane == 0) atomicMin(&fallen, j);
    }
    __syncthreads();
    const int kept = fallen, r = start + kept;
    const bool last = kept == n - 1;
    const Stat p = row_stat(false, r);
    auto answer = [&](int token) {  // a thread's
        for (int i = 0; i < n; ++i) a.out_tokens[start + i] = i < kept ? a.tokens[start + 1 + i] : i == kept ? token : -1;
        a.accepted[s] = kept;
    };
    if (greedy || p.top == kNone) {
        if (rank == 0 && tid == 0) answer(p.top == kNone ? -1 : p.index);
        return;  // the whole cluster does
    }
    const bool less = !last && a.draft != nullptr;
    Law<E> law = {Row<E>(logits_row<E>(a, false, s, r, kept), a.vocab), Row<E>(less ? logits_row<E>(a, true, s, r, kept) : logits_row<E>(a, false, s, r, kept), a.vocab),
                  p.top, 0.f, 0.0, 0.0, !last && !a.draft ? a.tokens[r + 1] : -1, less};
    if (less) law.q_top = row_stat(true, r).top;
    // the warp's words of a row, in order of (rank, warp)
    auto words_of = [&](const Row<E>& row, int& w1) {
        const int words = row.words(), each = (words + kCluster * kDrawWarps - 1) / (kCluster * kDrawWarps), w0 = (rank * kDrawWarps + warp) * each;
        w1 = min(words, w0 + each);
        return w0;
    };
    auto warp_total = [&](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    auto cta_total = [&](const double* sums) {  // of the warps, in order
        double v = 0.0;
#pragma unroll
        for (int w = 0; w < kDrawWarps; ++w) v += sums[w];
        return v;
    };
    // ── sums of the weights ──
    auto sum_row = [&](const Row<E>& row, float top) {
        double sum = 0.0;
        int w1;
        const int w0 = words_of(row, w1);
        if (top != kNone)
#pragma unroll 2
            for (int w = w0 + lane; w < w1; w += 32) {
                float v[N];
                row.load(w, v);
#pragma unroll
                for (int e = 0; e < N; ++e) sum += weight(v[e], top, scale, table);
            }
        return warp_total(sum);
    };
    law.p_rate = 1.0;  // without a draft's chances to take off, weights need no common measure
    if (less) {
        const double sp = sum_row(law.p, law.p_top), sq = sum_row(law.q, law.q_top);
        if (lane == 0) { warp_p[warp] = sp; warp_q[warp] = sq; }
        __syncthreads();
        if (tid == 0) {
            cta_p = cta_total(warp_p);
            cta_q = cta_total(warp_q);
        }
        cluster.sync();
        double x = 0.0, y = 0.0;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) { x += *cluster.map_shared_rank(&cta_p, c); y += *cluster.map_shared_rank(&cta_q, c); }
        law.p_rate = 1.0 / x;
        law.q_rate = y > 0.0 ? 1.0 / y : 0.0;
    }
    // What the elements of word w of p's row are drawn by (outside the row: 0).
    auto chances = [&](int w, bool drop, double (&c)[N]) {
        const int i0 = law.p.index(w);
        float v[N];
        law.p.load(w, v);
#pragma unroll
        for (int e = 0; e < N; ++e) c[e] = weight(v[e], law.p_top, scale, table) * law.p_rate;
        if (!drop) return;
        if (law.less) {
            if (law.q.skew == law.p.skew) {
                law.q.load(w, v);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = i0 + e >= 0 && i0 + e < a.vocab ? known(Logit<E>::at(law.q.row + i0 + e)) : kNone;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) c[e] = not_below_zero(fma(-law.q_rate, weight(v[e], law.q_top, scale, table), c[e]));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (i0 + e == law.without) c[e] = 0.0;
        }
    };
    int w1;
    const int w0 = words_of(law.p, w1);
    // ── max(p - q, 0); where that leaves nothing, p ──
    for (int drop = law.less || law.without >= 0 ? 1 : 0; drop >= 0; --drop) {
        double sum = 0.0;
        for (int w = w0 + lane; w < w1; w += 32) {
            double c[N];
            chances(w, drop, c);
#pragma unroll
            for (int e = 0; e < N; ++e) sum += c[e];
        }
        sum = warp_total(sum);
        if (lane == 0) warp_sums[warp] = sum;
        __syncthreads();
        if (tid == 0) cta_sum = cta_total(warp_sums);
        cluster.sync();
        double sums[kCluster], before = 0.0, total = 0.0;
        int owner = -1, last_with = -1;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) sums[c] = *cluster.map_shared_rank(&cta_sum, c);
#pragma unroll
        for (int c = 0; c < kCluster; ++c) total += sums[c];
        const double chance = (double)a.random[start + n - 1] * total;
        double run = 0.0;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
            const double x = sums[c];
            if (c == rank) before = run;
            run += x;
            if (x > 0.0) last_with = c;
            if (owner < 0 && run > chance) owner = c;
        }
        if (owner < 0) owner = last_with;
        cluster.sync();  // the sums have been read: they may be written again, and their CTA may end
        if (total > 0.0) {
            if (owner != rank) return;
            int mine = -1, with = -1;
            double at = before, at_mine = before;
#pragma unroll
            for (int w = 0; w < kDrawWarps; ++w) {
                if (warp_sums[w] > 0.0) with = w;
                if (mine < 0 && at + warp_sums[w] > chance) { mine = w; at_mine = at; }
                at += warp_sums[w];
            }
            if (mine < 0) {
                mine = with;
                at_mine = INFINITY;  // behind every border: the last index with a weight
            }
            if (warp != mine) return;
            // ── the index, 32 words at a time ──
            double base = at_mine;
            int found = -1, best = -1;
            for (int w = w0; w < w1 && found < 0; w += 32) {
                double c[N], lane_sum = 0.0;
#pragma unroll
                for (int e = 0; e < N; ++e) c[e] = 0.0;
                if (w + lane < w1) chances(w + lane, drop, c);
                int lane_best = -1;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    lane_sum += c[e];
                    if (c[e] > 0.0) lane_best = law.p.index(w + lane) + e;
                }
                double incl = lane_sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double x = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += x;
                }
                double run_e = base + (incl - lane_sum);
                int hit = 0x7fffffff;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    run_e += c[e];
                    if (hit == 0x7fffffff && c[e] > 0.0 && run_e > chance && at_mine != INFINITY) hit = law.p.index(w + lane) + e;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    hit = min(hit, __shfl_xor_sync(0xffffffffu, hit, o));
                    lane_best = max(lane_best, __shfl_xor_sync(0xffffffffu, lane_best, o));
                }
                if (hit != 0x7fffffff) found = hit;
                if (lane_best >= 0) best = lane_best;
                base += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) answer(found >= 0 ? found : best);
            return;
        }
    }
    if (rank == 0 && tid == 0) answer(-1);
}

template <class E>
cudaError_t go(const Launch& l, const VerifyArgs& a) {
    const int rows = (a.draft ? 2 : 1) * a.rows;
    const Stretches stretches = stretches_of(rows, a.vocab, Logit<E>::kPerWord);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * (unsigned)stretches.count);
    cfg.blockDim = dim3(kStatThreads);
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = l.pdl ? 1 : 0;
    cudaError_t e = prefer_max_shared(verify_stats_kernel<E>);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, verify_stats_kernel<E>, a, stretches);
    if (e == cudaSuccess) e = prefer_max_shared(verify_draw_kernel<E>);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned)a.n_seqs * kCluster);
    cfg.blockDim = dim3(kDrawThreads);
    return cudaLaunchKernelEx(&cfg, verify_draw_kernel<E>, a, stretches);
}

}  // namespace

size_t verify_workspace(LogitsType type, int rows, int vocab, bool draft) {
    const int all = (draft ? 2 : 1) * rows;
    return (size_t)all * stretches_of(all, vocab, type == kLogitsF32 ? 4 : 8).count * sizeof(Stat);
}

cudaError_t launch_verify(const Launch& l, LogitsType type, const VerifyArgs& a) {
    if (type == kLogitsF16) return go<__half>(l, a);
    if (type == kLogitsBf16) return go<__nv_bfloat16>(l, a);
    return go<float>(l, a);
}

}  // namespace smelt
