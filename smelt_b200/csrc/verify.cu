// Drafted tokens against the target's probabilities, from given random numbers.
//
// With p = softmax(target / T) and q = softmax(draft / T): draft x_j stands while u_j q_j(x_j) < p_j(x_j); at the first that does
// not the next token is drawn from max(p - q, 0), behind the last draft from p, as the first index whose running sum passes u times
// the whole.
//
// Two kernels.  verify_stats_kernel reads every row of logits once (the bytes that bound the operator): a CTA takes 1024 words of 16
// bytes of one row and leaves their maximum, the sum of exp((x - max) / T) and the lowest index of the maximum, in fp32 (a chance's
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

constexpr int kStatThreads = 256, kStatWords = 4;  // words of 16 bytes a thread
constexpr int kChunk = kStatThreads * kStatWords;
constexpr int kCluster = 8, kDrawThreads = 512, kDrawWarps = kDrawThreads / 32;
constexpr float kNone = -INFINITY;

struct Stat { float top, sum; int index, pad; };  // of a chunk or a row: largest logit, sum of exp((x - top) / T), lowest index of the largest

template <class E> struct Logit;
template <> struct Logit<__half> {
    static constexpr int kPerWord = 8;
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
    static __device__ __forceinline__ float at(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void word(const uint4& w, float (&v)[8]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
    }
};
template <> struct Logit<float> {
    static constexpr int kPerWord = 4;
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

__host__ __device__ inline int chunks_of(int vocab, int per_word) { return (vocab + 2 * per_word - 2) / per_word / kChunk + 1; }

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
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyArgs a, const int chunks) {
    constexpr int N = Logit<E>::kPerWord;
    __shared__ Stat warps[kStatThreads / 32];
    const int tid = threadIdx.x, chunk = blockIdx.x % chunks, y = blockIdx.x / chunks;
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
    const int words = row.words();
    float v[kStatWords][N];
    Stat mine = {kNone, 0.f, 0x7fffffff, 0};
#pragma unroll
    for (int i = 0; i < kStatWords; ++i) {
        const int w = chunk * kChunk + i * kStatThreads + tid;
        if (w < words) {
            row.load(w, v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[i][e] = kNone;
        }
    }
#pragma unroll
    for (int i = 0; i < kStatWords; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int at = row.index(chunk * kChunk + i * kStatThreads + tid) + e;
            if (v[i][e] > mine.top) { mine.top = v[i][e]; mine.index = at; }
        }
    if (mine.top != kNone && scale > 0.f) {
#pragma unroll
        for (int i = 0; i < kStatWords; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) mine.sum += v[i][e] == mine.top ? 1.f : v[i][e] == kNone ? 0.f : exp2f((v[i][e] - mine.top) * scale);
    }
    mine = warp_join(mine, scale);
    if ((tid & 31) == 0) warps[tid >> 5] = mine;
    __syncthreads();
    if (tid < 32) {
        Stat w = tid < kStatThreads / 32 ? warps[tid] : Stat{kNone, 0.f, 0x7fffffff, 0};
        w = warp_join(w, scale);
        if (tid == 0) static_cast<Stat*>(a.stats)[(size_t)y * chunks + chunk] = w;
    }
}

// exp((x - top) / T) in fp64; scale = log2(e) / T
__device__ __forceinline__ double weight(float x, float top, double scale) {
    return x == top ? 1.0 : x == kNone ? 0.0 : exp2(((double)x - (double)top) * scale);
}

// What a sequence draws its token from: max(p - q, 0), or p.
template <class E>
struct Law {
    Row<E> p, q;
    float p_top, q_top;
    double scale, p_rate, q_rate;  // rate: 1 / sum of the weights
    int without;                   // index that has no weight (a draft without probabilities), -1: none
    bool less;                     // q is taken off
};

template <class E>
__global__ void __launch_bounds__(kDrawThreads) __cluster_dims__(kCluster, 1, 1) verify_draw_kernel(const VerifyArgs a, const int chunks) {
    constexpr int N = Logit<E>::kPerWord;
    __shared__ int fallen;
    __shared__ double warp_p[kDrawWarps], warp_q[kDrawWarps], cta_p, cta_q, warp_sums[kDrawWarps], cta_sum;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster.block_rank(), s = blockIdx.x / kCluster;
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
    const double scale = greedy ? 0.0 : 1.4426950408889634074 / (double)T;
    const Stat* stats = static_cast<const Stat*>(a.stats);
    auto row_stat = [&](bool draft, int r) {  // a warp's
        Stat v = {kNone, 0.f, 0x7fffffff, 0};
        const Stat* from = stats + ((size_t)(draft ? a.rows : 0) + r) * chunks;
        for (int i = lane; i < chunks; i += 32) {
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
                const double px = p.sum > 0.f ? weight(known(Logit<E>::at(logits_row<E>(a, false, s, r, j) + x)), p.top, scale) / (double)p.sum : 0.0;
                double qx = 1.0;
                if (a.draft) {
                    const Stat q = row_stat(true, r);
                    qx = q.sum > 0.f ? weight(known(Logit<E>::at(logits_row<E>(a, true, s, r, j) + x)), q.top, scale) / (double)q.sum : 0.0;
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
                  p.top, 0.f, scale, 0.0, 0.0, !last && !a.draft ? a.tokens[r + 1] : -1, less};
    if (less) law.q_top = row_stat(true, r).top;
    // the warp's stretch of the vocabulary, in order of (rank, warp)
    const int stretch = (a.vocab + kCluster * kDrawWarps - 1) / (kCluster * kDrawWarps), v0 = min(a.vocab, (rank * kDrawWarps + warp) * stretch), v1 = min(a.vocab, v0 + stretch);
    // ── sums of the weights ──
    auto sum_row = [&](const Row<E>& row, float top) {
        double sum = 0.0;
        if (top == kNone) return sum;
        for (int w = (v0 + row.skew) / N + lane; row.index(w) < v1; w += 32) {
            float v[N];
            row.load(w, v);
            const int i0 = row.index(w);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (i0 + e >= v0 && i0 + e < v1) sum += weight(v[e], top, scale);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    };
    const double sp = sum_row(law.p, law.p_top), sq = less ? sum_row(law.q, law.q_top) : 0.0;
    if (lane == 0) { warp_p[warp] = sp; warp_q[warp] = sq; }
    __syncthreads();
    if (tid == 0) {
        double x = 0.0, y = 0.0;
        for (int w = 0; w < kDrawWarps; ++w) { x += warp_p[w]; y += warp_q[w]; }
        cta_p = x;
        cta_q = y;
    }
    cluster.sync();
    {
        double x = 0.0, y = 0.0;
        for (int c = 0; c < kCluster; ++c) { x += *cluster.map_shared_rank(&cta_p, c); y += *cluster.map_shared_rank(&cta_q, c); }
        law.p_rate = 1.0 / x;
        law.q_rate = y > 0.0 ? 1.0 / y : 0.0;
    }
    // The weights of 32 words that start at word w of p's row: this lane's, and 0 outside the stretch.
    auto chances = [&](int w, bool drop, double (&c)[N]) {
        const int i0 = law.p.index(w);
        float v[N];
        if (i0 < v1) law.p.load(w, v);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int i = i0 + e;
            c[e] = 0.0;
            if (i < v0 || i >= v1) continue;
            c[e] = weight(v[e], law.p_top, scale) * law.p_rate;
            if (!drop) continue;
            if (i == law.without) c[e] = 0.0;
        }
        if (drop && law.less && i0 < v1) {
            if (law.q.skew == law.p.skew) {
                law.q.load(w, v);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = i0 + e >= v0 && i0 + e < v1 ? known(Logit<E>::at(law.q.row + i0 + e)) : kNone;
            }
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (i0 + e >= v0 && i0 + e < v1) c[e] = fmax(c[e] - weight(v[e], law.q_top, scale) * law.q_rate, 0.0);
        }
    };
    // ── max(p - q, 0); where that leaves nothing, p ──
    for (int drop = law.less || law.without >= 0 ? 1 : 0; drop >= 0; --drop) {
        double sum = 0.0;
        const int w0 = (v0 + law.p.skew) / N;
        for (int w = w0 + lane; law.p.index(w) < v1; w += 32) {
            double c[N];
            chances(w, drop, c);
#pragma unroll
            for (int e = 0; e < N; ++e) sum += c[e];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) warp_sums[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            double x = 0.0;
            for (int w = 0; w < kDrawWarps; ++w) x += warp_sums[w];
            cta_sum = x;
        }
        cluster.sync();
        double before = 0.0, total = 0.0;
        int owner = -1, last_with = -1;
        for (int c = 0; c < kCluster; ++c) total += *cluster.map_shared_rank(&cta_sum, c);
        const double chance = (double)a.random[start + n - 1] * total;
        double run = 0.0;
        for (int c = 0; c < kCluster; ++c) {
            const double x = *cluster.map_shared_rank(&cta_sum, c);
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
            for (int w = w0; law.p.index(w) < v1 && found < 0; w += 32) {
                double c[N], lane_sum = 0.0;
                chances(w + lane, drop, c);
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
    const int chunks = chunks_of(a.vocab, Logit<E>::kPerWord);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.draft ? 2 : 1) * a.rows) * (unsigned)chunks);
    cfg.blockDim = dim3(kStatThreads);
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = l.pdl ? 1 : 0;
    cudaError_t e = prefer_max_shared(verify_stats_kernel<E>);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, verify_stats_kernel<E>, a, chunks);
    if (e == cudaSuccess) e = prefer_max_shared(verify_draw_kernel<E>);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned)a.n_seqs * kCluster);
    cfg.blockDim = dim3(kDrawThreads);
    return cudaLaunchKernelEx(&cfg, verify_draw_kernel<E>, a, chunks);
}

}  // namespace

size_t verify_workspace(LogitsType type, int rows, int vocab, bool draft) {
    return (size_t)(draft ? 2 : 1) * rows * chunks_of(vocab, type == kLogitsF32 ? 4 : 8) * sizeof(Stat);
}

cudaError_t launch_verify(const Launch& l, LogitsType type, const VerifyArgs& a) {
    if (type == kLogitsF16) return go<__half>(l, a);
    if (type == kLogitsBf16) return go<__nv_bfloat16>(l, a);
    return go<float>(l, a);
}

}  // namespace smelt
