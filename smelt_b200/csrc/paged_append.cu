// Queries and keys rotated by their positions, keys and values onto the pages of their sequences.
//
//   angle = position freq[pair],  (a, b) -> factor (a cos - b sin, b cos + a sin)
//
// for the pairs of the first rope_dim values of a head (adjacent values, or value i and value i + rope_dim / 2); the rest is copied.
// The angle is taken in turns, as a double: position (freq / 2 pi) less its nearest whole number, which is exact to 1e-16 of the angle
// however far the position is, and only what is left goes to 32 bits (float sincospi).  Products and sums are fp32, rounded once to the
// 16-bit type.
//
// A CTA takes one row, or two from 900 rows on (the chain row -> sequence -> length -> page and the sines are then paid for
// twice the bytes; us with one | two: 16 query and 4 key heads of 128, 600 rows 3.8 | 4.4, 900 5.3 | 5.3, 2400 8.9 | 7.8, 32768 114 | 91; 40 and 8 heads,
// 900 rows 6.9 | 7.7, 2400 18.2 | 18.5, 6000 37.8 | 36.7, 32768 182 | 170): a warp a row finds its sequence, all threads share the sines and cosines
// through shared memory, then a thread takes 16 bytes of a head and the 16 bytes they turn with.  Memory bounds it: 940 MB of 32768 rows go
// through in 170 us, 5.5 TB/s.
#include "attention.cuh"
#include "paged.h"

namespace smelt {
namespace {

using attn::TileElem;

constexpr int kThreads = 256, kMostRows = 2, kMostPairs = 128;

// Every eight pairs a gap of 16 bytes: the lanes of a load, 64 bytes apart, would meet in four banks.
__host__ __device__ constexpr int slot(int pair) { return pair + (pair >> 3) * 2; }

__device__ __forceinline__ float first_of(float a, float b, float2 t) { return __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y)); }
__device__ __forceinline__ float second_of(float a, float b, float2 t) { return __fadd_rn(__fmul_rn(b, t.x), __fmul_rn(a, t.y)); }

// WIDE: rows of 16 bytes that turn together with rows of 16 bytes (rope_dim a multiple of 8, in halves of 16)
template <int D, class E, bool HALVES, bool WIDE>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedAppendArgs a, const int rows_a_cta) {
    __shared__ __align__(16) float2 turn[kMostRows][slot(kMostPairs)];  // {cos, sin} factor of pair p at slot(p)
    __shared__ long long place[kMostRows];  // of the row's token in the pools (head 0), in elements; -1: nowhere, -2: not a row of the batch
    __shared__ int token[kMostRows];  // position, in tokens
    const PagedArgs& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, pairs = a.rope_dim / 2;
    const int row0 = blockIdx.x * rows_a_cta;
    pdl_trigger();
    pdl_wait();
    if (warp < rows_a_cta) {
        const int r = row0 + warp;
        const int total = min(c.row_start[c.n_seqs], c.rows);
        int start = 0;
        const int s = warp_find_seq(c.row_start, c.n_seqs, c.rows, r, &start);
        long long to = -2;
        int pos = 0;
        if (r < total && s >= 0) {
            const int n = min(max(c.row_start[s + 1], 0), c.rows) - start, i = r - start;
            if (i < n) {
                const int own = tokens_of(c, s) - n + i;  // [-n, table_tokens)
                to = -1;
                if (own >= 0) {
                    const int p = divide(own, c.page_div), page = c.table[(size_t)s * c.table_stride + p];
                    if ((uint32_t)page < (uint32_t)c.n_pages) to = (long long)page * c.page_stride + (long long)(own - p * c.page_size) * c.token_stride;
                }
                if (to < 0 && lane == 0 && c.err) atomicOr(c.err, KERR_BAD_PAGE);
                pos = a.position ? a.position[r] : c.prefix_length + max(own, 0);
            }
        }
        if (lane == 0) { place[warp] = to; token[warp] = pos; }
    }
    __syncthreads();
    for (int i = tid; i < rows_a_cta * pairs; i += kThreads) {
        const int r = i / pairs, p = i - r * pairs;
        const double turns = (double)token[r] * (a.freq[p] * 0.15915494309189533577);
        float sn, cs;
        sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
        turn[r][slot(p)] = make_float2(cs * a.factor, sn * a.factor);
    }
    __syncthreads();
    const int n_q = a.q ? c.n_q : 0, heads = n_q + c.n_kv;
    // a head of queries or keys: items that turn, then items that are copied
    constexpr int kItem = WIDE ? 8 : 2;  // values of an item's row of values
    const int turning = WIDE ? (HALVES ? a.rope_dim / 16 : a.rope_dim / 8) : pairs, rest = (D - a.rope_dim) / kItem, per_head = turning + rest;
    const int values = c.n_kv * (D / 8), items = heads * per_head + values;
    for (int r = 0; r < rows_a_cta; ++r) {
        const long long to = place[r];
        if (to == -2) continue;
        const size_t row = (size_t)(row0 + r);
#pragma unroll 2
        for (int i = tid; i < items; i += kThreads) {
            if (i >= heads * per_head) {
                if (to < 0) continue;
                const int j = i - heads * per_head, h = j / (D / 8), d = 8 * (j % (D / 8));
                const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const E*>(a.v_new) + row * a.v_stride + (size_t)h * D + d);
                *reinterpret_cast<uint4*>(static_cast<E*>(c.v) + to + (long long)h * c.head_stride + d) = v;
                continue;
            }
            const int h = i / per_head, j = i - h * per_head;
            const bool key = h >= n_q;
            if (key && to < 0) continue;
            const E* from = key ? static_cast<const E*>(a.k_new) + row * a.k_stride + (size_t)(h - n_q) * D : static_cast<const E*>(a.q) + row * a.q_stride + (size_t)h * D;
            E* dst = key ? static_cast<E*>(c.k) + to + (long long)(h - n_q) * c.head_stride : static_cast<E*>(a.q_out) + row * a.q_out_stride + (size_t)h * D;
            const float2* t = turn[r];
            if constexpr (WIDE) {
                if (j >= turning) {
                    const int d = a.rope_dim + 8 * (j - turning);
                    *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(from + d);
                } else if constexpr (HALVES) {
                    const int d = 8 * j;
                    const uint4 x = *reinterpret_cast<const uint4*>(from + d), y = *reinterpret_cast<const uint4*>(from + d + pairs);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
                    uint32_t u[4], w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 two = *reinterpret_cast<const float4*>(t + slot(d) + 2 * e);
                        const float2 p = TileElem<E>::unpack(xs[e]), q = TileElem<E>::unpack(ys[e]), t0 = make_float2(two.x, two.y), t1 = make_float2(two.z, two.w);
                        u[e] = TileElem<E>::pack(first_of(p.x, q.x, t0), first_of(p.y, q.y, t1));
                        w[e] = TileElem<E>::pack(second_of(p.x, q.x, t0), second_of(p.y, q.y, t1));
                    }
                    *reinterpret_cast<uint4*>(dst + d) = make_uint4(u[0], u[1], u[2], u[3]);
                    *reinterpret_cast<uint4*>(dst + d + pairs) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    const int d = 8 * j;
                    const uint4 x = *reinterpret_cast<const uint4*>(from + d);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
                    uint32_t u[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float4 two = *reinterpret_cast<const float4*>(t + slot(4 * j) + e);
                        const float2 p = TileElem<E>::unpack(xs[e]), q = TileElem<E>::unpack(xs[e + 1]), t0 = make_float2(two.x, two.y), t1 = make_float2(two.z, two.w);
                        u[e] = TileElem<E>::pack(first_of(p.x, p.y, t0), second_of(p.x, p.y, t0));
                        u[e + 1] = TileElem<E>::pack(first_of(q.x, q.y, t1), second_of(q.x, q.y, t1));
                    }
                    *reinterpret_cast<uint4*>(dst + d) = make_uint4(u[0], u[1], u[2], u[3]);
                }
            } else {
                const bool copied = j >= turning;
                const int d0 = copied ? a.rope_dim + 2 * (j - turning) : HALVES ? j : 2 * j, d1 = copied || !HALVES ? d0 + 1 : j + pairs;
                const E x = from[d0], y = from[d1];
                if (copied) {
                    dst[d0] = x;
                    dst[d1] = y;
                } else {
                    const float fx = (float)x, fy = (float)y;
                    const uint32_t v = TileElem<E>::pack(first_of(fx, fy, t[slot(j)]), second_of(fx, fy, t[slot(j)]));
                    reinterpret_cast<uint16_t*>(dst)[d0] = (uint16_t)v;
                    reinterpret_cast<uint16_t*>(dst)[d1] = (uint16_t)(v >> 16);
                }
            }
        }
    }
}

template <int D, class E>
cudaError_t go(const Launch& l, const PagedAppendArgs& a) {
    const int rows_a_cta = a.c.rows >= 900 ? kMostRows : 1;
    const bool halves = a.layout == 1, wide = halves ? a.rope_dim % 16 == 0 : a.rope_dim % 8 == 0;
    auto kernel = halves ? (wide ? paged_append_kernel<D, E, true, true> : paged_append_kernel<D, E, true, false>)
                         : (wide ? paged_append_kernel<D, E, false, true> : paged_append_kernel<D, E, false, false>);
    const cudaError_t e = prefer_max_shared(kernel);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.c.rows + rows_a_cta - 1) / rows_a_cta);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = l.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, rows_a_cta);
}

}  // namespace

cudaError_t launch_paged_append(const Launch& l, PagedType type, int head_dim, const PagedAppendArgs& a) {
    if (type == kPagedF16) return head_dim == 64 ? go<64, __half>(l, a) : head_dim == 128 ? go<128, __half>(l, a) : go<256, __half>(l, a);
    return head_dim == 64 ? go<64, __nv_bfloat16>(l, a) : head_dim == 128 ? go<128, __nv_bfloat16>(l, a) : go<256, __nv_bfloat16>(l, a);
}

}  // namespace smelt
