// Attention of a packed batch over a paged cache and a prefix that all its sequences share.
//
//   out[r, h] = sum_k softmax_k(scale q[r, h] . K[k, h / ratio]) V[k, h / ratio]   over the keys that row r sees,
//
// with the running maximum and sum of the softmax, so that keys and values are read once.  This file has the streaming kernel for blocks
// of few columns (a column is a row and a query head of the group that shares a key head) and the kernel that joins shared items.
//
// paged_narrow_kernel: one CTA a SM, each with as many steps of the line of work (paged.h).  A warp takes 16 keys of a step at a time as
// S^T = K Q^T and O^T += V^T P^T on mma.sync (the tile arithmetic of attention.cuh): the columns of the block are the narrow side of the
// product, so eight columns cost what one costs.  A tile's K and V halves are copied row by row with cp.async into a ring of the
// warp's own and read back by the lanes that copied them; the ring runs on across items, so that the pages of the next sequence are on
// their way while this one's warps join their sums.
// P goes into the product as two 16-bit parts: the kernel waits for memory, and rounding P once would cost up to half a step of the
// 16-bit type.  Keys outside an item are not read (zero fill), and a value row that is not finite reaches only the columns that see it.
#include "attention.cuh"
#include "paged_line.cuh"

namespace smelt {
namespace {

using namespace paged;
using attn::movmatrix_trans;
using attn::TileElem;
using attn::tile_scores;
using attn::tile_weighted_sum;

template <int D> constexpr int kWarps = D == 256 ? 4 : 8;
template <int D> constexpr int kUnits = D == 64 ? 10 : 5;  // of a warp's ring: a K or V half of a 16-key tile each, 20 KB (40 KB) a warp
template <int D> constexpr int kUnitBytes = 16 * D * 2;

template <int D>
constexpr size_t narrow_shared(int n_seqs) {  // rings, one column group's sums of all warps, their maxima and sums, the batch
    return (size_t)kWarps<D> * kUnits<D> * kUnitBytes<D> + (size_t)kWarps<D> * 8 * D * 4 + (size_t)kWarps<D> * 8 * 8 + batch_bytes(n_seqs);
}

__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(take ? 16 : 0) : "memory");
}

template <class E> __device__ __forceinline__ E round_to(float v);
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class E> __device__ __forceinline__ bool pair_not_finite(uint32_t v) {  // a pair of values with an exponent of all ones
    constexpr uint32_t m = sizeof(E) == 2 && std::is_same<E, __half>::value ? 0x7C00u : 0x7F80u;
    return (v & m) == m || ((v >> 16) & m) == m;
}

// O^T += V^T P^T where some value is not finite and not every column sees every key: column by column, with the rows that it does not
// see taken as zero.
template <int D, int NH>
struct MaskedTile {
    float o[NH][D / 16][4];
    uint32_t p[NH][4];
    Range keys[NH][2];
};
template <int D, int NH, class E>
__device__ __noinline__ void weighted_sum_masked(const unsigned char* vu, MaskedTile<D, NH>& m, int k0, int t) {
    constexpr int VC = D / 64;
    for (int nh = 0; nh < NH; ++nh)
        for (int col = 0; col < 8; ++col) {
            const int from = (threadIdx.x & 28) | (col >> 1);
            const int lo = __shfl_sync(0xffffffffu, m.keys[nh][col & 1].lo, from), hi = __shfl_sync(0xffffffffu, m.keys[nh][col & 1].hi, from);
            uint32_t keep[4];
            const int mine[4] = {k0 + 2 * t, k0 + 2 * t + 1, k0 + 2 * t + 8, k0 + 2 * t + 9};
            for (int i = 0; i < 4; ++i) keep[i] = mine[i] >= lo && mine[i] < hi ? 0xffffffffu : 0u;
            for (int c = 0; c < VC; ++c) {
                uint32_t r[4][4];
                for (int i = 0; i < 4; ++i) {
                    const uint4 v = *reinterpret_cast<const uint4*>(vu + (4 * c + i) * 512);
                    r[i][0] = v.x & keep[i]; r[i][1] = v.y & keep[i]; r[i][2] = v.z & keep[i]; r[i][3] = v.w & keep[i];
                }
                for (int e = 0; e < 4; ++e) {
                    float add[4] = {0.f, 0.f, 0.f, 0.f};
                    const uint32_t a0 = __byte_perm(r[0][e], r[1][e], 0x5410), a1 = __byte_perm(r[0][e], r[1][e], 0x7632);
                    const uint32_t a2 = __byte_perm(r[2][e], r[3][e], 0x5410), a3 = __byte_perm(r[2][e], r[3][e], 0x7632);
                    TileElem<E>::mma(add, a0, a1, a2, a3, m.p[nh][0], m.p[nh][1]);
                    TileElem<E>::mma(add, a0, a1, a2, a3, m.p[nh][2], m.p[nh][3]);
                    if ((col >> 1) == t) { m.o[nh][4 * c + e][col & 1] += add[col & 1]; m.o[nh][4 * c + e][2 + (col & 1)] += add[2 + (col & 1)]; }
                }
            }
        }
}

template <int D, int NH, class E>
__global__ void __launch_bounds__(kWarps<D> * 32, 1) paged_narrow_kernel(const PagedAttentionArgs a, const int which) {
    constexpr int W = kWarps<D>, THREADS = W * 32, NU = kUnits<D>, UNIT = kUnitBytes<D>, KEYS = W * 16, MT = D / 16, KJ = D / 32, VC = D / 64;
    extern __shared__ __align__(16) unsigned char smem[];
    float* sums = reinterpret_cast<float*>(smem + (size_t)W * NU * UNIT);   // [W][8][D]
    float2* state = reinterpret_cast<float2*>(sums + W * 8 * D);            // [W][8]
    const PagedArgs& c = a.c;
    const PagedLine& line = a.line[which];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_trigger();
    pdl_wait();
    Batch batch;
    scan_line<THREADS>(c, line, a.window, batch, reinterpret_cast<unsigned char*>(state + W * 8));
    const long long total = batch.cum[c.n_seqs + 1];
    const int ctas = line_ctas(total, line.ctas);
    if ((int)blockIdx.x >= ctas) return;
    const long long begin = line_begin(total, blockIdx.x, ctas), end = line_begin(total, blockIdx.x + 1, ctas);
    const E* K = static_cast<const E*>(c.k);
    const E* V = static_cast<const E*>(c.v);

    // ── the ring: unit u holds K (even) or V (odd) of this warp's tile of step begin + u / 2 ──
    unsigned char* ring = smem + (size_t)warp * NU * UNIT + lane * 16;
    Cursor ahead;  // the step whose page is looked up next
    long long at = begin;
    ahead.seek(c, line, a.window, batch, begin);
    int page = -1, key = 0, head = 0;  // lane i (and i + 16): page of key i of the tile that is issued next, -1 where it is outside the item
    auto look_up = [&]() {
        page = -1;
        if (at >= end) return;
        key = (ahead.first + ahead.step) * KEYS + warp * 16 + (lane & 15);
        head = ahead.head;
        if (key >= ahead.keys.lo && key < ahead.keys.hi) {
            const int32_t* table = ahead.source == 0 ? c.prefix_table : c.table + (size_t)(ahead.source - 1) * c.table_stride;
            page = table[divide(key, c.page_div)];
            if ((uint32_t)page >= (uint32_t)c.n_pages) { page = -1; if (c.err && lane < 16) atomicOr(c.err, KERR_BAD_PAGE); }
        }
        if (++at < end) ahead.advance(c, line, a.window, batch);
    };
    long long row = 0;  // of lane's key, in elements; -1: none
    auto issue_unit = [&](int u) {
        unsigned char* dst = ring + (size_t)(u % NU) * UNIT;
        if ((u & 1) == 0) {
            row = page < 0 ? -1ll : (long long)page * c.page_stride + (long long)(key - divide(key, c.page_div) * c.page_size) * c.token_stride + (long long)head * c.head_stride;
            look_up();
            const long long ra = __shfl_sync(0xffffffffu, row, g), rb = __shfl_sync(0xffffffffu, row, g + 8);
            const E *pa = K + max(ra, 0ll) + 8 * t, *pb = K + max(rb, 0ll) + 8 * t;
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                cp_async16_or_zero(dst + (2 * j) * 512, pa + 32 * j, ra >= 0);
                cp_async16_or_zero(dst + (2 * j + 1) * 512, pb + 32 * j, rb >= 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long r = __shfl_sync(0xffffffffu, row, 2 * t + (i & 1) + 8 * (i >> 1));
                const E* p = V + max(r, 0ll) + 8 * g;
#pragma unroll
                for (int cc = 0; cc < VC; ++cc) cp_async16_or_zero(dst + (4 * cc + i) * 512, p + 64 * cc, r >= 0);
            }
        }
        cp_async_commit();
    };
    look_up();
    const int n_units = 2 * (int)(end - begin);
    int issued = 0;
    for (; issued < NU - 1; ++issued) {
        if (issued < n_units) issue_unit(issued);
        else cp_async_commit();
    }

    Cursor cur;
    cur.seek(c, line, a.window, batch, begin);
    const E* q = static_cast<const E*>(a.q);
    uint32_t qf[NH][D / 8];
    float m_run[NH][2], l_run[NH][2], o[NH][MT][4];
    Range keys[NH][2];  // of this thread's columns 2t, 2t + 1
    int clear_lo = 0, clear_hi = 0;  // every column of the block sees the keys [clear_lo, clear_hi)
    Seq seq{0, 0, 0};
    int width = 0;  // columns of the block
    unsigned used = 0;

    for (long long pos = begin; pos < end;) {
        // ── an item: its columns' queries and key ranges ──
        const int f0 = cur.block * line.columns;
        if (cur.source == 0) seq = {0, batch.row[c.n_seqs], 0};
        else seq = batch.seq(cur.source - 1);
        width = min(line.columns, seq.n * c.ratio - f0);
        auto range_of = [&](int f) -> Range {
            if (f >= width) return {0, 0};
            const int i = (f0 + f) / c.ratio;
            if (cur.source) return own_keys(seq, i, a.window);
            const Seq s = batch.seq(seq_of_row(batch, c.n_seqs, i));
            return prefix_keys(s, i - s.row, c.prefix_length, a.window);
        };
        clear_lo = 0;
        clear_hi = 0x7fffffff;
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                keys[nh][x] = range_of(nh * 8 + 2 * t + x);
                if (nh * 8 + 2 * t + x < width) { clear_lo = max(clear_lo, keys[nh][x].lo); clear_hi = min(clear_hi, keys[nh][x].hi); }
                m_run[nh][x] = kLowest;
                l_run[nh][x] = 0.f;
            }
            const int f = nh * 8 + g;
            if (f < width) {
                const E* row_q = q + (size_t)(seq.row + (f0 + f) / c.ratio) * a.q_stride + (size_t)(cur.head * c.ratio + (f0 + f) % c.ratio) * D + 8 * t;
#pragma unroll
                for (int j = 0; j < KJ; ++j) {
                    const uint4 v = *reinterpret_cast<const uint4*>(row_q + 32 * j);
                    qf[nh][4 * j] = v.x; qf[nh][4 * j + 1] = v.y; qf[nh][4 * j + 2] = v.z; qf[nh][4 * j + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < D / 8; ++j) qf[nh][j] = 0u;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nh][i][0] = o[nh][i][1] = o[nh][i][2] = o[nh][i][3] = 0.f;
        }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
            clear_lo = max(clear_lo, __shfl_xor_sync(0xffffffffu, clear_lo, off));
            clear_hi = min(clear_hi, __shfl_xor_sync(0xffffffffu, clear_hi, off));
        }
        const Cursor item = cur;
        const long long item_at = pos - cur.step;  // the item's first step on the line

        // ── its steps in this CTA's stretch ──
        for (;;) {
            const int k0 = (cur.first + cur.step) * KEYS + warp * 16;
            const int u = 2 * (int)used;
            const unsigned char *ku = ring + (size_t)(u % NU) * UNIT, *vu = ring + (size_t)((u + 1) % NU) * UNIT;
            const bool active = k0 < cur.keys.hi && k0 + 16 > cur.keys.lo;
            uint32_t pb[NH][4];
            // K half
            if (issued < n_units) issue_unit(issued);
            else cp_async_commit();
            ++issued;
            cp_async_wait<NU - 1>();
            __syncwarp();
            bool clear = true;
            if (active) {
                float s[NH][4];
                tile_scores<D, NH, E>(ku, qf, s);
                clear = k0 >= clear_lo && k0 + 16 <= clear_hi;
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) {
                    bool valid[4] = {true, true, true, true};
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!clear) {
                            const int k = k0 + g + 8 * (i >> 1);
                            valid[i] = k >= keys[nh][i & 1].lo && k < keys[nh][i & 1].hi;
                        }
                        v[i] = valid[i] ? s[nh][i] * a.scale2 : kLowest;
                    }
                    float p[4];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float top = fmaxf(v[x], v[2 + x]);
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                        top = fmaxf(top, m_run[nh][x]);
                        const float keep = exp2f(m_run[nh][x] - top);
                        m_run[nh][x] = top;
                        p[x] = valid[x] ? exp2f(v[x] - top) : 0.f;
                        p[2 + x] = valid[2 + x] ? exp2f(v[2 + x] - top) : 0.f;
                        l_run[nh][x] = l_run[nh][x] * keep + (p[x] + p[2 + x]);
#pragma unroll
                        for (int i = 0; i < MT; ++i) { o[nh][i][x] *= keep; o[nh][i][2 + x] *= keep; }
                    }
                    const uint32_t pa = TileElem<E>::pack(p[0], p[1]), pc = TileElem<E>::pack(p[2], p[3]);
                    const float2 fa = TileElem<E>::unpack(pa), fc = TileElem<E>::unpack(pc);
                    pb[nh][0] = movmatrix_trans(pa);
                    pb[nh][1] = movmatrix_trans(pc);
                    pb[nh][2] = movmatrix_trans(TileElem<E>::pack(p[0] - fa.x, p[1] - fa.y));
                    pb[nh][3] = movmatrix_trans(TileElem<E>::pack(p[2] - fc.x, p[3] - fc.y));
                }
            }
            // V half
            if (issued < n_units) issue_unit(issued);
            else cp_async_commit();
            ++issued;
            cp_async_wait<NU - 1>();
            __syncwarp();
            if (active) {
                bool odd = false;
                if (!clear) {
#pragma unroll
                    for (int i = 0; i < 4 * VC; ++i) {
                        const uint4 v = *reinterpret_cast<const uint4*>(vu + i * 512);
                        odd = odd || pair_not_finite<E>(v.x) || pair_not_finite<E>(v.y) || pair_not_finite<E>(v.z) || pair_not_finite<E>(v.w);
                    }
                    odd = __any_sync(0xffffffffu, odd);
                }
                if (odd) {
                    MaskedTile<D, NH> rare;  // a copy: what is passed by address does not stay in registers
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh) {
                        rare.keys[nh][0] = keys[nh][0];
                        rare.keys[nh][1] = keys[nh][1];
#pragma unroll
                        for (int i = 0; i < 4; ++i) rare.p[nh][i] = pb[nh][i];
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) rare.o[nh][i][e] = o[nh][i][e];
                    }
                    weighted_sum_masked<D, NH, E>(vu, rare, k0, t);
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nh][i][e] = rare.o[nh][i][e];
                } else {
                    uint32_t b0[NH], b1[NH], l0[NH], l1[NH];
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh) { b0[nh] = pb[nh][0]; b1[nh] = pb[nh][1]; l0[nh] = pb[nh][2]; l1[nh] = pb[nh][3]; }
                    tile_weighted_sum<D, NH, E>(vu, o, b0, b1, l0, l1);
                }
            }
            ++used;
            ++pos;
            if (pos >= end) break;
            cur.advance(c, line, a.window, batch);
            if (!cur.same_item(item)) break;
        }

        // ── the warps' sums, eight columns at a time ──
        const bool here = item_at >= begin && item_at + item.steps <= end;
        const int slot = 2 * blockIdx.x + (item_at < begin ? 0 : 1);
        for (int nh = 0; nh < NH; ++nh) {
            if (nh * 8 >= width) break;
#pragma unroll
            for (int n2 = 0; n2 < NH; ++n2)
                if (n2 == nh) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float l = l_run[n2][x];
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
                        if (g == 0) state[warp * 8 + 2 * t + x] = make_float2(m_run[n2][x], l);
                        float* to = sums + (size_t)(warp * 8 + 2 * t + x) * D;
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int j = 2 * i + h;
                                to[64 * (j >> 3) + 8 * g + (j & 7)] = o[n2][i][2 * h + x];
                            }
                    }
                }
            __syncthreads();
            const int n = min(8, width - nh * 8);
            for (int i = tid; i < n * D; i += THREADS) {
                const int col = i / D, d = i % D, f = nh * 8 + col;
                float top = kLowest, sum = 0.f, l = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) top = fmaxf(top, state[w * 8 + col].x);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float keep = exp2f(state[w * 8 + col].x - top);
                    l += state[w * 8 + col].y * keep;
                    sum += sums[(size_t)(w * 8 + col) * D + d] * keep;
                }
                const size_t out_row = seq.row + (f0 + f) / c.ratio, out_head = item.head * c.ratio + (f0 + f) % c.ratio;
                if (!here) {
                    line.slot_o[((size_t)slot * line.columns + f) * D + d] = sum;
                    if (d == 0) line.slot_ml[(size_t)slot * line.columns + f] = make_float2(top, l);
                } else if (a.whole_o) {
                    const size_t at_row = ((item.source == 0 ? (size_t)c.rows : 0) + out_row) * c.n_q + out_head;
                    a.whole_o[at_row * D + d] = sum;
                    if (d == 0) a.whole_ml[at_row] = make_float2(top, l);
                } else {
                    static_cast<E*>(a.out)[out_row * a.out_stride + out_head * D + d] = round_to<E>(l > 0.f ? sum / l : (l == 0.f ? 0.f : l));
                }
            }
            __syncthreads();
        }
    }
    cp_async_wait<0>();
}

// ── the join ────────────────────────────────────────────────────────────────
// A warp a row and query head: the parts of its item of the sequence and of its item of the prefix, in the order of the line.
constexpr int kMergeWarps = 4;

template <int D>
struct Joined {
    float top = kLowest, l = 0.f, o[D / 32];
    __device__ __forceinline__ Joined() {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
    }
    __device__ __forceinline__ void add(const float2 ml, const float* part, int lane) {
        if (ml.y == 0.f) return;  // sees nothing of the part, whatever its sums are
        float v[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) v[i] = __ldcg(part + lane + 32 * i);
        const float m = fmaxf(top, ml.x), mine = exp2f(top - m), theirs = exp2f(ml.x - m);
        top = m;
        l = l * mine + ml.y * theirs;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = o[i] * mine + v[i] * theirs;
    }
};

template <int D, class E>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_merge_kernel(const PagedAttentionArgs a) {
    const PagedArgs& c = a.c;
    const int lane = threadIdx.x & 31;
    const long long id = (long long)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
    pdl_trigger();
    pdl_wait();
    if (id >= (long long)c.rows * c.n_q) return;
    const int r = (int)(id / c.n_q), h = (int)(id % c.n_q), head = h / c.ratio;
    if (r >= first_row(c, c.n_seqs)) return;
    int start = 0;
    const int s = warp_find_seq(c.row_start, c.n_seqs, c.rows, r, &start);
    if (s < 0) return;
    const Seq seq = load_seq(c, s);
    const int i = r - seq.row;
    if (i >= seq.n) return;
    Joined<D> sum;
    for (int x = 0; x < a.lines; ++x) {
        const PagedLine& line = a.line[x];
        const long long total = line.cum[c.n_seqs + 1];
        const int ctas = line_ctas(total, line.ctas);
        for (int prefix = line.with_prefix ? 1 : 0; prefix >= 0; --prefix) {
            if (!prefix && !line.with_own) continue;
            // the item of this row and head: its first step on the line, and its steps
            const int f = prefix ? r * c.ratio + h % c.ratio : i * c.ratio + h % c.ratio;
            const int block = f / line.columns, col = f % line.columns;
            long long at = prefix ? 0 : line.cum[s + 1];
            int steps;
            if (prefix) {
                steps = steps_of({(int)line.cum[c.n_seqs + 2], c.prefix_length}, line.keys);
                at += (long long)block * c.n_kv * steps;
            } else {
                for (int b = lane; b < block; b += 32) at += (long long)c.n_kv * steps_of(block_keys(seq, b, line.columns, c.ratio, a.window), line.keys);
                const long long base = line.cum[s + 1];
                at -= base;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) at += __shfl_xor_sync(0xffffffffu, at, o);
                at += base;
                steps = steps_of(block_keys(seq, block, line.columns, c.ratio, a.window), line.keys);
            }
            if (steps == 0) continue;
            at += (long long)head * steps;
            const int first = line_owner(total, at, ctas), last = line_owner(total, at + steps - 1, ctas);
            if (first == last) {
                if (!a.whole_o) return;  // written by the CTA that finished it
                const size_t row = ((prefix ? (size_t)c.rows : 0) + r) * c.n_q + h;
                sum.add(__ldcg(a.whole_ml + row), a.whole_o + row * D, lane);
                continue;
            }
#pragma unroll 4
            for (int cta = first; cta <= last; ++cta) {
                const size_t slot = (size_t)(2 * cta + (at < line_begin(total, cta, ctas) ? 0 : 1)) * line.columns + col;
                sum.add(__ldcg(line.slot_ml + slot), line.slot_o + slot * D, lane);
            }
        }
    }
    E* out = static_cast<E*>(a.out) + (size_t)r * a.out_stride + (size_t)h * D;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) out[lane + 32 * k] = round_to<E>(sum.l > 0.f ? sum.o[k] / sum.l : (sum.l == 0.f ? 0.f : sum.l));
}

template <class Kernel, class... Args>
cudaError_t launch(const Launch& l, Kernel kernel, int grid, int threads, size_t shared, Args... args) {
    cudaError_t e = allow_shared(kernel, shared);
    if (e == cudaSuccess) e = prefer_max_shared(kernel);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = l.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D, int NH>
cudaError_t narrow(const Launch& l, PagedType type, const PagedAttentionArgs& a, int line) {
    const size_t shared = narrow_shared<D>(a.c.n_seqs);
    if (type == kPagedF16) return launch(l, paged_narrow_kernel<D, NH, __half>, a.line[line].ctas, kWarps<D> * 32, shared, a, line);
    return launch(l, paged_narrow_kernel<D, NH, __nv_bfloat16>, a.line[line].ctas, kWarps<D> * 32, shared, a, line);
}

}  // namespace

int paged_narrow_columns(int head_dim, int64_t columns) {
    const int most = head_dim == 256 ? 16 : 32;
    return columns <= 8 ? 8 : columns <= 16 ? 16 : most;
}
int paged_narrow_keys(int head_dim) { return (head_dim == 256 ? kWarps<256> : head_dim == 128 ? kWarps<128> : kWarps<64>) * 16; }

cudaError_t launch_paged_narrow(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a, int line) {
    const int groups = a.line[line].columns / 8;
    if (head_dim == 64) return groups == 1 ? narrow<64, 1>(l, type, a, line) : groups == 2 ? narrow<64, 2>(l, type, a, line) : narrow<64, 4>(l, type, a, line);
    if (head_dim == 128) return groups == 1 ? narrow<128, 1>(l, type, a, line) : groups == 2 ? narrow<128, 2>(l, type, a, line) : narrow<128, 4>(l, type, a, line);
    return groups == 1 ? narrow<256, 1>(l, type, a, line) : narrow<256, 2>(l, type, a, line);
}

cudaError_t launch_paged_merge(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a) {
    const long long warps = (long long)a.c.rows * a.c.n_q;
    const int grid = (int)((warps + kMergeWarps - 1) / kMergeWarps);
    auto go = [&](auto f16, auto bf16) { return type == kPagedF16 ? launch(l, f16, grid, kMergeWarps * 32, 0, a) : launch(l, bf16, grid, kMergeWarps * 32, 0, a); };
    if (head_dim == 64) return go(paged_merge_kernel<64, __half>, paged_merge_kernel<64, __nv_bfloat16>);
    if (head_dim == 128) return go(paged_merge_kernel<128, __half>, paged_merge_kernel<128, __nv_bfloat16>);
    return go(paged_merge_kernel<256, __half>, paged_merge_kernel<256, __nv_bfloat16>);
}

}  // namespace smelt
