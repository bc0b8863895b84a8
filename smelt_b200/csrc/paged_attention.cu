// Attention of a packed batch over a paged cache and a prefix that all its sequences share.
//
//   out[r, h] = sum_k softmax_k(scale q[r, h] . K[k, h / ratio]) V[k, h / ratio]   over the keys that row r sees,
//
// with the running maximum and sum of the softmax, so that keys and values are read once.  This file has the streaming kernel for blocks
// of few columns (a column is a row and a query head of the group that shares a key head) and the kernel that joins shared items.
//
// paged_narrow_kernel: one CTA a SM, each warp with a stretch of the line of work (paged.h) of its own.  It takes 32 keys at a time as
// S^T = K Q^T and O^T += V^T P^T on mma.sync: the columns of the block are the narrow side of the product, so eight columns cost what one
// costs.  Rows come with cp.async, wherever their pages are, into a ring of the warp's own, 16 bytes more than their length apart, so
// that ldmatrix reads them without conflicts.  Nothing but the end of the stretch makes a warp wait for another: the ring runs on across
// items, and while one warp writes down an item or waits for the next one's queries the others keep the memory busy.  At the end the
// CTA joins what its warps have of the same item.
// P goes into the product as two 16-bit parts: the kernel waits for memory, and rounding P once would cost up to half a step of the
// 16-bit type.  Keys outside an item are not read (zeros), and a value row that is not finite reaches only the columns that see it; where an
// item's sums come out not finite, what infinite values make of them is put in afterwards (a part of P that is 0 times one is NaN).
// What several CTAs have of an item the last of them joins; with a prefix paged_merge_kernel does, behind the tensor-core kernel paged_join_kernel.
//
// Memory bounds it from some tens of MB on: 819 MB of two long sequences in 150 us (5.4 TB/s), 416 MB of a ragged batch in 82 (5.1 TB/s; a
// warp has 22 KB on its way, and 255 registers leave the SM eight warps).  Below that a call is a chain of waits, 10 to 15 us: the batch's
// lengths, page ids, first keys, the joins of warps and of CTAs.
#include "attention.cuh"
#include "paged_line.cuh"

namespace smelt {
namespace {

using namespace paged;
using attn::movmatrix_trans;
using attn::TileElem;

template <int D> constexpr int kWarps = D == 256 ? 4 : 8;
constexpr int kGroups = 2, kTile = 16 * kGroups;  // of 16 keys a tile: a chain of products, exchange and exponentials takes two as fast as one
template <int D, int NH> constexpr int kUnits = D == 64 ? (NH == 1 ? 10 : 8) : D == 128 ? (NH == 1 ? 5 : 4) : 5;  // of a warp's ring: the K or V rows of 16 keys each
template <int D> constexpr int kPitch = D * 2 + 16;
template <int D> constexpr int kUnitBytes = 16 * kPitch<D>;

// A warp's part of an item that it has not all of: from the steps before its stretch (0) or into those behind it (1).
struct Part { int valid, source, block, head, at, steps; };

template <int D, int NH>
constexpr size_t narrow_shared(int n_seqs) {  // rings (and at the end parts 1), parts 0, maxima and sums of both, rows of keys, parts, the batch
    return (size_t)kWarps<D> * (kUnits<D, NH> * kUnitBytes<D> + NH * 8 * (D + 1) * 4 + 2 * NH * 8 * 8 + kTile * 8 + 2 * sizeof(Part)) + batch_bytes(n_seqs);
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
constexpr uint32_t kHidden = 0x7FFFF00Du;  // a NaN of our own
// The largest weight is two to this power: an fp16 weight loses bits below 2^-14, and what many small ones add up to would be lost with them (a key
// that takes nearly all of the weight in front of thousands).  bf16 goes as far down as fp32.
template <class E> constexpr float kAbove = std::is_same<E, __half>::value ? 14.f : 0.f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }

template <class E> __device__ __forceinline__ E round_to(float v);
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class E> __device__ __forceinline__ bool pair_not_finite(uint32_t v) {  // a pair of values with an exponent of all ones
    constexpr uint32_t m = std::is_same<E, __half>::value ? 0x7C00u : 0x7F80u;
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
__device__ __noinline__ void weighted_sum_masked(uint32_t values, MaskedTile<D, NH>& m, int k0, int t) {
    for (int nh = 0; nh < NH; ++nh)
        for (int col = 0; col < 8; ++col) {
            const int from = (threadIdx.x & 28) | (col >> 1);
            const int lo = __shfl_sync(0xffffffffu, m.keys[nh][col & 1].lo, from), hi = __shfl_sync(0xffffffffu, m.keys[nh][col & 1].hi, from);
            auto sees = [&](int k) { return k >= lo && k < hi; };
            const int k = k0 + 2 * t;
            const uint32_t near = (sees(k) ? 0xffffu : 0u) | (sees(k + 1) ? 0xffff0000u : 0u), far = (sees(k + 8) ? 0xffffu : 0u) | (sees(k + 9) ? 0xffff0000u : 0u);
            for (int i = 0; i < D / 16; ++i) {
                uint32_t v[4];
                ldmatrix4_trans(v, values + 32 * i);
                float add[4] = {0.f, 0.f, 0.f, 0.f};
                TileElem<E>::mma(add, v[0] & near, v[1] & near, v[2] & far, v[3] & far, m.p[nh][0], m.p[nh][1]);
                TileElem<E>::mma(add, v[0] & near, v[1] & near, v[2] & far, v[3] & far, m.p[nh][2], m.p[nh][3]);
                if ((col >> 1) == t) { m.o[nh][i][col & 1] += add[col & 1]; m.o[nh][i][2 + (col & 1)] += add[2 + (col & 1)]; }
            }
        }
}

// Writes what an item's sums are where a value that a column sees is not finite, over what the warp has just written of the item: parts (part: [columns][D + 1]),
// sums beside a prefix or outputs (which stay NaN where the sum of weights l is).  In a function of its own and through memory, so that the sums' registers are not kept for it.
template <int D, int NH, class E>
__device__ __noinline__ void put_infinities(const PagedAttentionArgs& a, float* part, int source, int head, int row, int f0, int width, int from, int to, Range k0, Range k1, Range k2, Range k3,
                                           float l0, float l1, float l2, float l3) {
    const PagedArgs& c = a.c;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int32_t* table = source == 0 ? c.prefix_table : c.table + (size_t)(source - 1) * c.table_stride;
    Infinite<2 * NH> found;
    found.seen[0] = k0;
    found.seen[1] = k1;
    const float l[4] = {l0, l1, l2, l3};
    if constexpr (NH == 2) { found.seen[2] = k2; found.seen[3] = k3; }
    __syncwarp();
    for (int x = 0; x < D; x += 32) {
        look_for_infinities<E>(c, table, static_cast<const E*>(c.v) + (long long)head * c.head_stride + x, from, to, found);
        for (int col = 0; col < 2 * NH; ++col) {
            const int f = (col >> 1) * 8 + 2 * t + (col & 1), i = divide(f0 + f, c.ratio_div);
            if (f >= width) continue;
            const size_t out_head = head * c.ratio + f0 + f - i * c.ratio;
            for (int e = g; e < 32; e += 8) {
                if (!((found.pos[col] | found.neg[col]) >> e & 1u)) continue;
                const float v = found.sum(col, e, 0.f);
                if (part) part[f * (D + 1) + x + e] = v;
                else if (a.whole_o) a.whole_o[(((source == 0 ? (size_t)c.rows : 0) + row + i) * c.n_q + out_head) * D + x + e] = v;
                else if (l[col] == l[col]) static_cast<E*>(a.out)[(size_t)(row + i) * a.out_stride + out_head * D + x + e] = round_to<E>(v);
            }
        }
    }
}

template <int D> struct Sums { float v[D / 32]; };
template <int D> __device__ __forceinline__ Sums<D> load_part(const float* at, int lane) {  // a lane's values lie side by side
    Sums<D> s;
    if constexpr (D == 64) {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(at) + lane);
        s.v[0] = x.x; s.v[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(at) + lane * (D / 128) + i);
            s.v[4 * i] = x.x; s.v[4 * i + 1] = x.y; s.v[4 * i + 2] = x.z; s.v[4 * i + 3] = x.w;
        }
    }
    return s;
}
// A column's parts of an item, in the order of the line: where their sums and their maxima and sums of weights lie.
struct PartList {
    int n;
    const float *first, *others;  // part 0, part 1; the rest `stride` columns apart
    const float2 *first_ml, *others_ml;
    int stride;
    template <int D> __device__ __forceinline__ const float* at(int k) const { return k == 0 ? first : others + (size_t)(k - 1) * stride * D; }
    __device__ __forceinline__ const float2* ml(int k) const { return k == 0 ? first_ml : others_ml + (size_t)(k - 1) * stride; }
};
template <int D>
__device__ __forceinline__ PartList parts_from(const PagedLine& line, int slot0, int slot1, int n, int col) {
    const size_t at0 = (size_t)slot0 * line.columns + col, at1 = (size_t)slot1 * line.columns + col;
    return {n, line.slot_o + at0 * D, line.slot_o + at1 * D, line.slot_ml + at0, line.slot_ml + at1, 2 * line.columns};
}
template <int D>
__device__ __forceinline__ PartList shared_parts(const PagedLine& line, const Share& share, int at, int first, int last, int col) {
    return parts_from<D>(line, 2 * first + (at < share.cta_begin(first) ? 0 : 1), 2 * (first + 1), last - first + 1, col);
}
// One warp: the parts of two lists added up and written to a row of outputs.  A lane fetches a part's maximum and sum; then the parts' sums
// are added with their factors, eight on their way at a time.
template <int D, class E>
__device__ __forceinline__ void join_parts(const PartList& a, const PartList& b, E* out) {
    const int lane = threadIdx.x & 31, parts = a.n + b.n;
    float top = kLowest, l = 0.f, o[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] = 0.f;
#pragma unroll 1
    for (int base = 0; base < parts; base += 32) {
        const int k = base + lane;
        float2 ml = make_float2(kLowest, 0.f);
        if (k < parts) ml = __ldcg(k < a.n ? a.ml(k) : b.ml(k - a.n));
        const bool counts = ml.y != 0.f;  // a part that the row sees nothing of adds nothing, whatever its sums are
        const float m = fmaxf(top, warp_max(counts ? ml.x : kLowest)), mine = exp2_approx(top - m), factor = counts ? exp2_approx(ml.x - m) : 0.f;
        top = m;
        l = l * mine + warp_sum(counts ? ml.y * factor : 0.f);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= mine;
        const uint32_t used = __ballot_sync(0xffffffffu, counts);
        const int n = min(32, parts - base);
#pragma unroll 1
        for (int p = 0; p < n; p += 8) {
            Sums<D> v[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                const int q = base + p + y;
                if (p + y < n && (used >> (p + y) & 1u)) v[y] = load_part<D>(q < a.n ? a.at<D>(q) : b.at<D>(q - a.n), lane);
            }
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                const float w = __shfl_sync(0xffffffffu, factor, (p + y) & 31);
                if (p + y < n && (used >> (p + y) & 1u)) {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) o[i] += v[y].v[i] * w;
                }
            }
        }
    }
    const float rate = l > 0.f ? 1.f / l : l;  // l = 0: nothing was seen; NaN: what was seen is not a number
    uint32_t w[D / 64];
#pragma unroll
    for (int k = 0; k < D / 64; ++k) w[k] = l == 0.f ? 0u : TileElem<E>::pack(o[2 * k] * rate, o[2 * k + 1] * rate);
    out += lane * (D / 32);
    if constexpr (D == 64) *reinterpret_cast<uint32_t*>(out) = w[0];
    else if constexpr (D == 128) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <int D, int NH, class E>
__global__ void __launch_bounds__(kWarps<D> * 32, 1) paged_narrow_kernel(const __grid_constant__ PagedAttentionArgs a, const int which) {
    constexpr int W = kWarps<D>, THREADS = W * 32, NU = kUnits<D, NH>, UNIT = kUnitBytes<D>, PITCH = kPitch<D>, MT = D / 16, C = NH * 8;
    static_assert(kTile == 32, "a lane a key");
    static_assert(C * (D + 1) * 4 <= NU * UNIT && UNIT % 16 == 0, "parts 1 lie in the rings");
    extern __shared__ __align__(16) unsigned char smem[];
    float* fronts = reinterpret_cast<float*>(smem + (size_t)W * NU * UNIT);     // [W][C][D + 1]
    float2* state = reinterpret_cast<float2*>(fronts + W * C * (D + 1));        // [W][2][C]
    long long* rows_of = reinterpret_cast<long long*>(state + W * 2 * C);       // [W][kTile]
    Part* parts = reinterpret_cast<Part*>(rows_of + W * kTile);                 // [W][2]
    const PagedArgs& c = a.c;
    const PagedLine& line = a.line[which];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    long long* rows = rows_of + warp * kTile;
    pdl_trigger();
    pdl_wait();
    Batch batch;
    scan_line<THREADS>(c, line, a.window, batch, reinterpret_cast<unsigned char*>(parts + W * 2));
    const Share share(batch.cum[c.n_seqs + 1], line);
    if (a.counters)  // no join comes behind: blocks that see nothing get their zeros here
        for (int s = blockIdx.x * W + warp; s < c.n_seqs; s += gridDim.x * W) {
            const Seq seq = batch.seq(s);
            for (int b = 0, n = blocks_of(c, line, seq.n); b < n; ++b) {
                if (steps_of(block_keys(c, line, seq, b, a.window), line.keys)) continue;
                for (int f = b * line.columns; f < min((b + 1) * line.columns, seq.n * c.ratio); ++f) {
                    const int i = divide(f, c.ratio_div);
                    for (int h = 0; h < c.n_kv; ++h)
                        for (int d = 2 * lane; d < D; d += 64)
                            *reinterpret_cast<uint32_t*>(static_cast<E*>(a.out) + (size_t)(seq.row + i) * a.out_stride + (size_t)(h * c.ratio + f - i * c.ratio) * D + d) = 0u;
                }
            }
        }
    if ((int)blockIdx.x * W >= share.used) return;
    const int begin = share.begin(blockIdx.x * W + warp), end = share.begin(blockIdx.x * W + warp + 1);
    if (lane < 2) parts[warp * 2 + lane].valid = 0;

    if (begin < end) {
    // ── the ring: of every tile kGroups units of keys, then kGroups of values ──
    unsigned char* ring = smem + (size_t)warp * NU * UNIT;
    Cursor cur;
    cur.seek(c, line, a.window, batch, begin);
    Cursor ahead = cur;  // the step whose pages are looked up next
    bool more = false;   // there is a tile that is issued next
    int page = 0, slot = 0, head = 0;  // page and place of the lane's key of the tile that is issued next
    bool inside = false;               // ... which is one of the item's
    auto look_up = [&]() {
        inside = false;
        more = ahead.at < end;
        if (!more) return;
        const int key = (ahead.first + ahead.step) * kTile + lane;
        head = ahead.head;
        inside = key >= ahead.keys.lo && key < ahead.keys.hi;
        if (inside) {
            const int32_t* table = ahead.source == 0 ? c.prefix_table : c.table + (size_t)(ahead.source - 1) * c.table_stride;
            const int p = divide(key, c.page_div);
            slot = key - p * c.page_size;
            page = table[p];
        }
        ahead.advance(c, line, a.window, batch);
    };
    constexpr int LANES = D / 8 < 32 ? D / 8 : 32, TURN = 32 / LANES;  // lanes of a row of 16-byte pieces, rows of a turn of the warp
    const int turn_row = lane / LANES;
    const E *k_pool = static_cast<const E*>(c.k) + lane % LANES * 8, *v_pool = static_cast<const E*>(c.v) + lane % LANES * 8;
    const uint32_t ring_at = smem_u32(ring) + turn_row * PITCH + lane % LANES * 16;
    uint32_t there = 0;  // keys of the tile that are read; the others' rows are zeros
    bool tile = false;   // there is a tile that is issued
    auto issue_unit = [&](int w, int place) {  // unit w of a tile
        if (w == 0) {
            tile = more;
            bool take = inside && (uint32_t)page < (uint32_t)c.n_pages;
            if (inside && !take && c.err) atomicOr(c.err, KERR_BAD_PAGE);
            __syncwarp();  // the last tile's rows have been read by every lane: its last unit may have been issued just before
            rows[lane] = take ? (long long)page * c.page_stride + (long long)slot * c.token_stride + (long long)head * c.head_stride : 0;
            there = __ballot_sync(0xffffffffu, take);
            look_up();
        }
        if (!tile) return;
        __syncwarp();  // the rows are there, and the unit's last readers are through
        const E* pool = w < kGroups ? k_pool : v_pool;
        const uint32_t dst = ring_at + place * UNIT;
        const long long* row = rows + w % kGroups * 16 + turn_row;
        const uint32_t mine = there >> (w % kGroups * 16) & 0xffffu;
        if (mine == 0xffffu) {
#pragma unroll
            for (int i = 0; i < 16; i += TURN) cp_async16(dst + i * PITCH, pool + row[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i += TURN) cp_async16_or_zero(dst + i * PITCH, pool + row[i], mine >> (i + turn_row) & 1u);
        }
    };
    look_up();
    int issued = 0, issue_place = 0, freed = NU;  // the next unit to issue, its place in the ring, and up to which unit there is room

    const E* q = static_cast<const E*>(a.q);
    uint32_t qf[NH][D / 8];
    float m_run[NH][2], l_run[NH][2], o[NH][MT][4];
    Range keys[NH][2];  // of this thread's columns 2t, 2t + 1
    int clear_lo = 0, clear_hi = 0;  // every column of the block sees the keys [clear_lo, clear_hi)
    int use_place = 0;
    // ldmatrix: this lane's row of a tile of keys (as they are) and of values (turned)
    const uint32_t k_lane = smem_u32(ring) + ((lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + (lane >> 4) * 16;
    const uint32_t v_lane = smem_u32(ring) + ((lane & 7) + (lane >> 4) * 8) * PITCH + ((lane >> 3) & 1) * 16;
    auto seq_of = [&](int source) { return source == 0 ? Seq{0, batch.row[c.n_seqs], 0} : batch.seq(source - 1); };
    auto width_of = [&](const Cursor& x, const Seq& s) { return min(line.columns, s.n * c.ratio - x.block * line.columns); };
    auto load_queries = [&](const Cursor& x) {
        const Seq s = seq_of(x.source);
        const int width = width_of(x, s);
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
            const int f = x.block * line.columns + nh * 8 + g, i = divide(f, c.ratio_div);
            const E* row_q = q + (size_t)(s.row + i) * a.q_stride + (size_t)(x.head * c.ratio + f - i * c.ratio) * D + 2 * t;
            const bool live = nh * 8 + g < width;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) qf[nh][j] = live ? *reinterpret_cast<const uint32_t*>(row_q + 8 * j) : 0u;
        }
    };
    int unit[kGroups];  // places of the next units, which are there
    auto arrived = [&]() {  // in one place of the code: it is long, and short calls wait for instructions as for anything else
#pragma unroll 1
        for (; issued < freed; ++issued) {
            issue_unit(issued % (2 * kGroups), issue_place);
            cp_async_commit();
            if (++issue_place == NU) issue_place = 0;
        }
        cp_async_wait<NU - kGroups>();
        __syncwarp();
#pragma unroll
        for (int z = 0; z < kGroups; ++z) {
            unit[z] = use_place * UNIT;
            if (++use_place == NU) use_place = 0;
        }
        freed += kGroups;
    };

    if (cur.at < end) load_queries(cur);
    while (cur.at < end) {
        // ── an item: its columns' key ranges ──
        const Seq seq = seq_of(cur.source);
        const int f0 = cur.block * line.columns, width = width_of(cur, seq);
        auto range_of = [&](int f) -> Range {
            if (f >= width) return {0, 0};
            const int i = divide(f0 + f, c.ratio_div);
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
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nh][i][0] = o[nh][i][1] = o[nh][i][2] = o[nh][i][3] = 0.f;
        }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
            clear_lo = max(clear_lo, __shfl_xor_sync(0xffffffffu, clear_lo, off));
            clear_hi = min(clear_hi, __shfl_xor_sync(0xffffffffu, clear_hi, off));
        }
        const Cursor item = cur;
        const int item_at = cur.at - cur.step;  // the item's first step on the line

        // ── its steps in this warp's stretch: keys, then values ──
        uint32_t pb[kGroups][NH][4];
        bool clear = true, last = false;
        int k0 = 0;
#pragma unroll 1
        for (int phase = 0;; phase ^= 1) {
            arrived();
            if (phase == 0) {
                k0 = (cur.first + cur.step) * kTile;
                float s[kGroups][NH][4];
#pragma unroll
                for (int z = 0; z < kGroups; ++z)
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[z][nh][i] = 0.f;
#pragma unroll
                for (int j = 0; j < MT; ++j)
#pragma unroll
                    for (int z = 0; z < kGroups; ++z) {
                        uint32_t k[4];
                        ldmatrix4(k, k_lane + unit[z] + 32 * j);
#pragma unroll
                        for (int nh = 0; nh < NH; ++nh) TileElem<E>::mma(s[z][nh], k[0], k[1], k[2], k[3], qf[nh][2 * j], qf[nh][2 * j + 1]);
                    }
                clear = k0 >= clear_lo && k0 + kTile <= clear_hi;
                float top[NH][2];
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
                    for (int z = 0; z < kGroups; ++z)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[z][nh][i] *= a.scale2;
                            if (!clear) {  // NaN marks a key that the column does not see: a maximum passes it over
                                const int k = k0 + 16 * z + g + 8 * (i >> 1);
                                if (k < keys[nh][i & 1].lo || k >= keys[nh][i & 1].hi) s[z][nh][i] = __uint_as_float(kHidden);
                            }
                        }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        top[nh][x] = fmaxf(s[0][nh][x], s[0][nh][2 + x]);
#pragma unroll
                        for (int z = 1; z < kGroups; ++z) top[nh][x] = fmaxf(top[nh][x], fmaxf(s[z][nh][x], s[z][nh][2 + x]));
                    }
                }
                bool moved = false;
#pragma unroll
                for (int off = 4; off < 32; off <<= 1)
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                        for (int x = 0; x < 2; ++x) top[nh][x] = fmaxf(top[nh][x], __shfl_xor_sync(0xffffffffu, top[nh][x], off));
#pragma unroll
                for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        top[nh][x] -= kAbove<E>;
                        moved = moved || top[nh][x] > m_run[nh][x];
                    }
                if (__any_sync(0xffffffffu, moved)) {  // a new maximum: rare behind the first tiles
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float m = fmaxf(top[nh][x], m_run[nh][x]), keep = exp2_approx(m_run[nh][x] - m);
                            m_run[nh][x] = m;
                            l_run[nh][x] *= keep;
#pragma unroll
                            for (int i = 0; i < MT; ++i) { o[nh][i][x] *= keep; o[nh][i][2 + x] *= keep; }
                        }
                }
#pragma unroll
                for (int z = 0; z < kGroups; ++z)
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh) {
                        float p[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[i] = exp2_approx(s[z][nh][i] - m_run[nh][i & 1]);
                            if (!clear && __float_as_uint(s[z][nh][i]) == kHidden) p[i] = 0.f;
                        }
                        l_run[nh][0] += p[0] + p[2];
                        l_run[nh][1] += p[1] + p[3];
                        const uint32_t pa = TileElem<E>::pack(p[0], p[1]), pc = TileElem<E>::pack(p[2], p[3]);
                        const float2 fa = TileElem<E>::unpack(pa), fc = TileElem<E>::unpack(pc);
                        pb[z][nh][0] = movmatrix_trans(pa);
                        pb[z][nh][1] = movmatrix_trans(pc);
                        pb[z][nh][2] = movmatrix_trans(TileElem<E>::pack(p[0] - fa.x, p[1] - fa.y));
                        pb[z][nh][3] = movmatrix_trans(TileElem<E>::pack(p[2] - fc.x, p[3] - fc.y));
                    }
                last = cur.step + 1 == cur.steps || cur.at + 1 == end;
                cur.advance(c, line, a.window, batch);
                if (last && cur.at < end) load_queries(cur);  // of the next item, on their way meanwhile
            } else {
#pragma unroll
                for (int z = 0; z < kGroups; ++z) {
                    const uint32_t vu = v_lane + unit[z];
                    bool odd = false;
                    if (!clear) {
#pragma unroll 1
                        for (int i = 0; i < MT; ++i) {
                            uint32_t v[4];
                            ldmatrix4_trans(v, vu + 32 * i);
                            odd = odd || pair_not_finite<E>(v[0]) || pair_not_finite<E>(v[1]) || pair_not_finite<E>(v[2]) || pair_not_finite<E>(v[3]);
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
                            for (int i = 0; i < 4; ++i) rare.p[nh][i] = pb[z][nh][i];
#pragma unroll
                            for (int i = 0; i < MT; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) rare.o[nh][i][e] = o[nh][i][e];
                        }
                        weighted_sum_masked<D, NH, E>(vu, rare, k0 + 16 * z, t);
#pragma unroll
                        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                            for (int i = 0; i < MT; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[nh][i][e] = rare.o[nh][i][e];
                    } else {
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            uint32_t v[4];
                            ldmatrix4_trans(v, vu + 32 * i);
#pragma unroll
                            for (int nh = 0; nh < NH; ++nh) {
                                TileElem<E>::mma(o[nh][i], v[0], v[1], v[2], v[3], pb[z][nh][0], pb[z][nh][1]);
                                TileElem<E>::mma(o[nh][i], v[0], v[1], v[2], v[3], pb[z][nh][2], pb[z][nh][3]);
                            }
                        }
                    }
                }
                if (last) break;
            }
        }

        // ── the item's sums ──
        float odd[4] = {0.f, 0.f, 0.f, 0.f};  // NaN where a sum is not finite
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) odd[e] = fmaf(o[nh][i][e], 0.f, odd[e]);
        const bool infinite = __any_sync(0xffffffffu, odd[0] + odd[1] + odd[2] + odd[3] != 0.f);
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l_run[nh][x] += __shfl_xor_sync(0xffffffffu, l_run[nh][x], off);
        const bool before = item_at < begin, behind = item_at + item.steps > end;
        if (before || behind) {
            __syncwarp();  // behind: the ring has been read for the last time
            const int which_part = before ? 0 : 1;
            float* to = before ? fronts + warp * C * (D + 1) : reinterpret_cast<float*>(ring);
            if (lane == 0) parts[warp * 2 + which_part] = {1, item.source, item.block, item.head, item_at, item.steps};
#pragma unroll
            for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int col = nh * 8 + 2 * t + x;
                    if (g == 0) state[(warp * 2 + which_part) * C + col] = make_float2(m_run[nh][x], l_run[nh][x]);
                    if (col < width)
#pragma unroll
                        for (int i = 0; i < MT; ++i) { to[col * (D + 1) + 16 * i + g] = o[nh][i][x]; to[col * (D + 1) + 16 * i + 8 + g] = o[nh][i][2 + x]; }
                }
        } else if (a.whole_o) {
#pragma unroll
            for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int f = nh * 8 + 2 * t + x, i = divide(f0 + f, c.ratio_div);
                    if (f >= width) continue;
                    const size_t to = ((item.source == 0 ? (size_t)c.rows : 0) + seq.row + i) * c.n_q + item.head * c.ratio + f0 + f - i * c.ratio;
                    if (g == 0) a.whole_ml[to] = make_float2(m_run[nh][x], l_run[nh][x]);
#pragma unroll
                    for (int k = 0; k < MT; ++k) { a.whole_o[to * D + 16 * k + g] = o[nh][k][x]; a.whole_o[to * D + 16 * k + 8 + g] = o[nh][k][2 + x]; }
                }
        } else {
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) {
                float rate[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) rate[x] = l_run[nh][x] > 0.f ? 1.f / l_run[nh][x] : l_run[nh][x];
                const int f = nh * 8 + g, i = divide(f0 + f, c.ratio_div);  // after the turn this lane has two values of column g
                E* to = static_cast<E*>(a.out) + (size_t)(seq.row + i) * a.out_stride + (size_t)(item.head * c.ratio + f0 + f - i * c.ratio) * D + 2 * t;
#pragma unroll
                for (int k = 0; k < 2 * MT; ++k) {
                    const float v0 = o[nh][k >> 1][2 * (k & 1)], v1 = o[nh][k >> 1][2 * (k & 1) + 1];
                    const uint32_t w = movmatrix_trans(TileElem<E>::pack(l_run[nh][0] == 0.f ? 0.f : v0 * rate[0], l_run[nh][1] == 0.f ? 0.f : v1 * rate[1]));
                    if (f < width) *reinterpret_cast<uint32_t*>(to + 8 * k) = w;
                }
            }
        }
        if (infinite) {  // (worked out again, so that nothing more is kept over the item's steps)
            const Range of = item.source == 0 ? Range{batch.prefix_lo, c.prefix_length} : block_keys(c, line, seq_of(item.source), item.block, a.window);
            const int first = of.lo / kTile;
            put_infinities<D, NH, E>(a, before ? fronts + warp * C * (D + 1) : behind ? reinterpret_cast<float*>(ring) : nullptr, item.source, item.head, seq.row, f0, width,
                                     max((first + max(begin - item_at, 0)) * kTile, of.lo), min((first + min(end - item_at, item.steps)) * kTile, of.hi), keys[0][0], keys[0][1],
                                     keys[NH - 1][0], keys[NH - 1][1], l_run[0][0], l_run[0][1], l_run[NH - 1][0], l_run[NH - 1][1]);
        }
    }
    cp_async_wait<0>();
    }
    __syncthreads();

    // ── what the warps have of the same item, in order: a warp a column of an item ──
    const int cta_begin = share.cta_begin(blockIdx.x), cta_end = share.cta_begin(blockIdx.x + 1);
    const bool mine = lane < 2 * W && parts[lane & (2 * W - 1)].valid;  // lane p: part p
    const int at_mine = parts[lane & (2 * W - 1)].at;
    const uint32_t valid = __ballot_sync(0xffffffffu, mine), ahead_of_me = valid & ((1u << lane) - 1u);
    const int at_before = __shfl_sync(0xffffffffu, at_mine, ahead_of_me ? 31 - __clz(ahead_of_me) : 0);
    int turn = 0;
    Part edge[2] = {{0, 0, 0, 0, 0, 0}, {0, 0, 0, 0, 0, 0}};  // the items that this CTA shares with those in front and behind
    for (uint32_t first = __ballot_sync(0xffffffffu, mine && (!ahead_of_me || at_before != at_mine)); first; first &= first - 1u) {  // the first part of each item
        const int p0 = __ffs(first) - 1, p1 = first & (first - 1u) ? __ffs(first & (first - 1u)) - 1 : 32;
        const uint32_t members = valid & ~((1u << p0) - 1u) & (p1 < 32 ? (1u << p1) - 1u : 0xffffffffu);
        const Part part = parts[p0];
        const Seq seq = part.source == 0 ? Seq{0, batch.row[c.n_seqs], 0} : batch.seq(part.source - 1);
        const int f0 = part.block * line.columns, width = min(line.columns, seq.n * c.ratio - f0);
        const bool here = part.at >= cta_begin && part.at + part.steps <= cta_end;
        if (part.at < cta_begin) edge[0] = part;
        else if (!here) edge[1] = part;
        for (int f = 0; f < width; ++f) {
            if ((turn++ & (W - 1)) != warp) continue;
            const float2 ml = members >> lane & 1u ? state[lane * C + f] : make_float2(kLowest, 0.f);
            const bool counts = ml.y != 0.f;  // a part that the column sees nothing of adds nothing, whatever its sums are
            const float top = warp_max(counts ? ml.x : kLowest), factor = counts ? exp2_approx(ml.x - top) : 0.f, l = warp_sum(counts ? ml.y * factor : 0.f);
            float sum[D / 32];
#pragma unroll
            for (int k = 0; k < D / 32; ++k) sum[k] = 0.f;
            const uint32_t used = __ballot_sync(0xffffffffu, counts);
#pragma unroll 2
            for (uint32_t left = used; left; left &= left - 1u) {
                const int p = __ffs(left) - 1;
                const float w = __shfl_sync(0xffffffffu, factor, p);
                const float* from = (p & 1 ? reinterpret_cast<const float*>(smem + (size_t)(p >> 1) * NU * UNIT) : fronts + (p >> 1) * C * (D + 1)) + f * (D + 1) + lane;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) sum[k] += from[32 * k] * w;
            }
            const int ri = divide(f0 + f, c.ratio_div);
            const size_t out_row = seq.row + ri, out_head = part.head * c.ratio + f0 + f - ri * c.ratio;
            if (here && !a.whole_o) {
                const float rate = l > 0.f ? 1.f / l : l;  // l = 0: nothing was seen
                E* to = static_cast<E*>(a.out) + out_row * a.out_stride + out_head * D + lane;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) to[32 * k] = round_to<E>(sum[k] * rate);
            } else {
                const size_t to = here ? ((part.source == 0 ? (size_t)c.rows : 0) + out_row) * c.n_q + out_head : (size_t)(2 * blockIdx.x + (part.at < cta_begin ? 0 : 1)) * line.columns + f;
                float* o_to = (here ? a.whole_o : line.slot_o) + to * D + lane;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) o_to[32 * k] = sum[k];
                if (lane == 0) (here ? a.whole_ml : line.slot_ml)[to] = make_float2(top, l);
            }
        }
    }
    if (!a.counters || !(edge[0].valid || edge[1].valid)) return;
    // ── the last CTA of a shared item joins its parts; the item is counted at the CTA that it begins in ──
    __shared__ int join[2];
    __threadfence();
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            join[side] = 0;
            if (!edge[side].valid) continue;
            const int first = share.cta_of(edge[side].at), last = share.cta_of(edge[side].at + edge[side].steps - 1);
            if (atomicAdd(a.counters + first, 1) == last - first) {
                a.counters[first] = 0;
                join[side] = 1;
            }
        }
    }
    __syncthreads();
    __threadfence();
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
        if (!join[side]) continue;
        const Part part = side ? edge[1] : edge[0];
        const Seq seq = batch.seq(part.source - 1);
        const int f0 = part.block * line.columns, width = min(line.columns, seq.n * c.ratio - f0), first = share.cta_of(part.at), last = share.cta_of(part.at + part.steps - 1);
        for (int f = warp; f < width; f += W) {
            const int i = divide(f0 + f, c.ratio_div);
            join_parts<D, E>(shared_parts<D>(line, share, part.at, first, last, f), {0, nullptr, nullptr, nullptr, nullptr, 0},
                             static_cast<E*>(a.out) + (size_t)(seq.row + i) * a.out_stride + (size_t)(part.head * c.ratio + f0 + f - i * c.ratio) * D);
        }
    }
}

// ── the join ────────────────────────────────────────────────────────────────
// With a prefix: a warp some query heads of a row and key head, one or all of them: the parts of each one's item of the prefix and of its
// item of the sequence.  Looking for the sequence and its blocks costs more than the sums, so many rows have a warp do it once for a group's
// heads.
constexpr int kMergeWarps = 4;

template <int D, class E>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_merge_kernel(const __grid_constant__ PagedAttentionArgs a, const int heads) {
    const PagedArgs& c = a.c;
    const int lane = threadIdx.x & 31;
    const int id = blockIdx.x * kMergeWarps + (threadIdx.x >> 5), turns = c.n_q / heads, r = id / turns, h0 = (id - r * turns) * heads, head = divide(h0, c.ratio_div);
    const PagedLine &own = a.line[a.own_line], &ahead = a.line[a.prefix_line];
    pdl_trigger();
    pdl_wait();
    const int own_places = own.cum[c.n_seqs + 1], ahead_places = ahead.cum[c.n_seqs + 1], ahead_lo = ahead.cum[c.n_seqs + 2];  // (on their way while the sequence is looked for)
    if (ahead_lo == kDisordered || r >= c.rows || r >= first_row(c, c.n_seqs)) return;
    int start = 0;
    const int s = warp_find_seq(c.row_start, c.n_seqs, c.rows, r, &start);
    if (s < 0) return;
    const int own_at = own.cum[s + 1];
    const Seq seq = {start, max(first_row(c, s + 1) - start, 0), tokens_of(c, s)};
    const int i = r - start;
    if (i >= seq.n) return;
    // the parts of the item of this row and a head that begins at place `at`
    auto parts_of = [&](const PagedLine& line, int places, bool prefix, int h, int at, int steps, int col) -> PartList {
        if (steps == 0) return {0, nullptr, nullptr, nullptr, nullptr, 0};
        const Share share(places, line);
        const int first = share.cta_of(at), last = share.cta_of(at + steps - 1);
        if (first != last) return shared_parts<D>(line, share, at, first, last, col);
        const size_t to = ((prefix ? (size_t)c.rows : 0) + r) * c.n_q + h;
        return {1, a.whole_o + to * D, nullptr, a.whole_ml + to, nullptr, 0};
    };
    const int ahead_steps = steps_of({ahead_lo, c.prefix_length}, ahead.keys);
    int known = -1, steps = 0, before = 0;  // of the block that was looked at last
    for (int h = h0; h < h0 + heads; ++h) {
        const int g = h - head * c.ratio, f = i * c.ratio + g, block = divide(f, own.column_div);
        if (block != known) {
            known = block;
            steps = steps_of(block_keys(c, own, seq, block, a.window), own.keys);
            before = 0;
            if (block) {
                for (int b = lane; b < block; b += 32) before += c.n_kv * places_of(own, steps_of(block_keys(c, own, seq, b, a.window), own.keys));
#pragma unroll
                for (int k = 16; k > 0; k >>= 1) before += __shfl_xor_sync(0xffffffffu, before, k);
            }
        }
        const int af = r * c.ratio + g, ahead_block = divide(af, ahead.column_div);
        const PartList prefix = parts_of(ahead, ahead_places, true, h, (ahead_block * c.n_kv + head) * places_of(ahead, ahead_steps) + ahead.extra, ahead_steps, af - ahead_block * ahead.columns);
        const PartList mine = parts_of(own, own_places, false, h, own_at + before + head * places_of(own, steps) + own.extra, steps, f - block * own.columns);
        join_parts<D, E>(prefix, mine, static_cast<E*>(a.out) + (size_t)r * a.out_stride + (size_t)h * D);
    }
}

// Without one, behind the tensor-core kernel: the columns of the items that begin in a CTA of it and go on behind, shared out evenly.
constexpr int kJoinWarps = 8;
constexpr int kJoinCtas = 2;  // of an SM, with as many registers as the sums ask for (four, of 64: 1 us less of 120 at large calls, 4 more of 27 at small ones)

template <int D, class E>
__global__ void __launch_bounds__(kJoinWarps * 32, kJoinCtas) paged_join_kernel(const __grid_constant__ PagedAttentionArgs a) {
    __shared__ PagedShared items[kPagedCtas];
    __shared__ int owner[kPagedCtas], count[kPagedCtas / 32];
    static_assert(kPagedCtas == kJoinWarps * 32, "a thread a CTA");
    const PagedArgs& c = a.c;
    const PagedLine& line = a.line[0];
    const int tid = threadIdx.x, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    const PagedShared mine = tid < line.ctas ? line.shared[tid] : PagedShared{};
    const uint32_t some = __ballot_sync(0xffffffffu, mine.parts != 0);
    count[warp] = __popc(some);
    __syncthreads();
    int n = 0, at = __popc(some & ((1u << (tid & 31)) - 1u));
    for (int w = 0; w < kJoinWarps; ++w) {
        if (w < warp) at += count[w];
        n += count[w];
    }
    if (mine.parts) { items[at] = mine; owner[at] = tid; }
    __syncthreads();
    for (int k = blockIdx.x * kJoinWarps + warp; k < n * line.columns; k += gridDim.x * kJoinWarps) {
        const int which = divide(k, line.column_div), f = k - which * line.columns, first = owner[which];
        const PagedShared item = items[which];
        if (f >= item.width) continue;
        const int i = divide(item.f0 + f, c.ratio_div);
        join_parts<D, E>(parts_from<D>(line, 2 * first + 1, 2 * (first + 1), item.parts, f), {0, nullptr, nullptr, nullptr, nullptr, 0},
                         static_cast<E*>(a.out) + (size_t)(item.row + i) * a.out_stride + (size_t)(item.head * c.ratio + item.f0 + f - i * c.ratio) * D);
    }
}

template <class Kernel, class... Args>
cudaError_t launch(const Launch& l, Kernel kernel, dim3 grid, int threads, size_t shared, Args... args) {
    cudaError_t e = allow_shared(kernel, shared);
    if (e == cudaSuccess) e = prefer_max_shared(kernel);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
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
    const size_t shared = narrow_shared<D, NH>(a.c.n_seqs);
    if (type == kPagedF16) return launch(l, paged_narrow_kernel<D, NH, __half>, a.line[line].ctas, kWarps<D> * 32, shared, a, line);
    return launch(l, paged_narrow_kernel<D, NH, __nv_bfloat16>, a.line[line].ctas, kWarps<D> * 32, shared, a, line);
}

}  // namespace

int paged_narrow_columns(int head_dim, int64_t columns) { return columns <= 8 || head_dim == 256 ? 8 : 16; }
int paged_narrow_keys() { return 5; }
int paged_narrow_workers(int head_dim) { return head_dim == 256 ? kWarps<256> : kWarps<128>; }

cudaError_t launch_paged_narrow(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a, int line) {
    const int groups = a.line[line].columns / 8;
    if (head_dim == 64) return groups == 1 ? narrow<64, 1>(l, type, a, line) : narrow<64, 2>(l, type, a, line);
    if (head_dim == 128) return groups == 1 ? narrow<128, 1>(l, type, a, line) : narrow<128, 2>(l, type, a, line);
    return narrow<256, 1>(l, type, a, line);
}

cudaError_t launch_paged_merge(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a) {
    const int64_t all = (int64_t)a.c.rows * a.c.n_q;
    // A head a warp while 64 warps an SM hold them all, else a group (us of the call with a head | a group, 40 query and 8 key heads behind a prefix of
    // 2000: 100 rows 27 | 36, 200 37 | 41, 300 51 | 48, 1500 205 | 193).
    const int heads = all > (int64_t)a.line[0].ctas * 64 ? a.c.ratio : 1;
    const int grid = (int)((all / heads + kMergeWarps - 1) / kMergeWarps);
    auto go = [&](auto f16, auto bf16) { return type == kPagedF16 ? launch(l, f16, grid, kMergeWarps * 32, 0, a, heads) : launch(l, bf16, grid, kMergeWarps * 32, 0, a, heads); };
    if (head_dim == 64) return go(paged_merge_kernel<64, __half>, paged_merge_kernel<64, __nv_bfloat16>);
    if (head_dim == 128) return go(paged_merge_kernel<128, __half>, paged_merge_kernel<128, __nv_bfloat16>);
    return go(paged_merge_kernel<256, __half>, paged_merge_kernel<256, __nv_bfloat16>);
}

cudaError_t launch_paged_join(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a) {
    const int grid = kJoinCtas * a.line[0].ctas;
    auto go = [&](auto f16, auto bf16) { return type == kPagedF16 ? launch(l, f16, grid, kJoinWarps * 32, 0, a) : launch(l, bf16, grid, kJoinWarps * 32, 0, a); };
    if (head_dim == 64) return go(paged_join_kernel<64, __half>, paged_join_kernel<64, __nv_bfloat16>);
    if (head_dim == 128) return go(paged_join_kernel<128, __half>, paged_join_kernel<128, __nv_bfloat16>);
    return go(paged_join_kernel<256, __half>, paged_join_kernel<256, __nv_bfloat16>);
}

}  // namespace smelt
