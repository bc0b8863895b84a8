// Attention over pages for blocks of many columns (prompt chunks, drafts of wide groups, a prefix that a whole batch shares): the
// products on the fifth-generation tensor core.
//
// A block is up to 256 columns ((row, query head of the group) pairs of one key head; 128 with heads of 256) as two tiles of up to 128 lanes of
// tensor memory, whole rows where a group has no more than 128 heads, a step 128 keys (64).  Roles: four warps copy pages to shared memory (16-byte cp.async a row, so pages may have any size and strides;
// 128-byte swizzle), one warp issues the products S = Q K^T and O += P V, and two sets of four warps take a tile each: a thread has
// a column, so the softmax needs no exchange.  P overwrites S in tensor memory and is the product's operand from there.  While one
// set is at its exponentials (128 x 128 of them take the SM's 16 a clock 1024 clocks) the tensor core works for the other (1024 clocks a
// tile and step).  A block of 128 columns or fewer gives both sets the same tile and every other step, and their sums are joined at the
// end.  The maximum that P is relative to is the first step's, and moves only when a step's weights add up to more than 2^10 times the first step's largest: O is rescaled
// a few times an item at most, and behind the first step nobody looks for a maximum (1500 rows over 20000 tokens, as both were built: 594 us with it, 542 without).
// P is rounded once to the 16-bit type, the type of the values it is multiplied with; sums are fp32.  The streaming kernel, which waits for memory,
// multiplies with P in two parts and is as near to 64 bits as the rounded outputs are; here outputs are 1.2 to 1.35 times as far off (bf16, 4100
// tokens: 2.1e-3 of the norm against 1.6e-3), because a second part, rounded from what the first leaves, costs its products and as much again of the
// exponentials' warps: two ragged prompts of up to 1500 rows 172 | 225 us with one | two parts, 16 sequences of six drafts 30.6 | 36.3, 64 sequences behind a
// prefix of 8192 58.9 | 63.5.
//
// What bounds it: the way from a set's scores through its exponentials to its product and the next scores, 4000 clocks for two tiles and 128 keys, of
// which the tensor core works 2048 and the exponentials take as many beside it; the loads are hidden.  bf16, 40 query and 8 key heads of
// 128, pages of 32: 1500 rows over 20000 tokens in 527 us (1.12 PFLOP/s, 67 % of a library product's rate; 587 when a second of such calls has brought
// the clock down to what the power allows), 4 x 1500 rows over their own 1500 tokens in 191 (167 there; 136 with 32 query heads), where an item of six
// steps costs as much again for its beginning and end (lookups and first loads, the masked step, the sums).
//
// Value rows that are not finite and that not every column of the step sees are taken out of the product (as zeros) and added
// for the columns that see them alone, so that nothing reaches a row that it does not see.  An fp16 weight may round to 0, and 0 times infinity is
// NaN: where fp16 sums come out not finite, what infinite values make of them is put in afterwards.
#include <type_traits>

#include "attention.cuh"
#include "paged_line.cuh"
#include "tcgen05.cuh"

namespace smelt {
namespace {

using namespace paged;
using attn::TileElem;

template <int D>
struct Cfg {
    static constexpr int kSets = D == 256 ? 1 : 2;   // of four softmax warps, each with an accumulator of its own
    static constexpr int kKeys = D == 256 ? 64 : 128;
    static constexpr int kStages = D == 64 ? 3 : 2;
    static constexpr int kJoint = kSets == 2 ? 32 * 128 * 4 : 0;
    static constexpr int kQTile = 128 * D * 2, kTile = kKeys * D * 2;
    static constexpr int kLoadWarp = kSets * 4, kMmaWarp = kLoadWarp + 4, kThreads = (kMmaWarp + 4) * 32;
    // registers of a thread: the softmax holds a column's scores; 512 threads (384) are launched with 128 (168)
    static constexpr int kMany = kSets == 2 ? 192 : 232, kFew = kSets == 2 ? 64 : 120;
    static_assert(kSets * 128 * kMany + 256 * kFew <= kThreads * (65536 / kThreads / 8 * 8), "registers");
    static constexpr int kSum = 2 * kKeys;  // first column of the accumulators: behind two of scores
};

struct Shared {  // behind the tiles
    uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3], v_raw[3], s_full[2], p_ready[2], pv_done[2], q_full, q_empty;
    uint32_t tmem, dead;
    uint32_t keep[2];    // the first product of an item adds to what its set has put into the accumulator
    uint32_t odd[3][4];  // keys of a stage's step whose values are not finite, and were taken out
    float2 ml[2][128];
    long long row[2][128];  // of a step's keys in the pools, in elements (head 0); -1: none
};
template <int D>
constexpr size_t wide_shared(int n_seqs) {
    return (size_t)Cfg<D>::kSets * Cfg<D>::kQTile + 2 * Cfg<D>::kStages * Cfg<D>::kTile + Cfg<D>::kJoint + ((sizeof(Shared) + 15) & ~(size_t)15) + batch_bytes(n_seqs);
}

template <class E> struct Half16;  // of the products' 16-bit type: its code in a descriptor, its infinity, a value of it
template <> struct Half16<__half> {
    static constexpr uint32_t kType = 0u, kInf = 0x7C00u;
    static __device__ __forceinline__ float one(uint16_t v) { return __half2float(__ushort_as_half(v)); }
};
template <> struct Half16<__nv_bfloat16> {
    static constexpr uint32_t kType = (1u << 7) | (1u << 10), kInf = 0x7F80u;
    static __device__ __forceinline__ float one(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
};

// K-major operand: smem_desc_sw128 (tcgen05.cuh).  The values of a step are [key][64 values of a head] blocks of 128-byte rows: as the
// product's second operand that is the other major order, eight keys to an atom of 1024 bytes, the next 64 values one block further.
__device__ __forceinline__ uint64_t value_desc(uint32_t smem_addr, uint32_t block_bytes) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(block_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// D[128 x N] (+)= A[128 x 64] . B[64 x N], A from tensor memory, B values: four steps of 16 keys (2048 bytes).
__device__ __forceinline__ void umma_values_block(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, t;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
        "add.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}"
        ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
                   "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
                   "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(t)
                 : "memory");
}
// The lowest n bits.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// The loads behind v have arrived (v is named so that nothing is read of it earlier).
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                   "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]),
                   "+r"(v[29]), "+r"(v[30]), "+r"(v[31])::"memory");
}
// A column's scores, all on their way at once.
template <int KEYS> __device__ __forceinline__ void load_scores(uint32_t at, uint32_t (&v)[KEYS]) {
    uint32_t(&a)[KEYS / 32][32] = reinterpret_cast<uint32_t(&)[KEYS / 32][32]>(v);
#pragma unroll
    for (int x = 0; x < KEYS / 32; ++x) tmem_ld32(at + 32 * x, a[x]);
#pragma unroll
    for (int x = 0; x < KEYS / 32; ++x) tmem_wait_ld32(a[x]);
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// Not 0 where one of the eight values is not finite: an exponent of all ones, and one more, carries into the sign's place.
template <class E> __device__ __forceinline__ uint32_t not_finite(const uint4& w) {
    constexpr uint32_t m = Half16<E>::kInf * 0x10001u, one = (0x8000u - Half16<E>::kInf) * 0x10001u;
    return (((w.x & m) + one) | ((w.y & m) + one) | ((w.z & m) + one) | ((w.w & m) + one)) & 0x80008000u;
}

// What every role knows of an item.
struct Item {
    Seq seq;        // of the prefix: all rows
    int f0, width;  // first column of the block among the source's, and how many it has
    Range clear;    // keys that every column sees
};
__device__ __forceinline__ Item item_of(const PagedArgs& c, const PagedLine& line, uint32_t window, const Batch& b, const Cursor& cur) {
    Item it;
    it.seq = cur.source == 0 ? Seq{0, b.row[c.n_seqs], 0} : b.seq(cur.source - 1);
    it.f0 = cur.block * line.columns;
    it.width = min(line.columns, it.seq.n * c.ratio - it.f0);
    // of the prefix: without a window all columns, but for rows without a token, whose sums are dropped
    it.clear = cur.source ? Range{own_keys(it.seq, divide(it.f0 + it.width - 1, c.ratio_div), window).lo, own_keys(it.seq, divide(it.f0, c.ratio_div), window).hi} : window ? Range{0, 0} : Range{0, c.prefix_length};
    return it;
}

// 32 bytes; whole: on a boundary of as many
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8], bool whole) {
    if (whole) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
}

template <int REGS> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

// What the tensor maps read: boxes of `tokens` tokens, of which `boxes` make a step, and all query heads of a group of q_rows rows, which
// make a tile (0: a tile is 128 columns, from wherever in a row, and is copied column by column).
struct Pages {
    CUtensorMap k, v, q;
    int tokens, boxes, q_rows;
};

// TILED: pages come as boxes of a tensor map; else row by row.
template <int D, class E, bool TILED>
__global__ void __launch_bounds__(Cfg<D>::kThreads, 1) paged_wide_kernel(const __grid_constant__ PagedAttentionArgs a, const int which, const __grid_constant__ Pages pages) {
    using C = Cfg<D>;
    constexpr int KEYS = C::kKeys, S = C::kStages, CHUNKS = D / 8;  // 16-byte chunks of a row
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char *q_tiles = raw, *k_tiles = q_tiles + C::kSets * C::kQTile, *v_tiles = k_tiles + S * C::kTile;
    float* joint = reinterpret_cast<float*>(v_tiles + S * C::kTile);  // what the set of the other steps has, at the end of an item: [32][128]
    Shared& sh = *reinterpret_cast<Shared*>(reinterpret_cast<unsigned char*>(joint) + C::kJoint);
    const PagedArgs& c = a.c;
    const PagedLine& line = a.line[which];
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    volatile uint32_t* dead = &sh.dead;
    if (tid == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&sh.k_full[i], TILED ? 1 : 4); mbar_init(&sh.v_full[i], TILED ? 1 : 4); mbar_init(&sh.v_raw[i], 1);
            mbar_init(&sh.k_empty[i], 1); mbar_init(&sh.v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.s_full[i], 1); mbar_init(&sh.p_ready[i], 4); mbar_init(&sh.pv_done[i], 1); }
        mbar_init(&sh.q_full, 1);
        mbar_init(&sh.q_empty, 1);
        sh.dead = 0;
        if (TILED) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&pages.k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&pages.v) : "memory");
        }
        mbar_fence_init();
        fence_async_smem();
    }
    if (warp == C::kMmaWarp) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    pdl_trigger();
    pdl_wait();
    Batch batch;
    scan_line<C::kThreads>(c, line, a.window, batch, reinterpret_cast<unsigned char*>(&sh) + ((sizeof(Shared) + 15) & ~(size_t)15));
    tc_fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)sh.tmem);
    const Share share(batch.cum[c.n_seqs + 1], line);
    const int begin = share.cta_begin(blockIdx.x), end = share.cta_begin(blockIdx.x + 1);
    // A role that gives up a wait goes through the rest of its schedule without work, so that no barrier is short of a thread.
    bool alive = true;
    const int tile_columns = C::kSets == 2 ? line.columns >> 1 : line.columns;
    // An item's steps in this CTA: tasks, one a step, or with two tiles one a tile and step; task T of the CTA has score buffer T & 1.
    auto each_item = [&](auto&& body) {
        if (begin >= end) return;
        Cursor cur;
        cur.seek(c, line, a.window, batch, begin);
        uint32_t task = 0, step = 0;
        while (cur.at < end) {
            const int n = min(cur.steps - cur.step, end - cur.at);
            const Item it = item_of(c, line, a.window, batch, cur);
            const bool pair = it.width > tile_columns;
            const int tasks = pair ? 2 * n : n;
            body(cur, it, pair, n, tasks, task, step);
            task += tasks;
            step += n;
            cur.next_item(c, line, a.window, batch);
        }
    };

    if (warp >= C::kLoadWarp) {
    registers_down<C::kFew>();
    if (warp < C::kMmaWarp) {
        // ── pages to shared memory ──
        const int lt = tid - C::kLoadWarp * 32;
        constexpr int LANES = CHUNKS < 32 ? CHUNKS : 32, ROWS = 128 / LANES;  // lanes of a row, rows of a turn of the four warps
        const int ch = lt % LANES, r_first = lt / LANES;
        auto place = [](int rows, int row, int chunk) { return (uint32_t)((chunk >> 3) * rows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)); };
        auto warp_wait = [&](uint64_t* bar, uint32_t parity) { alive = __all_sync(0xffffffffu, alive && wait_alive_short(smem_u32(bar), parity, smem_u32(&sh.dead))) != 0; };
        auto arrive = [&](uint64_t* bar) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // Lanes of a tile behind its columns: no box writes their rows, and scores of what lies there by chance would look like new maxima.
        for (int i = 0; i < C::kSets; ++i)
            for (int f = tile_columns + r_first; f < 128; f += ROWS)
                for (int k = ch; k < CHUNKS; k += LANES) *reinterpret_cast<uint4*>(q_tiles + i * C::kQTile + place(128, f, k)) = make_uint4(0, 0, 0, 0);
        fence_async_smem();
        barrier(1, 128);  // the queries' barrier is passed on by one thread
        uint32_t items = 0;
        int v_behind = -1;        // stage of the values that were asked for last and not handed over yet
        bool v_check = false;     // ... that not every column sees all of
        Range v_rows = {0, KEYS}; // ... rows that are the item's (TILED)
        uint32_t v_bad = 0, raw_uses = 0;  // ... boxes whose page is none; parity of v_raw by stage
        auto zero_row = [&](unsigned char* tile, int r) {
            for (int k = ch; k < CHUNKS; k += LANES) *reinterpret_cast<uint4*>(tile + place(KEYS, r, k)) = make_uint4(0, 0, 0, 0);
        };
        auto hand_over_values = [&] {
            if (v_behind < 0) return;
            unsigned char* tile = v_tiles + v_behind * C::kTile;
            if (TILED) {
                warp_wait(&sh.v_raw[v_behind], raw_uses >> v_behind & 1u);
                raw_uses ^= 1u << v_behind;
                if (v_rows.lo > 0 || v_rows.hi < KEYS || v_bad)
                    for (int r = r_first; r < KEYS; r += ROWS)
                        if (r < v_rows.lo || r >= v_rows.hi || (v_bad >> (r / pages.tokens) & 1u)) zero_row(tile, r);
            }
            if (v_check) {
                barrier(1, 128);  // the stage's words of odd keys are zero
#pragma unroll 1
                for (int r0 = r_first; r0 < KEYS; r0 += 4 * ROWS) {
                    uint32_t odd[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) odd[i] = not_finite<E>(*reinterpret_cast<const uint4*>(tile + place(KEYS, r0 + i * ROWS, ch)));
                    if (__any_sync(0xffffffffu, odd[0] | odd[1] | odd[2] | odd[3]))
                        for (int i = 0; i < 4; ++i)
                            if (odd[i]) atomicOr(&sh.odd[v_behind][(r0 + i * ROWS) >> 5], 1u << ((r0 + i * ROWS) & 31));
                }
                barrier(1, 128);
                for (int r = r_first; r < KEYS; r += ROWS)
                    if (sh.odd[v_behind][r >> 5] >> (r & 31) & 1u) zero_row(tile, r);
            }
            if (TILED) {
                fence_async_smem();
                barrier(1, 128);
                if (lt == 0) mbar_arrive(&sh.v_full[v_behind]);
            } else {
                arrive(&sh.v_full[v_behind]);
            }
            v_behind = -1;
        };
        uint32_t all_steps = 0;
        each_item([&](const Cursor& cur, const Item& it, bool pair, int n, int, uint32_t, uint32_t step0) {
            // queries.  Where pages come as boxes the values before them are handed over behind this item's first keys: looking
            // through them would hold those up.
            if (!TILED) {
                cp_async_wait<0>();
                hand_over_values();
            }
            if (items > 0) warp_wait(&sh.q_empty, (items - 1) & 1);
            ++items;
            if (pages.q_rows) {
                if (warp == C::kLoadWarp && lane == 0 && alive) {
                    const int tiles = pair ? 2 : 1, row = it.seq.row + divide(it.f0, c.ratio_div);
                    arrive_expect_at(smem_u32(&sh.q_full), tiles * tile_columns * D * 2);
                    for (int i = 0; i < tiles; ++i)
#pragma unroll
                        for (int x = 0; x < D / 64; ++x)
                            tma_load_4d_at(smem_u32(q_tiles + i * C::kQTile) + x * (128 * 128), &pages.q, 64 * x, cur.head * c.ratio, row + i * pages.q_rows, 0, smem_u32(&sh.q_full));
                }
            } else if (alive) {
                for (int f = r_first; f < (pair ? 256 : 128); f += ROWS) {
                    const int ff = it.f0 + f, i = divide(ff, c.ratio_div);
                    const bool live = f < it.width;
                    const E* from = static_cast<const E*>(a.q) + (live ? (size_t)(it.seq.row + i) * a.q_stride + (size_t)(cur.head * c.ratio + ff - i * c.ratio) * D : 0);
                    const uint32_t to = smem_u32(q_tiles + (f >> 7) * C::kQTile);
                    for (int k = ch; k < CHUNKS; k += LANES) cp_async16_or_zero(to + place(128, f & 127, k), from + 8 * k, live);
                }
            }
            cp_async_commit();
            auto hand_over_queries = [&] {
                if (pages.q_rows) return;
                fence_async_smem();
                barrier(1, 128);
                if (lt == 0) mbar_arrive(&sh.q_full);
            };
            const int32_t* table = cur.source == 0 ? c.prefix_table : c.table + (size_t)(cur.source - 1) * c.table_stride;
            const long long head_at = (long long)cur.head * c.head_stride;
            if constexpr (TILED) {
                // lane p of each warp: the page of box p, a step ahead
                auto look_up = [&](int i) {
                    const int key = (cur.first + cur.step + i) * KEYS + lane * pages.tokens;
                    return lane < pages.boxes && i < n && key < cur.keys.hi && key + pages.tokens > cur.keys.lo ? table[divide(key, c.page_div)] : -1;
                };
                int ahead = look_up(0);
                for (int i = 0; i < n; ++i) {
                    const uint32_t step = step0 + i, s = step % S, use = step / S;
                    const int k0 = (cur.first + cur.step + i) * KEYS, key = k0 + lane * pages.tokens, page = ahead;
                    const bool in = lane < pages.boxes && key < cur.keys.hi && key + pages.tokens > cur.keys.lo, take = in && (uint32_t)page < (uint32_t)c.n_pages;
                    const uint32_t taken = __ballot_sync(0xffffffffu, take), bad = __ballot_sync(0xffffffffu, in && !take);
                    if (bad && lt == 0 && c.err) atomicOr(c.err, KERR_BAD_PAGE);
                    ahead = look_up(i + 1);
                    auto copy = [&](const CUtensorMap* map, unsigned char* tiles, uint64_t* bar) {
                        if (warp != C::kLoadWarp || !alive) return;
                        const uint32_t dst = smem_u32(tiles + s * C::kTile), at = smem_u32(bar);
                        if (lane == 0) arrive_expect_at(at, __popc(taken) * pages.tokens * D * 2);
                        __syncwarp();
#pragma unroll 1
                        for (uint32_t left = taken; left; left &= left - 1u) {
                            const int p = __ffs(left) - 1, id = __shfl_sync(0xffffffffu, page, p);
                            const int token = pages.boxes == 1 ? k0 - divide(k0, c.page_div) * c.page_size : 0;
                            if (lane == 0)
#pragma unroll
                                for (int x = 0; x < D / 64; ++x) tma_load_4d_at(dst + x * (KEYS * 128) + p * pages.tokens * 128, map, 64 * x, token, cur.head, id, at);
                        }
                    };
                    if (use > 0) warp_wait(&sh.k_empty[s], (use - 1) & 1);
                    if (bad) {
                        for (int r = r_first; r < KEYS; r += ROWS)
                            if (bad >> (r / pages.tokens) & 1u) zero_row(k_tiles + s * C::kTile, r);
                        fence_async_smem();
                        barrier(1, 128);
                    }
                    copy(&pages.k, k_tiles, &sh.k_full[s]);
                    hand_over_values();
                    if (use > 0) warp_wait(&sh.v_empty[s], (use - 1) & 1);
                    if (lt < 4) sh.odd[s][lt] = 0;
                    v_check = k0 < it.clear.lo || min(k0 + KEYS, cur.keys.hi) > it.clear.hi;
                    v_rows = {max(cur.keys.lo - k0, 0), min(cur.keys.hi - k0, KEYS)};
                    v_bad = bad;
                    const bool fix = v_check || v_rows.lo > 0 || v_rows.hi < KEYS || bad;
                    copy(&pages.v, v_tiles, fix ? &sh.v_raw[s] : &sh.v_full[s]);
                    if (fix) v_behind = (int)s;
                    if (i == 0) {
                        cp_async_wait<0>();
                        hand_over_queries();
                    }
                }
                all_steps = step0 + n;
                return;
            }
            // where the key of this thread lies, a step ahead
            auto look_up = [&](int i) {
                const int key = (cur.first + cur.step + i) * KEYS + lt;
                long long at = -1;
                if (lt < KEYS && i < n && key >= cur.keys.lo && key < cur.keys.hi) {
                    const int p = divide(key, c.page_div), page = table[p];
                    if ((uint32_t)page < (uint32_t)c.n_pages) at = (long long)page * c.page_stride + (long long)(key - p * c.page_size) * c.token_stride + head_at;
                    else if (c.err) atomicOr(c.err, KERR_BAD_PAGE);
                }
                return at;
            };
            long long ahead = look_up(0);
            for (int i = 0; i < n; ++i) {
                const uint32_t step = step0 + i, s = step % S, use = step / S;
                const int k0 = (cur.first + cur.step + i) * KEYS;
                long long* rows = sh.row[step & 1];
                if (lt < KEYS) rows[lt] = ahead;
                barrier(1, 128);  // ... and the rows of the step before have been read: the other half may be written
                ahead = look_up(i + 1);
                auto copy = [&](const void* pool, unsigned char* tiles) {
                    const uint32_t dst = smem_u32(tiles + s * C::kTile);
                    if (alive) {
#pragma unroll 4
                        for (int r = r_first; r < KEYS; r += ROWS) {
                            const long long at = rows[r];
                            for (int k = ch; k < CHUNKS; k += LANES) cp_async16_or_zero(dst + place(KEYS, r, k), static_cast<const E*>(pool) + max(at, 0ll) + 8 * k, at >= 0);
                        }
                    }
                    cp_async_commit();
                };
                if (use > 0) warp_wait(&sh.k_empty[s], (use - 1) & 1);
                copy(c.k, k_tiles);
                cp_async_wait<1>();  // the values of the step before (or the queries) have arrived
                if (i == 0) hand_over_queries();
                else hand_over_values();
                if (use > 0) warp_wait(&sh.v_empty[s], (use - 1) & 1);
                if (lt < 4) sh.odd[s][lt] = 0;
                copy(c.v, v_tiles);
                cp_async_wait<1>();
                arrive(&sh.k_full[s]);
                v_behind = (int)s;
                v_check = k0 < it.clear.lo || min(k0 + KEYS, cur.keys.hi) > it.clear.hi;
            }
        });
        cp_async_wait<0>();
        hand_over_values();
        if (TILED && !alive && warp == C::kLoadWarp)  // no copy may land after the CTA has left
            for (uint32_t s = 0; s < S && s < all_steps; ++s) {
                const uint32_t use = (all_steps - 1 - s) / S;
                mbar_poll_bounded(&sh.k_full[s], use & 1);
                mbar_poll_bounded(&sh.v_full[s], use & 1);
            }
    } else if (warp > C::kMmaWarp) {
        // ── without a prefix no join of all rows comes behind: the item that others finish is named for the join, and blocks that see
        // nothing, which have no item, get their zeros here ──
        if (!a.whole_o) {
            if (warp == C::kMmaWarp + 1) {
                PagedShared shared = {};
                each_item([&](const Cursor& cur, const Item& it, bool, int, int, uint32_t, uint32_t) {
                    const int item_at = cur.at - cur.step;
                    if (item_at >= begin && item_at + cur.steps > end) shared = {share.cta_of(item_at + cur.steps - 1) - (int)blockIdx.x + 1, it.seq.row, it.f0, it.width, cur.head};
                });
                if (lane == 0) line.shared[blockIdx.x] = shared;
            }
            for (int s = blockIdx.x * 3 + warp - C::kMmaWarp - 1; s < c.n_seqs; s += gridDim.x * 3) {
                const Seq seq = batch.seq(s);
                const int blocks = blocks_of(c, line, seq.n);
                for (int b0 = 0; b0 < blocks; b0 += 32) {
                    uint32_t none = __ballot_sync(0xffffffffu, b0 + lane < blocks && steps_of(block_keys(c, line, seq, b0 + lane, a.window), line.keys) == 0);
                    for (; none; none &= none - 1u) {
                        const int f0 = (b0 + __ffs(none) - 1) * line.columns, f1 = min(f0 + line.columns, seq.n * c.ratio);
                        for (int f = f0; f < f1; ++f) {
                            const int i = divide(f, c.ratio_div);
                            for (int h = 0; h < c.n_kv; ++h)
                                for (int x = 2 * lane; x < D; x += 64)
                                    *reinterpret_cast<uint32_t*>(static_cast<E*>(a.out) + (size_t)(seq.row + i) * a.out_stride + (size_t)(h * c.ratio + f - i * c.ratio) * D + x) = 0u;
                        }
                    }
                }
            }
        }
    } else if (warp == C::kMmaWarp) {
        // ── products ──
        constexpr uint32_t kScores = (1u << 4) | Half16<E>::kType | ((uint32_t)(KEYS >> 3) << 17) | ((128u >> 4) << 24);
        constexpr uint32_t kValues = (1u << 4) | Half16<E>::kType | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
        const uint64_t q_desc = smem_desc_sw128(smem_u32(q_tiles)), k_desc = smem_desc_sw128(smem_u32(k_tiles)), v_desc = value_desc(smem_u32(v_tiles), KEYS * 128);
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            alive = __all_sync(0xffffffffu, alive && wait_alive_short(smem_u32(bar), parity, smem_u32(&sh.dead))) != 0;
            tc_fence_after();
        };
        uint32_t items = 0, done = 0;
        each_item([&](const Cursor&, const Item&, bool pair, int, int tasks, uint32_t task0, uint32_t step0) {
            wait(&sh.q_full, items & 1);
            ++items;
            auto scores = [&](int t) {
                const uint32_t b = (task0 + t) & 1, step = step0 + (pair ? t >> 1 : t), s = step % S;
                const bool first = !pair || !(t & 1), last = !pair || (t & 1);
                if (first) wait(&sh.k_full[s], (step / S) & 1);
                if (!alive) return;
                const uint64_t q = q_desc + (uint64_t)((pair ? t & 1 : 0) * (C::kQTile / 16)), k = k_desc + (uint64_t)(s * (C::kTile / 16));
#pragma unroll
                for (int x = 0; x < D / 64; ++x) umma_f16_block(tmem + b * KEYS, q + x * (128 * 128 / 16), k + x * (KEYS * 128 / 16), kScores, x > 0);
                commit_elected(smem_u32(&sh.s_full[b]));
                if (last) commit_elected(smem_u32(&sh.k_empty[s]));
                if (t + 1 == tasks) commit_elected(smem_u32(&sh.q_empty));
            };
            scores(0);
            if (tasks > 1) scores(1);
#pragma unroll 1
            for (int t = 0; t < tasks; ++t) {
                const uint32_t T = task0 + t, b = T & 1, step = step0 + (pair ? t >> 1 : t), s = step % S;
                const bool first = !pair || !(t & 1), last = !pair || (t & 1);
                if (first) wait(&sh.v_full[s], (step / S) & 1);
                wait(&sh.p_ready[b], (T >> 1) & 1);
                if (alive) {
                    const uint32_t o = tmem + C::kSum + (C::kSets == 2 ? b * D : 0);
                    const bool add = t >= C::kSets || *(volatile uint32_t*)&sh.keep[b];
                    const uint64_t v = v_desc + (uint64_t)(s * (C::kTile / 16));
#pragma unroll
                    for (int x = 0; x < KEYS / 64; ++x) umma_values_block(o, tmem + b * KEYS + 32 * x, v + x * (64 * 128 / 16), kValues, x > 0 || add);
                    commit_elected(smem_u32(&sh.pv_done[b]));
                    if (last) commit_elected(smem_u32(&sh.v_empty[s]));
                    done = T + 1;
                }
                if (t + 2 < tasks) scores(t + 2);
            }
        });
        // the products in flight read shared memory and write tensor memory
        if (done > 0) mbar_poll_bounded(&sh.pv_done[(done - 1) & 1], ((done - 1) >> 1) & 1);
        if (done > 1) mbar_poll_bounded(&sh.pv_done[done & 1], ((done - 2) >> 1) & 1);
    }
    } else {
        registers_up<C::kMany>();
        // ── softmax: a thread a column ──
        const int set = warp >> 2, me = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), o_at = lanes + C::kSum + set * D;
        const float scale2 = fmaxf(fabsf(a.scale2), 1e-30f);  // the maximum wants a positive one, and so does -inf times it
        const bool negative = a.scale2 < 0.f;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            alive = __all_sync(0xffffffffu, alive && wait_alive_short(smem_u32(bar), parity, smem_u32(&sh.dead))) != 0;
            tc_fence_after();
        };
        float m = kLowest, l = 0.f;  // of the column: what its weights are relative to, and their sum
        // A task's scores to weights, in place.  all: every key is seen.
        auto weigh = [&](auto all, uint32_t s_at, int k0, const Range& keys, bool begun, uint32_t last) {
            uint32_t v[KEYS];
            load_scores<KEYS>(s_at, v);
            if (negative)
#pragma unroll
                for (int e = 0; e < KEYS; ++e) v[e] ^= 0x80000000u;
            if constexpr (!decltype(all)::value) {  // keys that the column does not see
#pragma unroll
                for (int x = 0; x < KEYS; x += 32) {
                    const uint32_t seen = below(keys.hi - k0 - x) & ~below(keys.lo - k0 - x);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1u)) v[x + e] = 0xFF800000u;
                }
            }
            auto largest = [&] {
                float most[4] = {kLowest, kLowest, kLowest, kLowest};
#pragma unroll
                for (int e = 0; e < KEYS; e += 8)
#pragma unroll
                    for (int i = 0; i < 4; ++i) most[i] = fmaxf(most[i], fmaxf(__uint_as_float(v[e + 2 * i]), __uint_as_float(v[e + 2 * i + 1])));
                const float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                return top == kLowest ? kLowest : top * scale2;
            };
            // An item's largest weights are 2^kAbove: fp16 loses bits below 2^-14, and with them what many small weights add up to.
            constexpr float kAbove = std::is_same<E, __half>::value ? 6.f : 0.f;
            if (!begun) {
                const float top = largest();
                m = top == kLowest ? kLowest : top - kAbove;
            }
            // Behind an item's first task the weights are relative to the maximum so far: the new one is looked for only where their sum is past
            // 1024 of the largest ones (what fp16 holds), and the task is done again.  Until then no weight is above that sum, which either
            // 16-bit type holds as well as 1, and a flat task's 128 of the largest ones stay below it.
            constexpr float kMost = std::is_same<E, __half>::value ? 65504.f : 1024.f;
            float added;
            auto exponentials = [&] {
                const uint64_t scales = pair_of(scale2, scale2), minus = pair_of(-m, -m);
                uint64_t sums[2] = {0ull, 0ull};
#pragma unroll
                for (int x = 0; x < KEYS; x += 32) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float y0, y1;
                        split(fma2(pair_of(__uint_as_float(v[x + e]), __uint_as_float(v[x + e + 1])), scales, minus), y0, y1);
                        const float p0 = exp2_approx(y0), p1 = exp2_approx(y1);
                        sums[e >> 1 & 1] = add2(sums[e >> 1 & 1], pair_of(p0, p1));
                        p[e / 2] = TileElem<E>::pack(p0, p1);
                    }
                    tmem_st16(s_at + x / 2, p);
                }
                float l0, l1;
                split(add2(sums[0], sums[1]), l0, l1);
                added = l0 + l1;
            };
            exponentials();
            if (begun && __any_sync(0xffffffffu, added > kMost)) {
                const float top = largest() - kAbove;
                const bool move = added > kMost;  // at least one weight is above 7 of the largest ones so far, so top is above m
                const float keep = move ? exp2_approx(m - top) : 1.f;
                if (move) m = top;
                l *= keep;
                wait(&sh.pv_done[last & 1], (last >> 1) & 1);
                if (alive) {
#pragma unroll 1
                    for (int x = 0; x < D; x += 16) {
                        uint32_t w[16];
                        tmem_ld16(o_at + x, w);
                        tmem_wait_ld16(w);
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * keep);
                        tmem_st16(o_at + x, w);
                    }
                }
                exponentials();
            }
            l += added;
        };
        each_item([&](const Cursor& cur, const Item& it, bool pair, int n, int tasks, uint32_t task0, uint32_t step0) {
            const int t_first = C::kSets == 1 ? 0 : (int)((task0 & 1) ^ set), f = me < tile_columns ? (pair ? t_first * tile_columns : 0) + me : 256, ff = it.f0 + f;
            Range keys = {0, 0};
            if (f < it.width) {
                const int i = divide(ff, c.ratio_div);
                if (cur.source) {
                    keys = own_keys(it.seq, i, a.window);
                } else {
                    const Seq s = batch.seq(seq_of_row(batch, c.n_seqs, i));
                    keys = prefix_keys(s, i - s.row, c.prefix_length, a.window);
                }
            }
            const bool blind = __any_sync(0xffffffffu, f < it.width && keys.hi == 0);  // a row of the prefix's block that sees nothing
            m = kLowest;
            l = 0.f;
            uint32_t last = 0;
            bool any = false;
            for (int t = t_first; t < tasks; t += C::kSets) {
                const uint32_t T = task0 + t, b = T & 1, use = T >> 1, step = step0 + (pair ? t >> 1 : t);
                const int k0 = (cur.first + cur.step + (pair ? t >> 1 : t)) * KEYS;
                const bool clear = k0 >= max(it.clear.lo, cur.keys.lo) && k0 + KEYS <= min(it.clear.hi, cur.keys.hi) && !blind;
                const bool checked = k0 < it.clear.lo || min(k0 + KEYS, cur.keys.hi) > it.clear.hi;
                const uint32_t s_at = lanes + b * KEYS;
                wait(&sh.s_full[b], use & 1);
                if (alive) {
                    const bool begun = any;
                    if (clear) weigh(std::true_type{}, s_at, k0, keys, begun, last);
                    else weigh(std::false_type{}, s_at, k0, keys, begun, last);
                    tmem_wait_st();
                    uint32_t keep_sum = 0;
                    if (checked) {  // values that were taken out of this step's product
                        const uint32_t s = step % S;
                        wait(&sh.v_full[s], (step / S) & 1);
                        uint32_t odd[4];
                        for (int i = 0; i < 4; ++i) odd[i] = i * 32 < KEYS ? *(volatile uint32_t*)&sh.odd[s][i] : 0u;
                        if (alive && (odd[0] | odd[1] | odd[2] | odd[3])) {
                            if (begun) {
                                wait(&sh.pv_done[last & 1], (last >> 1) & 1);
                            } else {
                                keep_sum = 1;
                                uint32_t zero[16] = {};
                                for (int x = 0; x < D; x += 16) tmem_st16(o_at + x, zero);
                                tmem_wait_st();
                            }
                            const int32_t* table = cur.source == 0 ? c.prefix_table : c.table + (size_t)(cur.source - 1) * c.table_stride;
                            for (int k = 0; k < KEYS; ++k) {
                                if (!(odd[k >> 5] >> (k & 31) & 1u)) continue;
                                const int key = k0 + k, page_at = divide(key, c.page_div), page = table[page_at];  // in the pool: its row was copied
                                const E* row = static_cast<const E*>(c.v) + (long long)page * c.page_stride + (long long)(key - page_at * c.page_size) * c.token_stride + (long long)cur.head * c.head_stride;
                                uint32_t pk[8];
                                tmem_ld8(s_at + ((k >> 1) & ~7), pk);
                                tmem_wait_ld();
                                float p = 0.f;
                                for (int e = 0; e < 8; ++e)
                                    if (e == ((k >> 1) & 7)) p = Half16<E>::one((uint16_t)(k & 1 ? pk[e] >> 16 : pk[e] & 0xffffu));
                                const bool sees = key >= keys.lo && key < keys.hi;
                                for (int x = 0; x < D; x += 16) {
                                    uint32_t v[16];
                                    tmem_ld16(o_at + x, v);
                                    tmem_wait_ld16(v);
                                    for (int e = 0; e < 16; ++e)
                                        if (sees) v[e] = __float_as_uint(__uint_as_float(v[e]) + p * (float)row[x + e]);
                                    tmem_st16(o_at + x, v);
                                    tmem_wait_st();
                                }
                            }
                        }
                    }
                    if (t < C::kSets) *(volatile uint32_t*)&sh.keep[b] = keep_sum;
                    tc_fence_before();
                    any = true;
                    last = T;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready[b]);
            }
            // ── the item's sums ──
            if (any) wait(&sh.pv_done[last & 1], (last >> 1) & 1);
            const int item_at = cur.at - cur.step;
            const bool here = item_at >= begin && item_at + cur.steps <= end;
            const bool both = C::kSets == 2 && !pair;
            float mine = 1.f;
            if (both) {
                sh.ml[set][me] = make_float2(m, l);
                barrier(2, 256);
                const float2 other = sh.ml[set ^ 1][me];
                const float top = fmaxf(m, other.x);
                mine = exp2_approx(m - top);
                l = l * mine + other.y * exp2_approx(other.x - top);
                m = top;
            }
            const bool writer = !both || t_first == 0;
            const size_t row = (size_t)it.seq.row + divide(ff, c.ratio_div), head = (size_t)cur.head * c.ratio + ff - divide(ff, c.ratio_div) * c.ratio;
            float* part = nullptr;
            float2* part_ml = nullptr;
            if (!here) {
                const size_t at = (size_t)(2 * blockIdx.x + (item_at < begin ? 0 : 1)) * line.columns + f;
                part = line.slot_o + at * D;
                part_ml = line.slot_ml + at;
            } else if (a.whole_o) {
                const size_t at = ((cur.source == 0 ? (size_t)c.rows : 0) + row) * c.n_q + head;
                part = a.whole_o + at * D;
                part_ml = a.whole_ml + at;
            }
            const bool write = writer && f < it.width && alive;
            if (write && part) *part_ml = make_float2(m, l);
            const float rate = part ? 1.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
            // 32 values of a column at a time.  A lane has a column to itself, and writes whole sectors of 32 bytes where the rows begin at one
            E* to = part ? nullptr : static_cast<E*>(a.out) + row * a.out_stride + head * D;
            const bool sectors = (reinterpret_cast<uintptr_t>(part ? (const void*)part : to) & 31) == 0;
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
                uint32_t v[32];
                if (any && alive) {
                    tmem_ld32(o_at + x, v);
                    tmem_wait_ld32(v);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = 0u;
                }
                if (both) {  // one set's to the other's: [32][128] in shared memory
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        v[e] = __float_as_uint(__uint_as_float(v[e]) * mine);
                        if (!writer) joint[e * 128 + me] = __uint_as_float(v[e]);
                    }
                    barrier(2, 256);
                    if (writer)
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + joint[e * 128 + me]);
                    barrier(2, 256);
                }
                if constexpr (std::is_same<E, __half>::value) {  // (a bf16 weight is zero only where the fp32 one is)
                    float odd[4] = {0.f, 0.f, 0.f, 0.f};  // NaN where a sum is not finite
#pragma unroll
                    for (int e = 0; e < 32; ++e) odd[e & 3] = fmaf(__uint_as_float(v[e]), 0.f, odd[e & 3]);
                    if (__any_sync(0xffffffffu, write && odd[0] + odd[1] + odd[2] + odd[3] != 0.f)) {
                        Infinite<1> found;
                        found.seen[0] = keys;
                        look_for_infinities<E>(c, cur.source == 0 ? c.prefix_table : c.table + (size_t)(cur.source - 1) * c.table_stride,
                                               static_cast<const E*>(c.v) + (long long)cur.head * c.head_stride + x, max((cur.first + cur.step) * KEYS, cur.keys.lo),
                                               min((cur.first + cur.step + n) * KEYS, cur.keys.hi), found);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(found.sum(0, e, __uint_as_float(v[e])));
                    }
                }
                if (!write) continue;
                if (part) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) store32(part + x + e, *reinterpret_cast<const uint32_t(*)[8]>(v + e), sectors);
                } else {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) w[e / 2] = l == 0.f ? 0u : TileElem<E>::pack(__uint_as_float(v[e]) * rate, __uint_as_float(v[e + 1]) * rate);
#pragma unroll
                    for (int e = 0; e < 16; e += 8) store32(to + x + 2 * e, *reinterpret_cast<const uint32_t(*)[8]>(w + e), sectors);
                }
            }
            tc_fence_before();
        });
    }
    __syncthreads();
    if (tid == 0 && c.err && *dead) atomicOr(c.err, 0x1000u);
    tc_fence_before();
    __syncthreads();
    if (warp == C::kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int D, class E, bool TILED>
cudaError_t run(const Launch& l, const PagedAttentionArgs& a, int line, const Pages& pages) {
    auto kernel = paged_wide_kernel<D, E, TILED>;
    const size_t shared = wide_shared<D>(a.c.n_seqs);
    cudaError_t e = allow_shared(kernel, shared);
    if (e == cudaSuccess) e = prefer_max_shared(kernel);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.line[line].ctas);
    cfg.blockDim = dim3(Cfg<D>::kThreads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = l.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, line, pages);
}

template <int D, class E>
cudaError_t go(const Launch& l, const PagedAttentionArgs& a, int line) {
    constexpr int KEYS = Cfg<D>::kKeys;
    const PagedArgs& c = a.c;
    // Boxes of a step: whole pages, or a part of one.  The swizzle's atoms are eight rows.
    Pages pages = {};
    pages.tokens = c.page_size < KEYS ? c.page_size : KEYS;
    pages.boxes = KEYS / pages.tokens;
    const bool tiled = pages.tokens % 8 == 0 && KEYS % pages.tokens == 0 && c.page_size % pages.tokens == 0 &&
                       encode_pages(&pages.k, c.k, D, c.page_size, c.n_kv, c.n_pages, c.token_stride, c.head_stride, c.page_stride, pages.tokens, 1) &&
                       encode_pages(&pages.v, c.v, D, c.page_size, c.n_kv, c.n_pages, c.token_stride, c.head_stride, c.page_stride, pages.tokens, 1);
    pages.q_rows = c.ratio <= 128 ? 128 / c.ratio : 0;
    if (pages.q_rows && !encode_pages(&pages.q, a.q, D, c.n_q, c.rows, 1, D, a.q_stride, 0, c.ratio, pages.q_rows)) return cudaErrorInvalidValue;
    return tiled ? run<D, E, true>(l, a, line, pages) : run<D, E, false>(l, a, line, pages);
}

}  // namespace

int paged_wide_columns(int head_dim, int ratio) { return (head_dim == 256 ? 1 : 2) * (ratio <= 128 ? 128 / ratio * ratio : 128); }
int paged_wide_keys(int head_dim) { return head_dim == 256 ? 6 : 7; }
bool paged_wide_takes(int head_dim, int n_seqs) {
    const size_t most = 227 * 1024 - 1024;  // less what the scan of the batch holds, up to the tiles' alignment
    return (head_dim == 64 ? wide_shared<64>(n_seqs) : head_dim == 128 ? wide_shared<128>(n_seqs) : wide_shared<256>(n_seqs)) <= most;
}
cudaError_t launch_paged_wide(const Launch& l, PagedType type, int head_dim, const PagedAttentionArgs& a, int line) {
    if (type == kPagedF16) return head_dim == 64 ? go<64, __half>(l, a, line) : head_dim == 128 ? go<128, __half>(l, a, line) : go<256, __half>(l, a, line);
    return head_dim == 64 ? go<64, __nv_bfloat16>(l, a, line) : head_dim == 128 ? go<128, __nv_bfloat16>(l, a, line) : go<256, __nv_bfloat16>(l, a, line);
}

}  // namespace smelt
