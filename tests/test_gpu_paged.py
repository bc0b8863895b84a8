"""A packed batch over a paged cache, and drafted tokens, against their formulas in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as cases
from smelt_b200 import capi

pytestmark = pytest.mark.gpu
CODE = {"f16": capi.PAGED_F16, "bf16": capi.PAGED_BF16}
LOGITS = {"f16": capi.LOGITS_F16, "bf16": capi.LOGITS_BF16, "f32": capi.LOGITS_F32}
WORD = {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context(0)
    yield c
    assert c.device_error_flags() == 0
    c.close()


class Device:
    """A batch of paged_cases on the GPU: its arrays and the two descriptions."""

    def __init__(self, ctx, b, kind, n_q, k, v, max_rows=None):
        self.ctx, self.b, self.kind = ctx, b, kind
        self.k, self.v = (ctx.to_device(cases.to_bits(b.memory(p), kind)) for p in (k, v))
        self.kept = [ctx.to_device(a) for a in (b.start, np.array(b.lengths, np.int32), b.table, b.prefix_table)]
        page, head, token = b.strides()
        self.cache = capi.PagedCache(CODE[kind], n_q, b.kv, b.dim, b.page, b.pages, page, head, token, self.k.ptr, self.v.ptr)
        self.batch = capi.PagedBatch(len(b.rows), b.total, max(b.rows) if max_rows is None else max_rows, b.table.shape[1], b.prefix, *[d.ptr for d in self.kept])

    def workspace(self):
        size = C.c_size_t()
        self.ctx.call("paged_attention_workspace", C.byref(self.cache), C.byref(self.batch), C.byref(size))
        return self.ctx.alloc(size.value).fill(0xFF), size.value

    def attend(self, q, scale, window=0, pad=0, in_place=False):
        """Outputs of all rows, those behind the last sequence among them."""
        rows, heads, dim = q.shape
        wide = heads * dim + pad
        put = np.full((rows, wide), 7.0)
        put[:, :heads * dim] = q.reshape(rows, -1)
        dq = self.ctx.to_device(cases.to_bits(put, self.kind))
        out = dq if in_place else self.ctx.to_device(cases.to_bits(np.full((rows, wide), 7.0), self.kind))
        work, size = self.workspace()
        self.ctx.call("paged_attention", C.byref(self.cache), C.byref(self.batch), dq.ptr, wide, out.ptr, wide, scale, window, work.ptr, size)
        got = cases.from_bits(out.download(WORD[self.kind], (rows, wide)), self.kind)
        assert (got[:, heads * dim:] == 7.0).all()
        return got[:, :heads * dim].reshape(q.shape)

    def pools(self):
        return [cases.from_bits(self.b.seen(d.download(WORD[self.kind], (self.b.pages * self.b.page * self.b.kv * self.b.dim,))), self.kind) for d in (self.k, self.v)]


def check_attention(ctx, g, kind, n_q, b, window=0, scale=None, spread=2.0, empty=np.nan, max_rows=None, **kw):
    scale = scale if scale is not None else spread / np.sqrt(b.dim)
    k, v, tokens = b.fill(g, empty)
    tokens = [cases.rounded(t, kind) for t in tokens]
    q = cases.rounded(g.standard_normal((b.total, n_q, b.dim)), kind)
    got = Device(ctx, b, kind, n_q, k, v, max_rows).attend(q, scale, window, **kw)
    want, size, reach = cases.attend(b, tokens, q, np.float32(scale), window)
    live = b.live
    behind = got[live:] == (q[live:] if kw.get("in_place") else 7.0)
    assert behind.all()
    off = np.abs(got[:live] - want[:live]) - cases.attend_bound(want, size, reach, kind, b.dim)[:live]
    assert off.max(initial=-1) <= 0, (np.unravel_index(off.argmax(), off.shape), off.max())
    return got


SHAPES = [  # n_q, n_kv, dim
    (4, 4, 64), (8, 2, 64), (5, 1, 128), (8, 2, 128), (32, 8, 128), (14, 2, 128), (4, 2, 256), (10, 1, 256)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim", SHAPES)
@pytest.mark.parametrize("page,order", [(16, "heads"), (7, "tokens")])
def test_one_token_a_sequence(ctx, kind, n_q, n_kv, dim, page, order):
    g = np.random.default_rng(n_q * dim + page)
    lengths = [1, 2, 15, 16, 17, 127, 128, 129, 300, 0, 64]
    check_attention(ctx, g, kind, n_q, cases.Batch(g, [1] * len(lengths), lengths, page, n_kv, dim, order=order, behind=2))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 50])
def test_drafts_and_empty_sequences(ctx, kind, n_q, n_kv, dim, window):
    g = np.random.default_rng(n_q + dim + window)
    b = cases.Batch(g, [5, 0, 1, 3, 2, 4, 6], [5, 10, 0, 131, 1, 260, 90], 20, n_kv, dim, behind=3)
    check_attention(ctx, g, kind, n_q, b, window)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim", SHAPES)
@pytest.mark.parametrize("prefix,window", [(1, 0), (130, 0), (500, 0), (500, 77), (300, 400)])
def test_shared_prefix(ctx, kind, n_q, n_kv, dim, prefix, window):
    g = np.random.default_rng(n_q + dim + prefix + window)
    b = cases.Batch(g, [1, 2, 0, 1, 4, 3], [30, 2, 9, 1, 3, 140], 16, n_kv, dim, prefix=prefix, order="tokens", behind=1)
    check_attention(ctx, g, kind, n_q, b, window)


@pytest.mark.parametrize("kind,n_q,n_kv,dim", [("f16", 8, 2, 64), ("bf16", 8, 2, 128), ("f16", 6, 1, 128), ("bf16", 4, 2, 256)])
@pytest.mark.parametrize("prefix,window", [(0, 0), (200, 0), (0, 60), (200, 150)])
def test_prompt_chunks(ctx, kind, n_q, n_kv, dim, prefix, window):
    g = np.random.default_rng(dim + prefix + window)
    b = cases.Batch(g, [70, 1, 200, 33], [70, 5, 333, 161], 24, n_kv, dim, prefix=prefix, behind=2)
    check_attention(ctx, g, kind, n_q, b, window)


@pytest.mark.parametrize("rows,lengths,hint", [([1] * 40, [3] * 40, 1), ([40, 1], [50, 200], 1), ([1, 2], [9, 300], 500), ([3], [4000], 0)])
def test_any_hint_gives_the_same(ctx, rows, lengths, hint):
    """max_rows says how the work is cut, whatever the sequences have."""
    g = np.random.default_rng(hint)
    check_attention(ctx, g, "f16", 8, cases.Batch(g, rows, lengths, 16, 2, 64), max_rows=hint)


def test_many_sequences(ctx):
    g = np.random.default_rng(5)
    rows = g.integers(0, 3, 1024).tolist()
    check_attention(ctx, g, "f16", 2, cases.Batch(g, rows, (np.array(rows) + g.integers(0, 40, 1024)).tolist(), 16, 1, 64, prefix=40))


@pytest.mark.parametrize("page", [1, 3, 100, 1000])
def test_page_sizes(ctx, page):
    g = np.random.default_rng(page)
    check_attention(ctx, g, "bf16", 4, cases.Batch(g, [1, 3, 2], [700, 99, 1001], page, 2, 128, prefix=101), window=900)


@pytest.mark.parametrize("page", [1, 8, 24, 32, 64, 128, 256, 1000])
@pytest.mark.parametrize("dim,order", [(64, "heads"), (128, "tokens"), (256, "heads")])
def test_page_sizes_under_many_columns(ctx, page, dim, order):
    g = np.random.default_rng(page + dim)
    check_attention(ctx, g, "bf16", 32, cases.Batch(g, [1, 30, 7], [700, 99, 1001], page, 2, dim, prefix=301, order=order), window=page % 64 * 10)


@pytest.mark.parametrize("prefix", [0, 90])
def test_strided_rows_and_outputs_in_the_place_of_queries(ctx, prefix):
    g = np.random.default_rng(8 + prefix)
    b = cases.Batch(g, [1, 4, 2], [700, 99, 3], 16, 2, 64, prefix=prefix, behind=2)
    one = check_attention(ctx, np.random.default_rng(1), "f16", 8, b, pad=24)
    two = check_attention(ctx, np.random.default_rng(1), "f16", 8, b, pad=24, in_place=True)
    assert np.array_equal(one[:b.live], two[:b.live])


def test_every_key_counts_once(ctx):
    """Equal scores: a key left out, doubled or read from a neighbour moves the mean by more than the bound allows."""
    g = np.random.default_rng(9)
    for lengths in ([40, 128, 129, 200], [1, 2, 3, 150]):
        b = cases.Batch(g, [1, 2, 1, 3], [max(n, 3) for n in lengths], 9, 2, 64, prefix=33)
        k, v, tokens = b.fill(g, np.nan)
        tokens = [cases.rounded(t, "f16") for t in tokens]
        got = Device(ctx, b, "f16", 4, k, v).attend(np.zeros((b.total, 4, 64)), 1.0)
        want, _, _ = cases.attend(b, tokens, np.zeros((b.total, 4, 64)), 1.0)
        assert np.abs(got - want).max() < 2.0 ** -11 * np.abs(want).max() + 2.0 ** -11  # half a step of the output and of the weights (values of order one)


@pytest.mark.parametrize("kind,rows", [("f16", 4), ("bf16", 4), ("f16", 40), ("bf16", 150)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, kind, rows, bad):
    """Keys and values that are not finite behind a row (drafts of later rows) and in front of its window."""
    g = np.random.default_rng(rows)
    b = cases.Batch(g, [rows, 1], [rows + 150, 20], 16, 2, 128)
    k, v, _ = b.fill(g, np.nan)
    q = cases.rounded(g.standard_normal((b.total, 8, 128)), kind)
    clean = Device(ctx, b, kind, 8, k, v).attend(q, 0.1, window=60)
    cut = 3  # the last rows' tokens are spoilt, and a few that only the first rows see
    for t in range(b.lengths[0] - cut, b.lengths[0]):
        p, i = b.place(0, t)
        k[p, :, i], v[p, :, i] = bad, bad
    p, i = b.place(0, 150 - 60 + 1)  # seen by the first row alone
    v[p, :, i] = bad
    got = Device(ctx, b, kind, 8, k, v).attend(q, 0.1, window=60)
    assert np.array_equal(got[1:rows - cut], clean[1:rows - cut]) and np.array_equal(got[rows:], clean[rows:])
    assert not np.isfinite(got[0]).any() and not np.isfinite(got[rows - cut:rows]).any()


@pytest.mark.parametrize("dim,n_q", [(64, 5), (128, 5), (128, 14), (256, 7)])
def test_queries_of_an_earlier_call_do_not_reach_the_next(ctx, dim, n_q):
    """Groups that do not fill a tile, behind a call whose queries were as large as the type holds."""
    g = np.random.default_rng(dim)
    b = cases.Batch(g, [300, 64], [900, 700], 16, 2, dim)
    k, v, _ = b.fill(g, 0.0)
    Device(ctx, b, "bf16", 16, k, v).attend(np.full((b.total, 16, dim), 3e38), 1.0)
    check_attention(ctx, g, "bf16", 2 * n_q, cases.Batch(g, [120, 33], [1500, 800], 16, 2, dim))


def test_large_scores_and_small_ones(ctx):
    g = np.random.default_rng(11)
    for scale in (40.0, 1e-6, 0.0, -3.0):
        check_attention(ctx, g, "bf16", 4, cases.Batch(g, [1, 3], [500, 77], 16, 2, 64, prefix=40), scale=scale)


@pytest.mark.parametrize("kind,n_q,n_kv,dim", [("f16", 8, 2, 64), ("bf16", 8, 2, 128), ("f16", 8, 2, 256)])
def test_maxima_that_move_under_many_columns(ctx, kind, n_q, n_kv, dim):
    """Scores so far apart that a later step's are many powers of two above the first's."""
    g = np.random.default_rng(dim)
    for spread in (40.0, -20.0, 0.0):
        check_attention(ctx, g, kind, n_q, cases.Batch(g, [90, 1], [1500, 77], 16, n_kv, dim), spread=spread)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("prefix,window", [(0, 0), (0, 30), (70, 0)])
def test_blocks_of_rows_without_tokens(ctx, dim, prefix, window):
    g = np.random.default_rng(dim + window)
    got = check_attention(ctx, g, "f16", 8, cases.Batch(g, [300, 2, 200], [40, 1, 0], 16, 2, dim, prefix=prefix, behind=3), window)
    assert (got[:260] == 0).all() and (got[300] == 0).all() and (got[302:502] == 0).all()


@pytest.mark.parametrize("n_q,n_kv,dim,rows", [(160, 1, 64, [1, 3]), (260, 2, 128, [2, 1]), (129, 1, 256, [1, 2])])
@pytest.mark.parametrize("prefix", [0, 200])
def test_more_heads_a_group_than_a_tile_has_columns(ctx, n_q, n_kv, dim, rows, prefix):
    g = np.random.default_rng(n_q + prefix)
    check_attention(ctx, g, "bf16", n_q, cases.Batch(g, rows, [700, 90], 16, n_kv, dim, prefix=prefix))


@pytest.mark.parametrize("prefix", [0, 90])
@pytest.mark.parametrize("shift", [0, 16])
def test_strided_rows_under_many_columns(ctx, prefix, shift):
    """Rows, outputs and workspace that begin at odd multiples of 16 bytes."""
    g = np.random.default_rng(prefix)
    b = cases.Batch(g, [100, 4, 60], [1700, 99, 60], 16, 2, 64, prefix=prefix)
    k, v, tokens = b.fill(g, np.nan)
    q, wide = cases.rounded(g.standard_normal((b.total, 8, 64)), "f16"), 8 * 64 + 8
    d = Device(ctx, b, "f16", 8, k, v)
    put = np.full((b.total, wide), 7.0)
    put[:, :512] = q.reshape(b.total, -1)
    data = ctx.to_device(np.concatenate([np.zeros(shift // 2, np.float16), cases.to_bits(put, "f16").ravel()]))
    size = C.c_size_t()
    ctx.call("paged_attention_workspace", C.byref(d.cache), C.byref(d.batch), C.byref(size))
    work = ctx.alloc(size.value + shift)
    ctx.call("paged_attention", C.byref(d.cache), C.byref(d.batch), data.at(shift), wide, data.at(shift), wide, 0.2, 0, work.at(shift), size.value)
    got = data.download(np.float16, (b.total * wide + shift // 2,))[shift // 2:].reshape(b.total, wide).astype(np.float64)
    assert (got[:, 512:] == 7.0).all()
    want, large, reach = cases.attend(b, [cases.rounded(t, "f16") for t in tokens], q, np.float32(0.2))
    assert (np.abs(got[:, :512].reshape(q.shape) - want) <= cases.attend_bound(want, large, reach, "f16", 64)).all()


@pytest.mark.parametrize("n_q,dim", [(32, 64), (32, 128), (16, 256)])
def test_many_sequences_under_many_columns(ctx, n_q, dim):
    g = np.random.default_rng(dim)
    rows = g.integers(0, 3, 1024).tolist()
    check_attention(ctx, g, "bf16", n_q, cases.Batch(g, rows, (np.array(rows) + g.integers(0, 20, 1024)).tolist(), 16, 1, dim))


# ── rotation and append ─────────────────────────────────────────────────────
def check_append(ctx, g, kind, n_q, b, rope_dim, layout, positions=None, factor=1.0, pad=0, queries=True, in_place=False, theta=1e4):
    kv, dim, rows = b.kv, b.dim, b.total
    wide = (n_q + 2 * kv) * dim + pad
    new = cases.rounded(g.standard_normal((rows, wide)), kind)
    k, v, _ = b.fill(g, 5.0)
    d = Device(ctx, b, kind, n_q, k, v)
    before = d.pools()
    freq, _ = capi.rope_frequencies(max(rope_dim, 2), theta)
    rows_dev, freq_dev = ctx.to_device(cases.to_bits(new, kind)), ctx.to_device(freq)
    out = rows_dev if in_place else ctx.to_device(cases.to_bits(np.full((rows, n_q * dim), 7.0), kind))
    at = ctx.to_device(np.asarray(positions, np.int32)) if positions is not None else None
    rope = capi.RopeDesc(rope_dim, layout, factor, freq_dev.ptr, at.ptr if at else None)
    item = 2
    ctx.call("paged_append", C.byref(d.cache), C.byref(d.batch), C.byref(rope), rows_dev.ptr if queries else None, wide, rows_dev.at(n_q * dim * item), wide,
             rows_dev.at((n_q + kv) * dim * item), wide, out.ptr, wide if in_place else n_q * dim)
    got_k, got_v = d.pools()
    want_k, want_v = before[0].copy(), before[1].copy()
    angle = np.zeros((rows, rope_dim // 2))
    for s, n in enumerate(b.rows):
        for i in range(n):
            r, t = b.start[s] + i, b.lengths[s] - n + i
            angle[r] = (positions[r] if positions is not None else b.prefix + t) * freq[:rope_dim // 2]
    heads = new[:, :wide - pad].reshape(rows, n_q + 2 * kv, dim)
    turned = cases.rotate(heads[:, :n_q + kv], angle, float(np.float32(factor)), layout)
    for s, n in enumerate(b.rows):
        for i in range(n):
            r, (p, slot) = b.start[s] + i, b.place(s, b.lengths[s] - n + i)
            want_k[p, :, slot], want_v[p, :, slot] = turned[r, n_q:], heads[r, n_q + kv:]
    assert np.array_equal(got_v, want_v)
    # one rounding to the type, and of the fp32 sine, cosine, products and sum: eight half steps of the pair's size (at most 6 here)
    room = cases.HALF_STEP[kind] * 1.01
    near = lambda a, w: (np.abs(a - w) <= room * np.abs(w) + 8 * 2.0 ** -24 * 12 * abs(factor) + 2.0 ** -24).all()  # noqa: E731
    assert near(got_k, want_k)
    if queries:
        got = cases.from_bits(out.download(WORD[kind], (rows, wide if in_place else n_q * dim)), kind)
        want = turned[:, :n_q].reshape(rows, -1)
        assert near(got[:b.live, :n_q * dim], want[:b.live])
        assert np.array_equal(got[b.live:, :n_q * dim], new[b.live:, :n_q * dim] if in_place else np.full((rows - b.live, n_q * dim), 7.0))
        if in_place:
            assert np.array_equal(got[:, n_q * dim:], new[:, n_q * dim:])
    return got_k, got_v


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("layout", [capi.ROPE_ADJACENT, capi.ROPE_HALVES])
@pytest.mark.parametrize("dim,rope_dim", [(64, 64), (64, 32), (64, 2), (128, 128), (128, 0), (128, 40), (128, 126), (256, 256), (256, 72), (256, 24)])
def test_append(ctx, kind, layout, dim, rope_dim):
    g = np.random.default_rng(dim + rope_dim)
    b = cases.Batch(g, [1, 0, 5, 2, 17], [1, 4, 40, 2, 100], 16, 2, dim, order="tokens" if layout else "heads", behind=2)
    check_append(ctx, g, kind, 6, b, rope_dim, layout, factor=1.25)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rope_dim", [64, 6])
def test_append_in_place_behind_a_prefix_and_of_many_rows(ctx, kind, rope_dim):
    g = np.random.default_rng(3)
    check_append(ctx, g, kind, 3, cases.Batch(g, [1, 2], [70, 9], 5, 1, 64, prefix=1000, behind=1), rope_dim, 1, pad=8, in_place=True)
    check_append(ctx, g, kind, 3, cases.Batch(g, [400, 0, 203], [500, 3, 203], 32, 1, 64, behind=3), rope_dim, 0, in_place=True)
    check_append(ctx, g, kind, 3, cases.Batch(g, [2, 2], [70, 9], 5, 1, 64), rope_dim, 1, queries=False)


@pytest.mark.parametrize("far", [131071, 5_000_000, 2 ** 31 - 1])
def test_far_positions(ctx, far):
    """fp32 angles would be off by far 2^-24 radians."""
    g = np.random.default_rng(4)
    check_append(ctx, g, "f16", 2, cases.Batch(g, [3], [20], 16, 1, 128), 128, 1, positions=[far, far - 1, far // 2], theta=1e6)


def test_lengths_that_leave_a_row_without_a_token(ctx):
    """More rows than tokens: those in front write nothing, and the error word says so."""
    g = np.random.default_rng(6)
    b = cases.Batch(g, [3], [2], 4, 1, 64)
    k, v, _ = b.fill(g, 5.0)
    d = Device(ctx, b, "f16", 1, k, v)
    rows = ctx.to_device(cases.to_bits(g.standard_normal((3, 64)), "f16"))
    ctx.call("paged_append", C.byref(d.cache), C.byref(d.batch), None, None, 0, rows.ptr, 64, rows.ptr, 64, None, 0)
    got = d.pools()[1]
    want = cases.from_bits(rows.download(np.float16, (3, 64)), "f16")
    seen = [got[b.place(0, t)[0], 0, b.place(0, t)[1]] for t in range(2)]
    assert np.array_equal(seen, want[1:])
    assert ctx.call_status("device_error", np.zeros(1, np.uint32)) == capi.OUT_OF_RANGE
    assert ctx.device_error_flags() == 0


@pytest.mark.parametrize("page", [16, 20, 128])
@pytest.mark.parametrize("n_q,dim", [(40, 64), (40, 128), (40, 256)])
def test_pages_outside_the_pool_under_many_columns(ctx, page, n_q, dim):
    g = np.random.default_rng(page + dim)
    for bad in (-1, 2 ** 31 - 1):
        b = cases.Batch(g, [6, 5], [700, 500], page, 1, dim)
        k, v, tokens = b.fill(g, np.nan)
        b.table[0, 1] = bad
        q = cases.rounded(g.standard_normal((11, n_q, dim)), "bf16")
        got = Device(ctx, b, "bf16", n_q, k, v).attend(q, 0.1)
        want, size, reach = cases.attend(b, [cases.rounded(t, "bf16") for t in tokens], q, np.float32(0.1))
        assert (np.abs(got - want) <= cases.attend_bound(want, size, reach, "bf16", dim))[6:].all() and np.isfinite(got).all()
        assert ctx.device_error_flags() == 0x10000


def test_pages_outside_the_pool_are_not_followed(ctx):
    g = np.random.default_rng(7)
    for bad in (-1, 2 ** 31 - 1, None):
        b = cases.Batch(g, [2, 1], [40, 30], 16, 1, 64, prefix=20)
        bad = b.pages if bad is None else bad
        k, v, tokens = b.fill(g, np.nan)
        b.table[0, 2] = bad
        d = Device(ctx, b, "f16", 2, k, v)
        q = cases.rounded(g.standard_normal((3, 2, 64)), "f16")
        got = d.attend(q, 0.2)
        want, size, reach = cases.attend(b, [cases.rounded(t, "f16") for t in tokens], q, np.float32(0.2))
        assert (np.abs(got - want) <= cases.attend_bound(want, size, reach, "f16", 64))[2].all()  # the other sequence
        assert np.isfinite(got).all()
        assert ctx.device_error_flags() == 0x10000
        before = d.pools()
        rows = ctx.to_device(cases.to_bits(np.ones((3, 64)), "f16"))
        ctx.call("paged_append", C.byref(d.cache), C.byref(d.batch), None, None, 0, rows.ptr, 64, rows.ptr, 64, None, 0)
        assert ctx.device_error_flags() == 0x10000
        changed = (np.nan_to_num(d.pools()[0]) != np.nan_to_num(before[0])).any((1, 3))
        assert changed.sum() == 1 and changed[b.place(1, 29)]


# ── drafted tokens ──────────────────────────────────────────────────────────
def run_verify(ctx, kind, start, target, draft, tokens, temperature, random, pad=0, shift=0):
    """target [rows, vocab] and draft [steps, seqs, vocab] as bits; rows pad apart, shift values into their buffer."""
    rows, V = target.shape
    put = lambda a: ctx.to_device(np.concatenate([np.zeros(shift, a.dtype), np.pad(a.reshape(-1, V), ((0, 0), (0, pad))).ravel()]))  # noqa: E731
    word = target.dtype.itemsize
    dt, dd = put(target), put(draft) if draft is not None else None
    kept = [ctx.to_device(a) for a in (np.asarray(start, np.int32), np.asarray(tokens, np.int32), np.asarray(temperature, np.float32), np.asarray(random, np.float32))]
    out, accepted = ctx.to_device(np.full(rows, -99, np.int32)), ctx.to_device(np.full(len(start) - 1, -99, np.int32))
    a = capi.VerifyArgs(precision=LOGITS[kind], n_seqs=len(start) - 1, rows=rows, vocab=V, target_stride=V + pad, row_start=kept[0].ptr, target=dt.at(shift * word), tokens=kept[1].ptr,
                        temperature=kept[2].ptr, random=kept[3].ptr, out_tokens=out.ptr, accepted=accepted.ptr)
    if draft is not None:
        a.draft, a.draft_step_stride, a.draft_seq_stride = dd.at(shift * word), (V + pad) * draft.shape[1], V + pad
    size = C.c_size_t()
    ctx.call("verify_drafts_workspace", C.byref(a), C.byref(size))
    work = ctx.alloc(size.value).fill(0xFF)
    a.workspace, a.workspace_bytes = work.ptr, size.value
    ctx.call("verify_drafts", C.byref(a))
    return out.download(np.int32, rows), accepted.download(np.int32, len(start) - 1)


def verify_case(g, kind, rows, V, near=0.7, peak=6.0):
    """Logits of a target and of a draft model near it, drafts drawn from the draft model."""
    start = np.concatenate([[0], np.cumsum(rows)])
    total, steps = int(start[-1]), max(1, max(rows) - 1)
    target = g.standard_normal((total, V))
    for r in range(total):
        target[r, g.integers(0, V, 4)] += peak
    draft = g.standard_normal((steps, len(rows), V))
    tokens = g.integers(0, V, total)
    for s, n in enumerate(rows):
        for j in range(n - 1):
            draft[j, s] = target[start[s] + j] + near * draft[j, s]
            tokens[start[s] + j + 1] = g.choice(V, p=cases.law(draft[j, s], 0.8))
    return start, cases.to_bits(target, kind), cases.to_bits(draft, kind), tokens, np.full(len(rows), 0.8, np.float32), g.random(total).astype(np.float32)


def check_verify(ctx, kind, start, target, draft, tokens, temperature, random, **kw):
    got = run_verify(ctx, kind, start, target, draft, tokens, temperature, random, **kw)
    want = cases.verify(start, cases.from_bits(target, kind), None if draft is None else cases.from_bits(draft, kind), tokens, temperature, random)
    live = start[-1]
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0][:live], want[0][:live]) and (got[0][live:] == -99).all()
    return got


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 7, 1000, 8193, 40001])
@pytest.mark.parametrize("drafted", [True, False])
def test_verify(ctx, kind, V, drafted):
    g = np.random.default_rng(V)
    start, target, draft, tokens, temperature, random = verify_case(g, kind, [1, 5, 0, 2, 8, 3, 1, 4], V)
    temperature[:] = g.random(8) + 0.3
    temperature[3], temperature[4] = 0, -1
    _, kept = check_verify(ctx, kind, start, target, draft if drafted else None, tokens, temperature, random)
    if V == 1:
        assert kept.tolist() == [0, 4, 0, 1, 7, 2, 0, 3]


@pytest.mark.parametrize("kind,pad,shift", [("f16", 3, 1), ("bf16", 8, 5), ("f32", 1, 3), ("f16", 0, 7)])
def test_verify_rows_at_any_address(ctx, kind, pad, shift):
    g = np.random.default_rng(pad + shift)
    check_verify(ctx, kind, *verify_case(g, kind, [4, 2, 6], 5003), pad=pad, shift=shift)


def test_verify_large_vocabulary(ctx):
    g = np.random.default_rng(21)
    check_verify(ctx, "f16", *verify_case(g, "f16", [3, 1, 5], 151936))
    flat = verify_case(g, "f32", [1] * 12, 151936, peak=0.0)  # every index is a likely answer
    check_verify(ctx, "f32", *flat)


def test_verify_draws_at_the_ends(ctx):
    g = np.random.default_rng(22)
    start, target, draft, tokens, temperature, random = verify_case(g, "f32", [2, 1, 1, 2], 3000)
    for value in (0.0, np.float32(1) - np.float32(2.0 ** -24)):
        random[:] = value
        check_verify(ctx, "f32", start, target, draft, tokens, temperature, random)
    target[:, :1000] = -np.inf
    target[:, 2500:] = np.nan
    out, kept = check_verify(ctx, "f32", start, target, draft, tokens, temperature, random)
    drawn = out[start[:-1] + kept]
    assert (drawn == 2499).all()


def test_verify_masked_rows_bad_ids_and_equal_models(ctx):
    g = np.random.default_rng(23)
    start, target, draft, tokens, temperature, random = verify_case(g, "f16", [3, 3, 3, 3, 2], 4001)
    target[start[0]:start[1]] = -np.inf          # no token has a chance
    tokens[start[1] + 1], tokens[start[2] + 2] = -1, 4001
    for j in range(2):
        draft[j, 3] = target[start[3] + j]       # the draft model is the target: every draft stands
        tokens[start[3] + 1 + j] = int(np.argmax(target[start[3] + j]))
    draft[0, 4] = np.float16(-np.inf)            # a draft model that says nothing: q = 0, p > 0 stands
    tokens[start[4] + 1] = 17
    out, kept = check_verify(ctx, "f16", start, target, draft, tokens, temperature, random)
    assert kept[0] == 0 and out[start[0]] == -1 and kept[1] == 0 and kept[2] <= 1 and kept[3] == 2 and kept[4] == 1
    check_verify(ctx, "f16", start, target, None, tokens, temperature, random)


@pytest.mark.parametrize("kind,pad,shift", [("f16", 0, 0), ("f16", 3, 1), ("f32", 1, 2)])
def test_verify_bad_ids_under_equal_models_draw_from_the_target(ctx, kind, pad, shift):
    """p - q leaves nothing but rounding, in rows that begin at different addresses too."""
    g = np.random.default_rng(25)
    start, target, draft, tokens, temperature, random = verify_case(g, kind, [2, 3, 2], 40001)
    for s in range(3):
        draft[0, s] = target[start[s]]
        tokens[start[s] + 1] = -1
    out, kept = check_verify(ctx, kind, start, target, draft, tokens, temperature, random, pad=pad, shift=shift)
    assert kept.tolist() == [0, 0, 0] and (out[start[:-1]] >= 0).all()


@pytest.mark.parametrize("drafted", [True, False])
def test_verify_many_sequences(ctx, drafted):
    g = np.random.default_rng(26)
    start, target, draft, tokens, temperature, random = verify_case(g, "bf16", g.integers(0, 4, 120).tolist(), 9001)
    check_verify(ctx, "bf16", start, target, draft if drafted else None, tokens, temperature, random)


def test_verify_without_end_of_temperature_every_token_is_alike(ctx):
    g = np.random.default_rng(27)
    V = 4096
    target = g.standard_normal((5, V)).astype(np.float32)
    target[:, 1000:2000] = -np.inf
    random = np.array([0.25, 0.5, 0.999, 1e-4, 0.75], np.float32)
    out, kept = run_verify(ctx, "f32", [0, 1, 2, 5], target, None, [0, 0, 0, 5, 7], [np.inf] * 3, random)
    left = np.r_[0:1000, 2000:V]
    assert kept.tolist() == [0, 0, 0]  # u = 0.999 and 1 / 3096
    assert out[0] == left[int(0.25 * left.size)] and out[1] == left[int(0.5 * left.size)]
    assert out[2] == np.delete(left, 5)[int(0.75 * (left.size - 1))] and out[3:].tolist() == [-1, -1]
    random[2], random[3] = 1e-4, 3e-4
    out, kept = run_verify(ctx, "f32", [0, 1, 2, 5], target, None, [0, 0, 0, 5, 7], [np.inf] * 3, random)
    assert kept.tolist() == [0, 0, 2] and out[2:4].tolist() == [5, 7] and out[4] == left[int(0.75 * left.size)]


def test_verify_of_no_rows(ctx):
    out, kept = run_verify(ctx, "f16", [0, 0, 0], np.zeros((0, 50), np.float16), None, [], [1.0, 1.0], [])
    assert kept.tolist() == [0, 0] and out.size == 0


def test_verify_greedy_ties_take_the_lowest_index(ctx):
    target = np.zeros((4, 300), np.float16)
    target[0, [40, 90, 299]] = 2
    target[1, [3]] = -0.0
    target[2, :] = -np.inf
    target[2, 7] = np.inf
    target[2, 5] = np.inf
    out, kept = run_verify(ctx, "f16", [0, 4], target, None, [0, 40, 0, 5], [0.0], [0.9] * 4)
    assert kept.tolist() == [3] and out.tolist() == [40, 0, 5, 0]


def test_verify_draws_follow_the_target(ctx):
    """Many sequences with the same laws: what is drawn is distributed as the target says."""
    g = np.random.default_rng(24)
    V, n, t = 50, 4000, 0.9
    p, q = np.float16(g.standard_normal(V) * 1.5), np.float16(g.standard_normal(V) * 1.5)
    x = g.choice(V, n, p=cases.law(q, t))
    start = np.arange(0, 2 * n + 1, 2)
    out, kept = run_verify(ctx, "f16", start, np.tile(p, (2 * n, 1)), np.tile(q, (1, n, 1)), np.stack([np.zeros(n, int), x], 1).ravel(), np.full(n, t), g.random(2 * n))
    seen = np.bincount(out[0::2], minlength=V) / n
    assert np.abs(seen - cases.law(p, t)).max() < 5 * np.sqrt(0.25 / n)
    assert abs(kept.mean() - np.minimum(cases.law(p, t), cases.law(q, t)).sum()) < 5 * np.sqrt(0.25 / n)


# ── together ────────────────────────────────────────────────────────────────
def test_a_servers_step_captured_and_replayed(ctx):
    """Append, attention and verification in one capture; lengths, tables and drafts change on the device between replays."""
    g = np.random.default_rng(31)
    n_q, kv, dim, page, V, seqs, most, P = 8, 2, 64, 16, 5000, 4, 3, 50
    b = cases.Batch(g, [most] * seqs, [200] * seqs, page, kv, dim, prefix=P)
    k, v, _ = b.fill(g, 0.0)
    d = Device(ctx, b, "f16", n_q, k, v)
    total, wide = b.total, (n_q + 2 * kv) * dim
    new, q_out, out = ctx.alloc(total * wide * 2), ctx.alloc(total * n_q * dim * 2), ctx.alloc(total * n_q * dim * 2)
    freq = ctx.to_device(capi.rope_frequencies(dim, 1e4)[0])
    rope = capi.RopeDesc(dim, 1, 1.0, freq.ptr, None)
    work, size = d.workspace()
    logits, tokens, random = ctx.alloc(total * V * 2), ctx.alloc(total * 4), ctx.alloc(total * 4)
    said, kept = ctx.alloc(total * 4), ctx.alloc(seqs * 4)
    args = capi.VerifyArgs(precision=LOGITS["f16"], n_seqs=seqs, rows=total, vocab=V, target_stride=V, row_start=d.kept[0].ptr, target=logits.ptr, tokens=tokens.ptr, random=random.ptr,
                           out_tokens=said.ptr, accepted=kept.ptr)
    need = C.c_size_t()
    ctx.call("verify_drafts_workspace", C.byref(args), C.byref(need))
    stats = ctx.alloc(need.value)
    args.workspace, args.workspace_bytes = stats.ptr, need.value

    def step():
        ctx.call("paged_append", C.byref(d.cache), C.byref(d.batch), C.byref(rope), new.ptr, wide, new.at(n_q * dim * 2), wide, new.at((n_q + kv) * dim * 2), wide, q_out.ptr, n_q * dim)
        ctx.call("paged_attention", C.byref(d.cache), C.byref(d.batch), q_out.ptr, n_q * dim, out.ptr, n_q * dim, 0.125, 0, work.ptr, size)
        ctx.call("verify_drafts", C.byref(args))

    ctx.call("capture_begin")
    step()
    ctx.call("capture_end")
    ms = C.c_float()
    history = [[] for _ in range(seqs)]
    angle = lambda t: (P + t) * capi.rope_frequencies(dim, 1e4)[0][None]  # noqa: E731
    ahead = [np.zeros((P, kv, dim)), np.zeros((P, kv, dim))]
    for t in range(P):
        ahead[0][t], ahead[1][t] = (cases.rounded(p, "f16")[b.prefix_table[t // page], :, t % page] for p in (k, v))
    lengths = [0] * seqs
    for turn in range(4):
        rows = [int(g.integers(0, most + 1)) for _ in range(seqs)]
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        lengths = [n + r for n, r in zip(lengths, rows)]
        d.kept[0].upload(start)
        d.kept[1].upload(np.array(lengths, np.int32))
        x = cases.rounded(g.standard_normal((total, wide)), "f16")
        new.upload(np.float16(x))
        out.upload(np.full(total * n_q * dim, 7, np.float16))
        target, ids, u = np.float16(3 * g.standard_normal((total, V))), g.integers(0, V, total), g.random(total).astype(np.float32)
        for r in range(total - 1):
            target[r, ids[r + 1]] += 9
        logits.upload(target), tokens.upload(ids.astype(np.int32)), random.upload(u)
        ctx.call("capture_replay", turn % 2, 1 + turn % 2, C.byref(ms))
        heads = x.reshape(total, n_q + 2 * kv, dim)
        q = np.zeros((total, n_q, dim))
        got_q = q_out.download(np.float16, (total, n_q, dim)).astype(np.float64)
        for s in range(seqs):
            for i in range(rows[s]):
                r, t = start[s] + i, lengths[s] - rows[s] + i
                turned = cases.rotate(heads[r:r + 1, :n_q + kv], angle(t), 1.0, 1)[0]
                assert np.abs(turned[:n_q] - got_q[r]).max() < 2.0 ** -10 * 4
                p, slot = b.place(s, t)
                history[s].append((d.pools()[0][p, :, slot], heads[r, n_q + kv:]))
                assert np.abs(history[s][-1][0] - turned[n_q:]).max() < 2.0 ** -10 * 4
                q[r] = got_q[r]
        tokens_now = [np.stack([np.concatenate([ahead[i]] + [np.stack([h[i] for h in history[s]])] if history[s] else [ahead[i]]) for i in range(2)]) for s in range(seqs)]
        b.start, b.rows, b.lengths = start, rows, lengths
        want, reach_v, reach = cases.attend(b, tokens_now, q, 0.125)
        got = out.download(np.float16, (total, n_q, dim)).astype(np.float64)
        live = start[-1]
        assert (np.abs(got - want) <= cases.attend_bound(want, reach_v, reach, "f16", dim))[:live].all() and (got[live:] == 7).all()
        want_said, want_kept = cases.verify(start, target.astype(np.float64), None, ids, [1.0] * seqs, u)
        assert np.array_equal(said.download(np.int32, total)[:live], want_said[:live]) and np.array_equal(kept.download(np.int32, seqs), want_kept)


def test_refusals(ctx):
    g = np.random.default_rng(41)
    b = cases.Batch(g, [2, 1], [20, 10], 16, 2, 64, prefix=16)
    k, v, _ = b.fill(g, 0.0)
    d = Device(ctx, b, "f16", 4, k, v)
    q, out = ctx.alloc(3 * 256 * 2 + 16), ctx.alloc(3 * 256 * 2 + 16)
    work, size = d.workspace()
    ok = dict(q=q.ptr, qs=256, out=out.ptr, os=256, scale=0.1, work=work.ptr, size=size)

    def attend(cache={}, batch={}, **kw):
        c, t, a = capi.PagedCache.from_buffer_copy(d.cache), capi.PagedBatch.from_buffer_copy(d.batch), {**ok, **kw}
        for s, change in ((c, cache), (t, batch)):
            for n, x in change.items():
                setattr(s, n, x)
        first = ctx.call_status("paged_attention", C.byref(c), C.byref(t), a["q"], a["qs"], a["out"], a["os"], a["scale"], 0, a["work"], a["size"])
        if (cache or batch) and first in (capi.BAD_ARGUMENT, capi.OUT_OF_RANGE):  # the append refuses the same descriptions
            assert ctx.call_status("paged_append", C.byref(c), C.byref(t), None, None, 0, k_dev.ptr, 128, k_dev.ptr, 128, None, 0) == first
        return first

    k_dev = ctx.alloc(3 * 128 * 2)
    assert attend() == capi.OK
    bad = capi.BAD_ARGUMENT
    for change in (dict(precision=2), dict(n_q=3), dict(n_q=0), dict(n_kv=0), dict(page_size=0), dict(n_pages=0), dict(page_stride=-8), dict(head_stride=12), dict(token_stride=32), dict(k=None), dict(v=None),
                   dict(k=d.k.ptr + 2)):
        assert attend(cache=change) == bad, change
    assert attend(cache=dict(head_dim=96)) == capi.UNSUPPORTED
    for change in (dict(n_seqs=-1), dict(rows=-1), dict(max_rows=-1), dict(table_stride=-1), dict(prefix_length=-1), dict(row_start=None), dict(length=None), dict(table=None), dict(prefix_table=None)):
        assert attend(batch=change) == bad, change
    assert attend(batch=dict(rows=2 ** 30)) == capi.OUT_OF_RANGE
    assert attend(batch=dict(n_seqs=1025)) == capi.UNSUPPORTED
    for change in (dict(q=None), dict(q=q.ptr + 2), dict(qs=128), dict(qs=260), dict(out=None), dict(os=255), dict(scale=float("nan")), dict(scale=float("inf")), dict(work=None), dict(work=work.ptr + 4),
                   dict(size=size - 1), dict(out=q.ptr, os=264)):
        assert attend(**change) == bad, change
    assert attend(batch=dict(n_seqs=0)) == capi.OK and attend(batch=dict(rows=0)) == capi.OK
    freq = ctx.to_device(np.ones(32))
    for change in (dict(rope_dim=-2), dict(rope_dim=3), dict(rope_dim=66), dict(layout=2), dict(freq=None)):
        rope = capi.RopeDesc(64, 1, 1.0, freq.ptr, None)
        for n, x in change.items():
            setattr(rope, n, x)
        assert ctx.call_status("paged_append", C.byref(d.cache), C.byref(d.batch), C.byref(rope), None, 0, k_dev.ptr, 128, k_dev.ptr, 128, None, 0) == bad, change
    for change in (dict(k=None), dict(k=k_dev.ptr + 8), dict(ks=64), dict(ks=130), dict(v=None), dict(q_out=None), dict(qs=100), dict(q_out=q.ptr, qos=264)):
        a = dict(k=k_dev.ptr, ks=128, v=k_dev.ptr, q=q.ptr, qs=256, q_out=out.ptr, qos=256) | change
        assert ctx.call_status("paged_append", C.byref(d.cache), C.byref(d.batch), None, a["q"], a["qs"], a["k"], a["ks"], a["v"], 128, a["q_out"], a["qos"]) == bad, change
    assert ctx.call_status("paged_attention_workspace", C.byref(d.cache), C.byref(d.batch), None) == bad


def test_verify_refusals(ctx):
    buf, need = ctx.alloc(1 << 16), C.c_size_t()
    good = dict(precision=0, n_seqs=1, rows=2, vocab=100, target_stride=100, row_start=buf.ptr, target=buf.at(1024), tokens=buf.at(4096), random=buf.at(5120), out_tokens=buf.at(6144),
                accepted=buf.at(7168), workspace=buf.at(8192), workspace_bytes=8192)
    buf.upload(np.array([0, 2], np.int32))

    def status(**change):
        return ctx.call_status("verify_drafts", C.byref(capi.VerifyArgs(**{**good, **change})))

    assert status() == capi.OK
    for change in (dict(precision=3), dict(n_seqs=-1), dict(rows=-1), dict(vocab=0), dict(target_stride=99), dict(row_start=None), dict(target=None), dict(target=buf.at(1025)), dict(tokens=None),
                   dict(random=None), dict(out_tokens=None), dict(out_tokens=buf.at(4096)), dict(accepted=None), dict(workspace=None), dict(workspace=buf.at(8196)), dict(workspace_bytes=16),
                   dict(draft=buf.at(1025)), dict(draft=buf.at(1024), draft_seq_stride=-1)):
        assert status(**change) == capi.BAD_ARGUMENT, change
    assert status(vocab=1 << 25, target_stride=1 << 25) == capi.OUT_OF_RANGE and status(rows=1 << 21) == capi.OUT_OF_RANGE
    assert status(n_seqs=0) == capi.OK and status(rows=0) == capi.OK
    assert ctx.call_status("verify_drafts_workspace", C.byref(capi.VerifyArgs(**good)), None) == capi.BAD_ARGUMENT
