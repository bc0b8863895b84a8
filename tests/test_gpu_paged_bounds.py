"""The batch over pages at its bounds: calls repeated, arrays that say what they should not, infinite values, plans that only large calls take."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as cases
import paged_pairs as pairs
from smelt_b200 import capi
from test_gpu_paged import CODE, LOGITS, WORD, Device, check_append, check_attention, check_verify, run_verify, verify_case  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context(0)
    yield c
    assert c.device_error_flags() == 0
    c.close()


@pytest.mark.parametrize("kind,n_q,n_kv,dim", [("f16", 4, 2, 64), ("bf16", 24, 2, 64), ("f16", 8, 2, 128), ("bf16", 32, 2, 128), ("f16", 6, 1, 256)])
@pytest.mark.parametrize("page", [1, 20])
def test_the_same_call_gives_the_same_bits(ctx, kind, n_q, n_kv, dim, page):
    """Every row is fetched from where its own page lies, whichever lane of a warp runs ahead: rings of an odd and of an even number of units,
    first fills that begin a second tile, items of a single tile and of many."""
    g = np.random.default_rng(dim + page)
    b = cases.Batch(g, [1] * 6, [1000, 33, 4, 257, 64, 1500], page, n_kv, dim, order="tokens")
    k, v, tokens = b.fill(g, np.nan)
    q = cases.rounded(g.standard_normal((b.total, n_q, dim)), kind)
    d = Device(ctx, b, kind, n_q, k, v)
    first = d.attend(q, 0.1)
    want, size, reach = cases.attend(b, [cases.rounded(t, kind) for t in tokens], q, np.float32(0.1))
    assert (np.abs(first - want) <= cases.attend_bound(want, size, reach, kind, dim)).all()
    for _ in range(10):
        assert np.array_equal(d.attend(q, 0.1), first)


@pytest.mark.parametrize("length", [-2 ** 31, -2 ** 31 + 1, -1, 0, 2 ** 31 - 1])
@pytest.mark.parametrize("rows", [1, 3])
def test_append_cuts_lengths_at_both_ends(ctx, length, rows):
    """Without tokens nothing is written; tokens past the table are its last ones."""
    g = np.random.default_rng(6)
    b = cases.Batch(g, [rows, 2], [8, 6], 4, 1, 64)
    b.table = np.ascontiguousarray(b.table[:, :2])  # eight tokens a sequence
    k, v, _ = b.fill(g, 5.0)
    d = Device(ctx, b, "f16", 1, k, v)
    before = d.pools()[1]
    d.kept[1].upload(np.array([length, 6], np.int32))
    new = ctx.to_device(cases.to_bits(g.standard_normal((rows + 2, 64)), "f16"))
    ctx.call("paged_append", C.byref(d.cache), C.byref(d.batch), None, None, 0, new.ptr, 64, new.ptr, 64, None, 0)
    want, put = before.copy(), cases.from_bits(new.download(np.float16, (rows + 2, 64)), "f16")
    for s, at in ((0, 8 - rows if length > 0 else None), (1, 4)):
        for i in range(b.rows[s]):
            if at is not None:
                p, slot = b.place(s, at + i)
                want[p, 0, slot] = put[b.start[s] + i]
    assert np.array_equal(d.pools()[1], want)
    assert ctx.device_error_flags() == (0 if length > 0 else 0x10000)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("steps", [1, 3, 6])
@pytest.mark.parametrize("t", [0.8, 0.0])
def test_drafts_behind_the_steps_of_a_draft_are_not_judged(ctx, kind, steps, t):
    """Row starts that give a sequence more drafts than the draft model left logits for: those of the array are judged, and the token behind
    them is drawn from the target.  (What lies behind the array here would let every draft stand.)"""
    g = np.random.default_rng(steps)
    rows, V = [7, 1, 2, 5, 0, 7, 7], 3001
    start, target, draft, tokens, temperature, random = verify_case(g, kind, rows, V, near=0.2, peak=9.0)
    temperature[:] = t
    for s in (0, 5):  # drafts that stand, as far as anybody looks
        for j in range(rows[s] - 1):
            draft[j, s] = target[start[s] + j]
            tokens[start[s] + 1 + j] = int(np.argmax(cases.from_bits(target[start[s] + j], kind)))
    word, total = target.dtype.itemsize, int(start[-1])
    dt, dd = ctx.to_device(target), ctx.to_device(draft)
    kept = [ctx.to_device(np.asarray(a, w)) for a, w in ((start, np.int32), (tokens, np.int32), (temperature, np.float32), (random, np.float32))]
    out, accepted = ctx.to_device(np.full(total, -99, np.int32)), ctx.to_device(np.full(len(rows), -99, np.int32))
    a = capi.VerifyArgs(precision=LOGITS[kind], draft_steps=steps, n_seqs=len(rows), rows=total, vocab=V, target_stride=V, row_start=kept[0].ptr, target=dt.ptr, draft=dd.ptr,
                        draft_step_stride=len(rows) * V, draft_seq_stride=V, tokens=kept[1].ptr, temperature=kept[2].ptr, random=kept[3].ptr, out_tokens=out.ptr, accepted=accepted.ptr)
    size = C.c_size_t()
    ctx.call("verify_drafts_workspace", C.byref(a), C.byref(size))
    work = ctx.alloc(size.value).fill(0xFF)
    a.workspace, a.workspace_bytes = work.ptr, size.value
    ctx.call("verify_drafts", C.byref(a))
    said, stood = out.download(np.int32, total), accepted.download(np.int32, len(rows))
    for s, n in enumerate(rows):
        cut = min(n, steps + 1)
        at = np.arange(start[s], start[s] + cut)
        u = random[at].copy()
        if cut:
            u[-1] = random[start[s] + n - 1]
        want, full = cases.verify([0, cut], cases.from_bits(target, kind)[at], cases.from_bits(draft, kind)[:, s:s + 1], np.asarray(tokens)[at], [t], u)
        assert stood[s] == full[0] and np.array_equal(said[start[s]:start[s] + n], np.concatenate([want, np.full(n - cut, -1)])), (s, said, want)
    assert stood[0] == min(6, steps) and stood[5] == min(6, steps)


@pytest.mark.parametrize("n_q,dim,rows", [(4, 64, 4), (32, 128, 40), (16, 256, 30)])  # streaming and tensor-core kernel
@pytest.mark.parametrize("prefix,window", [(0, 0), (100, 0), (100, 60)])
def test_row_starts_that_go_down_compute_nothing(ctx, n_q, dim, rows, prefix, window):
    g = np.random.default_rng(dim + prefix)
    b = cases.Batch(g, [rows] * 5, [rows + 50] * 5, 16, 2, dim, prefix=prefix)
    k, v, tokens = b.fill(g, 0.0)
    q = cases.rounded(g.standard_normal((b.total, n_q, dim)), "f16")
    d = Device(ctx, b, "f16", n_q, k, v)
    good = d.attend(q, 0.1, window)
    for starts in ([0, 5 * rows, 0, 5 * rows, 0, 5 * rows], [0, rows, 2 * rows, 2 * rows - 1, 4 * rows, 5 * rows], [1, 0, 2, 3, 4, 5], [0, rows, 3 * rows, 4 * rows, 5 * rows, -(2 ** 31)]):
        d.kept[0].upload(np.array(starts, np.int32))
        assert (d.attend(q, 0.1, window) == 7.0).all()
        assert ctx.device_error_flags() == 0x10000
    d.kept[0].upload(np.minimum(b.start.astype(np.int64) * 2 ** 20, 2 ** 31 - 1).astype(np.int32))  # cut to the rows there are: all are the first sequence's, whose last tokens they are
    d.attend(q, 0.1, window)
    assert ctx.device_error_flags() == 0
    d.kept[0].upload(b.start)
    assert np.array_equal(d.attend(q, 0.1, window), good)


def test_graphs_that_the_caller_captures_run_side_by_side(ctx):
    """Two calls captured from the context's stream, each with a workspace of its own, replayed on two streams, and eager calls beside them."""
    torch = pytest.importorskip("torch")
    g = np.random.default_rng(51)
    calls = []
    for lengths, n_q in (([600], 8), ([900, 40, 3], 4), ([500, 2], 8)):
        b = cases.Batch(g, [1] * len(lengths), lengths, 16, 2, 128)
        k, v, _ = b.fill(g, 0.0)
        q = cases.rounded(g.standard_normal((b.total, n_q, 128)), "f16")
        d = Device(ctx, b, "f16", n_q, k, v)
        want = d.attend(q, 0.1)
        dq, out = ctx.to_device(np.float16(q)), ctx.to_device(np.full(q.shape, 7, np.float16))
        work, size = d.workspace()
        args = (C.byref(d.cache), C.byref(d.batch), dq.ptr, n_q * 128, out.ptr, n_q * 128, 0.1, 0, work.ptr, size)
        calls.append((args, out, want, (d, dq, work)))
    torch.cuda.set_device(0)
    torch.zeros(1, device="cuda")
    own = torch.cuda.ExternalStream(ctx.lib.smelt_cuda_stream(ctx.h))
    graphs, sides = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for args, _, _, _ in calls[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(own):
            graph.capture_begin(capture_error_mode="thread_local")
            ctx.call("paged_attention", *args)
            graph.capture_end()
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for _, out, want, _ in calls:
            out.upload(np.full(want.shape, 7, np.float16))
        for _ in range(10):
            for graph, side in zip(graphs, sides):
                with torch.cuda.stream(side):
                    graph.replay()
            ctx.call("paged_attention", *calls[2][0])
        torch.cuda.synchronize()
        for _, out, want, _ in calls:
            assert np.array_equal(out.download(np.float16, want.shape).astype(np.float64), want)
    del graphs


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("t", [1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-8, 1e-30, 1e-40])
@pytest.mark.parametrize("drafted", [True, False])
def test_small_temperatures(ctx, kind, t, drafted):
    """Almost greedy: a draft that is the only likely token of both models stands, whatever u below 1, and so does the draw."""
    g = np.random.default_rng(61)
    rows, V = [4] * 40, 4099
    start, target, draft, tokens, temperature, random = verify_case(g, "f32", rows, V)
    target, draft = np.minimum(target, 6.0), np.minimum(draft, 6.0)
    for r in range(int(start[-1])):  # one token far above the rest, at any height
        target[r, tokens[r + 1] if r + 1 < len(tokens) else 0] = g.uniform(8, 30)
    for s, n in enumerate(rows):
        for j in range(n - 1):
            draft[j, s, tokens[start[s] + j + 1]] = g.uniform(8, 30)
        tokens[start[s]] = 0
    target[3::4] = np.minimum(target[3::4], 6.0)
    for r in range(3, int(start[-1]), 4):
        target[r, g.integers(0, V)] = g.uniform(8, 30)
    random[:] = np.float32(1) - np.float32(2.0 ** -24)
    random[3::4] = g.random(40)  # the draw's
    target, draft = cases.to_bits(target, kind), cases.to_bits(draft, kind)
    temperature[:] = t
    out, kept = check_verify(ctx, kind, start, target, draft if drafted else None, tokens, temperature, random)
    assert (kept == 3).all() and np.array_equal(out.reshape(40, 4)[:, :3], np.asarray(tokens).reshape(40, 4)[:, 1:])


@pytest.mark.parametrize("t", [1e-3, 1e-6])
def test_small_temperatures_share_what_is_close(ctx, t):
    """Two tokens a fraction of T apart at the height where T is far below a logit's last place in the product with 1 / T."""
    g = np.random.default_rng(62)
    V, n = 1000, 64
    target = np.full((2 * n, V), -50.0, np.float32)
    step = np.float32(2.0 ** -20) if t < 1e-4 else np.float32(2.0 ** -11)
    target[:, 10], target[:, 700] = np.float32(13.0), np.float32(13.0) + step  # exact in fp32
    chance = 1 / (1 + np.exp(-float(step) / float(np.float32(t))))  # of token 700
    random = np.repeat(np.linspace(0.01, 0.99, n), 2).astype(np.float32)
    assert np.abs(random - chance).min() > 1e-5  # none within the error of fp32 sums
    tokens = np.tile([0, 700], n)
    start = np.arange(0, 2 * n + 1, 2)
    out, kept = check_verify(ctx, "f32", start, target, None, tokens, np.full(n, t, np.float32), random)
    assert np.array_equal(kept, (random[0::2] < chance).astype(np.int32))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim,rows", [(2, 2, 64, 1), (10, 1, 64, 1), (8, 2, 128, 2), (4, 1, 128, 4), (4, 1, 256, 2), (8, 2, 64, 40), (16, 2, 128, 33), (40, 1, 256, 5)])
@pytest.mark.parametrize("prefix,window", [(0, 0), (300, 0), (300, 500)])
def test_infinite_values_that_a_row_sees(ctx, kind, n_q, n_kv, dim, rows, prefix, window):
    """A weight times an infinite value is infinite, however small the weight is and however many CTAs have a part of the item; infinities of both
    signs, or what is not a number, give NaN; every other value of the row stays what it is."""
    g = np.random.default_rng(dim + rows + prefix)
    b = cases.Batch(g, [rows, rows, 1], [rows + 700, rows + 3, 150], 16, n_kv, dim, prefix=prefix)
    k, v, tokens = b.fill(g, np.nan)
    tokens = [cases.rounded(t, kind) for t in tokens]
    odd = [np.zeros(t[1].shape) for t in tokens]  # what is not finite of every sequence's values

    def put(s, t, head, d, x):
        p, slot = (b.prefix_table[t // 16], t % 16) if t < prefix else b.place(s, t - prefix)
        v[p, head, slot, d] = x
        for o in odd if t < prefix else odd[s:s + 1]:
            o[t, head, d] = x

    far = prefix + b.lengths[0]
    for n, (t, x) in enumerate([(far - rows, np.inf), (far - 1, -np.inf), (far - rows - 1, np.nan), (prefix + 5, np.inf), (prefix + 400, -np.inf), (prefix + 128, np.inf), (prefix + 131, np.inf)]):
        put(0, t, n % n_kv, 3 * n + 1, x)
    for t, x in ((prefix + 300, np.inf), (prefix + 301, -np.inf)):
        put(0, t, 0, dim - 1, x)
    put(1, prefix + 1, 0, 7, -np.inf)  # in front of every row of the second sequence
    if prefix:
        put(0, 17, 0, 40, np.inf), put(0, 299, 0, 41, np.nan), put(0, 250, n_kv - 1, dim - 2, -np.inf)
    q = cases.rounded(g.standard_normal((b.total, n_q, dim)), kind)
    scale = np.float32(4 / np.sqrt(dim))  # weights from 1 down to 2^-40 and below
    with np.errstate(invalid="ignore"):
        got = Device(ctx, b, kind, n_q, k, v).attend(q, scale, window)
        clean = [np.stack([t[0], np.where(o == 0, t[1], 0)]) for t, o in zip(tokens, odd)]
        want, size, reach = cases.attend(b, clean, q, scale, window)
        bound = cases.attend_bound(want, size, reach, kind, dim)
        for s, n in enumerate(b.rows):
            for i in range(n):
                at = prefix + b.lengths[s] - n + i
                seen = odd[s][max(0, at + 1 - window) if window else 0:at + 1].repeat(n_q // n_kv, 1)
                bad = np.where(seen == 0, 0, seen).sum(0)  # finite: 0
                r = b.start[s] + i
                assert np.array_equal(np.isnan(got[r]), np.isnan(bad)) and np.array_equal(got[r][np.isinf(bad)], bad[np.isinf(bad)]), (s, i)
                fine = bad == 0
                assert (np.abs(got[r] - want[r]) <= bound[r])[fine].all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim,rows,below", [(4, 2, 64, 1, 10.0), (4, 2, 64, 1, 17.0), (12, 1, 128, 1, 14.0), (4, 1, 256, 2, 17.0), (8, 2, 64, 6, 10.0), (8, 2, 128, 6, 13.0), (16, 2, 256, 3, 13.0)])
@pytest.mark.parametrize("prefix", [0, 200])
def test_many_small_weights_behind_a_large_one(ctx, kind, n_q, n_kv, dim, rows, below, prefix):
    """The first key takes nearly all of the weight and has no value: what is left of the output is what thousands of weights of e^-below add up to."""
    g = np.random.default_rng(dim + rows)
    b = cases.Batch(g, [rows, 1], [rows + 1500, 30], 16, n_kv, dim, prefix=prefix)
    k, v, tokens = b.fill(g, 0.0)
    q = np.full((b.total, n_q, dim), 1.0)
    for pool in [k, v]:
        pool[:] = 0
    tokens = [t * 0 for t in tokens]

    def put(s, t, key, value):
        p, slot = (b.prefix_table[t // 16], t % 16) if t < prefix else b.place(s, t - prefix)
        k[p, :, slot], v[p, :, slot] = key, value
        for u in tokens if t < prefix else [tokens[s]]:
            u[0, t], u[1, t] = key, value

    for s in range(2):
        for t in range(prefix if s else 0, prefix + b.lengths[s]):
            put(s, t, 0.0, float(1 + t % 3))
        if s == 0 or not prefix:
            put(s, 0, 1.0, 0.0)
    check = Device(ctx, b, kind, n_q, k, v)
    scale = np.float32(below / dim)
    got = check.attend(q, scale)
    want, size, reach = cases.attend(b, tokens, q, scale)
    # a score is exact but for its product with the scale and log2(e), 2^-23 of `below` each; all else as everywhere
    off = np.abs(got - want) - cases.attend_bound(want, size, reach, kind, dim)
    assert off.max() <= 0, (off.max(), got[0, 0, 0], want[0, 0, 0])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim,rows", [(4, 2, 64, 2), (16, 1, 64, 1), (4, 1, 128, 2), (8, 2, 128, 4), (8, 1, 256, 1)])
@pytest.mark.parametrize("prefix", [0, 12])
def test_streamed_weights_have_two_parts(ctx, kind, n_q, n_kv, dim, rows, prefix):
    """One rounding of the weights would be several times what the bound allows (tests/test_paged_pairs.py)."""
    g = np.random.default_rng(dim + prefix)
    b = cases.Batch(g, [1, rows, 1], [16, 24, 8], 16, n_kv, dim, prefix=prefix)
    k, v, tokens = pairs.fill(g, b, kind)
    q, scale = pairs.queries(g, b.total, n_q, dim), np.float32(0.75 / np.sqrt(dim))
    got = Device(ctx, b, kind, n_q, k, v).attend(q, scale)
    want, size, _ = cases.attend(b, tokens, q, scale)
    off = np.abs(got - want) / pairs.bound(want, size, prefix + 24, pairs.largest_score(b, tokens, q, scale), kind)
    assert off.max() <= 1, off.max()


# ── plans that only large calls take ────────────────────────────────────────
def merged_bytes(ctx, columns, n_seqs, rows, n_q, dim):
    """The workspace of a call with a prefix whose lines have blocks of so many columns."""
    pad, sm = lambda n: -(-n // 32) * 32, ctx.lib.smelt_cuda_sm_count(ctx.h)  # noqa: E731
    lines = sum(pad(4 * (n_seqs + 3)) + pad(8 * sm * c * dim) + pad(16 * sm * c) + pad(20 * sm) for c in columns)
    return lines + pad(8 * rows * n_q * dim) + pad(16 * rows * n_q)


@pytest.mark.parametrize("kind,n_q,n_kv,dim,rows,prefix", [("bf16", 16, 4, 64, 70, 2300), ("f16", 4, 1, 128, 70, 8600), ("bf16", 10, 2, 128, 60, 4300), ("f16", 8, 2, 256, 70, 1200)])
@pytest.mark.parametrize("window", [0, 700])
def test_a_long_prefix_beside_streamed_sequences(ctx, kind, n_q, n_kv, dim, rows, prefix, window):
    """The prefix on the tensor core, the sequences on the streaming kernel, and every row's parts of both joined."""
    g = np.random.default_rng(prefix + window)
    lengths = g.integers(1, 60, rows)
    lengths[0], lengths[3] = 300, 1
    b = cases.Batch(g, [1] * rows, lengths.tolist(), 16, n_kv, dim, prefix=prefix, behind=2)
    ratio = n_q // n_kv
    k, v, _ = b.fill(g, 0.0)
    _, size = Device(ctx, b, kind, n_q, k, v).workspace()
    assert size == merged_bytes(ctx, ((1 if dim == 256 else 2) * (128 // ratio * ratio), 8), rows, b.total, n_q, dim)
    check_attention(ctx, g, kind, n_q, b, window)


@pytest.mark.parametrize("n_q,n_kv,dim,prefix,window", [(16, 4, 64, 40, 0), (32, 1, 64, 200, 0), (20, 4, 128, 40, 30), (16, 4, 256, 33, 0)])
def test_the_parts_of_a_groups_heads_joined_by_a_warp(ctx, n_q, n_kv, dim, prefix, window):
    """Rows and heads past 64 warps an SM, behind a prefix: in blocks of one and of many rows, and a sequence that ends inside a block."""
    g = np.random.default_rng(n_q + dim)
    rows = 64 * ctx.lib.smelt_cuda_sm_count(ctx.h) // n_q + 9
    b = cases.Batch(g, [rows - 100, 1, 0, 99], [rows - 100, 70, 4, 60], 16, n_kv, dim, prefix=prefix, behind=1)
    check_attention(ctx, g, "bf16", n_q, b, window)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rope_dim,layout", [(64, 0), (64, 1), (6, 1), (40, 0)])
@pytest.mark.parametrize("last", [0, 1])
def test_append_of_two_rows_a_cta(ctx, kind, rope_dim, layout, last):
    """900 rows and more: even and odd numbers of them, CTAs whose rows are of two sequences, rows behind the last sequence."""
    g = np.random.default_rng(rope_dim)
    b = cases.Batch(g, [401, 0, 503 + last], [500, 3, 503 + last], 32, 1, 64, prefix=10, behind=1)
    check_append(ctx, g, kind, 3, b, rope_dim, layout, in_place=bool(last))


def test_misaligned_arrays_are_refused(ctx):
    g = np.random.default_rng(71)
    b = cases.Batch(g, [2, 1], [20, 10], 16, 2, 64, prefix=16)
    k, v, _ = b.fill(g, 0.0)
    d = Device(ctx, b, "f16", 4, k, v)
    q, out = ctx.alloc(3 * 256 * 2), ctx.alloc(3 * 256 * 2)
    work, size = d.workspace()
    freq, position = ctx.to_device(np.ones(34)), ctx.to_device(np.zeros(4, np.int32))
    for field in (None, "row_start", "length", "table", "prefix_table"):
        t = capi.PagedBatch.from_buffer_copy(d.batch)
        if field:
            setattr(t, field, getattr(t, field) + 2)
        status = capi.BAD_ARGUMENT if field else capi.OK
        assert ctx.call_status("paged_attention", C.byref(d.cache), C.byref(t), q.ptr, 256, out.ptr, 256, 0.1, 0, work.ptr, size) == status, field
        assert ctx.call_status("paged_append", C.byref(d.cache), C.byref(t), None, None, 0, q.ptr, 128, q.ptr, 128, None, 0) == status, field
    for f, p, status in ((freq.ptr, position.ptr, capi.OK), (freq.at(4), position.ptr, capi.BAD_ARGUMENT), (freq.ptr, position.at(2), capi.BAD_ARGUMENT)):
        rope = capi.RopeDesc(64, 1, 1.0, f, p)
        assert ctx.call_status("paged_append", C.byref(d.cache), C.byref(d.batch), C.byref(rope), None, 0, q.ptr, 128, q.ptr, 128, None, 0) == status
    buf = ctx.alloc(1 << 16).fill(0)
    buf.upload(np.array([0, 2], np.int32))
    good = dict(n_seqs=1, rows=2, vocab=100, target_stride=100, row_start=buf.ptr, target=buf.at(1024), tokens=buf.at(4096), temperature=buf.at(4608), random=buf.at(5120), out_tokens=buf.at(6144),
                accepted=buf.at(7168), workspace=buf.at(8192), workspace_bytes=8192)
    assert ctx.call_status("verify_drafts", C.byref(capi.VerifyArgs(**good))) == capi.OK
    for field in ("row_start", "tokens", "temperature", "random", "out_tokens", "accepted"):
        assert ctx.call_status("verify_drafts", C.byref(capi.VerifyArgs(**{**good, field: good[field] + 1}))) == capi.BAD_ARGUMENT, field


@pytest.mark.parametrize("n_q,n_kv,dim", [(16, 1, 64), (4, 2, 128), (16, 1, 128), (8, 1, 256)])
@pytest.mark.parametrize("prefix", [0, 30])
def test_as_many_sequences_as_a_call_takes(ctx, n_q, n_kv, dim, prefix):
    """The streaming kernel's rings beside the starts and lengths of 1024 sequences."""
    g = np.random.default_rng(dim + prefix)
    lengths = g.integers(0, 12, 1024)
    lengths[[0, 511, 1023]] = 70, 200, 41
    check_attention(ctx, g, "bf16", n_q, cases.Batch(g, [1] * 1024, lengths.tolist(), 8, n_kv, dim, prefix=prefix))


PLANS = [("streaming", 8, 2, 64, 0, 2), ("tensor core", 32, 2, 64, 0, 8), ("one line with a prefix", 8, 2, 64, 100, 2), ("tensor core with a prefix", 32, 2, 128, 300, 8), ("two lines", 16, 4, 64, 2600, 1)]


@pytest.mark.parametrize("name,n_q,n_kv,dim,prefix,most", PLANS, ids=[p[0] for p in PLANS])
def test_a_captured_call_follows_lengths_and_tables(ctx, name, n_q, n_kv, dim, prefix, most):
    """Every plan, captured once: starts, lengths and pages of each replay as an eager call has them, bit for bit."""
    g = np.random.default_rng(dim + prefix)
    seqs = 70
    b = cases.Batch(g, [most] * seqs, [most + 90] * seqs, 16, n_kv, dim, prefix=prefix)
    k, v, _ = b.fill(g, 0.0)
    d = Device(ctx, b, "f16", n_q, k, v)
    q = ctx.to_device(np.float16(g.standard_normal((b.total, n_q, dim))))
    outs = [ctx.alloc(b.total * n_q * dim * 2) for _ in range(2)]
    (work, size), (other, _) = d.workspace(), d.workspace()

    def call(out, memory):
        ctx.call("paged_attention", C.byref(d.cache), C.byref(d.batch), q.ptr, n_q * dim, out.ptr, n_q * dim, 0.1, 0, memory.ptr, size)

    ctx.call("capture_begin")
    call(outs[0], work)
    call(outs[0], work)  # and one behind the other, over the same workspace
    ctx.call("capture_end")
    ms = C.c_float()
    for turn in range(5):
        rows = g.integers(0, most + 1, seqs)
        d.kept[0].upload(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
        d.kept[1].upload(np.array([rows + g.integers(0, 90, seqs), rows, np.zeros(seqs)][turn % 3], np.int32))
        d.kept[2].upload(g.permutation(b.table.reshape(-1)).reshape(b.table.shape) if turn == 4 else b.table)
        for out in outs:
            out.upload(np.full(b.total * n_q * dim, 7, np.float16))
        ctx.call("capture_replay", turn % 2, 1 + turn % 2, C.byref(ms))
        call(outs[1], other)
        first, second = (out.download(np.uint16, b.total * n_q * dim) for out in outs)
        assert np.array_equal(first, second)
        assert (first.reshape(b.total, -1)[rows.sum():] == np.float16(7).view(np.uint16)).all()
        assert ctx.device_error_flags() in ((0, 0x10000) if turn == 4 else (0,))


def test_two_contexts_side_by_side(ctx):
    """Calls of two contexts, on their two streams, with a workspace each."""
    other = capi.Context(0)
    try:
        sides = []
        for c, (n_q, n_kv, dim, prefix, rows) in zip((ctx, other) * 2, ((8, 2, 128, 0, 1), (8, 2, 128, 0, 1), (32, 2, 64, 0, 9), (16, 2, 64, 200, 3))):
            g = np.random.default_rng(rows + dim)
            b = cases.Batch(g, [rows, 1], [700, 60], 16, n_kv, dim, prefix=prefix)
            k, v, _ = b.fill(g, 0.0)
            d, q = Device(c, b, "f16", n_q, k, v), cases.rounded(g.standard_normal((b.total, n_q, dim)), "f16")
            want = d.attend(q, 0.1)
            dq, out, (work, size) = c.to_device(np.float16(q)), c.to_device(np.full(q.shape, 7, np.float16)), d.workspace()
            sides.append((c, (C.byref(d.cache), C.byref(d.batch), dq.ptr, n_q * dim, out.ptr, n_q * dim, 0.1, 0, work.ptr, size), out, want, (d, dq, work)))
        for _ in range(30):
            for c, args, _, _, _ in sides:
                c.call("paged_attention", *args)
        for _, _, out, want, _ in sides:
            assert np.array_equal(out.download(np.float16, want.shape).astype(np.float64), want)
        assert other.device_error_flags() == 0
        del sides
    finally:
        other.close()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim,rows", [(2, 2, 64, 1), (8, 2, 128, 2), (4, 1, 256, 2), (8, 2, 64, 40), (16, 1, 256, 9)])
@pytest.mark.parametrize("prefix", [0, 50])
@pytest.mark.parametrize("length", [20, 900])
def test_scores_that_are_not_numbers_beside_infinite_values(ctx, kind, n_q, n_kv, dim, rows, prefix, length):
    """A key that is not a number makes NaN of every output of the rows that see it, infinite values or not; the other rows do not notice."""
    g = np.random.default_rng(dim + rows)
    b = cases.Batch(g, [rows, 1], [rows + length, 30], 16, n_kv, dim, prefix=prefix)
    k, v, tokens = b.fill(g, 0.0)
    q = cases.rounded(g.standard_normal((b.total, n_q, dim)), kind)
    clean = Device(ctx, b, kind, n_q, k, v).attend(q, 0.1)
    for t in (length // 2, length // 2 + 7):
        p, i = b.place(0, t)
        v[p, :, i, 3], v[p, :, i, dim - 1] = np.inf, -np.inf
    p, i = b.place(0, 2)
    k[p, 0, i, 5] = np.nan
    got = Device(ctx, b, kind, n_q, k, v).attend(q, 0.1)
    ratio = n_q // n_kv
    assert np.isnan(got[:rows, :ratio]).all() and np.array_equal(got[rows:], clean[rows:])
    other = got[:rows, ratio:]
    assert (other[..., 3] == np.inf).all() and (other[..., dim - 1] == -np.inf).all()
    rest = [d for d in range(dim) if d not in (3, dim - 1)]
    # a key whose values are not finite is added apart where not every column sees it, so these are not the clean call's bits: two sums of the same
    # terms in another order, each within the bound of the one in 64 bits
    want, size, reach = cases.attend(b, [cases.rounded(t, kind) for t in tokens], q, np.float32(0.1))
    assert (np.abs(other - want[:rows, ratio:]) <= cases.attend_bound(want, size, reach, kind, dim)[:rows, ratio:])[..., rest].all()
