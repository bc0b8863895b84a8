"""The batch over pages at its bounds: calls repeated, arrays that say what they should not, infinite values, plans that only large calls take."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as cases
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
