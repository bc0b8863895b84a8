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
