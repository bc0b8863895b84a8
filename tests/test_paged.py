"""A packed batch over a paged cache, and drafted tokens: what needs no GPU."""
import ctypes as C
import math

import numpy as np
import pytest

import paged_cases as cases
from smelt_b200 import capi


@pytest.mark.parametrize("kind", [capi.ROPE_PLAIN, capi.ROPE_LINEAR, capi.ROPE_BASE, capi.ROPE_RAMP, capi.ROPE_BANDS])
@pytest.mark.parametrize("n", [2, 64, 128, 130])
def test_frequencies(kind, n):
    theta, s, known, slow, fast = 1e4, 8.0, 4096.0, 1.0, 32.0
    freq, factor = capi.rope_frequencies(n, theta, kind, s, known, slow, fast)
    i = np.arange(n // 2)
    plain = theta ** (-2.0 * i / n)
    if kind == capi.ROPE_PLAIN:
        want = plain
    elif kind == capi.ROPE_LINEAR:
        want = plain / s
    elif kind == capi.ROPE_BASE:
        want = (theta * s ** (n / (n - 2) if n > 2 else 0)) ** (-2.0 * i / n)
    else:
        if kind == capi.ROPE_RAMP:
            at = [n * math.log(known / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (fast, slow)]
            low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
            keep = 1 - np.clip((i - low) / max(high - low, 1e-3), 0, 1)
        else:
            keep = np.clip((known * plain / (2 * math.pi) - slow) / (fast - slow), 0, 1)
        want = plain * keep + plain / s * (1 - keep)
        if n > 2:
            assert want[0] == plain[0] and abs(want[-1] * s / plain[-1] - 1) < 1e-12  # the ends of the ramp
    assert np.allclose(freq, want, rtol=1e-12, atol=0)
    assert factor == np.float32(0.1 * math.log(s) + 1 if kind == capi.ROPE_RAMP else 1)


@pytest.mark.parametrize("bad", [dict(rope_dim=0), dict(rope_dim=7), dict(theta=1.0), dict(theta=float("nan")), dict(kind=9), dict(kind=capi.ROPE_LINEAR, factor=0.5),
                                 dict(kind=capi.ROPE_RAMP, factor=2.0, known_positions=0.0), dict(kind=capi.ROPE_BANDS, factor=2.0, known_positions=100.0, fast_turns=1.0)])
def test_bad_scalings_are_refused(bad):
    with pytest.raises(capi.SmeltError) as e:
        capi.rope_frequencies(**{"rope_dim": 64, "theta": 1e4, **bad})
    assert e.value.status == capi.BAD_ARGUMENT


def test_no_context_is_a_refusal():
    lib, size = capi.load(), C.c_size_t()
    cache, batch, args = capi.PagedCache(), capi.PagedBatch(), capi.VerifyArgs()
    assert lib.smelt_cuda_paged_append(None, C.byref(cache), C.byref(batch), None, None, 0, None, 0, None, 0, None, 0) == capi.BAD_ARGUMENT
    assert lib.smelt_cuda_paged_attention(None, C.byref(cache), C.byref(batch), None, 0, None, 0, 1.0, 0, None, 0) == capi.BAD_ARGUMENT
    assert lib.smelt_cuda_paged_attention_workspace(None, C.byref(cache), C.byref(batch), C.byref(size)) == capi.BAD_ARGUMENT
    assert lib.smelt_cuda_verify_drafts(None, C.byref(args)) == capi.BAD_ARGUMENT
    assert lib.smelt_cuda_verify_drafts_workspace(None, C.byref(args), C.byref(size)) == capi.BAD_ARGUMENT


def test_structures_match_the_header():
    assert [C.sizeof(t) for t in (capi.PagedCache, capi.PagedBatch, capi.RopeDesc, capi.RopeScaling, capi.VerifyArgs)] == [64, 56, 32, 48, 120]
    assert capi.PagedCache.page_stride.offset == 24 and capi.PagedBatch.row_start.offset == 24 and capi.RopeDesc.freq.offset == 16 and capi.VerifyArgs.row_start.offset == 40


# ── the restatements the GPU tests compare with ─────────────────────────────
def test_attention_of_equal_scores_is_the_mean_of_what_is_seen():
    g = np.random.default_rng(0)
    b = cases.Batch(g, [2, 0, 3], [5, 4, 2], 3, 1, 8, prefix=4)
    _, _, tokens = b.fill(g, np.nan)
    out, _, _ = cases.attend(b, tokens, np.zeros((5, 2, 8)), 1.0, window=6)
    assert np.allclose(out[0, 0], tokens[0][1][2:8, 0].mean(0)) and np.allclose(out[1, 1], tokens[0][1][3:9, 0].mean(0))
    assert (out[2] == 0).all()  # three rows, two tokens
    assert np.allclose(out[3, 0], tokens[2][1][0:5, 0].mean(0)) and np.allclose(out[4, 0], tokens[2][1][0:6, 0].mean(0))


def test_verification_keeps_the_targets_law():
    """Whatever the draft, the first token is distributed as the target says."""
    g = np.random.default_rng(1)
    V, n = 6, 40000
    p, q = g.standard_normal(V), g.standard_normal(V)
    law_p, law_q = cases.law(p, 0.7), cases.law(q, 0.7)
    x = g.choice(V, n, p=law_q)
    target, draft = np.tile(p, (2 * n, 1)), np.tile(q, (1, n, 1))
    tokens = np.stack([np.zeros(n, int), x], 1).ravel()
    out, kept = cases.verify(np.arange(0, 2 * n + 1, 2), target, draft, tokens, np.full(n, 0.7), g.random(2 * n).astype(np.float32))
    seen = np.bincount(out[0::2], minlength=V) / n
    assert np.abs(seen - law_p).max() < 5 * math.sqrt(0.25 / n)
    assert abs(kept.mean() - np.minimum(law_p, law_q).sum()) < 5 * math.sqrt(0.25 / n)


def test_a_rounding_is_half_a_step():
    for kind, top in (("f16", 2.0 ** -11), ("bf16", 2.0 ** -8)):
        a = np.random.default_rng(2).standard_normal(1000)
        assert np.abs(cases.rounded(a, kind) / a - 1).max() <= top
