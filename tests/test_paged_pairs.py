"""What the bound of paged_pairs tells apart, without a GPU."""
import numpy as np
import pytest

import paged_cases as cases
import paged_pairs as pairs


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim", [(4, 2, 64), (4, 1, 128), (8, 1, 256)])
@pytest.mark.parametrize("prefix", [0, 12])
def test_one_rounding_of_the_weights_shows(kind, n_q, n_kv, dim, prefix):
    g = np.random.default_rng(dim + prefix)
    b = cases.Batch(g, [1, 2, 1], [16, 24, 8], 16, n_kv, dim, prefix=prefix)
    _, _, tokens = pairs.fill(g, b, kind)
    q, scale = pairs.queries(g, b.total, n_q, dim), np.float32(0.75 / np.sqrt(dim))
    want, size, _ = cases.attend(b, tokens, q, scale)
    room = pairs.bound(want, size, prefix + 24, pairs.largest_score(b, tokens, q, scale), kind)
    off = [np.abs(pairs.rounded_attention(b, tokens, q, scale, kind, parts) - want) / room for parts in (1, 2)]
    assert off[0].max() > 2 and (off[0] > 1).mean() > 0.05 and off[1].max() <= 1, [x.max() for x in off]
