"""Attention over e4m3 codes where rows see little, scales lie far apart or one token takes most of the weight.  Tolerances as in
`test_cache8_gpu`, but where a test says more."""

import math

import pytest
import torch

import plain_cache8 as pc
from test_cache8_gpu import BF16, DEV, _attention

pytestmark = pytest.mark.gpu


def _split(monkeypatch, splits):
    from bare_cuda_4gib_b200.kernels import cache8
    monkeypatch.setattr(cache8, "prompt_splits", lambda *a: splits)
    monkeypatch.setattr(cache8, "decode_splits", lambda *a: splits)


# ------------------------------------------------------------------------------ blocks and queries without a number

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("more", [dict(window=1), dict(window=2), dict(chunk=4), dict(chunk=12), dict(chunk=20), dict(chunk=100), dict(window=1, sink=True)])
def test_rows_that_see_few_keys_of_a_block_without_a_number(monkeypatch, dim, splits, more):
    """Wherever in the block they lie, those keys make the row NaN, and no other row is."""
    _split(monkeypatch, splits)

    def spoil(setup, plain):
        for s, cache in enumerate(plain):
            cache.scales[0, 0, 1::2] = math.nan
            setup.fill(s, cache)

    requests = [(0, 100), (130, 61), (250, 2), (37, 1), (20, 1), (600, 30)]
    setup, _q, out = _attention(requests, 2, 4, dim, 16, seed=8, edit=spoil, **more)
    lost = out[: setup.rows].view(setup.rows, 8, dim).isnan().all(-1)
    assert lost[:, :4].any() and not lost[:, :4].all() and not lost[:, 4:].any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("more", [dict(window=1), dict(window=2), dict(chunk=4)])
@pytest.mark.parametrize("entry", [math.nan, math.inf, -math.inf])
def test_queries_without_a_number_that_see_few_keys(monkeypatch, dim, splits, more, entry):
    """At every place of a block of 16 positions: the query's own row is NaN (an infinite entry's product with a code of zero is one), the
    others are as they were."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import AttentionExtras
    _split(monkeypatch, splits)

    def with_zeros(k, v):      # a zero in every key, so that an infinite entry of a query has no score
        return torch.where(torch.arange(dim) == 3, 0.0, k), v

    setup, q, out = _attention([(0, 90), (77, 40)], 2, 4, dim, 16, seed=2, keys=with_zeros, **more)
    bad, again = q.clone(), torch.zeros_like(out)
    rows = list(range(0, setup.rows, 7))
    for i, r in enumerate(rows):
        bad[r, (i % 8) * dim + 3] = entry
    extras = AttentionExtras(more["chunk"]) if "chunk" in more else None
    cache8.attention(bad, again, setup.view, setup.maps, 8, 1 / math.sqrt(dim), more.get("window", 0), extras)
    wrong = again[: setup.rows].view(setup.rows, 8, dim).isnan().all(-1)
    assert wrong.nonzero().tolist() == [[r, i % 8] for i, r in enumerate(rows)]
    good = ~wrong
    assert torch.equal(again[: setup.rows].view(setup.rows, 8, dim)[good], out[: setup.rows].view(setup.rows, 8, dim)[good])
