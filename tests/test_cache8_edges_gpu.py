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


# ------------------------------------------------------------------------------ factors of the scores at the ends of float32's range

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("q_scale", [1e-20, 1e-30, 1e-37])
def test_small_queries_over_keys_of_zero(monkeypatch, dim, splits, q_scale):
    """A key block of zeros has the least scale, which times a small query's own is below float32: hidden keys stay hidden, the row is the
    mean of the values that it sees."""
    _split(monkeypatch, splits)

    def keys(k, v):
        return k * (torch.arange(k.shape[0])[:, None, None] // 16 % 3 == 1).double(), v

    _attention([(0, 90), (100, 70), (30, 1), (64, 3)], 2, 4, dim, 16, seed=4, keys=keys, q_scale=q_scale)
    _attention([(0, 90), (100, 70), (30, 1), (64, 3)], 2, 4, dim, 16, seed=4, keys=keys, q_scale=q_scale, window=20)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 4])
def test_large_queries_over_large_keys_that_are_hidden(monkeypatch, dim, splits):
    """The first key is zero, the others so large that a query's scores of them are beyond float32: the first row sees only the zero, and is the
    first value."""
    from bare_cuda_4gib_b200.kernels import cache8
    _split(monkeypatch, splits)
    kept = []

    def keys(k, v):
        return k * (torch.arange(k.shape[0])[:, None, None] > 0).double() * 2.0 ** 100, v

    requests = [(0, 30), (0, 2), (0, 3)]        # of the prompt kernel and of the decode kernel
    setup, q, out = _attention(requests, 2, 4, dim, 16, seed=4, keys=keys, q_scale=2.0 ** 70, check=False, edit=lambda _s, plain: kept.extend(plain))
    row = 0
    for s, (_c, n) in enumerate(requests):
        v = kept[s].values()[1][:, 0].repeat_interleave(4, 0)         # [heads, dim]
        got = out[row].double().cpu().view(8, dim)
        assert ((got - v).abs() <= (2.0 ** -8 + 2.0 ** -9) * v.abs()).all(), s
        row += n


# ------------------------------------------------------------------------------ values far apart

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 2, 4])
@pytest.mark.parametrize("more", [dict(), dict(window=20), dict(chunk=48), dict(window=40, sink=True)])
def test_small_values_count_for_rows_that_see_no_larger_ones(monkeypatch, dim, splits, more):
    """Values of ordinary size between values 2^-72 of them: rows ahead of the ordinary ones, and rows whose window has left them behind, are made of
    the small ones alone, rows that see both take the small ones' share of the sum into account."""
    _split(monkeypatch, splits)

    def keys(k, v):
        ordinary = (torch.arange(k.shape[0])[:, None, None] // 16 % 8 == 3).double()
        return k, v * torch.where(ordinary > 0, 1.0, 2.0 ** -72)

    _attention([(0, 90), (100, 170), (0, 17), (30, 1), (44, 6), (300, 1)], 2, 4, dim, 16, seed=5, keys=keys, **more)
    _attention([(500, 61), (0, 130)], 1, 8, dim, 64, seed=6, keys=keys, **more)


@pytest.mark.parametrize("dim", [64, 128])
def test_later_tokens_change_no_earlier_row(dim):
    """Behind them a token's values are 2^90 times as large or not: the rows are the same, but for a sum that is taken from other terms (2^-16 of
    it at most), so that an output may be the other neighbour in bfloat16.  (Rows that see keys of the large values' own block are another
    matter: the block's codes are off by 2^-10 of its scale.)"""
    outs = []
    for size in (1.0, 2.0 ** 90):
        def keys(k, v):
            return k, v * torch.where(torch.arange(k.shape[0])[:, None, None] >= 50, size, 1.0)

        _setup, _q, out = _attention([(0, 60)], 2, 4, dim, 16, seed=7, keys=keys, check=size == 1.0)
        outs.append(out[:48].double())
    assert ((outs[0] - outs[1]).abs() <= 2.0 ** -7 * outs[0].abs()).all()


# ------------------------------------------------------------------------------ one token that takes most of the weight

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("sink", [False, True])
def test_a_first_token_that_takes_most_of_the_weight(monkeypatch, dim, splits, sink):
    """Its value is next to nothing, so that the other tokens, each 8 to 20 nats below it, make the output.  A weight is a half in units of 2^-7 of
    the row's largest or more: where it lies below the half's normal range it is off by at most 2^-25 of that, 2^-32 of the largest weight."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import AttentionExtras
    _split(monkeypatch, splits)
    kept, requests = [], [(0, 1), (2000, 1), (500, 3), (1500, 40), (0, 200)]

    def keys(k, v):
        t = torch.arange(k.shape[0])[:, None, None]
        u = torch.rand(v.shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
        return torch.where(t == 0, 2.0, 0.0) + 0 * k, torch.where(t == 0, 2.0 ** -9, 1 + 0.7 * u)

    setup, _q, out = _attention(requests, 2, 4, dim, 16, seed=1, keys=keys, check=False, edit=lambda _s, plain: kept.extend(plain))
    gen = torch.Generator().manual_seed(5)
    gap = 8 + 12 * torch.rand(setup.rows, 8, 1, generator=gen)                       # nats
    q = (gap / (2 * math.sqrt(dim)) * (0.5 + torch.rand(setup.rows, 8, dim, generator=gen))).view(setup.rows, -1).to(BF16).to(DEV)
    sinks = (torch.rand(8, generator=gen) * 20).to(DEV) if sink else None
    again = torch.zeros_like(out)
    cache8.attention(q, again, setup.view, setup.maps, 8, 1 / math.sqrt(dim), 0, AttentionExtras(sink=sinks) if sink else None)
    row = 0
    for s, (c, n) in enumerate(requests):
        k, v = kept[s].values()
        want, bound = pc.attention(q[row: row + n].double().cpu().view(n, 8, dim), k, v, c, 1 / math.sqrt(dim), 0, 0, sinks.double().cpu() if sink else None, None)
        got = again[row: row + n].double().cpu().view(n, 8, dim)
        # (the sum of a row's weights is at least the largest of them)
        lost = 2.0 ** -32 * v.abs().sum(1).repeat_interleave(4, 0)
        off = (got - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -9 * bound + lost)
        assert (off <= 0).all(), (s, float(((got - want).abs() / want.abs()).max()))
        row += n


# ------------------------------------------------------------------------------ a captured call that is the first one

def test_a_view_makes_what_a_captured_call_reports_to(monkeypatch):
    """A graph that made the error word itself would set it to zero at every replay."""
    from bare_cuda_4gib_b200.kernels import cache8, gemm
    from test_cache8_gpu import Setup
    monkeypatch.setattr(gemm, "_error_words", {})
    setup = Setup([(40, 1)], 2, 4, 64, 16)
    assert list(gemm._error_words) == [setup.codes.device]
    word = gemm._error_words[setup.codes.device]
    q = torch.zeros(1, 8 * 64, dtype=BF16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache8.attention(q, q, setup.view, setup.maps, 8, 0.125)
    word.fill_(46)
    graph.replay()
    assert gemm._error_words[setup.codes.device] is word and int(word) == 46


# ------------------------------------------------------------------------------ bounds beyond 32 bits

@pytest.mark.parametrize("window,chunk,scale", [(1 << 31, 0, 0.125), ((1 << 32) + 5, 0, 0.125), (0, 1 << 31, 0.125), (0, (1 << 32) + 16, 0.125), (0, -16, 0.125),
                                                (0, 0, 1e-50), (0, 0, 1e39)])
def test_bounds_and_scales_beyond_32_bits_are_refused(window, chunk, scale):
    """They went to the kernel modulo 2^32, as zero or as infinity: a window of 2^32 + 5 positions was one of 5."""
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import AttentionExtras
    setup, q, out = _attention([(40, 1), (0, 30)], 2, 4, 64, 16)
    with pytest.raises(KernelLaunchError, match="in 32 bits"):
        cache8.attention(q, out, setup.view, setup.maps, 8, scale, window, AttentionExtras(chunk) if chunk else None)
    again = torch.zeros_like(out)
    most = (1 << 31) - 1
    for args in ((most, None), (0, AttentionExtras(most))):
        cache8.attention(q, again, setup.view, setup.maps, 8, 1 / 8, *args)
        assert torch.equal(again[: setup.rows], out[: setup.rows])


# ------------------------------------------------------------------------------ twice

@pytest.mark.parametrize("dim", [64, 128])
def test_a_call_repeats_itself(dim):
    """The same call twice, also split over a cluster: the same to the bit."""
    from bare_cuda_4gib_b200.kernels import cache8
    setup, q, out = _attention([(2000, 1), (700, 3), (1500, 61), (0, 300)], 2, 4, dim, 16, window=900, sink=False)
    for _ in range(5):
        again = torch.zeros_like(out)
        cache8.attention(q, again, setup.view, setup.maps, 8, 1 / math.sqrt(dim), 900)
        assert torch.equal(again[: setup.rows], out[: setup.rows])


# ------------------------------------------------------------------------------ far positions

def _far(page, length, new, width):
    """One request of `length` positions of which only the last two pages are held, and the plain statement of its new rows."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import Partials
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    dim = 128
    maps = StepMaps(new, 1, width, page, group=1, tile_rows=cache8.tile_rows(dim), few_rows=16, device=DEV)
    blocks = -(-(length + new) // page)
    pages = torch.full((blocks,), -1, dtype=torch.int32)
    pages[-2:] = torch.tensor([1, 0])
    maps.build(torch.tensor([length], dtype=torch.int32, device=DEV), torch.tensor([new], dtype=torch.int32, device=DEV), pages.to(DEV), new, new, new)
    codes = torch.zeros(2, 2, 1, page, dim, dtype=torch.uint8, device=DEV)
    scales = torch.full((2, 2, 1, page // 16), 2.0 ** -100, device=DEV)
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float().to(DEV)
    qkv = torch.randn(new, 3 * dim, generator=torch.Generator().manual_seed(length)).to(DEV)
    q = torch.zeros(new, dim, dtype=BF16, device=DEV)
    cache8.append(Partials(qkv), q, cache8.view(codes, scales, maps.table), maps, inv_freq, 1)
    want = pc.rotate(qkv.double().cpu().view(new, 3, dim)[:, :2], torch.arange(length, length + new), inv_freq.cpu())
    return q.double().cpu(), want[:, 0], (maps, codes, scales, inv_freq, qkv)


@pytest.mark.parametrize("length", [1000, 130001, 1 << 20, 3000001, (1 << 23) - 9, (1 << 23) + 12345, (1 << 24) - 40])
def test_append_turns_by_the_angle_of_far_positions(length):
    """To the last position that a float32 holds: 2^-20 of the entries a rotation mixes, and the rounding to bfloat16."""
    q, want, _ = _far(128, length, 37, (1 << 24) // 128)
    assert ((q - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * (1 + want.abs().amax())).all()


def test_append_refuses_angles_of_positions_beyond_that():
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import Partials
    with pytest.raises(KernelLaunchError, match="angles are taken for"):
        _far(128, 1000, 2, (1 << 24) // 128 + 1)
    _q, _want, (maps, codes, scales, _inv_freq, qkv) = _far(128, 1000, 2, 100)
    q = torch.zeros(2, 128, dtype=BF16, device=DEV)
    cache8.append(Partials(qkv), q, cache8.view(codes, scales, maps.table), maps, None, 1)       # without angles there is no such bound
    assert torch.equal(q, qkv[:, :128].to(BF16))


# ------------------------------------------------------------------------------ infinite queries

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("entry", [math.inf, -math.inf])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_a_query_with_an_infinite_entry_is_lost_whatever_the_keys_signs(dim, entry, sign):
    """Rows of the decode kernel and of the prompt kernel alike, also where every score of the row would be minus infinity."""
    from bare_cuda_4gib_b200.kernels import cache8
    setup, q, out = _attention([(100, 1), (40, 3), (0, 40), (0, 1)], 2, 4, dim, 16, seed=3, keys=lambda k, v: (sign * (k.abs() + 1), v))
    bad, again = q.clone(), torch.zeros_like(out)
    rows = [0, 2, 4 + 17, 44]
    for i, r in enumerate(rows):
        bad[r, i * dim + 5] = entry
    cache8.attention(bad, again, setup.view, setup.maps, 8, 1 / math.sqrt(dim))
    wrong = again[: setup.rows].view(setup.rows, 8, dim).isnan().all(-1)
    assert wrong.nonzero().tolist() == [[r, i] for i, r in enumerate(rows)]
    good = ~wrong
    assert torch.equal(again[: setup.rows].view(setup.rows, 8, dim)[good], out[: setup.rows].view(setup.rows, 8, dim)[good])
