"""The cache of e4m3 codes on the GPU: a step's maps, the append and attention over the codes, each against the plain statement in 64
bits, a run of them together, and the engine with such a cache.

Tolerances, from what each kernel rounds.  A code is at most half a step from its number: 2^-4 of it, or 2^-10 of the scale
below the normal range; the entries themselves are float32 sums (2^-22 of the largest of the two that a rotation mixes).  Attention's
output is rounded to bfloat16 (2^-8 of it at most); its weights are halves (2^-11), its scores float32 sums of at most 128 exact products
(128 * 2^-24 of the sum of their sizes, which here stays below 60 in the exponent: 2^-11), once in the weights and once in their sum: 2^-9
of the weighted sizes of the values."""

import math
import random

import pytest
import torch

import plain_cache8 as pc

pytestmark = pytest.mark.gpu
DEV, BF16, F32, F64, I32 = "cuda", torch.bfloat16, torch.float32, torch.float64, torch.int32
CODES = torch.float8_e4m3fn


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


class Setup:
    """A pool of pages, its scales, the requests' pages in a shuffled order and the step's maps."""

    def __init__(self, requests, kv_heads, group, dim, page, seed=0, caches=1, index=0, width=None, dropped=None, spare=2, garbage=True):
        """requests: (cached, new) each, cached < 0 for an idle row; dropped: pages given back at the front, per request."""
        from bare_cuda_4gib_b200.kernels import cache8
        from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
        self.requests, self.kv_heads, self.group, self.dim, self.page = requests, kv_heads, group, dim, page
        rng = random.Random(seed)
        counts = [0 if c < 0 else -(-(c + n) // page) for c, n in requests]
        n_pages = sum(counts) + spare
        order = list(range(n_pages))
        rng.shuffle(order)
        self.lists, at = [], 0
        for s, k in enumerate(counts):
            mine = order[at: at + k]
            at += k
            gone = dropped[s] if dropped else 0
            self.lists.append([-1] * gone + mine[gone:])
        self.rows = sum(n for _, n in requests)
        self.width = width or max(counts + [1])
        shape = (n_pages, caches, 2, kv_heads, page, dim)
        # what earlier requests left: NaN codes and scales among it
        gen = torch.Generator().manual_seed(seed)
        self.codes = (torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8) if garbage else torch.zeros(shape, dtype=torch.uint8)).to(DEV)
        self.scales = torch.full(shape[:4] + (page // 16,), math.nan if garbage else 1.0, device=DEV)
        self.caches, self.index = caches, index
        self.maps = StepMaps(self.rows, len(requests), self.width, page, group=group, tile_rows=cache8.tile_rows(dim), few_rows=16, device=DEV)
        self.build()
        self.view = cache8.view(self.codes, self.scales, self.maps.table, index)

    def build(self, requests=None):
        requests = requests or self.requests
        self.maps.build(i32([c for c, _ in requests]), i32([n for _, n in requests]), i32([p for mine in self.lists for p in mine] or [0]),
                        sum(n for _, n in requests), max(n for _, n in requests), min(n for _, n in requests))

    def fill(self, s, cache, upto=None):
        """Writes a plain cache's codes and scales into the pages of request s."""
        codes = cache.codes.to(F32).to(CODES).view(torch.uint8)
        upto = cache.length if upto is None else upto
        for b, p in enumerate(self.lists[s]):
            lo, hi = b * self.page, min((b + 1) * self.page, upto)
            if p < 0 or hi <= lo:
                continue
            self.codes[p, self.index, :, :, : hi - lo] = codes[:, :, lo:hi].to(DEV)
            k = -(-(hi - lo) // 16)
            self.scales[p, self.index, :, :, :k] = cache.scales[:, :, lo // 16: lo // 16 + k].to(F32).to(DEV)

    def read(self, s, length):
        """(codes' numbers, scales) of request s's first positions, float64 on the host."""
        codes, scales = [], []
        for p in self.lists[s]:
            codes.append(pc.NUMBERS[self.codes[p, self.index].cpu().long()])
            scales.append(self.scales[p, self.index].double().cpu())
        return torch.cat(codes, 2)[:, :, :length], torch.cat(scales, 2)[:, :, : -(-length // 16)]


# ------------------------------------------------------------------------------ maps

MAPS = [([(0, 1)], 16, 1), ([(15, 1), (16, 1), (17, 1), (-1, 1)], 16, 4), ([(100, 3), (0, 70), (33, 1)], 32, 8), ([(0, 16), (0, 17), (16, 16)], 48, 3),
        ([(5, 200), (-1, 1), (-1, 1)], 64, 16), ([(k * 7 % 90, 1 + k % 5) for k in range(300)], 16, 7), ([(1000, 1)] * 8 + [(1, 389), (0, 100)], 128, 8),
        ([(40, 1), (0, 1), (40, 1), (39, 2)], 16, 2)]


@pytest.mark.parametrize("requests,page,group", MAPS)
def test_step_maps(requests, page, group):
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    rng = random.Random(len(requests))
    pages = [rng.randrange(-1, 5000) for c, n in requests if c >= 0 for _ in range(-(-(c + n) // page))]
    width = max(-(-(c + n) // page) for c, n in requests) + 3
    rows = sum(n for _, n in requests)
    maps = StepMaps(rows + 5, len(requests) + 2, width, page, group=group, tile_rows=128, few_rows=16, device=DEV)
    for extra in (0, 3):            # rows behind the last request
        n_rows = rows + extra
        maps.build(i32([c for c, _ in requests]), i32([n for _, n in requests]), i32(pages or [0]), n_rows, max(n for _, n in requests),
                   min(n for _, n in requests))
        want = pc.maps([c for c, _ in requests], [n for _, n in requests], pages, page, group, 128, 16, width, n_rows)
        for name, value in want.items():
            got = getattr(maps, name)
            assert got.tolist() == value, name
    assert maps.slots.dtype == torch.int64 and maps.table.data_ptr() == maps.block_table.data_ptr()


def test_step_maps_of_large_pools_and_short_tables():
    """Slots pass 32 bits; a request longer than its table has slots and entries up to the table's end only."""
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    maps = StepMaps(40, 2, 2, 128, device=DEV)
    big = (1 << 31) - 1
    maps.build(i32([250, 0]), i32([10, 30]), i32([big, 5, 9, big - 1]), 40, 30, 10)
    assert maps.slots.tolist() == [5 * 128 + 122 + i for i in range(6)] + [-1] * 4 + [(big - 1) * 128 + i for i in range(30)]
    assert maps.block_table.tolist() == [[big, 5], [big - 1, -1]]


def test_step_maps_of_lengths_that_are_not_the_steps():
    """More rows than the step has are cut off at its end; pages that are not listed are not held."""
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    maps = StepMaps(20, 3, 4, 16, device=DEV)
    maps.build(i32([3, 0, 7]), i32([5, 40, 6]), i32([4, 9]), 20, 20, 1)
    assert maps.seq_q_start.tolist() == [0, 5, 25] and maps.seq_q_len.tolist() == [5, 15, 0] and maps.seq_kv_len.tolist() == [8, 15, 7]
    assert maps.row_seq.tolist() == [0] * 5 + [1] * 15 and maps.slots.tolist() == [67, 68, 69, 70, 71] + [144 + i for i in range(15)]
    assert maps.block_table.tolist() == [[4, -1, -1, -1], [9, -1, -1, -1], [-1] * 4]


def test_step_maps_refuse():
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    maps = StepMaps(64, 4, 8, 16, device=DEV)
    a, p = i32([3, 4]), i32([0, 1])
    for args in ((a, i32([1]), p, 2, 1, 1), (a, a, p, 65, 1, 1), (a, a, p, 0, 1, 1), (a.long(), a, p, 2, 1, 1), (a, a.cpu(), p, 2, 1, 1),
                 (i32([1] * 5), i32([1] * 5), p, 5, 1, 1), (a, a, p, 2, 1, 2), (a, a, p, 2, 3, 1), (a, a, i32([[0, 1], [2, 3]])[:, 0], 2, 1, 1)):
        with pytest.raises(KernelLaunchError, match="step maps"):
            maps.build(*args)


# ------------------------------------------------------------------------------ append

def _rows(setup, seed, wide, partials, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    heads = setup.kv_heads * setup.group
    x = torch.randn(partials, setup.rows, (heads + 2 * setup.kv_heads) * setup.dim, generator=gen) * scale
    return x.to(F32 if wide else BF16).to(DEV)


def _appended(setup, qkv, inv_freq, write=True):
    """Runs the append; returns q and, per request, the plain (k, v) before rounding."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import Partials
    heads = setup.kv_heads * setup.group
    q = torch.full((setup.rows, heads * setup.dim), 7.0, dtype=BF16, device=DEV)
    cache8.append(Partials(qkv if qkv.shape[0] > 1 else qkv[0], qkv.shape[0]), q, setup.view, setup.maps, inv_freq, heads, write)
    x = qkv.double().cpu().sum(0).view(setup.rows, heads + 2 * setup.kv_heads, setup.dim)
    out, row = [], 0
    for c, n in setup.requests:
        mine = x[row: row + n]
        turned = mine[:, : heads + setup.kv_heads]
        if inv_freq is not None:
            turned = pc.rotate(turned, torch.arange(max(c, 0), max(c, 0) + n), inv_freq.cpu())
        out.append((turned[:, :heads].reshape(n, -1), turned[:, heads:], mine[:, heads + setup.kv_heads:]))
        row += n
    return q.double().cpu(), out


APPENDS = [([(0, 1)], 1, 64, 16, False, 1), ([(15, 1), (16, 1), (17, 1)], 4, 128, 16, False, 1), ([(0, 16), (3, 13), (8, 40)], 8, 64, 48, False, 1),
           ([(100, 3), (0, 70), (33, 1), (31, 2)], 4, 128, 32, True, 3), ([(1, 1), (30, 5), (64, 64)], 7, 64, 64, True, 1), ([(5, 2), (0, 129)], 16, 128, 128, False, 2),
           ([(47, 1)] * 5, 1, 128, 16, True, 4), ([(2, 31)], 32, 64, 16, False, 1)]


@pytest.mark.parametrize("requests,group,dim,page,wide,partials", APPENDS)
def test_append_without_rotation_is_the_definition(requests, group, dim, page, wide, partials):
    """Codes and scales to the bit (sums of a few partial results are exact enough in float32 to be compared so only where there is
    one); what earlier steps filled is rescaled where the new entries are larger, the rest of the pool left as it was."""
    setup = Setup(requests, 3, group, dim, page, seed=dim + group, caches=3, index=1)
    plain, gen = [], torch.Generator().manual_seed(1)
    for s, (c, n) in enumerate(requests):
        cache = pc.Cache(3, dim)
        if c:        # smaller entries than the new ones in some heads, larger in others
            size = torch.tensor([0.01, 1.0, 30.0], dtype=F64).view(1, 3, 1)
            cache.append(torch.randn(c, 3, dim, generator=gen, dtype=F64).float().double() * size, torch.randn(c, 3, dim, generator=gen, dtype=F64).float().double() / size)
        setup.fill(s, cache)
        plain.append(cache)
    before, scales_before = setup.codes.clone(), setup.scales.clone()
    qkv = _rows(setup, 2, wide, 1)
    if partials > 1:          # parts that add up exactly
        qkv = torch.cat([qkv * 0.5] * 2 + [torch.zeros_like(qkv)] * (partials - 2))
    q, parts = _appended(setup, qkv, None)
    row = 0
    for s, (c, n) in enumerate(requests):
        want_q, k, v = parts[s]
        assert torch.equal(q[row: row + n], want_q.to(F32).to(BF16).double())
        plain[s].append(k, v)
        codes, scales = setup.read(s, c + n)
        assert torch.equal(scales, plain[s].scales)
        assert torch.equal(codes, plain[s].codes)
        row += n
    # everything else of the pool is as it was
    touched = torch.zeros_like(setup.codes, dtype=torch.bool)
    touched_scales = torch.zeros_like(setup.scales, dtype=torch.bool)
    for s, (c, n) in enumerate(requests):
        for p in range(c // 16 * 16, c + n):
            touched[setup.lists[s][p // page], 1, :, :, p % page] = True
            touched_scales[setup.lists[s][p // page], 1, :, :, p % page // 16] = True
    assert torch.equal(setup.codes[~touched], before[~touched])
    assert torch.equal(setup.scales[~touched_scales].nan_to_num(-1), scales_before[~touched_scales].nan_to_num(-1))


@pytest.mark.parametrize("requests,group,dim,page,wide,partials", APPENDS + [([(120000, 2), (9000, 17)], 4, 128, 64, False, 1)])
def test_append_with_rotation(requests, group, dim, page, wide, partials):
    """Also at far positions, whose angle a float32 product alone would miss by 2^-7."""
    setup = Setup(requests, 2, group, dim, page, seed=3)
    for s, (c, n) in enumerate(requests):
        if c % 16:          # the open block's scale is a number
            for w in range(c // 16 * 16, c):
                p = setup.lists[s][w // page]
                setup.codes[p, 0, :, :, w % page] = 0
                setup.scales[p, 0, :, :, w % page // 16] = 2.0 ** -100
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, dtype=F64) / dim)).to(F32).to(DEV)
    qkv = _rows(setup, 4, wide, partials)
    q, parts = _appended(setup, qkv, inv_freq)
    row = 0
    for s, (c, n) in enumerate(requests):
        want_q, k, v = parts[s]
        near = 2.0 ** -20 * (1 + want_q.abs().amax())
        assert ((q[row: row + n] - want_q).abs() <= 2.0 ** -8 * want_q.abs() + near).all()
        codes, scales = setup.read(s, c + n)
        got = (codes * scales.repeat_interleave(16, -1)[..., : c + n, None])[:, :, c:]
        want = torch.stack([k, v]).transpose(1, 2)
        step = scales.repeat_interleave(16, -1)[..., c: c + n, None]
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -10 * step * (1 + 2.0 ** -10) + near).all()
        row += n


@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-30, 3e-2, 448.0, 6e4, 1e20, 3.38e38])
def test_append_of_any_size(size):
    setup = Setup([(0, 20)], 1, 1, 64, 32)
    qkv = torch.zeros(1, 20, 192, device=DEV)
    qkv[0, :, 64:] = (torch.rand(20, 128, device=DEV, generator=torch.Generator(DEV).manual_seed(1)) * 2 - 1) * size
    if size:
        qkv[0, 3, 70], qkv[0, 17, 130] = size, -size
    _q, parts = _appended(setup, qkv, None)
    cache = pc.Cache(1, 64)
    cache.append(parts[0][1], parts[0][2])
    codes, scales = setup.read(0, 20)
    assert torch.equal(scales, cache.scales) and torch.equal(codes, cache.codes)


def test_append_of_numbers_that_are_none():
    """A NaN or an infinity, as key or value, makes the keys' scale of its block and head NaN, until a page is opened anew; codes and the
    values' scales stay numbers."""
    setup = Setup([(4, 40)], 2, 1, 64, 64)
    old = pc.Cache(2, 64)
    old.append(torch.randn(4, 2, 64, dtype=F64).float().double(), torch.randn(4, 2, 64, dtype=F64).float().double())
    setup.fill(0, old)
    qkv = torch.randn(1, 40, (2 + 4) * 64, device=DEV)
    view = qkv[0].view(40, 6, 64)
    view[2, 2, 5] = math.nan         # position 6, key, head 0
    view[20, 5, 1] = math.inf        # position 24, value, head 1
    view[39, 3, 63] = -math.inf      # position 43, key, head 1
    _q, parts = _appended(setup, qkv, None)
    old.append(parts[0][1], parts[0][2])
    codes, scales = setup.read(0, 44)
    assert torch.equal(scales.isnan(), old.scales.isnan()) and torch.equal(scales.nan_to_num(), old.scales.nan_to_num())
    assert scales.isnan().nonzero().tolist() == [[0, 0, 0], [0, 1, 1], [0, 1, 2]]
    assert torch.equal(codes, old.codes)
    # the next token of the spoilt open block: the block stays without a number
    setup.requests = [(44, 1)]
    setup.rows = 1
    setup.build()
    _q, parts = _appended(setup, torch.randn(1, 1, 6 * 64, device=DEV), None)
    _codes, scales = setup.read(0, 45)
    assert scales[0, 1, 2].isnan() and not scales[0, 0, 2].isnan()
    # another request takes the page: nothing of it is left
    setup.requests = [(0, 3)]
    setup.rows = 3
    setup.build()
    _appended(setup, torch.randn(1, 3, 6 * 64, device=DEV), None)
    assert not setup.read(0, 3)[1].isnan().any()


def test_append_leaves_alone_what_is_not_its_own():
    """Idle rows, rows behind the last request, a borrowed cache, a block whose page is not held."""
    setup = Setup([(20, 1), (-1, 1), (40, 1)], 2, 4, 64, 16, dropped=[0, 0, 0])
    setup.lists[2][2] = -1
    setup.build()
    before, scales = setup.codes.clone(), setup.scales.clone()
    qkv = _rows(setup, 1, False, 1)
    q, parts = _appended(setup, qkv, None)
    assert (q[1] == 7.0).all() and torch.equal(q[0], parts[0][0][0]) and torch.equal(q[2], parts[2][0][0])
    page = setup.lists[0][1]
    assert torch.equal(setup.codes[:page], before[:page]) and torch.equal(setup.codes[page + 1:], before[page + 1:])
    after = setup.codes.clone()
    scales = setup.scales.clone()
    q, _ = _appended(setup, _rows(setup, 2, False, 1), None, write=False)
    assert torch.equal(setup.codes, after) and torch.equal(setup.scales.nan_to_num(-1), scales.nan_to_num(-1)) and not (q[0] == 7.0).any()


def test_append_refuses():
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import CacheView, Partials
    setup = Setup([(0, 4)], 2, 4, 64, 16)
    good, q = torch.zeros(4, 12 * 64, device=DEV), torch.zeros(4, 8 * 64, dtype=BF16, device=DEV)
    freq = torch.zeros(32, device=DEV)
    half = CacheView(0, 0, setup.maps.table, 0, 1, 16, 2, 64, BF16)
    for t, out, view, inv, heads in ((good[:3], q, setup.view, freq, 8), (good[:, :-1], q, setup.view, freq, 8), (good.half(), q, setup.view, freq, 8),
                                     (good, q.float(), setup.view, freq, 8), (good, q[:3], setup.view, freq, 8), (good, q, setup.view, freq[:31], 8),
                                     (good, q, setup.view, freq.double(), 8), (good, q, setup.view, freq, 6), (good, q, half, freq, 8),
                                     (good.cpu(), q, setup.view, freq, 8), (torch.zeros(4, 24 * 64, device=DEV)[:, : 12 * 64], q, setup.view, freq, 8)):
        with pytest.raises(KernelLaunchError):
            cache8.append(Partials(t), out, view, setup.maps, inv, heads)
    for n in (0, 2):           # two axes hold one result
        with pytest.raises(KernelLaunchError):
            cache8.append(Partials(good, n), q, setup.view, setup.maps, freq, 8)
    parts = torch.zeros(2 * 4 * 12 * 64 + 4, dtype=BF16, device=DEV)        # partial results a whole number of 16 bytes apart, or refused
    with pytest.raises(KernelLaunchError):
        cache8.append(Partials(parts.as_strided((2, 4, 12 * 64), (4 * 12 * 64 + 4, 12 * 64, 1)), 2), q, setup.view, setup.maps, freq, 8)
    with pytest.raises(KernelLaunchError, match="have not been built"):
        from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
        cache8.append(Partials(good), q, setup.view, StepMaps(4, 1, 1, 16, group=4, device=DEV), freq, 8)
    for codes, scales in ((setup.codes.float(), setup.scales), (setup.codes, setup.scales.double()), (setup.codes[..., :48], setup.scales),
                          (setup.codes, setup.scales[:1]), (setup.codes[:, :, :, :, :, ::2], setup.scales)):
        with pytest.raises(KernelLaunchError, match="cache8"):
            cache8.view(codes, scales, setup.maps.table)
    with pytest.raises(KernelLaunchError, match="no cache 1"):
        cache8.view(setup.codes, setup.scales, setup.maps.table, 1)


# ------------------------------------------------------------------------------ attention

def _attention(requests, kv_heads, group, dim, page, seed=0, window=0, chunk=0, sink=False, gate=False, q_scale=1.0, keys=None, dropped=None,
               caches=2, check=True, edit=None):
    """Fills a cache, runs attention over it and compares every row; returns (setup, q, out)."""
    from bare_cuda_4gib_b200.kernels import cache8, gemm
    from bare_cuda_4gib_b200.kernels.lib import AttentionExtras
    setup = Setup(requests, kv_heads, group, dim, page, seed, caches=caches, index=caches - 1, dropped=dropped, width=max(1, max(-(-(c + n) // page) for c, n in requests)) + 1)
    gen, heads = torch.Generator().manual_seed(seed), kv_heads * group
    plain = []
    for s, (c, n) in enumerate(requests):
        cache = pc.Cache(kv_heads, dim)
        if c >= 0:
            k, v = torch.randn(2, c + n, kv_heads, dim, generator=gen, dtype=F64).float().double()
            if keys is not None:
                k, v = keys(k, v)
            cache.append(k, v)
            setup.fill(s, cache)
        plain.append(cache)
    if edit is not None:
        edit(setup, plain)
    q = (torch.randn(setup.rows, heads * dim, generator=gen) * q_scale).to(BF16).to(DEV)
    gates = torch.randn(setup.rows, heads + 3, generator=gen).to(BF16).to(DEV)[:, 1: heads + 1] if gate else None
    sinks = torch.randn(heads, generator=gen).to(DEV) if sink else None
    out = torch.full((setup.rows + 2, heads * dim), 7.0, dtype=BF16, device=DEV)
    scale = 1 / math.sqrt(dim)
    extras = AttentionExtras(chunk, sinks, gates) if chunk or sink or gate else None
    cache8.attention(q, out, setup.view, setup.maps, heads, scale, window, extras)
    torch.cuda.synchronize()
    gemm.check_errors()
    assert (out[setup.rows:] == 7.0).all()
    row = 0
    for s, (c, n) in enumerate(requests):
        got = out[row: row + n].double().cpu().view(n, heads, dim)
        if c < 0:
            assert (got == 7.0).all()
        elif check:
            k, v = plain[s].values()
            want, bound = pc.attention(q[row: row + n].double().cpu().view(n, heads, dim), k, v, c, scale, window, chunk,
                                       sinks.double().cpu() if sink else None, gates[row: row + n].double().cpu() if gate else None)
            assert torch.equal(got.isnan(), want.isnan()), f"request {s}"
            off = (got - want).abs().nan_to_num(0.0) - (2.0 ** -8 * want.abs() + 2.0 ** -9 * bound).nan_to_num(0.0)
            assert (off <= 0).all(), f"request {s}: {int((off > 0).sum())} of {off.numel()} off, worst {float(off.max()):.3e}"
        row += n
    return setup, q, out


@pytest.mark.parametrize("group", [1, 3, 4, 8, 16])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_lengths(dim, group):
    """One new token behind every number of cached ones around the blocks' borders; pages of 48; an idle row in between."""
    lengths = [0, 1, 14, 15, 16, 17, 31, 32, 47, 48, 49, 63, 127, 128, 129, 300]
    _attention([(c, 1) for c in lengths[:8]] + [(-1, 1)] + [(c, 1) for c in lengths[8:]], 2, group, dim, 48, seed=group)


@pytest.mark.parametrize("dim,group,each", [(64, 4, 2), (128, 4, 4), (64, 8, 2), (128, 1, 16), (64, 5, 3), (128, 2, 7)])
def test_decode_of_several_tokens(dim, group, each):
    _attention([(c, each) for c in (0, 1, 13, 16, 30, 100, 257)], 3, group, dim, 16, seed=each)


@pytest.mark.parametrize("dim,group", [(64, 8), (128, 8), (64, 5), (128, 3), (128, 16), (64, 1)])
@pytest.mark.parametrize("window", [0, 70])
def test_few_rows_beside_prompts(dim, group, window):
    """Requests of every number of packed rows up to 16 and just above beside prompts and idle rows: a block of 8 rows each, two for some."""
    few = [(50 + 37 * n, n) for n in range(1, 18 // group + 2)]
    _attention([(100, 1), (0, 90), *few, (-1, 1), (0, 1), (333, 1), (64, 20)], 2, group, dim, 32, seed=group, window=window, sink=True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
def test_decode_long_and_split(monkeypatch, dim, splits):
    """Every number of blocks that may share a request, requests shorter than they have warps, and more scale blocks a warp than the
    lanes know at a time."""
    from bare_cuda_4gib_b200.kernels import cache8
    monkeypatch.setattr(cache8, "decode_splits", lambda *a: splits)
    _attention([(5000, 1), (37, 1), (0, 1), (2047, 1), (129, 1)], 1, 4, dim, 32, seed=splits)


def test_decode_of_more_requests_than_run_at_once():
    """Longest requests first: every row lands at its own place."""
    rng = random.Random(5)
    _attention([(rng.randrange(0, 200), 1) for _ in range(90)], 8, 1, 64, 16, seed=9)


PROMPTS = [(64, 4, [(0, 17)], 16), (64, 8, [(0, 129), (5, 3)], 32), (128, 4, [(0, 300)], 64), (128, 8, [(100, 61), (0, 40)], 48), (64, 1, [(0, 257), (17, 33)], 128),
           (128, 16, [(130, 20), (3, 2)], 16), (64, 7, [(64, 64), (0, 1), (1, 90)], 16), (128, 32, [(0, 1), (9, 5)], 64), (128, 1, [(200, 130)], 96)]


@pytest.mark.parametrize("dim,group,requests,page", PROMPTS)
def test_prompts(dim, group, requests, page):
    _attention(requests, 2, group, dim, page, seed=dim + group)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
def test_prompts_split(monkeypatch, dim, splits):
    """Every number of blocks that may share a tile's keys; tiles with fewer key blocks than that."""
    from bare_cuda_4gib_b200.kernels import cache8
    monkeypatch.setattr(cache8, "prompt_splits", lambda *a: splits)
    _attention([(1500, 61), (0, 20), (127, 70), (513, 1)], 2, 4, dim, 32, seed=splits, sink=True)
    _attention([(700, 61), (0, 150)], 1, 8, dim, 16, seed=splits, window=100)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("more", [dict(window=1), dict(window=5), dict(window=16), dict(window=17), dict(window=100), dict(chunk=16), dict(chunk=40),
                                  dict(chunk=100), dict(sink=True), dict(gate=True), dict(window=70, chunk=64, sink=True, gate=True)])
def test_windows_blocks_sinks_gates(dim, more):
    """Requests of few rows beside prompts, in one call."""
    _attention([(c, 1) for c in (0, 15, 16, 17, 39, 40, 130)] + [(0, 150), (77, 90), (250, 2)], 2, 4, dim, 16, seed=3, **more)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 4])
def test_infinite_sinks(monkeypatch, dim, splits):
    """A sink of -inf is none, one of +inf leaves nothing of its head, and a row without a key is zero whatever its sink."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import AttentionExtras
    monkeypatch.setattr(cache8, "prompt_splits", lambda *a: splits)
    monkeypatch.setattr(cache8, "decode_splits", lambda *a: splits)
    setup, q, out = _attention([(700, 1), (600, 60), (0, 1)], 2, 4, dim, 16, seed=9)
    again, sinks = torch.zeros_like(out), torch.tensor([-math.inf, math.inf] * 4, device=DEV)
    cache8.attention(q, again, setup.view, setup.maps, 8, 1 / math.sqrt(dim), 0, AttentionExtras(sink=sinks))
    got, want = (x[: setup.rows].double().view(setup.rows, 8, dim) for x in (again, out))
    assert (got[:, 1::2] == 0).all() and ((got - want)[:, ::2].abs() <= 2.0 ** -7 * want[:, ::2].abs() + 2.0 ** -12).all()
    setup.maps.table.fill_(-1)
    for sink in (None, sinks, torch.zeros(8, device=DEV)):
        cache8.attention(q, again, setup.view, setup.maps, 8, 1 / math.sqrt(dim), 0, AttentionExtras(sink=sink) if sink is not None else None)
        assert (again[: setup.rows] == 0).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_pages_that_a_window_gave_back(dim):
    """Blocks without a page in front of the window; the pool is full of NaN codes and scales."""
    _attention([(100, 1), (85, 3), (200, 40), (16, 1)], 2, 4, dim, 16, window=33, dropped=[4, 3, 10, 0])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("entry", [-1, -7, 2 ** 31 - 1, "first behind the pool"])
def test_pages_outside_the_pool(dim, entry):
    """A block whose entry of the table names no page of the pool: its positions are seen by no query, and the append writes nothing there."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import Partials
    requests, kept = [(200, 1), (150, 40), (300, 4), (64, 1), (70, 200)], []

    def spoil(setup, plain):
        kept.extend(plain)
        setup.maps.table[:, 3] = setup.codes.shape[0] if isinstance(entry, str) else entry

    setup, q, out = _attention(requests, 2, 4, dim, 16, seed=7, edit=spoil, check=False)
    row = 0
    for s, (c, n) in enumerate(requests):
        k, v = (torch.cat([x[:, :48], x[:, 64:]], 1) for x in kept[s].values())      # [heads, positions, entries]
        want, bound = pc.attention(q[row: row + n].double().cpu().view(n, 8, dim), k, v, c - 16, 1 / math.sqrt(dim), 0, 0, None, None)
        off = (out[row: row + n].double().cpu().view(n, 8, dim) - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -9 * bound)
        assert (off <= 0).all(), s
        row += n
    requests = [(48, 3), (40, 20), (63, 1)]                # writes to blocks 2, 3 and (the second's) 3 again
    setup = Setup(requests, 2, 4, dim, 16, seed=8)
    setup.maps.table[:, 3] = setup.codes.shape[0] if isinstance(entry, str) else entry
    before, scales = setup.codes.clone(), setup.scales.clone()
    qkv = torch.randn(setup.rows, 12 * dim, device=DEV)
    out = torch.zeros(setup.rows, 8 * dim, dtype=BF16, device=DEV)
    cache8.append(Partials(qkv), out, setup.view, setup.maps, None, 8)
    assert torch.equal(out, qkv[:, : 8 * dim].to(BF16))
    page = setup.lists[1][2]                                # the one block that is held and written
    others = [p for p in range(setup.codes.shape[0]) if p != page]
    assert torch.equal(setup.codes[others], before[others]) and torch.equal(setup.scales[others].nan_to_num(-1), scales[others].nan_to_num(-1))
    assert (setup.codes[page] != before[page]).any()


@pytest.mark.parametrize("dim", [64, 128])
def test_scales_far_apart(dim):
    """Value blocks 2^20 apart and key blocks 2^12 apart, so that large and small ones meet in a row's sum and rows see small ones alone; values of
    1e30 and of 1e-28."""
    def keys(k, v):
        t = torch.arange(k.shape[0])[:, None, None]
        return k * 2.0 ** -(t // 16 % 3 * 6).double(), v * 2.0 ** (20 - t // 16 % 5 * 10).double()

    _attention([(0, 1), (30, 1), (200, 1), (0, 100), (150, 70)], 2, 4, dim, 16, seed=1, keys=keys)
    _attention([(40, 1), (0, 90)], 2, 4, dim, 16, seed=2, keys=lambda k, v: (k, v * 1e30), check=True)
    _attention([(40, 1), (0, 90)], 2, 4, dim, 16, seed=2, keys=lambda k, v: (k, v * 1e-28), check=True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e9, 1e16])
def test_zeros_beside_large_values(dim, size):
    """Three of four blocks hold values of zero (their scale is the least one) and keys of zero: many keys, each 2^-10 or so of the largest weight,
    which add nothing to the output but their share of the sum."""
    def keys(k, v):
        holds = (torch.arange(k.shape[0])[:, None, None] // 16 % 4 == 1).double()
        return k * holds * 4, v * holds * size

    _attention([(900, 1), (30, 1), (500, 40), (0, 200), (100, 4)], 2, 4, dim, 16, seed=5, keys=keys)
    _attention([(400, 1), (300, 90)], 2, 8, dim, 64, seed=6, window=130, keys=keys)


@pytest.mark.parametrize("dim", [64, 128])
def test_growing_scores(dim):
    """Keys that grow along the sequence move the running maximum in most blocks; constant ones never."""
    def growing(k, v):
        direction = torch.randn(1, 1, dim, generator=torch.Generator().manual_seed(2), dtype=F64)
        return direction * torch.arange(1, k.shape[0] + 1)[:, None, None] / 60 + 0 * k, v

    _attention([(400, 1), (100, 200), (0, 130)], 1, 8, dim, 32, seed=4, keys=growing, q_scale=1.0)
    _attention([(400, 1), (100, 200)], 1, 8, dim, 32, seed=4, keys=lambda k, v: (k * 0 + 0.5, v))


@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_without_numbers_reach_only_the_rows_that_see_them(dim):
    """A block whose keys' scale is NaN: rows that see one of its keys are NaN, rows of the same tile that do not are right (a window hides
    it from later rows, causality from earlier ones)."""
    def spoil(setup, plain):
        for s, (c, n) in enumerate(setup.requests):
            block = min(4, (c + n - 1) // 16)
            plain[s].scales[0, 0, block] = math.nan
            setup.fill(s, plain[s])

    setup, _q, out = _attention([(20, 100), (63, 4), (200, 1), (10, 1), (66, 120)], 2, 4, dim, 32, seed=6, window=50, edit=spoil)
    seen = out[: setup.rows].isnan().any(1)
    assert seen.any() and not seen.all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-3, 300.0])
def test_query_sizes(dim, size):
    if size == 300.0:       # scores of hundreds: the largest key takes all; only its rounding matters, exponents grow with the scores
        setup, q, out = _attention([(100, 1), (0, 80)], 2, 4, dim, 16, q_scale=size, check=False)
        assert out[: setup.rows].isfinite().all()
        return
    _attention([(100, 1), (0, 80)], 2, 4, dim, 16, q_scale=size)


@pytest.mark.parametrize("dim", [64, 128])
def test_queries_that_are_no_numbers(dim):
    """A NaN or infinite query entry makes its own row NaN and no other."""
    from bare_cuda_4gib_b200.kernels import cache8
    setup, q, out = _attention([(100, 1), (40, 1), (0, 80)], 2, 4, dim, 16)
    bad = q.clone()
    bad[0, 3], bad[2 + 50, dim + 1], bad[2 + 7, 5 * dim] = math.nan, math.inf, -math.inf
    again = torch.zeros_like(out)
    cache8.attention(bad, again, setup.view, setup.maps, 8, 1 / math.sqrt(dim))
    wrong = again[: setup.rows].view(setup.rows, 8, dim).isnan().all(-1)
    assert wrong.nonzero().tolist() == [[0, 0], [9, 5], [52, 1]]
    good = ~wrong
    assert torch.equal(again[: setup.rows].view(setup.rows, 8, dim)[good], out[: setup.rows].view(setup.rows, 8, dim)[good])


def test_pool_beyond_32_bits():
    """The same pages at the end of a pool of 5 GB: the same outputs, and the same codes from the append."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import Partials
    requests = [(200, 1), (150, 40), (63, 2)]
    setup, q, out = _attention(requests, 2, 4, 128, 64, seed=3, caches=1)
    small, total = setup.codes.shape[0], (5 << 30) // (2 * 2 * 64 * 128)
    codes = torch.empty((total, 2, 2, 64, 128), dtype=torch.uint8, device=DEV)
    scales = torch.empty((total, 2, 2, 4), device=DEV)
    codes[total - small:], scales[total - small:] = setup.codes[:, 0], setup.scales[:, 0]
    near, table = setup.view, setup.maps.table
    far_table = torch.where(table >= 0, table + (total - small), table)
    far = cache8.view(codes, scales, far_table)
    again = torch.zeros_like(out)
    cache8.attention(q, again, far, setup.maps, 8, 1 / math.sqrt(128))
    assert torch.equal(again[: setup.rows], out[: setup.rows])
    qkv = torch.randn(setup.rows, 12 * 128, device=DEV) * 3
    for view in (near, far):
        cache8.append(Partials(qkv), again, view, setup.maps, None, 8)
    assert torch.equal(codes[total - small:], setup.codes[:, 0])
    assert torch.equal(scales[total - small:].nan_to_num(-1), setup.scales[:, 0].nan_to_num(-1))


def test_attention_refuses():
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import AttentionExtras
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    setup = Setup([(0, 4)], 2, 4, 64, 16)
    q = torch.zeros(4, 8 * 64, dtype=BF16, device=DEV)
    wide = torch.zeros(4, 9 * 64, dtype=BF16, device=DEV)[:, 64:]
    for a, b, heads, scale, window, extras in ((q[:3], q, 8, 0.1, 0, None), (q, q[:3], 8, 0.1, 0, None), (q.float(), q, 8, 0.1, 0, None), (q, wide, 8, 0.1, 0, None),
                                               (q, q, 4, 0.1, 0, None), (q, q, 8, 0.0, 0, None), (q, q, 8, -1.0, 0, None), (q, q, 8, math.nan, 0, None),
                                               (q, q, 8, 0.1, -1, None), (q.cpu(), q, 8, 0.1, 0, None), (q, q, 8, 0.1, 0, AttentionExtras(sink=torch.zeros(7, device=DEV))),
                                               (q, q, 8, math.inf, 0, None), (q, q, 8, 0.1, 0, AttentionExtras(gate=torch.zeros(3, 8, dtype=BF16, device=DEV))),
                                               (q, q, 8, 0.1, 0, AttentionExtras(gate=torch.zeros(8, dtype=BF16, device=DEV)))):
        with pytest.raises(KernelLaunchError):
            cache8.attention(a, b, setup.view, setup.maps, heads, scale, window, extras)
    other = StepMaps(4, 1, 1, 16, group=4, tile_rows=128, few_rows=16, device=DEV)
    other.build(i32([0]), i32([4]), i32([0]), 4, 4, 4)
    with pytest.raises(KernelLaunchError, match="tile_rows"):
        cache8.attention(q, q, setup.view, other, 8, 0.1)


# ------------------------------------------------------------------------------ together

@pytest.mark.parametrize("dim,group,page", [(64, 8, 16), (128, 4, 64)])
def test_steps_of_requests_together(dim, group, page):
    """Maps, append and attention as a program runs them: a prompt, portions of it, single tokens and several, requests joining, over two
    caches of one pool, on a stream of its own; every row against the plain cache that grew the same way."""
    from bare_cuda_4gib_b200.kernels import cache8, gemm
    from bare_cuda_4gib_b200.kernels.lib import Partials
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    kv_heads, heads, most = 2, 2 * group, 200
    width = -(-most // page)
    gen = torch.Generator().manual_seed(dim)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        codes = torch.zeros(3 * width + 1, 2, 2, kv_heads, page, dim, dtype=torch.uint8, device=DEV).view(CODES)
        scales = torch.zeros(3 * width + 1, 2, 2, kv_heads, page // 16, device=DEV)
        maps = StepMaps(256, 3, width, page, group=group, tile_rows=cache8.tile_rows(dim), few_rows=16, device=DEV)
        views = [cache8.view(codes, scales, maps.table, i) for i in range(2)]
        pages = torch.randperm(3 * width, generator=gen).view(3, width).tolist()
        inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, dtype=F64) / dim)).to(F32).to(DEV)
        lengths, plain = [0, 0, 0], [[pc.Cache(kv_heads, dim) for _ in range(3)] for _ in range(2)]
        q = torch.zeros(256, heads * dim, dtype=BF16, device=DEV)
        for step, news in enumerate([(37, 0, 0), (1, 90, 0), (1, 1, 0), (1, 1, 33), (16, 2, 1), (1, 1, 1), (3, 1, 2)]):
            live = [s for s in range(3) if news[s]]
            rows = sum(news)
            maps.build(i32([lengths[s] for s in live]), i32([news[s] for s in live]),
                       i32([p for s in live for p in pages[s][: -(-(lengths[s] + news[s]) // page)]]), rows, max(news[s] for s in live), min(news[s] for s in live))
            for layer in range(2):
                qkv = (torch.randn(rows, (heads + 2 * kv_heads) * dim, generator=gen) * 2.0 ** step).to(DEV)
                out = torch.zeros(rows, heads * dim, dtype=BF16, device=DEV)
                cache8.append(Partials(qkv), q, views[layer], maps, inv_freq, heads)
                cache8.attention(q, out, views[layer], maps, heads, 0.02)
                stream.synchronize()
                gemm.check_errors()
                x, row = qkv.double().cpu().view(rows, -1, dim), 0
                for s in live:
                    n, c = news[s], lengths[s]
                    mine = x[row: row + n]
                    k = pc.rotate(mine[:, heads: heads + kv_heads], torch.arange(c, c + n), inv_freq.cpu())
                    plain[layer][s].append(k, mine[:, heads + kv_heads:])
                    # the cache: scales are the plain one's, codes but for ones that float32 rounds to their neighbour
                    held = [(pc.NUMBERS[codes.view(torch.uint8)[p, layer].cpu().long()], scales[p, layer].double().cpu()) for p in pages[s]]
                    got = torch.cat([a for a, _ in held], 2)[:, :, : c + n]
                    got_scales = torch.cat([b for _, b in held], 2)[:, :, : -(-(c + n) // 16)]
                    assert torch.equal(got_scales, plain[layer][s].scales)
                    other = got != plain[layer][s].codes
                    assert ((got - plain[layer][s].codes).abs() <= 2.0 ** -3 * got.abs() + 2.0 ** -9).all() and other.double().mean() < 1e-3
                    plain[layer][s].codes = got
                    kk, vv = plain[layer][s].values()
                    qq = q[row: row + n].double().cpu().view(n, heads, dim)
                    want, bound = pc.attention(qq, kk, vv, c, 0.02)
                    # The entries grow from step to step, and the scores with them beyond what the module's bound allows for, so the scores' part is
                    # counted out: 128 products a sum and its scaling, 130 * 2^-24 of the sum of their sizes, and entries of q below 2^-9 of
                    # the row's largest, 2^-17 of that largest; once in the weights and once in their sum.
                    per_head = kk.abs().repeat_interleave(heads // kv_heads, 0)
                    sizes = torch.einsum("nhd,hld->nhl", qq.abs(), per_head).amax(-1) * 0.02
                    most = qq.abs().amax(-1, keepdim=True)
                    tiny = torch.einsum("nhd,hld->nhl", (qq.abs() < 2.0 ** -9 * most) * most * 2.0 ** -17, per_head).amax(-1) * 0.02
                    slack = torch.expm1(2 * (130 * 2.0 ** -24 * sizes + tiny))[..., None]
                    off = (out[row: row + n].double().cpu().view(n, heads, dim) - want).abs()
                    # weights far below the row's largest, which is at least 1, are halves with a step of 2^-24: half of that each
                    lost = 2.0 ** -25 * vv.abs().sum(1).repeat_interleave(heads // kv_heads, 0)
                    assert (off <= 2.0 ** -8 * want.abs() + (2.0 ** -10 + slack) * bound + lost).all(), (step, layer, s)
                    row += n
            for s in live:
                lengths[s] += news[s]


def test_a_captured_step_is_replayed_while_its_requests_grow():
    """The append and attention in a graph, the maps built anew ahead of every replay."""
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import Partials
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    dim, kv_heads, group, page, S = 64, 2, 4, 16, 3
    heads = kv_heads * group

    def program(graph):
        gen = torch.Generator(DEV).manual_seed(1)
        codes = torch.zeros(3 * 8, 2, kv_heads, page, dim, dtype=torch.uint8, device=DEV)
        scales = torch.zeros(3 * 8, 2, kv_heads, 1, device=DEV)
        maps = StepMaps(S, S, 8, page, group=group, tile_rows=cache8.tile_rows(dim), few_rows=16, device=DEV)
        qkv = torch.zeros(S, (heads + 2 * kv_heads) * dim, device=DEV)
        q, out = torch.zeros(S, heads * dim, dtype=BF16, device=DEV), torch.zeros(S, heads * dim, dtype=BF16, device=DEV)
        lengths, outs, captured = [0, 5, 30], [], None

        def step():
            cache8.append(Partials(qkv), q, view, maps, None, heads)
            cache8.attention(q, out, view, maps, heads, 0.125)

        for i in range(40):
            maps.build(i32(lengths), i32([1] * S), i32([s * 8 + b for s in range(S) for b in range(lengths[s] // page + 1)]), S, 1, 1)
            view = cache8.view(codes, scales, maps.table) if i == 0 else view
            qkv.copy_(torch.randn(qkv.shape, generator=gen, device=DEV) * (1 + i))
            if not graph or i < 2:
                step()
            else:
                if captured is None:
                    captured = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(captured):
                        step()
                captured.replay()
            outs.append(out.clone())
            lengths = [n + 1 for n in lengths]
        return torch.stack(outs), codes, scales

    for a, b in zip(program(False), program(True)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------ the engine

WIDE = dict(vocab_size=515, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=352,
            max_position_embeddings=512)
BROAD = dict(vocab_size=300, hidden_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=1, head_dim=128, intermediate_size=384,
             max_position_embeddings=512)


def _engine_and_plain(tmp_path, monkeypatch, sizes):
    import plain_llama as pl
    from bare_cuda_4gib_b200.models.presets import preset_config
    from bare_cuda_4gib_b200.weights.random_init import write_random_model
    write_random_model(tmp_path, preset_config("tinyA", **sizes), 3)
    plain = pl.read_model_folder(tmp_path)

    def held(x):        # [T, kv heads, dim] -> what a cache of codes stands for
        cache = pc.Cache(x.shape[1], x.shape[2])
        cache.append(x, x)
        return cache.values()[1].transpose(0, 1)

    scores, values = pl.attention_scores, pl.attention_values
    monkeypatch.setattr(pl, "attention_scores", lambda q, k, *a, **b: scores(q, held(k), *a, **b))
    monkeypatch.setattr(pl, "attention_values", lambda p, v: values(p, held(v)))
    return plain, pl


@pytest.mark.parametrize("sizes,page", [(WIDE, 16), (BROAD, 64)])
def test_engine_cut_into_steps(tmp_path, monkeypatch, sizes, page):
    """Whole prompts, portions, single tokens, mixed batches, padded decode steps and replayed graphs against the plain model whose cache
    holds codes, within the suite's bfloat16 tolerance."""
    from bare_cuda_4gib_b200.cache.manager import CacheManager
    from bare_cuda_4gib_b200.engine.model import cache_type, load_model
    from bare_cuda_4gib_b200.engine.step import StepEntry, StepRunner
    from bare_cuda_4gib_b200.kernels import gemm
    from helpers import TOLERANCE, row_error
    plain, pl = _engine_and_plain(tmp_path, monkeypatch, sizes)
    model, _config = load_model(tmp_path, "bfloat16", "cuda")
    cache = CacheManager(model.cache_demands(), page_tokens=page, max_seqs=6, max_tokens=256, num_pages=6 * 256 // page,
                         dtype=cache_type("float8_e4m3", model), device="cuda")
    for g in cache.groups:
        g.pool.shuffle_free_list(3)
    runner = StepRunner(model, cache, max_step_tokens=300, max_batch_seqs=6)
    rng = random.Random(7)
    texts = [[rng.randrange(sizes["vocab_size"]) for _ in range(n)] for n in (200, 61, 33, 20, 5)]
    want = [pl.forward_logits(plain, t) for t in texts]
    slots = [cache.acquire_slot() for _ in texts]
    at = [0] * len(texts)

    def step(news):
        entries = [StepEntry(slots[s], texts[s][at[s]: at[s] + n], [n - 1]) for s, n in enumerate(news) if n]
        logits = runner.step(entries)
        cache.check_consistency()
        row = 0
        for s, n in enumerate(news):
            if n:
                at[s] += n
                assert row_error(logits[row], want[s][at[s] - 1]) <= TOLERANCE["bfloat16"], (news, s)
                row += 1

    step((120, 0, 0, 0, 0))
    step((30, 61 - 25, 0, 0, 0))
    step((1, 1, 17, 0, 0))
    step((2, 1, 1, 10, 1))
    for _ in range(4):
        step((1, 1, 1, 1, 1))
    for _ in range(6):
        step((1, 1, 1, 1, 0))
    step((3, 2, 4, 0, 0))
    gemm.check_errors()
    assert any(k[0] == "decode" for k in runner._graphs)


def test_engine_generates_and_reports(tmp_path, monkeypatch):
    """The entry points with such a cache: half the cache's bytes and a little, greedy ids that the plain model agrees with up to near ties,
    the same ids from a batch, sampling, and refusals."""
    from bare_cuda_4gib_b200.engine.engine import LLMEngine
    from bare_cuda_4gib_b200.errors import EngineError
    from bare_cuda_4gib_b200.sampling.params import SamplingParams
    plain, pl = _engine_and_plain(tmp_path, monkeypatch, WIDE)
    rng = random.Random(2)
    prompts = [[rng.randrange(515) for _ in range(n)] for n in (70, 9, 33)]
    engine = LLMEngine(tmp_path, max_tokens=128, max_seqs=4, cache_dtype="float8_e4m3")
    half = LLMEngine(tmp_path, max_tokens=128, max_seqs=4)
    assert sum(g.bytes for g in engine.cache.groups) * 2 == sum(g.bytes for g in half.cache.groups) * (1 + 4 / (16 * 64))
    got = engine.generate_batch(prompts, 24)
    for prompt, tokens in zip(prompts, got):
        logits = pl.forward_logits(plain, prompt + tokens[:-1])
        for i, t in enumerate(tokens):
            row = logits[len(prompt) - 1 + i]
            assert float(row.max() - row[t]) <= 3e-2 * float(row.abs().max())
    assert engine.generate(prompts[0], 6, sampling=SamplingParams(temperature=0.8, seed=5)) == engine.generate(
        prompts[0], 6, sampling=SamplingParams(temperature=0.8, seed=5))
    with pytest.raises(EngineError, match="bfloat16 runs"):
        LLMEngine(tmp_path, max_tokens=128, dtype="float32", cache_dtype="float8_e4m3")
    with pytest.raises(EngineError, match="e4m3"):
        LLMEngine(tmp_path, max_tokens=128, page_tokens=8, cache_dtype="float8_e4m3")


def test_tools(tmp_path, monkeypatch):
    """`llm-infer`, `llm-ppl`, `llm-bench` and `llm-kernel-bench` with such a cache, and the refusal of a float32 run."""
    import json
    import os
    import pathlib
    import subprocess
    import sys
    root = pathlib.Path(__file__).resolve().parents[1]

    def run(tool, *args):
        return subprocess.run([sys.executable, str(root / "bin" / tool), *map(str, args)], capture_output=True, text=True, timeout=600,
                              env=dict(os.environ, PYTHONDONTWRITEBYTECODE="1"))

    plain, pl = _engine_and_plain(tmp_path, monkeypatch, WIDE)
    rng = random.Random(4)
    prompt = [rng.randrange(515) for _ in range(40)]
    args = ("--model", tmp_path, "--prompt", ",".join(map(str, prompt)), "--tokens", 9, "--cache-dtype", "float8_e4m3")
    done = run("llm-infer", *args)
    assert done.returncode == 0, done.stderr[-2000:]
    tokens = [int(t) for t in next(line for line in done.stdout.splitlines() if line.startswith("generated:")).split(":")[1].split()]
    logits = pl.forward_logits(plain, prompt + tokens[:-1])
    assert len(tokens) == 9 and all(float(logits[39 + i].max() - logits[39 + i, t]) <= 3e-2 * float(logits[39 + i].abs().max()) for i, t in enumerate(tokens))
    done = run("llm-infer", *args, "--dtype", "float32")
    assert done.returncode == 1 and "bfloat16 runs" in done.stderr
    (tmp_path / "text.ids").write_bytes(b"".join(rng.randrange(515).to_bytes(4, "little") for _ in range(140)))
    args = ("--model", tmp_path, "--ids", tmp_path / "text.ids", "--ctx", 65, "--cache-dtype", "float8_e4m3")
    done = run("llm-ppl", *args)
    assert done.returncode == 0, done.stderr[-2000:]
    done = run("llm-ppl", *args, "--dtype", "float32")
    assert done.returncode == 1 and done.stderr.strip().splitlines()[-1].startswith("[llm] ") and "Traceback" not in done.stderr
    done = run("llm-bench", "--model", tmp_path, "--prompt-len", 40, "--tokens", 3, "--runs", 1, "--warmup", 1, "--batch", 2, "--kernels",
               "--cache-dtype", "float8_e4m3")
    assert done.returncode == 0 and all(f"  {label}  " in done.stdout for label in ("step maps", "append (codes)", "attention (codes)")), done.stderr[-2000:]
    for kernel, sizes, name in (("attention", ("--batch", 2, "--context", 100), "attention over e4m3 codes"), ("rope", ("--rows", 70), "append to e4m3 codes"),
                                ("attention", ("--batch", 1, "--q-len", 50, "--context", 300, "--head-dim", 128, "--page", 16), "attention over e4m3 codes")):
        done = run("llm-kernel-bench", kernel, *sizes, "--iters", 2, "--cache-dtype", "float8_e4m3")
        assert done.returncode == 0, done.stderr[-2000:]
        line = json.loads(done.stdout.strip().splitlines()[-1])
        assert line["kernel"].startswith(name) and line["us"] > 0
