"""The cache of e4m3 codes on the host: the plain statement of it, the cache manager's storage and refusals, which models take it, and how
many blocks the kernels share a request's keys among."""

import math

import pytest
import torch

import plain_cache8 as pc


def test_numbers_and_rounding_of_the_plain_statement():
    assert float(pc.NUMBERS[126]) == 448.0 and math.isnan(float(pc.NUMBERS[127])) and float(pc.NUMBERS[1]) == 2.0 ** -9
    assert torch.equal(torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().nan_to_num(), pc.NUMBERS.nan_to_num())
    x = torch.cat([torch.randn(4000, dtype=torch.float64) * 2.0 ** e for e in range(-12, 7)])
    x = x[x.abs() <= 448.0].float().double()
    assert torch.equal(pc.nearest(x), x.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("largest,want", [(0.0, -100), (448.0, 0), (448.0001, 1), (449.0, 1), (896.0, 1), (447.0, 0), (224.0, -1), (224.1, 0),
                                          (3.3e38, 119), (1e-45, -100), (1.0, -8), (1.75, -8), (1.76, -7)])
def test_scale_exponent(largest, want):
    assert pc.exponent(largest) == want
    assert want in (-100, 119) or (largest <= 448 * 2.0 ** want and largest > 448 * 2.0 ** (want - 1))


def _demands(head_dim=64, kv_heads=2, layers=3, **more):
    from bare_cuda_4gib_b200.cache.manager import CacheDemand
    from bare_cuda_4gib_b200.parts.base import KVCacheRequest
    return [CacheDemand(KVCacheRequest(kv_heads, head_dim, **more)) for _ in range(layers)]


def test_storage_of_codes_and_scales():
    from bare_cuda_4gib_b200.cache.manager import CacheManager
    m = CacheManager(_demands(), page_tokens=32, max_seqs=2, max_tokens=100, num_pages=5, dtype=torch.float8_e4m3fn, device="cpu")
    g = m.groups[0]
    assert g.storage.dtype == torch.uint8 and tuple(g.storage.shape) == (5, 3 * 2 * 2 * 32 * 64)
    assert g.scales.dtype == torch.float32 and tuple(g.scales.shape) == (5, 3 * 2 * 2 * 2)
    assert g.bytes == g.storage.numel() + 4 * g.scales.numel()
    table = torch.zeros(2, 4, dtype=torch.int32)
    for run in range(3):
        v = m.cache_view(run, table)
        assert v.dtype == torch.float8_e4m3fn and v.maps is None
        assert v.k_ptr - g.storage.data_ptr() == run * 2 * 2 * 32 * 64 and v.v_ptr - v.k_ptr == 2 * 32 * 64
        assert v.k_scale_ptr - g.scales.data_ptr() == 4 * run * 8 and v.v_scale_ptr - v.k_scale_ptr == 4 * 4 and v.scale_stride == 24
    half = CacheManager(_demands(), page_tokens=32, max_seqs=2, max_tokens=100, num_pages=5, dtype=torch.bfloat16, device="cpu").groups[0]
    assert half.scales is None and half.bytes == 2 * g.storage.numel()


@pytest.mark.parametrize("head_dim,page,more", [(16, 16, {}), (96, 16, {}), (64, 8, {}), (64, 24, {}), (64, 16, {"v_head_dim": 128})])
def test_storage_refusals(head_dim, page, more):
    from bare_cuda_4gib_b200.cache.manager import CacheManager
    from bare_cuda_4gib_b200.errors import CacheError
    with pytest.raises(CacheError, match="e4m3"):
        CacheManager(_demands(head_dim, **more), page_tokens=page, max_seqs=1, max_tokens=64, dtype=torch.float8_e4m3fn, allocate=False)


def test_pages_of_a_slot():
    from bare_cuda_4gib_b200.cache.manager import CacheManager
    m = CacheManager(_demands(window=40), page_tokens=16, max_seqs=2, max_tokens=400, num_pages=9, dtype=torch.float8_e4m3fn, allocate=False)
    s = m.acquire_slot()
    for n in (30, 50, 1, 40):
        m.reserve(s, n)
        length = m.length(s) + n
        assert m.pages_of(0, s, length) == m.groups[0].tables[s][: -(-length // 16)]
        m.commit(s, n)
    assert m.pages_of(0, s, 121)[0] == -1 and len(m.pages_of(0, s, 121)) == 8


def _model(preset, dtype=torch.bfloat16):
    import bare_cuda_4gib_b200.models  # noqa: F401
    from bare_cuda_4gib_b200.config.registry import resolve_architecture
    from bare_cuda_4gib_b200.engine.model import Model
    from bare_cuda_4gib_b200.models.presets import preset_config
    config = preset_config(preset)
    model = Model(resolve_architecture(config.to_dict()).build_spec(config))
    model.dtype = dtype
    return model


def test_which_models_take_codes():
    from bare_cuda_4gib_b200.engine.model import cache_type
    from bare_cuda_4gib_b200.errors import ConfigError
    llama = _model("tinyllama")
    assert cache_type(None, llama) == torch.bfloat16 == cache_type("bfloat16", llama)
    assert cache_type("float8_e4m3", llama) == torch.float8_e4m3fn == cache_type(torch.float8_e4m3fn, llama)
    for name in ("float32", "int8", torch.float16):
        with pytest.raises(ConfigError, match="not supported"):
            cache_type(name, llama)
    with pytest.raises(ConfigError, match="bfloat16 runs"):
        cache_type("float8_e4m3", _model("tinyllama", torch.float32))
    for other in ("zadurax-tiny", "dopudra-tiny", "gurolix-tiny", "fuzazen-tiny", "pudulorn-tiny", "sizitar-tiny"):
        with pytest.raises(ConfigError, match="not supported by the mixer"):
            cache_type("float8_e4m3", _model(other))


def test_blocks_that_share_keys():
    from bare_cuda_4gib_b200.kernels import cache8
    for rule in (cache8.decode_splits, cache8.prompt_splits):
        for n in (1, 2, 8, 37, 64, 300):
            for heads in (1, 4, 8, 32):
                for keys in (16, 128, 2048, 8192, 131072):
                    splits = rule(n, heads, keys)
                    assert splits in (1, 2, 4, 8)
                    assert splits == 1 or (splits // 2) * 128 < keys          # every block has keys to look at
    assert cache8.decode_splits(1, 4, 2048) == 8 and cache8.decode_splits(64, 8, 2048) == 1 and cache8.decode_splits(64, 8, 8192) == 2
    assert cache8.prompt_splits(1, 8, 8192) == 8 and cache8.prompt_splits(65, 4, 2048) == 1


@pytest.mark.parametrize("sizes", [dict(page_tokens=24), dict(page_tokens=8), dict(max_rows=0), dict(max_seqs=0), dict(group=0), dict(max_seqs=5000),
                                   dict(max_rows=1 << 30, group=4), dict(max_blocks=1 << 28)])
def test_step_maps_refuse_sizes(sizes):
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels.step_maps import StepMaps
    args = dict(max_rows=64, max_seqs=4, max_blocks=8, page_tokens=16) | sizes
    with pytest.raises(KernelLaunchError, match="step maps"):
        StepMaps(**args)


def test_a_launcher_turns_bad_sizes_away():
    """The C entries check sizes and alignment before they touch the device."""
    import ctypes
    from bare_cuda_4gib_b200.kernels import cache8, step_maps
    from bare_cuda_4gib_b200.kernels.step_maps import StepLists
    lists = StepLists(0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 1)
    at = ctypes.addressof(lists)

    def cache(**more):
        c = dict(k=4096, v=8192, k_scale=0, v_scale=0, block_table=0, page_stride=4096, scale_stride=4, n_pages=1, table_stride=1, page_tokens=16,
                 kv_heads=2, head_dim=64) | more
        return cache8._Cache8(*(c[name] for name, _ in cache8._Cache8._fields_))

    def append(c, dtype=1, partials=1, heads=4, qkv=4096):
        return cache8._append().llm_cache8_append(qkv, dtype, partials, 0, 4096, ctypes.addressof(c), at, 0, heads, 1, 0)

    assert append(cache(head_dim=96)) == 2 and append(cache(page_tokens=24)) == 2 and append(cache(), heads=3) == 2
    assert append(cache(), partials=0) == 2 and append(cache(), dtype=7) == 1 and append(cache(), qkv=4098) == 3 and append(cache(k=4100)) == 3

    def decode(c, splits=1, rows=4, q=4096):
        return cache8._decode(64).llm_cache8_attention_decode(q, 4096, ctypes.addressof(c), 0, 4096, at, splits, 0, rows, 1, 4, 0.125, 0, 0, 0, 0, 0, 0, 0)

    assert decode(cache(head_dim=128)) == 2 and decode(cache(), splits=3) == 2 and decode(cache(), rows=17) == 2 and decode(cache(), q=4104) == 3
    assert decode(cache(k=1024)) == 3                                   # ahead of the pool's base

    def prompt(c, splits=1, box=16, scale=0.125):
        return cache8._prompt(64).llm_cache8_attention_prompt(4096, 4096, ctypes.addressof(c), 0, 4096, box, at, splits, 4, scale, 0, 0, 0, 0, 0, 0, 0)

    assert prompt(cache(head_dim=128)) == 2 and prompt(cache(), splits=16) == 2 and prompt(cache(), box=32) == 2 and prompt(cache(), box=8) == 2
    assert prompt(cache(), scale=0.0) == 2 and prompt(cache(v=8208)) == 3
    for seqs, page in ((5000, 16), (1, 24), (1, 0)):
        args = step_maps.MapsArgs(0, 0, seqs, 0, 0, 1, page, 1, 128, 16, 1, 1, 1, *[0] * 12)
        assert step_maps.lib().llm_step_maps(ctypes.addressof(args), 0) == 2
    map_at = ctypes.addressof((ctypes.c_ubyte * 128)())
    for base, rows, box in ((4096, 1 << 40, 16), (4104, 64, 16), (4096, 0, 16), (4096, 64, 24), (4096, 64, 8)):
        assert cache8._prompt(64).llm_cache8_prompt_pool_map(map_at, base, rows, box) == 2
    assert cache8._decode(64).llm_cache8_decode_pool_map(map_at, 4096, 1 << 31) == 2


def test_every_device_has_an_error_word_of_its_own(monkeypatch):
    """What a kernel reports to lies on its own device; a report on any of them is found, once."""
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels import gemm
    monkeypatch.setattr(gemm, "_error_words", {}, raising=False)
    monkeypatch.setattr(gemm, "_error_word", None, raising=False)
    first, second = (gemm.error_word(d) for d in (torch.device("cpu"), torch.device("cpu", 0)))
    assert first is not second and gemm.error_word(torch.device("cpu", 0)) is second
    gemm.check_errors()
    second.fill_(46)
    with pytest.raises(KernelLaunchError, match="decode attention over 8-bit codes"):
        gemm.check_errors()
    gemm.check_errors()


def test_a_view_refuses_parts_of_tables():
    """A request longer than its table's columns must find no page there; in a part of a wider table it would find the neighbouring columns', and
    behind the last row what lies behind the table."""
    from bare_cuda_4gib_b200.errors import KernelLaunchError
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import CacheView
    codes, scales = torch.zeros(4, 2, 1, 16, 64, dtype=torch.uint8), torch.zeros(4, 2, 1, 1)
    table = torch.zeros(3, 8, dtype=torch.int32)
    for part in (table[:, 2:], table[:, :4], table.t(), table[::2], table[0], table.long(), table[:1].expand(3, 8)):
        with pytest.raises(KernelLaunchError, match="block table must be contiguous"):
            cache8.view(codes, scales, part)
        with pytest.raises(KernelLaunchError, match="block table must be contiguous"):      # a view made by a cache's manager, at its first use
            cache8._Launch(CacheView(0, 0, part, 4096, 8, 16, 1, 64, cache8.DTYPE))
    for whole in (table, table[:2], table[1:2]):
        with pytest.raises(KernelLaunchError, match="one CUDA device"):
            cache8.view(codes, scales, whole)
