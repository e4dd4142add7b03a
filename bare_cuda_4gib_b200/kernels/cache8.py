"""A paged cache held in 8 bits: e4m3 codes with a power-of-two scale for every 16 positions, key/value head and keys or values each
(the format: `csrc/cache8.cuh`).  `append` writes a step's keys and values (`csrc/cache8_append.cu`), `attention` reads them
(`csrc/cache8_attention_decode.cu` for requests that bring at most 16 packed rows, `csrc/cache8_attention_tcgen05.cu` for the others).
Both go by the step's `StepMaps`.  Head sizes 64 and 128, bfloat16 queries and outputs."""

from __future__ import annotations

import ctypes
import functools
import math
from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Dict, Optional

import torch

from . import build, gemm
from ..errors import KernelLaunchError
from .lib import AttentionExtras, CacheView, Partials, _check, _ptr, dtype_code, sm_count
from .step_maps import SCALE_TOKENS, StepMaps

DTYPE = torch.float8_e4m3fn
HEAD_DIMS = (64, 128)
FEW_ROWS = 16            # packed rows up to which the decode kernel takes a request
KEY_BLOCK = 128          # positions that the prompt kernel takes at a time
BLOCKS_AT_ONCE = {2: 148, 4: 132, 8: 120}     # of the prompt kernel on a B200, one an SM, by the size of a cluster (cudaOccupancyMaxActiveClusters)
LEAST_SCALE, MOST_SCALE = 2.0 ** -126, 2.0 ** 127      # of the scores: what float32 has
MOST_POSITIONS = 1 << 24       # that angles are taken for: float32 has their numbers
DECODE_WARPS = 8         # warps of a block of the decode kernel, which a request's scale blocks are dealt to
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_append_lib = None
_decode_libs: Dict[int, object] = {}
_prompt_libs: Dict[int, object] = {}


class _Cache8(ctypes.Structure):
    """struct Cache8 of csrc/cache8.cuh."""

    _fields_ = [("k", c_void_p), ("v", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p), ("block_table", c_void_p),
                ("page_stride", c_longlong), ("scale_stride", c_longlong), ("n_pages", c_int), ("table_stride", c_int),
                ("page_tokens", c_int), ("kv_heads", c_int), ("head_dim", c_int)]


def supports(head_dim: int, v_dim: Optional[int] = None, page_tokens: int = SCALE_TOKENS) -> bool:
    return head_dim in HEAD_DIMS and (v_dim is None or v_dim == head_dim) and page_tokens > 0 and page_tokens % SCALE_TOKENS == 0


def _append():
    global _append_lib
    if _append_lib is None:
        l = build.load_library("cache8_append.cu")
        P, I, L = c_void_p, c_int, c_longlong
        l.llm_cache8_append.argtypes = [P, I, I, L, P, P, P, P, I, I, P]
        l.llm_cache8_append.restype = c_int
        _append_lib = l
    return _append_lib


def _decode(head_dim: int):
    l = _decode_libs.get(head_dim)
    if l is None:
        l = build.load_library("cache8_attention_decode.cu", (f"-DHEAD_DIM={head_dim}",))
        P, I, L, F = c_void_p, c_int, c_longlong, c_float
        l.llm_cache8_attention_decode.argtypes = [P, P, P, P, P, P, I, I, I, I, I, F, I, I, P, P, L, P, P]
        l.llm_cache8_attention_decode.restype = c_int
        l.llm_cache8_decode_pool_map.argtypes = [P, P, L]
        l.llm_cache8_decode_pool_map.restype = c_int
        _decode_libs[head_dim] = l
    return l


def _prompt(head_dim: int):
    l = _prompt_libs.get(head_dim)
    if l is None:
        l = build.load_library("cache8_attention_tcgen05.cu", (f"-DHEAD_DIM={head_dim}",))
        P, I, L, F = c_void_p, c_int, c_longlong, c_float
        l.llm_cache8_attention_prompt.argtypes = [P, P, P, P, P, I, P, I, I, F, I, I, P, P, L, P, P]
        l.llm_cache8_attention_prompt.restype = c_int
        l.llm_cache8_attention_prompt_rows.restype = c_int
        l.llm_cache8_prompt_pool_map.argtypes = [P, P, L, I]
        l.llm_cache8_prompt_pool_map.restype = c_int
        l.tile_rows = int(l.llm_cache8_attention_prompt_rows())
        _prompt_libs[head_dim] = l
    return l


def tile_rows(head_dim: int) -> int:
    """The `tile_rows` that a `StepMaps` for this head size is made with."""
    return _prompt(head_dim).tile_rows


def prepare(head_dim: int) -> None:
    """Builds and loads the kernels for this head size."""
    _append(), _decode(head_dim), _prompt(head_dim)


def _check_table(table: torch.Tensor) -> None:
    # (in a part of a wider table a request longer than the part would find its neighbours' entries, or what lies behind the table)
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
        raise KernelLaunchError("cache8: the block table must be contiguous int32 with two axes")


def view(codes: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor, index: int = 0) -> CacheView:
    """The cache that lies in `codes` (uint8 or float8_e4m3fn, [pages, (caches,) keys | values, kv heads, page tokens, head size])
    and `scales` (float32, [pages, (caches,) keys | values, kv heads, page tokens / 16]): with caches, the one at `index`."""
    if codes.dim() == 5:
        codes, scales = codes.unsqueeze(1), scales.unsqueeze(1)
    if codes.dim() != 6 or scales.dim() != 5 or codes.dtype not in (torch.uint8, DTYPE) or scales.dtype != torch.float32:
        raise KernelLaunchError("cache8: codes must be uint8 or float8_e4m3fn with five or six axes, scales float32 with one less")
    pages, caches, two, kv_heads, page_tokens, head_dim = codes.shape
    if tuple(scales.shape) != (pages, caches, two, kv_heads, page_tokens // SCALE_TOKENS) or two != 2 or not 0 <= index < caches:
        raise KernelLaunchError(f"cache8: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not belong together, or there is "
                                f"no cache {index}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise KernelLaunchError("cache8: codes and scales must be contiguous")
    if not supports(head_dim, None, page_tokens):
        raise KernelLaunchError(f"cache8: head size {head_dim} in pages of {page_tokens} positions is not supported (head sizes "
                                f"{HEAD_DIMS}, pages of a multiple of {SCALE_TOKENS})")
    _check_table(block_table)
    if not codes.is_cuda or scales.device != codes.device or block_table.device != codes.device:
        raise KernelLaunchError("cache8: codes, scales and block table must lie on one CUDA device")
    per_cache, per_cache_scales = 2 * kv_heads * page_tokens * head_dim, 2 * kv_heads * (page_tokens // SCALE_TOKENS)
    k = codes.data_ptr() + index * per_cache
    s = scales.data_ptr() + index * per_cache_scales * 4
    out = CacheView(k, k + per_cache // 2, block_table, caches * per_cache, block_table.shape[1], page_tokens, kv_heads, head_dim,
                    DTYPE, codes.data_ptr(), codes.numel(), k_scale_ptr=s, v_scale_ptr=s + per_cache_scales // 2 * 4,
                    scale_stride=caches * per_cache_scales)
    out.keeps = (codes, scales)
    gemm.error_word(codes.device)      # made here, so that a captured call, if it is the first, need not
    return out


class _Launch:
    """What the launchers hand on of a cache, made at its first use and kept with its view: the struct's address, the kernels' tensor maps
    over the pool, and the kernels' entries."""

    def __init__(self, cache: CacheView):
        if cache.dtype != DTYPE:
            raise KernelLaunchError(f"cache8: a cache of {cache.dtype} is not one of e4m3 codes")
        _check_table(cache.block_table)
        d = cache.head_dim
        self._struct = _Cache8(cache.k_ptr, cache.v_ptr, cache.k_scale_ptr, cache.v_scale_ptr, cache.block_table.data_ptr(),
                               cache.page_stride, cache.scale_stride, cache.pool_elems // cache.page_stride, cache.table_stride, cache.page_tokens,
                               cache.kv_heads, d)
        self.cache = ctypes.addressof(self._struct)
        self.box_rows, rows = math.gcd(KEY_BLOCK, cache.page_tokens), cache.pool_elems // d
        self._maps = (ctypes.c_ubyte * 128)(), (ctypes.c_ubyte * 128)()
        self.decode_map, self.prompt_map = (ctypes.addressof(m) for m in self._maps)
        _check(_decode(d).llm_cache8_decode_pool_map(self.decode_map, cache.pool_ptr, rows), "cache8 pool map")
        _check(_prompt(d).llm_cache8_prompt_pool_map(self.prompt_map, cache.pool_ptr, rows, self.box_rows), "cache8 pool map")
        self.append, self.decode, self.prompt = (_append().llm_cache8_append, _decode(d).llm_cache8_attention_decode,
                                                 _prompt(d).llm_cache8_attention_prompt)
        self.tile_rows, self.keys = tile_rows(d), cache.table_stride * cache.page_tokens
        self.device, self.table_rows = cache.block_table.get_device(), cache.block_table.shape[0]
        self.error_word = gemm.error_word(cache.block_table.device).data_ptr()


def _check_step(what: str, cache: CacheView, maps: StepMaps, q_heads: int, a: torch.Tensor, b: torch.Tensor) -> _Launch:
    """Whether cache, maps and the two tensors belong together (this and what follows runs for every layer of a step)."""
    launch = cache.launch
    if launch is None:
        launch = cache.launch = _Launch(cache)
    if q_heads <= 0 or maps.group * cache.kv_heads != q_heads or maps.page_tokens != cache.page_tokens:
        raise KernelLaunchError(f"{what}: the step's maps are for pages of {maps.page_tokens} positions and {maps.group} heads a key/value "
                                f"head, the cache has pages of {cache.page_tokens} and {cache.kv_heads} key/value heads for {q_heads} heads")
    if maps.longest == 0:
        raise KernelLaunchError(f"{what}: the step's maps have not been built")
    if launch.table_rows < maps.n_seqs:
        raise KernelLaunchError(f"{what}: {maps.n_seqs} requests, and a block table of {launch.table_rows} rows")
    index = maps.index
    if launch.device != index or a.get_device() != index or b.get_device() != index:
        raise KernelLaunchError(f"{what}: maps, cache and tensors must lie on one CUDA device")
    if index != _current_device():
        raise KernelLaunchError(f"{what}: the tensors lie on {maps.device}, the current device is cuda:{torch.cuda.current_device()}")
    return launch


def _bf16_rows(t: torch.Tensor, rows: int, width: int) -> bool:
    return t.dtype == torch.bfloat16 and t.dim() == 2 and t.size(1) == width and t.size(0) >= rows and t.is_contiguous()


def append(qkv: Partials, q_out: torch.Tensor, cache: CacheView, maps: StepMaps, inv_freq: Optional[torch.Tensor], q_heads: int,
           write_cache: bool = True, stream=None) -> None:
    """Rows [q | k | v] of the step (`qkv`, dense, bfloat16 or float32, possibly a sum of partial results): q turned by
    position into `q_out` (bfloat16 [rows, q_heads * head size]), k turned by position and v into the cache (left alone unless
    `write_cache`).  `inv_freq` (float32 [head size / 2]) None: no rotation.  Positions of a written block that earlier steps filled
    keep their numbers, but for a rounding where the new ones need a larger scale.  Requests may share pages that they read, not
    pages that a step writes.  Rows of no request and idle ones are left as they were in `q_out`.  With `inv_freq` the block table has columns for
    2^24 positions at most."""
    t = qkv.tensor
    width, d = (q_heads + 2 * cache.kv_heads) * cache.head_dim, cache.head_dim
    launch = _check_step("cache8_append", cache, maps, q_heads, t, q_out)
    shape = t.shape
    if t.dim() not in (2, 3) or shape[-1] != width or shape[-2] < maps.n_rows or t.stride(-1) != 1 or t.stride(-2) != width or (
            qkv.n != 1 and (qkv.n < 1 or t.dim() != 3 or shape[0] < qkv.n)):
        raise KernelLaunchError(f"cache8_append: projections of {tuple(shape)} for {maps.n_rows} dense rows of {width}")
    if not _bf16_rows(q_out, maps.n_rows, q_heads * d):
        raise KernelLaunchError(f"cache8_append: queries go to contiguous bfloat16 [rows, {q_heads * d}], not {tuple(q_out.shape)} of {q_out.dtype}")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() != d // 2 or not inv_freq.is_contiguous()
                                 or inv_freq.get_device() != maps.index):
        raise KernelLaunchError(f"cache8_append: the inverse frequencies must be {d // 2} contiguous float32 numbers")
    if inv_freq is not None and launch.keys > MOST_POSITIONS:
        raise KernelLaunchError(f"cache8_append: a block table for {launch.keys} positions, angles are taken for {MOST_POSITIONS}")
    _check(launch.append(
        t.data_ptr(), dtype_code(t.dtype), qkv.n, qkv.stride, q_out.data_ptr(), launch.cache, maps.lists, _ptr(inv_freq), q_heads,
        1 if write_cache else 0, stream if stream is not None else _current_stream(maps.index)), "cache8_append")


@functools.lru_cache(maxsize=256)
def decode_splits(n_seqs: int, kv_heads: int, max_keys: int) -> int:
    """How many blocks of the decode kernel share a request's keys: a power of two up to 8, about two blocks an SM in all, and no more
    than have a scale block for every warp.  With long caches twice that: requests of different lengths then leave fewer SMs idle at the
    end than a block's start and merge cost (one / two blocks: 64 requests of 2,000 to 8,191 positions, 8 heads of 128, 128 / 118 us; of 500 to
    2,047 positions 37 / 44).  `max_keys` is what the block table has columns for, not the lengths at hand, so that a captured graph stays valid: short
    requests in wide tables are split for nothing (8 of 100 positions, 4 heads of 64: 4.0 us in a table for 128, 5.8 in one for 8,192)."""
    splits = 1
    while splits < 8 and max_keys > splits * DECODE_WARPS * SCALE_TOKENS and (
            n_seqs * kv_heads * splits * 2 <= 2 * sm_count() or (max_keys >= splits * 2 * 2560 and n_seqs * kv_heads * splits <= 4 * sm_count())):
        splits *= 2
    return splits


@functools.lru_cache(maxsize=256)
def prompt_splits(n_tiles: int, kv_heads: int, max_keys: int) -> int:
    """How many blocks of the prompt kernel share a tile's keys: a power of two up to 8, as many as the SMs take at once in clusters of
    that size (more start only when others have ended: 128 blocks by eights 27.6 us, by fours 64 of them 18.8), and none over four key blocks, where the
    merge costs more than they save (389 tokens, 4 heads of 64, one block / two 11.9 / 13.4 us; behind 1,000 more 28.0 / 21.5).  `max_keys` is what
    the block table has columns for: a short prompt in a wide table is split all the same (61 tokens behind nothing, 8 heads of 128: 11.4 us in a table
    for 64 positions, 16.0 in one for 8,192)."""
    splits = 1
    while splits < 8 and n_tiles * kv_heads * splits * 2 <= BLOCKS_AT_ONCE[splits * 2] and max_keys > max(splits, 4) * KEY_BLOCK:
        splits *= 2
    return splits


def attention(q: torch.Tensor, out: torch.Tensor, cache: CacheView, maps: StepMaps, q_heads: int, scale: float, window: int = 0,
              extras: Optional[AttentionExtras] = None, stream=None) -> None:
    """out = softmax(scale * q k^T) v over each request's cached positions up to the query's own (with `window` > 0 the newest
    `window` of them), q and out contiguous bfloat16 [rows, q_heads * head size].  `extras`: blocks of positions, sink, gate.
    Requests of few packed rows go to the decode kernel, the others to the prompt kernel, which a step may launch both of; rows
    of no request and idle ones are left as they were in `out`, a row that sees no key is zero.  A position whose page is not held (an entry of the
    block table outside the pool) is seen by no query.

    Positions below the step's first new ones are read ahead of the wait for the kernels before, so between what wrote them and this call there has to
    be an ordinary operation of the stream (a copy, a kernel of torch's, the step's own `build`).  The step's maps are that where they are built
    behind the appends of the step before; a program that builds the maps of two steps ahead of both puts a copy or a synchronisation there.

    Weights are halves: 2^-32 of a row's largest is lost of any one of them, where a bfloat16 cache's kernels keep eight bits."""
    launch = _check_step("cache8_attention", cache, maps, q_heads, q, out)
    width = q_heads * cache.head_dim
    if not _bf16_rows(q, maps.n_rows, width) or not _bf16_rows(out, maps.n_rows, width):
        raise KernelLaunchError(f"cache8_attention: queries and outputs must be contiguous bfloat16 [{maps.n_rows} rows, {width}], not "
                                f"{tuple(q.shape)} of {q.dtype} and {tuple(out.shape)} of {out.dtype}")
    if not LEAST_SCALE <= scale < MOST_SCALE or not 0 <= window < 1 << 31 or extras is not None and not 0 <= extras.chunk < 1 << 31:
        raise KernelLaunchError(f"cache8_attention: scale {scale}, window {window} and blocks of {extras.chunk if extras is not None else 0} are not "
                                f"supported (above zero; zero or more; in 32 bits)")
    if maps.few_rows != FEW_ROWS or maps.tile_rows != launch.tile_rows:
        raise KernelLaunchError(f"cache8_attention: the step's maps must be made with few_rows {FEW_ROWS} and tile_rows {launch.tile_rows}")
    more = (0, 0, 0, 0)
    if extras is not None:
        more = extras.arguments(q_heads, q.dtype)
        if any(t is not None and t.get_device() != maps.index for t in (extras.sink, extras.gate)) or (
                extras.gate is not None and (extras.gate.dim() != 2 or extras.gate.size(0) < maps.n_rows)):
            raise KernelLaunchError(f"cache8_attention: sink and gate must lie on {maps.device}, the gate have two axes and {maps.n_rows} rows")
    stream = stream if stream is not None else _current_stream(maps.index)
    q_at, out_at, error_word, group = q.data_ptr(), out.data_ptr(), launch.error_word, maps.group
    if maps.shortest * group <= FEW_ROWS:
        splits = decode_splits(maps.n_seqs, cache.kv_heads, launch.keys)
        ordered = 1 if maps.n_seqs * cache.kv_heads * splits > 2 * sm_count() else 0
        # beside prompts only the shortest request is known: then most are taken to be like it, and one with more than 8 rows is read twice
        parts = 2 if maps.longest * group > FEW_ROWS and maps.shortest * group <= FEW_ROWS // 2 else 1
        _check(launch.decode(q_at, out_at, launch.cache, launch.decode_map, cache.pool_ptr, maps.lists, splits, ordered,
                             min(maps.longest * group, FEW_ROWS), parts, q_heads, scale, window, *more, error_word, stream), "cache8_attention_decode")
    if maps.longest * group > FEW_ROWS:
        # the list of tiles has room for a last one of every request; taken as if all were like the longest they are fewer
        tiles = min(maps.n_tiles, -(-maps.n_rows * -(-maps.longest * group // launch.tile_rows) // maps.longest))
        _check(launch.prompt(q_at, out_at, launch.cache, launch.prompt_map, cache.pool_ptr, launch.box_rows, maps.lists,
                             prompt_splits(tiles, cache.kv_heads, launch.keys), q_heads, scale, window, *more, error_word, stream),
               "cache8_attention_prompt")
