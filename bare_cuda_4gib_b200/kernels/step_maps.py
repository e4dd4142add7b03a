"""Launcher of `csrc/step_maps.cu`: the maps of a step, built on the device from the requests' lengths and pages.

A program that keeps its requests' lengths and page lists on the device, or that would rather send those few numbers than
padded tables and one position a row, makes a `StepMaps` once for its largest step and calls `build` for
every step; the arrays it then offers are what the kernels of that step read."""

from __future__ import annotations

import ctypes
from ctypes import c_int, c_void_p

import torch

from . import build
from ..errors import KernelLaunchError
from .lib import _check, stream_handle

SCALE_TOKENS = 16       # positions that share a scale in a cache of 8-bit codes: the blocks that `write_block` counts
_lib = None


def lib():
    global _lib
    if _lib is None:
        l = build.load_library("step_maps.cu")
        l.llm_step_maps.argtypes = [c_void_p, c_void_p]
        l.llm_step_maps.restype = c_int
        l.llm_step_maps_max_seqs.restype = c_int
        _lib = l
    return _lib


class MapsArgs(ctypes.Structure):
    """struct MapsArgs of csrc/step_maps.cu."""

    _fields_ = [("cached", c_void_p), ("q_len", c_void_p), ("n_seqs", c_int), ("pages", c_void_p)] + [(name, c_int) for name in (
        "n_pages", "n_rows", "page_tokens", "group", "tile_rows", "few_rows", "max_blocks", "n_writes", "n_tiles")] + [(name, c_void_p) for name in (
            "seq_q_start", "seq_q_len", "seq_kv_len", "order", "positions", "row_seq", "slots", "block_table", "write_seq", "write_block",
            "tile_seq", "tile_index")]


class StepLists(ctypes.Structure):
    """struct StepLists of csrc/cache8.cuh."""

    _fields_ = [(name, c_void_p) for name in ("seq_q_start", "seq_q_len", "seq_kv_len", "write_seq", "write_block", "order",
                                              "tile_seq", "tile_index")] + [(name, c_int) for name in ("n_seqs", "n_writes", "n_tiles")]


class StepMaps:
    """Device arrays for steps of at most `max_rows` rows and `max_seqs` requests of at most `max_blocks` pages of `page_tokens`
    positions (a multiple of 16).  Every array lies at an address of its own that `build` keeps, so graphs may hold them.

    `group` query heads share a key/value head: a request with more than `few_rows` packed rows (tokens x group) is cut into tiles
    of `tile_rows`.

    A `StepMaps` serves one stream: `build` writes what the kernels of the step before read, and waits for them in its stream's order.

    After `build`, for that step (S requests, T rows):

    * seq_q_start, seq_q_len, seq_kv_len, order  int32 [S]: first row, new tokens, length after the step; the requests, longest first
    * positions, row_seq  int32 [T]; slots int64 [T] = page * page_tokens + place in the page, -1 where no page is held
    * block_table  int32 [S, max_blocks], -1 behind a request's last page
    * write_seq, write_block  int32: the blocks of 16 positions that the step writes (request, number of the block in it)
    * tile_seq, tile_index  int32: the tiles

    The lists of blocks and tiles are as long as a step of that many rows and requests can make them; entries behind the
    last are -1 and 0.  Rows behind the last request have position 0, request -1 and slot -1."""

    def __init__(self, max_rows: int, max_seqs: int, max_blocks: int, page_tokens: int, *, group: int = 1, tile_rows: int = 128,
                 few_rows: int = 16, device="cuda"):
        if min(max_rows, max_seqs, max_blocks, page_tokens, group, tile_rows) <= 0 or few_rows < 0:
            raise KernelLaunchError("step maps: sizes must be positive")
        if page_tokens % SCALE_TOKENS:
            raise KernelLaunchError(f"step maps: pages of {page_tokens} positions are not supported (a multiple of {SCALE_TOKENS})")
        if max_seqs > int(lib().llm_step_maps_max_seqs()):
            raise KernelLaunchError(f"step maps: {max_seqs} requests in one step, the kernel takes {int(lib().llm_step_maps_max_seqs())}")
        if max_rows * group >= 1 << 31 or max_blocks * page_tokens >= 1 << 31:
            raise KernelLaunchError("step maps: rows and positions are counted in 32 bits")
        self.max_rows, self.max_seqs, self.max_blocks, self.page_tokens = max_rows, max_seqs, max_blocks, page_tokens
        self.group, self.tile_rows, self.few_rows = group, tile_rows, few_rows
        self.device = torch.device(device)
        i32 = dict(dtype=torch.int32, device=self.device)
        writes, tiles = self._list_lengths(max_rows, max_seqs)
        self._seqs = torch.zeros(4, max_seqs, **i32)
        self._rows = torch.zeros(2, max_rows, **i32)
        self._slots = torch.full((max_rows,), -1, dtype=torch.int64, device=self.device)
        self._table = torch.full((max_seqs, max_blocks), -1, **i32)
        self._writes = torch.full((2, writes), -1, **i32)
        self._tiles = torch.full((2, tiles), -1, **i32)
        self.device = self._table.device
        self.index = self.device.index
        self.table = self._table                       # the block tables whole, at the address that `block_table` keeps
        self._args = MapsArgs(0, 0, 0, 0, 0, 0, page_tokens, group, tile_rows, few_rows, max_blocks, 0, 0,
                              *(t.data_ptr() for t in (*self._seqs, *self._rows, self._slots, self._table, *self._writes, *self._tiles)))
        self._args_at = ctypes.addressof(self._args)
        self._shape = None
        self.longest = self.shortest = 0

    def _list_lengths(self, rows: int, seqs: int):
        return min(rows, rows // SCALE_TOKENS + 2 * seqs), rows * self.group // self.tile_rows + seqs

    def _arrays(self, seqs: int, rows: int) -> None:
        self.n_seqs, self.n_rows = seqs, rows
        self.n_writes, self.n_tiles = self._list_lengths(rows, seqs)
        self.seq_q_start, self.seq_q_len, self.seq_kv_len, self.order = (t[:seqs] for t in self._seqs)
        self.positions, self.row_seq = (t[:rows] for t in self._rows)
        self.slots, self.block_table = self._slots[:rows], self._table[:seqs]
        self.write_seq, self.write_block = (t[:self.n_writes] for t in self._writes)
        self.tile_seq, self.tile_index = (t[:self.n_tiles] for t in self._tiles)
        self._shape = (seqs, rows)
        a = self._args
        a.n_seqs, a.n_rows, a.n_writes, a.n_tiles = seqs, rows, self.n_writes, self.n_tiles
        self._lists = StepLists(*(t.data_ptr() for t in (self.seq_q_start, self.seq_q_len, self.seq_kv_len, self.write_seq,
                                                         self.write_block, self.order, self.tile_seq,
                                                         self.tile_index)),
                                seqs, self.n_writes, self.n_tiles)
        self.lists = ctypes.addressof(self._lists)      # what the launchers of the step's kernels hand on

    def build(self, cached: torch.Tensor, q_len: torch.Tensor, pages: torch.Tensor, n_rows: int, longest: int, shortest: int,
              stream=None) -> None:
        """`cached`, `q_len` (int32 [S]): every request's positions before the step and its new ones; `cached` < 0: an idle row that pads
        a decode step, which holds nothing.  `pages` (int32): request after request, the ceil(length after the step /
        page_tokens) pages of its blocks, -1 for one that was given back.  `n_rows`: the sum of q_len.  `longest`, `shortest`:
        the most and the fewest new tokens that a request of the step brings; they decide which kernels of the step
        are launched and are the only lengths that the host has to know."""
        seqs = cached.numel()
        if not 0 < seqs <= self.max_seqs or q_len.numel() != seqs:
            raise KernelLaunchError(f"step maps: {seqs} cached lengths and {q_len.numel()} new ones, made for {self.max_seqs} requests")
        if not 0 < n_rows <= self.max_rows:
            raise KernelLaunchError(f"step maps: {n_rows} rows in one step, made for {self.max_rows}")
        if not 0 < shortest <= longest <= n_rows:
            raise KernelLaunchError(f"step maps: requests of {shortest} to {longest} new tokens in a step of {n_rows}")
        for t in (cached, q_len, pages):
            if t.dtype != torch.int32 or t.get_device() != self.index or not t.is_contiguous():
                raise KernelLaunchError(f"step maps: lengths and pages must be contiguous int32 on {self.device}")
        if self.index != torch.cuda.current_device():
            raise KernelLaunchError(f"step maps: made for {self.device}, the current device is cuda:{torch.cuda.current_device()}")
        if self._shape != (seqs, n_rows):
            self._arrays(seqs, n_rows)
        self.longest, self.shortest = int(longest), int(shortest)
        a = self._args
        a.cached, a.q_len, a.pages, a.n_pages = cached.data_ptr(), q_len.data_ptr(), pages.data_ptr(), pages.numel()
        _check(lib().llm_step_maps(self._args_at, stream if stream is not None else stream_handle()), "step_maps")
