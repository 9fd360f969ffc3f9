"""Host side of a paged KV cache: one layer's pages, the batch of sequences that live in them, and the three operators over them.

    append            the projected rows of a step: queries and keys rotated to their positions, keys and values stored in the pages
    attention         of a ragged batch over its pages: single tokens, drafts, prompts, all of them in one call
    prefix attention  the same for a batch that shares the pages of a long prefix, which are read once for all of it (head_dim 64 and 128; 256: once
                      per 16 rows)

The reference keeps one contiguous cache per sequence (its ROPE, SET_ROWS and FLASH_ATTN_EXT nodes, adapters/llama/ggml-ameva/ggml-ameva.cpp:
4008-4111, 5140-5285); a server of several users needs their keys in pages that are handed out one at a time. Everything that changes from
step to step (tables, lengths, the prefix) is read on the device, so that a recorded batch can be replayed for every step whose numbers stay
within the announced maxima.

All functions record dispatches into a `runtime.Batch`; arguments are checked by the library's launchers, which the batch reports when it is
submitted or instantiated. What the device finds wrong in the step's numbers (a page that is none of the cache's, a length past the
table) is left out and counted in `status`: two 32-bit words, the count (to be zeroed by the caller; a page counts for every tile that
meets it) and the lowest `node` number that met one (to be set to 0xFFFFFFFF).
"""
from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Optional, Tuple

from . import runtime as rt


def _bits(v: float) -> int:
    return struct.unpack("<I", struct.pack("<f", float(v)))[0]


@dataclass
class Cache:
    """One layer's keys and values, f16, in pages of `page_size` tokens, two ranges that do not meet. layout "token": [page][token][head][head_dim], a token's heads
    beside one another; "head": [page][head][token][head_dim], a head's tokens beside one another (longer runs for the attention)."""
    k: rt.Buffer
    v: rt.Buffer
    n_pages: int
    page_size: int
    kv_heads: int
    head_dim: int
    layout: str = "token"

    @property
    def strides(self) -> Tuple[int, int, int]:
        """Elements between two pages, two tokens of a page, two heads."""
        page = self.page_size * self.kv_heads * self.head_dim
        if self.layout == "token":
            return page, self.kv_heads * self.head_dim, self.head_dim
        if self.layout == "head":
            return page, self.head_dim, self.page_size * self.head_dim
        raise ValueError(f"layout {self.layout!r} is neither 'token' nor 'head'")

    @staticmethod
    def nbytes(n_pages: int, page_size: int, kv_heads: int, head_dim: int) -> int:
        """Bytes of the keys (and as many of the values)."""
        return 2 * n_pages * page_size * kv_heads * head_dim


@dataclass
class Sequences:
    """A batch. table: i32 [n_seqs][table_stride], the pages of every sequence; q_start: i32 [n_seqs + 1], sequence s has the rows
    q_start[s] .. q_start[s + 1] - 1 of the step (not decreasing); kv_len: i32 [n_seqs], the keys of every sequence, this step's among them. rows, max_q and
    max_kv announce the most rows of a step, of one sequence, and the most keys of one: launches are sized by them."""
    table: rt.Buffer
    q_start: rt.Buffer
    kv_len: rt.Buffer
    n_seqs: int
    table_stride: int
    rows: int
    max_q: int
    max_kv: int


@dataclass
class Rope:
    """The rotation's parameters, as of ameva_rope: angle = position * theta_scale^j of pair j (divided by its frequency factor), YaRN
    mixing between the pairs `corr`. neox: pairs (j, j + n_dims / 2) instead of (2 j, 2 j + 1)."""
    n_dims: int
    theta_scale: float
    neox: bool = False
    freq_scale: float = 1.0
    ext_factor: float = 0.0
    attn_factor: float = 1.0
    corr: Tuple[float, float] = (0.0, 0.0)


def record_append(batch: rt.Batch, cache: Cache, seqs: Sequences, q: rt.Buffer, k: rt.Buffer, v: rt.Buffer, q_out: rt.Buffer,
                  status: rt.Buffer, *, heads: int, rope: Rope, positions: Optional[rt.Buffer] = None, factors: Optional[rt.Buffer] = None,
                  q_stride: Optional[int] = None, k_stride: Optional[int] = None, v_stride: Optional[int] = None,
                  q_out_stride: Optional[int] = None, node: int = 0) -> None:
    """q f32 [rows][heads x head_dim], k and v f32 [rows][kv_heads x head_dim] (strides in floats: the three may be column ranges of one
    product) -> q_out f16 rotated, k rotated and v in the cache. positions: i32 [rows] instead of the keys' places, which are counted from
    a sequence's first own key: behind a shared prefix they have to be given, the prefix's number of keys added. factors: f32
    [n_dims / 2]. Rows behind the last sequence are left as they are; tokens whose place has no page are not written, and counted."""
    D, w, kw = cache.head_dim, heads * cache.head_dim, cache.kv_heads * cache.head_dim
    flags = (1 if positions is not None else 0) | (2 if factors is not None else 0)
    push = [D, heads, cache.kv_heads, seqs.n_seqs, seqs.rows, cache.page_size, cache.n_pages, seqs.table_stride, *cache.strides,
            w if q_stride is None else q_stride, kw if k_stride is None else k_stride, kw if v_stride is None else v_stride,
            w if q_out_stride is None else q_out_stride, rope.n_dims, int(rope.neox), flags, _bits(rope.theta_scale), _bits(rope.freq_scale),
            _bits(rope.ext_factor), _bits(rope.attn_factor), _bits(rope.corr[0]), _bits(rope.corr[1]), node]
    batch.dispatch(batch.ctx.kernel("ameva_paged_append"),
                   [q, k, v, seqs.table, seqs.q_start, seqs.kv_len, positions or seqs.kv_len, factors or seqs.kv_len, q_out, cache.k, cache.v, status],
                   push)


def _attention_push(cache: Cache, seqs: Sequences, heads, scale, softcap, f16_out, q_stride, dst_stride):
    w = heads * cache.head_dim
    return [cache.head_dim, heads, cache.kv_heads, seqs.n_seqs, seqs.rows, seqs.max_q, seqs.max_kv, cache.page_size, cache.n_pages,
            seqs.table_stride, *cache.strides, w if q_stride is None else q_stride, w if dst_stride is None else dst_stride, int(f16_out),
            _bits(scale), _bits(softcap)]


def record_attention(batch: rt.Batch, cache: Cache, seqs: Sequences, q: rt.Buffer, dst: rt.Buffer, scratch: rt.Buffer, status: rt.Buffer, *,
                     heads: int, scale: float, softcap: float = 0.0, window: int = 0, f16_out: bool = False, q_stride: Optional[int] = None,
                     dst_stride: Optional[int] = None, node: int = 0) -> None:
    """q f16 [rows][heads x head_dim] -> dst f32 (f16_out: the same, rounded to f16 once) [rows][heads x head_dim]. Query j of a sequence's n sees the keys up to its
    own place kv_len - n + j (window: that many of them); one that sees none is zero, rows behind the last sequence are left as they
    are. scratch: see `scratch_bytes`; a smaller one means fewer CTAs, not another result than rounding makes. Launches behind one another
    may share it, batches that run at the same time may not."""
    push = _attention_push(cache, seqs, heads, scale, softcap, f16_out, q_stride, dst_stride) + [window, node]
    batch.dispatch(batch.ctx.kernel("ameva_paged_attn"), [q, cache.k, cache.v, seqs.table, seqs.q_start, seqs.kv_len, dst, scratch, status], push)


def record_prefix_attention(batch: rt.Batch, cache: Cache, seqs: Sequences, q: rt.Buffer, dst: rt.Buffer, scratch: rt.Buffer,
                            status: rt.Buffer, *, prefix: rt.Buffer, max_prefix: int, heads: int, scale: float, softcap: float = 0.0,
                            f16_out: bool = False, q_stride: Optional[int] = None, dst_stride: Optional[int] = None, node: int = 0) -> None:
    """`record_attention` for sequences whose keys begin with a prefix that all of them share. prefix: i32 [1 + pages], its number of keys
    (at most max_prefix) and its pages; `seqs` describes the keys behind it, which are appended with the positions that they have behind
    it (`record_append`: positions). The rows begin at 0, and a batch with a sequence that does not
    fit its numbers is left out altogether."""
    push = _attention_push(cache, seqs, heads, scale, softcap, f16_out, q_stride, dst_stride) + [max_prefix, node]
    batch.dispatch(batch.ctx.kernel("ameva_paged_prefix_attn"),
                   [q, cache.k, cache.v, seqs.table, seqs.q_start, seqs.kv_len, dst, scratch, status, prefix], push)


def scratch_bytes(ctx: rt.Context, seqs: Sequences, *, heads: int, head_dim: int, prefix: bool = False, sms: Optional[int] = None) -> int:
    """Bytes of scratch with which the attention of this batch takes the whole GPU of `ctx` (or `sms` SMs): per SM two row tiles of 16 rows of
    eight KV heads and two of 256 rows, and for a shared prefix the rows' results over their own keys."""
    sms = ctx.sm_count if sms is None else sms
    row = (head_dim + 4) * 4
    own = seqs.rows * heads * row + 256 if prefix else 0
    return own + sms * (2 * (8 * 16 + 256) * row + 128) + 8192
