"""Attention over an 8-bit cache on MI355X: what a decoder layer does between its qkv projection and its
output projection.

* `norm_rope`: per-head RMS norms of queries and keys and the position rotation, one pass;
* `append`: keys and values into a cache of 8-bit codes (int8 or e4m3) with a scale for each block of 64 tokens
  and head, norms and rotation on the way where asked, queries with them: one launch;
* `read`: the last tokens of a cache back in fp32, fp16 or bf16;
* `attend`: softmax(q K^T) V over the cache, from one token of one sequence to prompts.

A sequence's blocks stand in its row of a table, anywhere in the pool (`new_cache`). Functions return None when
the library declines a shape or dtype; every check happens before a launch, and none waits for the GPU.

Calls whose arguments fit as they are go through `_bind` (csrc/python/bind.cpp); what is below makes the others.
"""
import math
from typing import NamedTuple

import torch

from . import _bind, _lib
from ._torch import DTYPES, ptr, require_cuda, stream

BLOCK = 64
FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}


class Cache(NamedTuple):
    """A pool of blocks: codes of keys [blocks, heads, 64, dim] and of values [blocks, heads, dim, 64] (int8 or
    float8_e4m3fn), scales [blocks, heads] fp32 of either."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class Batch(NamedTuple):
    """The sequences of a call: `table` [sequences, width] int32 block numbers, `lengths` [sequences] int32 tokens in
    the cache with the call's own, `starts` [sequences + 1] int32 first rows. `max_rows` and `max_length` bound the
    rows and tokens of a sequence (host numbers: a captured call follows the tensors up to them)."""
    table: torch.Tensor
    lengths: torch.Tensor
    starts: torch.Tensor
    max_rows: int
    max_length: int


def new_cache(blocks, heads, dim, dtype=torch.int8, device="cuda"):
    """An empty pool. A block's scale is written when its first token is."""
    if dtype not in FORMATS:
        raise ValueError("a cache holds int8 or float8_e4m3fn codes")
    return Cache(torch.zeros((blocks, heads, BLOCK, dim), dtype=torch.int8, device=device).view(dtype),
                 torch.zeros((blocks, heads, dim, BLOCK), dtype=torch.int8, device=device).view(dtype),
                 torch.zeros((blocks, heads), device=device), torch.zeros((blocks, heads), device=device))


def turns(dim=None, base=10000.0, inv_freq=None, device="cuda"):
    """The rotation's table [dim / 2]: each pair's turns a position as a fraction of 2^64 (an int64 tensor of those
    bits). `inv_freq` (radians a position) for rescaled frequencies, else base ** (-2 i / dim)."""
    if inv_freq is None:
        inv_freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    bits = [round(math.fmod(float(f) / (2 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64) for f in inv_freq]
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64, device=device)


def _heads(x, what):
    """x [rows, heads, dim] as the kernels take it, and its strides: rows and heads on 16 bytes, else copied. The stride of
    a single row or head counts for nothing: slices keep odd ones there, and contiguous() leaves them as they are."""
    if x.dim() != 3:
        raise ValueError(f"{what} must be [rows, heads, dim]")
    rows, heads, dim = x.shape
    row, head, last = x.stride()
    row, head = row if rows > 1 else heads * dim, head if heads > 1 else dim
    step = 16 // x.element_size()
    if last != 1 or row % step or head % step or x.data_ptr() & 15:
        x = x.contiguous()
        if x.data_ptr() & 15:
            x = x.clone()
        row, head = heads * dim, dim
    return x, row, head


def _weight(w, dim):
    if w is not None and (w.dtype is not torch.float32 or w.shape != (dim,) or not w.is_contiguous()):
        raise ValueError(f"a norm's weight must be {dim} contiguous fp32 values")
    return ptr(w)


def _turn(positions, table, rows):
    if table is None:
        return None, None, 0
    if table.dtype is not torch.int64 or not table.is_contiguous() or table.dim() != 1:
        raise ValueError("turns must be a contiguous int64 table (attention.turns)")
    if positions is None or positions.dtype is not torch.int32 or positions.shape != (rows,) or not positions.is_contiguous():
        raise ValueError(f"a rotation needs {rows} contiguous int32 positions")
    return positions.data_ptr(), table.data_ptr(), 2 * table.shape[0]


def _cache(c):
    """(pointers and format, blocks, heads, dim) of a pool whose tensors fit each other."""
    k, v, ks, vs = c
    blocks, heads, size, dim = k.shape
    if (size != BLOCK or v.shape != (blocks, heads, dim, BLOCK) or ks.shape != (blocks, heads) or vs.shape != ks.shape
            or v.dtype is not k.dtype or ks.dtype is not torch.float32 or vs.dtype is not torch.float32
            or not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous())):
        raise ValueError("a cache is k [blocks, heads, 64, dim], v [blocks, heads, dim, 64] and fp32 scales [blocks, heads]")
    require_cuda(k, v, ks, vs)
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), FORMATS.get(k.dtype, -1), blocks, heads, dim)


def _batch(b):
    """(table, width, lengths, starts, sequences) of a call's sequences."""
    table, lengths, starts = b.table, b.lengths, b.starts
    n = lengths.shape[0]
    if (table.dtype is not torch.int32 or lengths.dtype is not torch.int32 or starts.dtype is not torch.int32
            or table.dim() != 2 or table.shape[0] != n or starts.shape != (n + 1,)
            or not (table.is_contiguous() and lengths.is_contiguous() and starts.is_contiguous())):
        raise ValueError("a batch is int32 table [sequences, width], lengths [sequences] and starts [sequences + 1]")
    require_cuda(table, lengths, starts)
    return table.data_ptr(), table.shape[1], lengths.data_ptr(), starts.data_ptr(), n


def norm_rope(q, k, positions=None, turns=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, factor=1.0):
    """(q, k) [rows, heads, dim] normed over each head (where a weight is given) and turned by their positions
    (where `turns` is), computed in fp32 and rounded once to their dtype; None if declined."""
    out = _bind.norm_rope(q, k, positions, turns, q_weight, k_weight, eps, interleaved, factor)
    if out is not NotImplemented:
        return out
    require_cuda(q, k, positions, turns, q_weight, k_weight)
    q, q_row, q_head = _heads(q, "q")
    k, k_row, k_head = _heads(k, "k")
    rows, heads, dim = q.shape
    kv = k.shape[1]
    if k.shape != (rows, kv, dim) or k.dtype is not q.dtype:
        raise ValueError(f"k {tuple(k.shape)} beside q {tuple(q.shape)}")
    at, table, rot = _turn(positions, turns, rows)
    q_out = torch.empty((rows, heads, dim), dtype=q.dtype, device=q.device)
    k_out = torch.empty((rows, kv, dim), dtype=q.dtype, device=q.device)
    rc = _lib.lib().ishz_norm_rope(q.data_ptr(), q_row, q_head, heads, k.data_ptr(), k_row, k_head, kv,
                                   DTYPES.get(q.dtype, -1), rows, dim, at, table, rot, int(interleaved), factor,
                                   _weight(q_weight, dim), _weight(k_weight, dim), eps, q_out.data_ptr(),
                                   k_out.data_ptr(), stream())
    return (q_out, k_out) if _lib.check(rc, "norm_rope") else None


def append(k, v, cache, batch, q=None, positions=None, turns=None, q_weight=None, k_weight=None, eps=1e-6,
           interleaved=False, factor=1.0):
    """Writes k and v [rows, heads, dim] behind what the batch's sequences hold (rows past a sequence's table nowhere),
    k normed and turned first as in `norm_rope` where asked. Returns q [rows, q heads, dim] normed and turned (True where there is no q); None if
    declined."""
    out = _bind.append(k, v, cache, batch, q, positions, turns, q_weight, k_weight, eps, interleaved, factor)
    if out is not NotImplemented:
        return out
    require_cuda(k, v, q, positions, turns, q_weight, k_weight)
    pointers = _cache(cache)
    heads, dim = pointers[6:]
    rows = k.shape[0]
    if k.shape != (rows, heads, dim) or v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} into a cache of {heads} heads of {dim}")
    k, k_row, k_head = _heads(k, "k")
    v, v_row, v_head = _heads(v, "v")
    at, table, rot = _turn(positions, turns, rows)
    blocks, width, lengths, starts, sequences = _batch(batch)
    q_out, q_row, q_head, q_heads = None, 0, 0, 0
    if q is not None:
        q, q_row, q_head = _heads(q, "q")
        q_heads = q.shape[1]
        if q.shape != (rows, q_heads, dim) or q.dtype is not k.dtype:
            raise ValueError(f"q {tuple(q.shape)} beside k {tuple(k.shape)}")
        q_out = torch.empty((rows, q_heads, dim), dtype=q.dtype, device=q.device)
    rc = _lib.lib().ishz_kv_append(k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head, DTYPES.get(k.dtype, -1), rows,
                                   *pointers, blocks, width, lengths, starts, sequences, batch.max_rows, ptr(q), q_row,
                                   q_head, q_heads, at, table, rot, int(interleaved), factor, _weight(q_weight, dim),
                                   _weight(k_weight, dim), eps, ptr(q_out), stream())
    if not _lib.check(rc, "kv_append"):
        return None
    return True if q is None else q_out


def read(cache, batch, tail=None, dtype=torch.float16):
    """(k, v) [sequences, tail, heads, dim]: the last `tail` tokens (None: max_length) of each sequence, zeros where
    it has fewer or its table ends before; None if declined."""
    out = _bind.read(cache, batch, tail, dtype)
    if out is not NotImplemented:
        return out
    pointers = _cache(cache)
    heads, dim = pointers[6:]
    table, width, lengths, _, sequences = _batch(batch)
    tail = batch.max_length if tail is None else tail
    if tail < 0:
        raise ValueError("a tail of a negative length")
    k = torch.empty((sequences, tail, heads, dim), dtype=dtype, device=cache.k.device)
    v = torch.empty((sequences, tail, heads, dim), dtype=dtype, device=cache.k.device)
    rc = _lib.lib().ishz_kv_read(*pointers, table, width, lengths, sequences, tail, DTYPES.get(dtype, -1), k.data_ptr(),
                                 v.data_ptr(), stream())
    return (k, v) if _lib.check(rc, "kv_read") else None


def attend(q, cache, batch, scale=None, causal=True, window=0):
    """[rows, q heads, dim]: attention of the batch's rows over their sequences' tokens in the cache, weights
    softmax(scale q K^T) (`scale` None: dim ** -0.5; q fp16 or bf16). Causal: a row sees the tokens up to its own
    (`window` > 0: the last `window` of them); else all of its sequence's. A row that sees none gives zeros. Rows of no
    sequence, and those of a sequence beyond `max_rows`, are not written: they hold whatever the memory held. The work is
    divided by the most rows of a sequence: prompts and single tokens are faster in a call each. None if declined."""
    out = _bind.attend(q, cache, batch, scale, causal, window)
    if out is not NotImplemented:
        return out
    require_cuda(q)
    pointers = _cache(cache)
    heads, dim = pointers[6:]
    q, q_row, q_head = _heads(q, "q")
    rows, q_heads, width_q = q.shape
    if width_q != dim:
        raise ValueError(f"q of heads of {width_q} over a cache of heads of {dim}")
    table, width, lengths, starts, sequences = _batch(batch)
    L = _lib.lib()
    out = torch.empty((rows, q_heads, dim), dtype=q.dtype, device=q.device)
    ws_bytes = L.ishz_kv_attend_workspace_size(rows, q_heads, heads, dim, sequences, batch.max_rows, batch.max_length)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    rc = L.ishz_kv_attend(q.data_ptr(), q_row, q_head, q_heads, DTYPES.get(q.dtype, -1), rows, *pointers, table, width,
                          lengths, starts, sequences, batch.max_rows, batch.max_length,
                          dim ** -0.5 if scale is None else scale, int(causal), window, out.data_ptr(), ptr(ws), ws_bytes,
                          stream())
    return out if _lib.check(rc, "kv_attend") else None
