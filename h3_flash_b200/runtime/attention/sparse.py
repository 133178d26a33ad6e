"""Block-sparse attention on B200: every block of queries attends to its own list of key blocks.

``select_key_blocks`` picks the lists by a cheap score (the product of the blocks' mean query
and mean key), ``block_sparse_attention`` attends over given lists, and ``sparse_attention`` /
``packed_sparse_attention`` do both: the sparse counterparts of ``dense.attention_bshd`` and
``dense.packed_attention``, with the same [B, S, H, D] views and packed buffer. The reference's
attention is dense (src/h3_flash/runtime/parallel/packed_ulysses.py:201-209).

A query block is 128 or 256 rows, a key block 64 or 128. Query heads may share key heads
(``heads`` a multiple of ``kv_heads``). ``q_lens`` / ``k_lens`` (int32 [B] on the device) give
the rows of each batch entry that exist; what a padded batch holds behind them is never read
into a result. All ops are inference only and run on the current stream of the tensors' device.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from ..._torch import call, call_on, check_inputs, require_cuda
from .dense import HEAD_DIM

BLOCK_Q = (128, 256)
BLOCK_K = (64, 128)
HEAD_DIMS = (64, 128)
_TYPES = (torch.bfloat16, torch.float16)


def _check_shapes(op: str, q: torch.Tensor, k: torch.Tensor, block_q: int, block_k: int) -> None:
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"{op}: expected [batch, seq, heads, head_dim] tensors")
    b, _, h, d = q.shape
    kb, _, hk, kd = k.shape
    if kb != b or kd != d:
        raise ValueError(f"{op}: q {tuple(q.shape)} and k {tuple(k.shape)} disagree")
    if d not in HEAD_DIMS:
        raise RuntimeError(f"{op}: head_dim must be one of {HEAD_DIMS}, got {d}")
    if block_q not in BLOCK_Q or block_k not in BLOCK_K:
        raise ValueError(f"{op}: block_q must be one of {BLOCK_Q} and block_k one of {BLOCK_K}, got "
                         f"{block_q} and {block_k}")
    if hk == 0 or h % hk:
        raise ValueError(f"{op}: {h} query heads are not a multiple of {hk} key heads")


def _strides(op: str, name: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(batch, row, head) strides of a view the kernels can address."""

    *strides, last = t.stride()
    if last != 1:
        raise ValueError(f"{op}: {name}: head_dim must be contiguous")
    if t.data_ptr() % 16:
        raise ValueError(f"{op}: {name}: base address must be 16-byte aligned")
    return strides


def _side_tensor(op: str, name: str, t: torch.Tensor | None, dtype: torch.dtype, shape: tuple[int, ...],
                 device: torch.device) -> torch.Tensor | None:
    """A contiguous int32 or bool argument on the right device, or None."""

    if t is None:
        return None
    require_cuda(op, t)
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        raise ValueError(f"{op}: {name} must be a {dtype} tensor of shape {shape} on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t.contiguous()


def _opt(t: torch.Tensor | None) -> int | None:
    return t.data_ptr() if t is not None else None


@functools.lru_cache(maxsize=256)
def _bytes(name: str, *shape: int) -> int:
    """Workspace bytes of a shape on B200."""

    value = ctypes.c_int64(0)
    call(name, *shape, ctypes.byref(value))
    return value.value


def select_key_blocks(q: torch.Tensor, k: torch.Tensor, top_k: int, *, block_q: int = 128, block_k: int = 128,
                      q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None,
                      keep: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``top_k`` key blocks (all of them if there are fewer) of every query block, by the
    product of the block's mean query with the block's mean key.

    q [B, Sq, H, D], k [B, Sk, Hk, D]. ``keep``: bool [ceil(Sk / block_k)], blocks that every
    list holds before any other (audio or text rows, say). Returns ``indices`` int32
    [B, H, ceil(Sq / block_q), top_k], ascending and -1 behind the last, and ``counts`` int32
    [B, H, ceil(Sq / block_q)]. Scores are compared in 64 bits, ties go to the lowest index:
    equal inputs give equal lists on any device and in any batch."""

    op = "select_key_blocks"
    dtype = check_inputs(op, _TYPES, (q, k))
    _check_shapes(op, q, k, block_q, block_k)
    (b, sq, h, d), (_, sk, hk, _) = q.shape, k.shape
    nq, nk = -(-sq // block_q), -(-sk // block_k)
    if isinstance(top_k, bool) or not isinstance(top_k, int) or top_k < 1:
        raise ValueError(f"{op}: top_k must be a positive integer, got {top_k!r}")
    top_k = min(top_k, max(nk, 1))
    q_lens = _side_tensor(op, "q_lens", q_lens, torch.int32, (b,), q.device)
    k_lens = _side_tensor(op, "k_lens", k_lens, torch.int32, (b,), q.device)
    keep = _side_tensor(op, "keep", keep, torch.bool, (nk,), q.device)
    if b and sq and h and not sk:
        raise ValueError(f"{op}: empty key sequence")
    indices = torch.empty((b, h, nq, top_k), dtype=torch.int32, device=q.device)
    counts = torch.empty((b, h, nq), dtype=torch.int32, device=q.device)
    if counts.numel() == 0:
        return indices, counts
    need = _bytes("h3b_select_key_blocks_workspace_size", b, sq, sk, h, hk, d, block_q, block_k)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    call_on(q, "h3b_select_key_blocks", indices.data_ptr(), counts.data_ptr(), q.data_ptr(), k.data_ptr(), b, sq, sk,
            h, hk, d, block_q, block_k, top_k, *_strides(op, "q", q), *_strides(op, "k", k), _opt(q_lens),
            _opt(k_lens), _opt(keep), dtype, ws.data_ptr(), need)
    return indices, counts


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, indices: torch.Tensor,
                           counts: torch.Tensor | None = None, *, block_q: int = 128, block_k: int = 128,
                           softmax_scale: float | None = None, q_lens: torch.Tensor | None = None,
                           k_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
                           return_lse: bool = False):
    """softmax(q k^T * scale) v over the keys of every query block's listed key blocks.

    q [B, Sq, H, D], k and v [B, Sk, Hk, D] (strided views with a contiguous, 16-byte aligned
    head_dim of 64 or 128; bf16 or fp16). ``indices`` int32 [B, H, ceil(Sq / block_q), n]: the
    first ``counts`` entries of a list count (all of them without ``counts``), in any order. An
    entry outside the key blocks adds nothing, an entry that is there twice counts twice. Query
    rows that have no key, and rows behind ``q_lens``, get zeros (lse -inf). Returns
    [B, Sq, H, D] (``out`` if given), and with ``return_lse`` the fp32 [B, H, Sq] logarithms of
    the softmax sums."""

    op = "block_sparse_attention"
    dtype = check_inputs(op, _TYPES, (q, k, v) if out is None else (q, k, v, out))
    _check_shapes(op, q, k, block_q, block_k)
    if v.shape != k.shape:
        raise ValueError(f"{op}: k {tuple(k.shape)} and v {tuple(v.shape)} disagree")
    (b, sq, h, d), (_, sk, hk, _) = q.shape, k.shape
    nq = -(-sq // block_q)
    if not isinstance(indices, torch.Tensor) or indices.dim() != 4:
        raise ValueError(f"{op}: indices must be [batch, heads, query blocks, entries]")
    entries = indices.shape[3]
    indices = _side_tensor(op, "indices", indices, torch.int32, (b, h, nq, entries), q.device)
    counts = _side_tensor(op, "counts", counts, torch.int32, (b, h, nq), q.device)
    q_lens = _side_tensor(op, "q_lens", q_lens, torch.int32, (b,), q.device)
    k_lens = _side_tensor(op, "k_lens", k_lens, torch.int32, (b,), q.device)
    if out is None:
        out = torch.empty((b, sq, h, d), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise ValueError(f"{op}: out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
    lse = torch.empty((b, h, sq), dtype=torch.float32, device=q.device) if return_lse else None
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(d)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{op}: softmax_scale must be positive and finite, got {scale}")
    if out.numel() and (sk == 0 or entries == 0):
        out.zero_()
        if lse is not None:
            lse.fill_(-math.inf)
    elif out.numel():
        need = _bytes("h3b_block_sparse_attention_workspace_size", b, sq, h, d, block_k, entries)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        call_on(q, "h3b_block_sparse_attention", out.data_ptr(), _opt(lse), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                indices.data_ptr(), _opt(counts), entries, b, sq, sk, h, hk, d, block_q, block_k,
                *_strides(op, "q", q), *_strides(op, "k", k), *_strides(op, "v", v), *_strides(op, "out", out),
                _opt(q_lens), _opt(k_lens), scale, dtype, _opt(ws), need)
    return (out, lse) if return_lse else out


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, top_k: int, *, block_q: int = 128,
                     block_k: int = 128, softmax_scale: float | None = None, q_lens: torch.Tensor | None = None,
                     k_lens: torch.Tensor | None = None, keep: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, return_lse: bool = False):
    """``select_key_blocks`` and then ``block_sparse_attention`` over its lists."""

    indices, counts = select_key_blocks(q, k, top_k, block_q=block_q, block_k=block_k, q_lens=q_lens,
                                        k_lens=k_lens, keep=keep)
    return block_sparse_attention(q, k, v, indices, counts, block_q=block_q, block_k=block_k,
                                  softmax_scale=softmax_scale, q_lens=q_lens, k_lens=k_lens, out=out,
                                  return_lse=return_lse)


def packed_sparse_attention(packed: torch.Tensor, top_k: int, head_dim: int = HEAD_DIM, *, block_q: int = 128,
                            block_k: int = 128, softmax_scale: float | None = None,
                            keep: torch.Tensor | None = None, out: torch.Tensor | None = None,
                            return_lse: bool = False):
    """``sparse_attention`` over the packed receive buffer ``[S, hl, 3*D]`` (q | k | v per
    head), read in place. Returns ``[S, hl, D]`` (and lse ``[hl, S]``)."""

    if packed.dim() != 3 or packed.shape[-1] != 3 * head_dim:
        raise ValueError(f"packed attention expects [S, hl, 3*{head_dim}], got {tuple(packed.shape)}")
    if packed.stride(-1) != 1 or packed.stride(-2) != 3 * head_dim:
        packed = packed.contiguous()
    q, k, v = (packed[..., i * head_dim : (i + 1) * head_dim].unsqueeze(0) for i in range(3))
    if out is None:
        out = torch.empty((packed.shape[0], packed.shape[1], head_dim), dtype=packed.dtype, device=packed.device)
    result = sparse_attention(q, k, v, top_k, block_q=block_q, block_k=block_k, softmax_scale=softmax_scale,
                              keep=keep, out=out.unsqueeze(0), return_lse=return_lse)
    return (out, result[1][0]) if return_lse else out
