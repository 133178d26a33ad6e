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
from dataclasses import dataclass
from typing import Any

import torch

from ..._torch import call, call_on, check_inputs, require_cuda, scratch
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


def _view(op: str, name: str, t: torch.Tensor) -> tuple[int, ...]:
    """(address, batch stride, row stride, head stride) of a view the kernels can address."""

    batch, row, head, last = t.stride()
    address = t.data_ptr()
    if last != 1:
        raise ValueError(f"{op}: {name}: head_dim must be contiguous")
    if address % 16:
        raise ValueError(f"{op}: {name}: base address must be 16-byte aligned")
    return address, batch, row, head


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


def _new_out(q: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor like q. (empty_like of a contiguous one takes half empty's host time.)"""

    return torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _list_length(op: str, top_k: int, blocks: int) -> int:
    if isinstance(top_k, bool) or not isinstance(top_k, int) or top_k < 1:
        raise ValueError(f"{op}: top_k must be a positive integer, got {top_k!r}")
    return min(top_k, max(blocks, 1))


def _select(dims, q, k, lists, lens, keep, code, workspace, need, device) -> None:
    """One selection. dims: (batch, seq_q, seq_k, heads, kv_heads, head_dim, block_q, block_k,
    top_k); q, k: ``_view``s; lists: the addresses of indices and counts."""

    call_on(device, "h3b_select_key_blocks", *lists, q[0], k[0], *dims, *q[1:], *k[1:], *lens, keep, code,
            workspace, need)


def _attend(dims, entries, q, k, v, out, lse, lists, lens, scale, code, workspace, need, device) -> None:
    """One attention over lists of ``entries``; dims as for ``_select`` without top_k."""

    call_on(device, "h3b_block_sparse_attention", out[0], lse, q[0], k[0], v[0], *lists, entries, *dims, *q[1:],
            *k[1:], *v[1:], *out[1:], *lens, scale, code, workspace, need)


def _scale(op: str, softmax_scale: float | None, head_dim: int) -> float:
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(head_dim)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{op}: softmax_scale must be positive and finite, got {scale}")
    return scale


def select_key_blocks(q: torch.Tensor, k: torch.Tensor, top_k: int, *, block_q: int = 128, block_k: int = 128,
                      q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None,
                      keep: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``top_k`` key blocks (all of them if there are fewer) of every query block, by the
    product of the block's mean query with the block's mean key.

    q [B, Sq, H, D], k [B, Sk, Hk, D]. ``keep``: bool [ceil(Sk / block_k)], blocks that every
    list holds before any other (audio or text rows, say). Returns ``indices`` int32
    [B, H, ceil(Sq / block_q), top_k], ascending and -1 behind the last, and ``counts`` int32
    [B, H, ceil(Sq / block_q)]. Scores are compared in 64 bits, ties go to the lowest index:
    equal inputs give equal lists in any batch (bf16: as long as the nonzero values of a column
    of a block lie within a factor of 2^37; beyond that its 64-bit sum may round differently)."""

    op = "select_key_blocks"
    code = check_inputs(op, _TYPES, (q, k))
    _check_shapes(op, q, k, block_q, block_k)
    (b, sq, h, d), (_, sk, hk, _) = q.shape, k.shape
    nq, nk = -(-sq // block_q), -(-sk // block_k)
    top_k = _list_length(op, top_k, nk)
    q_lens = _side_tensor(op, "q_lens", q_lens, torch.int32, (b,), q.device)
    k_lens = _side_tensor(op, "k_lens", k_lens, torch.int32, (b,), q.device)
    keep = _side_tensor(op, "keep", keep, torch.bool, (nk,), q.device)
    indices = torch.empty_strided((b, h, nq, top_k), (h * nq * top_k, nq * top_k, top_k, 1), dtype=torch.int32,
                                  device=q.device)
    counts = torch.empty_strided((b, h, nq), (h * nq, nq, 1), dtype=torch.int32, device=q.device)
    if counts.numel() == 0:
        return indices, counts
    if not sk:
        raise ValueError(f"{op}: empty key sequence")
    need = _bytes("h3b_select_key_blocks_workspace_size", b, sq, sk, h, hk, d, block_q, block_k)
    ws = scratch(need, q.device)
    _select((b, sq, sk, h, hk, d, block_q, block_k, top_k), _view(op, "q", q), _view(op, "k", k),
            (indices.data_ptr(), counts.data_ptr()), (_opt(q_lens), _opt(k_lens)), _opt(keep), code, ws.data_ptr(),
            need, q.get_device())
    return indices, counts


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, indices: torch.Tensor,
                           counts: torch.Tensor | None = None, *, block_q: int = 128, block_k: int = 128,
                           softmax_scale: float | None = None, q_lens: torch.Tensor | None = None,
                           k_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
                           return_lse: bool = False):
    """softmax(q k^T * scale) v over the keys of every query block's listed key blocks.

    q [B, Sq, H, D], k and v [B, Sk, Hk, D] (strided views with a contiguous, 16-byte aligned
    head_dim of 64 or 128, no expanded dimensions; bf16 or fp16). ``indices`` int32 [B, H, ceil(Sq / block_q), n]: the
    first ``counts`` entries of a list count (all of them without ``counts``), in any order. An
    entry outside the key blocks adds nothing, an entry that is there twice counts twice. Query
    rows that have no key, and rows behind ``q_lens``, get zeros (lse -inf). Returns
    [B, Sq, H, D] (``out`` if given, which must not overlap an input), and with ``return_lse`` the
    fp32 [B, H, Sq] logarithms of the softmax sums."""

    op = "block_sparse_attention"
    code = check_inputs(op, _TYPES, (q, k, v) if out is None else (q, k, v, out))
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
        out = _new_out(q)
    elif out.shape != q.shape:
        raise ValueError(f"{op}: out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
    lse = torch.empty_strided((b, h, sq), (h * sq, sq, 1), dtype=torch.float32,
                              device=q.device) if return_lse else None
    scale = _scale(op, softmax_scale, d)
    if b * sq * h and (sk == 0 or entries == 0):
        out.zero_()
        if lse is not None:
            lse.fill_(-math.inf)
    elif b * sq * h:
        need = _bytes("h3b_block_sparse_attention_workspace_size", b, sq, h, d, block_k, entries)
        ws = scratch(need, q.device) if need else None
        _attend((b, sq, sk, h, hk, d, block_q, block_k), entries, _view(op, "q", q), _view(op, "k", k),
                _view(op, "v", v), _view(op, "out", out), _opt(lse), (indices.data_ptr(), _opt(counts)),
                (_opt(q_lens), _opt(k_lens)), scale, code, _opt(ws), need, q.get_device())
    return (out, lse) if return_lse else out


def _select_and_attend(dims, top_k, q, k, v, out, lse, lens, keep, scale, code, device) -> None:
    """Both steps; the lists and the workspaces are parts of one allocation that the two share."""

    b, sq, sk, h, hk, d, block_q, block_k = dims
    rows = b * h * -(-sq // block_q)
    lists = (4 * rows * (top_k + 1) + 255) // 256 * 256
    first = _bytes("h3b_select_key_blocks_workspace_size", *dims)
    second = _bytes("h3b_block_sparse_attention_workspace_size", b, sq, h, d, block_k, top_k)
    ws = scratch(lists + max(first, second), device)
    at = ws.data_ptr()
    pair = (at, at + 4 * rows * top_k)
    _select((*dims, top_k), q, k, pair, lens, keep, code, at + lists, first, device.index)
    _attend(dims, top_k, q, k, v, out, lse, pair, lens, scale, code, at + lists, second, device.index)


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, top_k: int, *, block_q: int = 128,
                     block_k: int = 128, softmax_scale: float | None = None, q_lens: torch.Tensor | None = None,
                     k_lens: torch.Tensor | None = None, keep: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, return_lse: bool = False):
    """``select_key_blocks`` and then ``block_sparse_attention`` over its lists."""

    op = "sparse_attention"
    code = check_inputs(op, _TYPES, (q, k, v) if out is None else (q, k, v, out))
    _check_shapes(op, q, k, block_q, block_k)
    if v.shape != k.shape:
        raise ValueError(f"{op}: k {tuple(k.shape)} and v {tuple(v.shape)} disagree")
    (b, sq, h, d), (_, sk, hk, _) = q.shape, k.shape
    nk = -(-sk // block_k)
    top_k = _list_length(op, top_k, nk)
    q_lens = _side_tensor(op, "q_lens", q_lens, torch.int32, (b,), q.device)
    k_lens = _side_tensor(op, "k_lens", k_lens, torch.int32, (b,), q.device)
    keep = _side_tensor(op, "keep", keep, torch.bool, (nk,), q.device)
    if out is None:
        out = _new_out(q)
    elif out.shape != q.shape:
        raise ValueError(f"{op}: out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
    lse = torch.empty_strided((b, h, sq), (h * sq, sq, 1), dtype=torch.float32,
                              device=q.device) if return_lse else None
    scale = _scale(op, softmax_scale, d)
    if b * sq * h:
        if not sk:
            raise ValueError(f"{op}: empty key sequence")
        _select_and_attend((b, sq, sk, h, hk, d, block_q, block_k), top_k, _view(op, "q", q), _view(op, "k", k),
                           _view(op, "v", v), _view(op, "out", out), _opt(lse), (_opt(q_lens), _opt(k_lens)),
                           _opt(keep), scale, code, q.device)
    return (out, lse) if return_lse else out


def packed_sparse_attention(packed: torch.Tensor, top_k: int, head_dim: int = HEAD_DIM, *, block_q: int = 128,
                            block_k: int = 128, softmax_scale: float | None = None,
                            keep: torch.Tensor | None = None, out: torch.Tensor | None = None,
                            return_lse: bool = False):
    """``sparse_attention`` over the packed receive buffer ``[S, hl, 3*D]`` (q | k | v per
    head), read in place. Returns ``[S, hl, D]`` (and lse ``[hl, S]``)."""

    op = "packed_sparse_attention"
    code = check_inputs(op, _TYPES, (packed,) if out is None else (packed, out))
    if packed.dim() != 3 or packed.shape[-1] != 3 * head_dim:
        raise ValueError(f"packed attention expects [S, hl, 3*{head_dim}], got {tuple(packed.shape)}")
    if head_dim not in HEAD_DIMS:
        raise RuntimeError(f"{op}: head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    if block_q not in BLOCK_Q or block_k not in BLOCK_K:
        raise ValueError(f"{op}: block_q must be one of {BLOCK_Q} and block_k one of {BLOCK_K}, got "
                         f"{block_q} and {block_k}")
    s, hl, _ = packed.shape
    row, head, last = packed.stride()
    if last != 1 or head != 3 * head_dim or row % 8:
        packed = packed.contiguous()
        row, head, last = packed.stride()
    nk = -(-s // block_k)
    top_k = _list_length(op, top_k, nk)
    keep = _side_tensor(op, "keep", keep, torch.bool, (nk,), packed.device)
    if out is None:
        out = torch.empty((s, hl, head_dim), dtype=packed.dtype, device=packed.device)
    elif out.shape != (s, hl, head_dim):
        raise ValueError(f"{op}: out must have shape {(s, hl, head_dim)}, got {tuple(out.shape)}")
    lse = torch.empty((hl, s), dtype=torch.float32, device=packed.device) if return_lse else None
    scale = _scale(op, softmax_scale, head_dim)
    out_row, out_head, out_last = out.stride()
    base, to = packed.data_ptr(), out.data_ptr()
    if out_last != 1 or base % 16 or to % 16:
        raise ValueError(f"{op}: packed and out must have a contiguous, 16-byte aligned last dimension")
    if s * hl:
        # (Sizes of one never step: any positive batch stride will do.)
        views = [(base + 2 * i * head_dim, s * row, row, head) for i in range(3)]
        _select_and_attend((1, s, s, hl, hl, head_dim, block_q, block_k), top_k, *views,
                           (to, s * hl * head_dim, out_row, out_head), _opt(lse), (None, None), _opt(keep), scale,
                           code, packed.device)
    return (out, lse) if return_lse else out


# Where ``install_sparse_attention`` leaves its settings on an attention module, and the packed
# attention forward looks for them.
SPARSE_ATTRIBUTE = "_h3b_sparse_attention"


@dataclass
class SparseAttention:
    """How the packed attention of one transformer is made sparse: every block of ``block_q``
    queries attends to a ``density`` share of the blocks of ``block_k`` keys (at least
    ``min_blocks``), and among them always to all blocks that hold any of the first
    ``keep_first_rows`` or the last ``keep_last_rows`` rows. The rows are those of the whole sequence:
    ``H3Transformer`` has text first, then video, then audio, so its text is kept by
    ``keep_first_rows`` and its audio by ``keep_last_rows``."""

    density: float
    block_q: int = 128
    block_k: int = 128
    keep_last_rows: int = 0
    min_blocks: int = 1
    keep_first_rows: int = 0
    calls: int = 0

    def __post_init__(self) -> None:
        if not 0.0 < self.density <= 1.0:
            raise ValueError(f"sparse attention: density must be in (0, 1], got {self.density}")
        if self.block_q not in BLOCK_Q or self.block_k not in BLOCK_K:
            raise ValueError(f"sparse attention: block_q must be one of {BLOCK_Q} and block_k one of {BLOCK_K}, got "
                             f"{self.block_q} and {self.block_k}")
        if self.keep_first_rows < 0 or self.keep_last_rows < 0 or self.min_blocks < 1:
            raise ValueError("sparse attention: keep_first_rows and keep_last_rows must not be negative, min_blocks at "
                             "least 1")

    def list_length(self, rows: int) -> int:
        """Key blocks per list for a sequence of ``rows``."""

        blocks = -(-rows // self.block_k)
        share = math.ceil(self.density * blocks - 1e-9)  # 0.1 * 30 is a little more than 3
        return min(blocks, max(share, self.min_blocks, self._kept(rows)))

    def _kept_ends(self, rows: int) -> tuple[int, int]:
        """Kept key blocks at the start and at the end of a sequence of ``rows``."""

        last = min(self.keep_last_rows, rows)
        return (-(-min(self.keep_first_rows, rows) // self.block_k),
                -(-rows // self.block_k) - (rows - last) // self.block_k if last else 0)

    def _kept(self, rows: int) -> int:
        return min(sum(self._kept_ends(rows)), -(-rows // self.block_k))

    def _keep_mask(self, rows: int, device: torch.device) -> torch.Tensor | None:
        """The kept blocks, made anew on the current stream by every call: a mask that outlived its call
        could be replaced while another stream, or a captured graph, still reads it."""

        first, last = self._kept_ends(rows)
        if not first and not last:
            return None
        mask = torch.zeros(-(-rows // self.block_k), dtype=torch.bool, device=device)
        if first:
            mask[:first] = True
        if last:
            mask[-last:] = True
        return mask

    def attend(self, packed: torch.Tensor, head_dim: int) -> torch.Tensor:
        """``packed_sparse_attention`` over the receive buffer [S, hl, 3*D]."""

        rows = packed.shape[0]
        self.calls += 1
        # (A sequence without rows has lists of no blocks, and the op answers it as the dense one does.)
        return packed_sparse_attention(packed, max(self.list_length(rows), 1), head_dim, block_q=self.block_q,
                                       block_k=self.block_k, keep=self._keep_mask(rows, packed.device))


def install_sparse_attention(transformer: Any, *, density: float = 0.1, block_q: int = 128, block_k: int = 128,
                             keep_last_rows: int = 0, min_blocks: int = 1, keep_first_rows: int = 0) -> dict[str, Any]:
    """Make the packed attention of every block sparse (see ``SparseAttention``).

    Call it after ``install_transformer_fusions`` (with ``qknorm_rope``) or
    ``install_packed_ulysses``: their attention forwards read the settings, also when they are
    installed again later. On several ranks each selects for its own heads over the whole
    sequence, so the ranks need not agree on anything. Returns the installation's metadata; its
    ``"runtime"`` counts calls. ``remove_sparse_attention`` goes back to dense attention."""

    runtime = SparseAttention(density, block_q, block_k, keep_last_rows, min_blocks, keep_first_rows)
    modules = [block.attn for block in transformer.transformer_blocks]
    for attention in modules:
        if not getattr(attention.__dict__.get("forward"), "h3b_packed", False):
            raise RuntimeError("sparse attention needs the packed attention forward: call install_transformer_fusions "
                               "or install_packed_ulysses first")
        if attention.head_dim not in HEAD_DIMS:
            raise RuntimeError(f"sparse attention: head_dim must be one of {HEAD_DIMS}, got {attention.head_dim}")
    for attention in modules:
        setattr(attention, SPARSE_ATTRIBUTE, runtime)
    return {"backend": "h3b_block_sparse", "semantics": "sparse", "modules": len(modules), "density": density,
            "block_q": block_q, "block_k": block_k, "keep_first_rows": keep_first_rows, "keep_last_rows": keep_last_rows,
            "runtime": runtime}


def remove_sparse_attention(transformer: Any) -> None:
    """Dense attention again."""

    for block in transformer.transformer_blocks:
        if hasattr(block.attn, SPARSE_ATTRIBUTE):
            delattr(block.attn, SPARSE_ATTRIBUTE)
