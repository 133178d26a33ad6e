"""Argument checks of the block-sparse and sandwich-norm entry points: they return before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from h3_flash_b200 import _lib

FAKE = 1 << 20  # a 16-byte aligned address, never read


def _select(batch=1, sq=256, sk=256, heads=2, kv=2, d=128, bq=128, bk=128, top=1, strides=(8,) * 6, dtype=0, ws=FAKE, ws_bytes=1 << 30,
            q=FAKE):
    _lib.call("h3b_select_key_blocks", FAKE, FAKE, q, FAKE, batch, sq, sk, heads, kv, d, bq, bk, top, *strides, None, None, None, dtype,
              ws, ws_bytes, None)


def _attend(batch=1, sq=256, sk=256, heads=2, kv=2, d=128, bq=128, bk=128, n=1, strides=(8,) * 12, scale=1.0, dtype=0, q=FAKE, idx=FAKE):
    _lib.call("h3b_block_sparse_attention", FAKE, None, q, FAKE, FAKE, idx, None, n, batch, sq, sk, heads, kv, d, bq, bk, *strides, None,
              None, scale, dtype, None, 0, None)


def _sandwich(rows=1, cols=8, n_index=1, n_table=1, dtype=0, normed=None, weight=None, gate=FAKE):
    _lib.call("h3b_sandwich_residual_rmsnorm_modulate", FAKE, normed, FAKE, FAKE, FAKE, gate, weight, None, None, FAKE, rows, cols,
              n_index, n_table, 8, 8, 8, 8, 8, 8, 1.0, 1e-6, 1e-6, dtype, None)


@pytest.mark.parametrize("call", [_select, _attend])
def test_unsupported_shapes(call):
    for bad in (dict(d=96), dict(bq=64), dict(bk=256), dict(dtype=2)):
        with pytest.raises(RuntimeError, match="needs bf16 or fp16"):
            call(**bad)
    with pytest.raises(ValueError, match="negative shape"):
        call(batch=-1)
    with pytest.raises(ValueError, match="empty key sequence"):
        call(sk=0)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        call(heads=3)
    with pytest.raises(ValueError, match="launch limits"):
        call(sq=2**31)
    with pytest.raises(ValueError, match="null argument"):
        call(q=None)
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(q=FAKE + 2)


def test_select_refusals():
    for top in (0, 3):
        with pytest.raises(ValueError, match=r"top_k \(%d\) must be 1..2" % top):
            _select(top=top)
    with pytest.raises(ValueError, match="multiples of 8"):
        _select(strides=(8, 8, 8, 8, 12, 8))
    need = ctypes.c_int64(-1)
    _lib.call("h3b_select_key_blocks_workspace_size", 1, 256, 256, 2, 2, 128, 128, 128, ctypes.byref(need))
    assert need.value > 0
    with pytest.raises(ValueError, match="workspace of %d bytes" % need.value):
        _select(ws_bytes=need.value - 1)
    with pytest.raises(ValueError, match="workspace"):
        _select(ws=FAKE + 8)


def test_attend_refusals():
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="positive and finite"):
            _attend(scale=scale)
    with pytest.raises(ValueError, match="empty lists"):
        _attend(n=0)
    with pytest.raises(ValueError, match="launch limits"):
        _attend(n=2**20 + 1)
    with pytest.raises(ValueError, match="positive multiples of 8"):
        _attend(strides=(8, 8, 8, 8, 0, 8, 8, 8, 8, 8, 8, 8))
    with pytest.raises(ValueError, match="null argument"):
        _attend(idx=None)


def test_sandwich_refusals():
    for bad, match in ((dict(rows=-1), "negative shape"), (dict(dtype=3), "unknown dtype"), (dict(n_index=0), "empty index"),
                       (dict(n_table=0), "empty index or table"), (dict(normed=FAKE), "needs weight"), (dict(gate=None), "null argument")):
        with pytest.raises(ValueError, match=match):
            _sandwich(**bad)


def test_calls_without_rows_launch_nothing():
    _lib.reset_launch_count()
    _select(sq=0)
    _attend(batch=0)
    _sandwich(rows=0)
    assert _lib.launch_count() == 0


def test_python_ops_refuse_cpu_tensors():
    from h3_flash_b200.runtime.attention.sparse import select_key_blocks, sparse_attention
    from h3_flash_b200.runtime.kernels.fusions import fused_sandwich_residual

    x = torch.zeros(1, 8, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        select_key_blocks(x, x, 1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        sparse_attention(x, x, x, 1)
    row = torch.zeros(1, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fused_sandwich_residual(row, row, row[0], row[0], None, 1e-6)
