"""Host side of sparse attention and the sandwich-norm block, without a GPU."""

from __future__ import annotations

import pytest
import torch

from h3_flash_b200.runtime.attention import install_sparse_attention, remove_sparse_attention
from h3_flash_b200.runtime.attention.sparse import SPARSE_ATTRIBUTE, SparseAttention
from h3_flash_b200.runtime.h3_block import H3BlockStack, H3TransformerBlock


def _stack(**kw):
    block = H3TransformerBlock(dim=256, heads=2, head_dim=128, ffn_inner=512, **kw)
    return H3BlockStack([block])


def test_list_length():
    s = SparseAttention(0.1)
    assert [s.list_length(n) for n in (1, 128, 129, 1280, 51200)] == [1, 1, 1, 1, 40]
    assert SparseAttention(0.1).list_length(30 * 128) == 3
    s = SparseAttention(0.1, block_k=64, keep_last_rows=130, min_blocks=5)
    assert s.list_length(64 * 100) == 10
    assert s.list_length(64 * 10) == 5
    assert s.list_length(64 * 2) == 2
    # rows 510..639 lie in blocks 7 to 9, rows 511..640 in blocks 7 to 10
    assert s._kept(640) == 3 and s._kept(641) == 4 and s._kept(100) == 2
    assert SparseAttention(0.01, keep_last_rows=1280).list_length(51200) == 10


def test_no_mask_outlives_its_call():
    """A mask that is kept for later calls could be replaced under a stream or a graph that reads it."""

    s = SparseAttention(0.1, block_k=64, keep_last_rows=130)
    before = dict(vars(s))
    first = s._keep_mask(640, torch.device("cpu"))
    assert first.tolist() == [False] * 7 + [True] * 3
    assert s._keep_mask(640, torch.device("cpu")) is not first
    assert s._keep_mask(64, torch.device("cpu")).tolist() == [True]
    s.keep_last_rows = 1
    assert s._keep_mask(640, torch.device("cpu")).tolist() == [False] * 9 + [True]
    assert vars(s) == {**before, "keep_last_rows": 1}
    assert s._keep_mask(0, torch.device("cpu")) is None


def test_rows_at_both_ends_are_kept():
    """Text stands first in the sequence, audio last."""

    s = SparseAttention(0.1, block_k=64, keep_first_rows=65, keep_last_rows=1)
    cpu = torch.device("cpu")
    assert s._keep_mask(641, cpu).tolist() == [True] * 2 + [False] * 8 + [True]
    assert s.list_length(641) == 3 and s.list_length(6400) == 10
    assert s._keep_mask(128, cpu).tolist() == [True] * 2 and s.list_length(128) == 2
    assert s._keep_mask(3, cpu).tolist() == [True] and s.list_length(3) == 1
    assert SparseAttention(0.1, keep_first_rows=1)._keep_mask(256, cpu).tolist() == [True, False]
    assert SparseAttention(0.1, keep_first_rows=10**6, keep_last_rows=10**6).list_length(51200) == 400
    assert SparseAttention(0.1)._keep_mask(256, cpu) is None
    with pytest.raises(ValueError, match="keep_first_rows"):
        SparseAttention(0.1, keep_first_rows=-1)
    stack = _stack()
    from h3_flash_b200.runtime.kernels.transformer import _patch_attention

    _patch_attention(stack, {})
    meta = install_sparse_attention(stack, keep_first_rows=77, keep_last_rows=5)
    assert meta["keep_first_rows"] == meta["runtime"].keep_first_rows == 77
    assert meta["keep_last_rows"] == meta["runtime"].keep_last_rows == 5


@pytest.mark.parametrize("bad", [dict(density=0.0), dict(density=1.5), dict(density=0.1, block_q=64), dict(density=0.1, block_k=32),
                                 dict(density=0.1, keep_last_rows=-1), dict(density=0.1, min_blocks=0)])
def test_settings_are_checked(bad):
    with pytest.raises(ValueError, match="sparse attention"):
        SparseAttention(**bad)


def test_install_needs_the_packed_forward():
    stack = _stack()
    with pytest.raises(RuntimeError, match="packed attention forward"):
        install_sparse_attention(stack)
    attention = stack.transformer_blocks[0].attn
    attention.forward = lambda *a: None
    with pytest.raises(RuntimeError, match="packed attention forward"):
        install_sparse_attention(stack)
    from h3_flash_b200.runtime.kernels.transformer import _patch_attention

    _patch_attention(stack, {})
    meta = install_sparse_attention(stack, density=0.25, block_k=64)
    assert getattr(attention, SPARSE_ATTRIBUTE) is meta["runtime"] and meta["modules"] == 1
    _patch_attention(stack, {})  # installing the forward again keeps the settings
    assert getattr(attention, SPARSE_ATTRIBUTE) is meta["runtime"]
    remove_sparse_attention(stack)
    assert not hasattr(attention, SPARSE_ATTRIBUTE)
    remove_sparse_attention(stack)


def test_peer_exchange_runs_sparse_attention_locally_and_scatters():
    """With sparse attention the fused output exchange is left: local rows, then the scatter."""

    from h3_flash_b200.runtime.parallel.packed_ulysses import _peer_exchange_rest

    log = []

    class Peer:
        def barrier(self):
            log.append("barrier")

        def attention(self, *args):
            log.append("dense")
            return "merged"

        def recv_view(self, rows, heads, head_dim):
            return ("packed", rows, heads, head_dim)

        def scatter(self, output, counts):
            log.append(("scatter", output, tuple(counts)))
            return "merged"

    class Runtime:
        peer, fuse_output_exchange = Peer(), True

    class Sparse:
        def attend(self, packed, head_dim):
            log.append(("sparse", packed, head_dim))
            return "rows"

    assert _peer_exchange_rest(Runtime(), [3, 4], 2, 128, Sparse()) == "merged"
    assert log == ["barrier", ("sparse", ("packed", 7, 2, 128), 128), ("scatter", "rows", (3, 4)), "barrier"]
    log.clear()
    _peer_exchange_rest(Runtime(), [3, 4], 2, 128)
    assert log == ["barrier", "dense", "barrier"]


def test_sandwich_block_eager_math():
    torch.manual_seed(0)
    block = H3TransformerBlock(dim=64, heads=1, head_dim=64, ffn_inner=128, sandwich_norm=True, residual_scale=0.5)
    with torch.no_grad():
        for p in block.parameters():
            p.copy_(torch.randn_like(p) * 0.2)
    x, idx = torch.randn(1, 6, 64), torch.tensor([0, 1, 2, 0, 1, 2])
    norm = lambda t, m: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + m.eps) * m.weight  # noqa: E731
    shift1, scale1, gate1, shift2, scale2, gate2 = (t[idx] for t in block.adaln_proj())
    a = block.attn(norm(x, block.norm1) * (1 + scale1) + shift1)
    h = 0.5 * x + gate1 * norm(a, block.norm1_post)
    f = block.ff(norm(h, block.norm2) * (1 + scale2) + shift2)
    want = 0.5 * h + gate2 * norm(f, block.norm2_post)
    torch.testing.assert_close(block(x, None, idx, None), want, rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError, match="needs sandwich_norm"):
        H3TransformerBlock(dim=64, heads=1, head_dim=64, ffn_inner=128, residual_scale=0.5)
    assert block.norm1_post is not None and H3TransformerBlock(dim=64, heads=1, head_dim=64, ffn_inner=128).norm1_post is None


@pytest.mark.parametrize("missing", ["norm1_post", "norm2_post"])
@pytest.mark.parametrize("gone", [False, True])
def test_a_block_with_one_post_norm_is_refused_when_installed(missing, gone):
    """Not in the middle of a forward pass (norm2_post missing), and not run without its norm (norm1_post missing)."""

    from h3_flash_b200.runtime.kernels.transformer import _patch_blocks

    stack = H3BlockStack([H3TransformerBlock(dim=64, heads=1, head_dim=64, ffn_inner=128, sandwich_norm=True) for _ in range(2)])
    last = stack.transformer_blocks[1]
    if gone:
        delattr(last, missing)
    else:
        setattr(last, missing, None)
    with pytest.raises(RuntimeError, match="norm1_post and norm2_post together"):
        _patch_blocks(stack, True, True, {"gate": {}})
    assert all("forward" not in vars(block) for block in stack.transformer_blocks)
    _patch_blocks(H3BlockStack([stack.transformer_blocks[0]]), True, True, {"gate": {}})
    assert "forward" in vars(stack.transformer_blocks[0])
