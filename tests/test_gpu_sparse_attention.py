"""Block selection and block-sparse attention against their fp64 definitions.

Bounds. Weights p are rounded once to the operand type (relative u = eps/2) and the output
once more, so |out - ref| <= u * sum p|v| + u * |ref| plus what fp32 leaves: a score is a sum
of D products, off by at most D * 2^-23 * |q|.|k| * scale (accumulation that truncates), which
moves p and lse by that much; exp2, the softmax sum and the division stay within 2^-18.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import sparse_ref

pytestmark = pytest.mark.gpu


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _randn(shape, seed, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _lists(b, h, nq, nk, n, seed, lo=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    indices = torch.rand(b, h, nq, nk, generator=g, device="cuda").argsort(-1)[..., :n].to(torch.int32)
    counts = torch.randint(lo, n + 1, (b, h, nq), generator=g, device="cuda").to(torch.int32)
    return indices, counts


def _check(out, lse, q, k, v, indices, counts, **kw):
    ref, ref_lse, weight_abs, score_abs = sparse_ref.attend(q, k, v, indices, counts, **kw)
    u = _half_step(out.dtype)
    slack = q.shape[-1] * 2.0**-23 * score_abs + 2.0**-18
    bound = (u + 2 * slack.transpose(1, 2)[..., None]) * weight_abs + u * ref.abs() * (1 + 2.0**-6) + 2.0**-24
    err = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound).all(), float((err - bound).max())
    if lse is not None:
        got = lse.double().cpu()
        empty = ref_lse == -math.inf
        assert torch.equal(got == -math.inf, empty)
        tol = slack + 2.0**-21 * ref_lse.abs().nan_to_num(posinf=0.0)
        assert ((got - ref_lse).abs()[~empty] <= tol[~empty]).all()


@pytest.fixture(autouse=True)
def _status():
    from h3_flash_b200 import _lib

    yield
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("block_q,block_k", [(128, 128), (128, 64), (256, 128), (256, 64)])
def test_attend(dtype, d, block_q, block_k):
    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    b, sq, sk, h, hk = 2, 700, 901, 4, 2
    q, k, v = _randn((b, sq, h, d), 1, dtype), _randn((b, sk, hk, d), 2, dtype), _randn((b, sk, hk, d), 3, dtype)
    nq, nk = -(-sq // block_q), -(-sk // block_k)
    indices, counts = _lists(b, h, nq, nk, nk - 1, 4)
    out, lse = block_sparse_attention(q, k, v, indices, counts, block_q=block_q, block_k=block_k, return_lse=True)
    _check(out, lse, q, k, v, indices, counts, block_q=block_q, block_k=block_k)


@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 5000), (2, 64), (3, 1300), (33, 3000), (128, 127), (128, 2500), (129, 129), (255, 65), (257, 1025), (1000, 3)])
@pytest.mark.parametrize("block_k", [64, 128])
def test_lengths(sq, sk, block_k):
    """From one row and one key; a single query block is split along its list and joined."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    q, k, v = _randn((1, sq, 3, 128), 1), _randn((1, sk, 3, 128), 2), _randn((1, sk, 3, 128), 3)
    nq, nk = -(-sq // 128), -(-sk // block_k)
    indices, _ = _lists(1, 3, nq, nk, nk, 4)
    out, lse = block_sparse_attention(q, k, v, indices, block_k=block_k, return_lse=True)
    _check(out, lse, q, k, v, indices, None, block_k=block_k)


@pytest.mark.parametrize("sq,block_k", [(1, 128), (5, 64), (128, 128)])
def test_many_single_tiles(sq, block_k):
    """More one-tile queries than SMs with long lists: two ranges per item and no more, counts of
    every size, and a list of one entry beside them."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    b, h, sk = 16, 10, 1700
    q, k, v = _randn((b, sq, h, 64), 1), _randn((b, sk, 1, 64), 2), _randn((b, sk, 1, 64), 3)
    nk = -(-sk // block_k)
    indices, counts = _lists(b, h, 1, nk, nk, 4)
    out, lse = block_sparse_attention(q, k, v, indices, counts, block_k=block_k, return_lse=True)
    _check(out, lse, q, k, v, indices, counts, block_k=block_k)
    out, lse = block_sparse_attention(q, k, v, indices[..., :1].contiguous(), block_k=block_k, return_lse=True)
    _check(out, lse, q, k, v, indices[..., :1], None, block_k=block_k)


def test_many_items_per_cta():
    """More pairs of tiles than SMs, lists of very different lengths (none among them)."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    b, s, h = 2, 2100, 40
    q, k, v = (_randn((b, s, h, 64), i) for i in (1, 2, 3))
    nq = nk = -(-s // 128)
    indices, counts = _lists(b, h, nq, nk, nk, 4)
    counts[:, ::3] = 0
    counts[0, 1::3] = torch.where(torch.rand(h // 3 + 1, nq, device="cuda")[: counts[0, 1::3].shape[0]] < 0.5, 1, counts[0, 1::3])
    out, lse = block_sparse_attention(q, k, v, indices, counts, return_lse=True)
    _check(out, lse, q, k, v, indices, counts)
    # neighbouring tiles at the same entries read one copy: the same rows, bit for bit
    same = indices[:, :, :1].expand(-1, -1, nq, -1).contiguous()
    n = torch.full_like(counts, nk)
    whole = block_sparse_attention(q, k, v, same, n)
    shifted = same.clone()
    shifted[:, :, 1::2] = same[:, :, 1::2].roll(1, -1)
    _check(whole, None, q, k, v, same, n)
    _check(block_sparse_attention(q, k, v, shifted, n), None, q, k, v, shifted, n)


@pytest.mark.parametrize("block_q", [128, 256])
@pytest.mark.parametrize("block_k", [64, 128])
def test_short_lists_over_and_over(block_q, block_k):
    """Items of one to three units, many per CTA, many calls: every wait ends, the bits repeat."""

    from h3_flash_b200 import _lib
    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    s, h = 148 * 256, 2
    q, k, v = (_randn((1, s, h, 128), i) for i in (1, 2, 3))
    nq, nk = s // block_q, s // block_k
    for n in (1, 2, 3):
        indices = torch.randint(0, nk, (1, h, nq, n), device="cuda", generator=torch.Generator("cuda").manual_seed(n)).int()
        for counts in (None, torch.randint(0, n + 1, (1, h, nq), device="cuda").int()):
            first = block_sparse_attention(q, k, v, indices, counts, block_q=block_q, block_k=block_k)
            for _ in range(40):
                again = block_sparse_attention(q, k, v, indices, counts, block_q=block_q, block_k=block_k)
            assert torch.equal(first, again)
            assert _lib.device_status() == 0
            rows = slice(0, 512)
            part = indices[:, :, : 512 // block_q].contiguous()
            n_part = None if counts is None else counts[:, :, : 512 // block_q].contiguous()
            _check(first[:, rows], None, q[:, rows], k, v, part, n_part, block_q=block_q, block_k=block_k)


@pytest.mark.parametrize("sq,block_k", [(1, 128), (1, 64), (40, 128), (300, 64)])
def test_long_lists_over_cold_keys(sq, block_k):
    """Lists of many units over keys that come from HBM: loads land out of order, and a tile
    may reach a slot before the other tile's rows in it have landed."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    s, h = 60000, 24
    k, v = _randn((1, s, h, 128), 2), _randn((1, s, h, 128), 3)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    nq, nk = -(-sq // 128), -(-s // block_k)
    for seed in range(3):
        q = _randn((1, sq, h, 128), 10 + seed)
        indices, counts = _lists(1, h, nq, nk, 100, seed)
        flush.zero_()
        out, lse = block_sparse_attention(q, k, v, indices, counts, block_k=block_k, return_lse=True)
        few = slice(0, 3)
        _check(out[:, :, few], lse[:, few], q[:, :, few], k[:, :, few], v[:, :, few], indices[:, few], counts[:, few], block_k=block_k)


@pytest.mark.parametrize("sq,block_k,padded", [(2944, 64, False), (2944, 128, True), (640, 64, True)])
def test_lists_per_256_rows_without_a_second_tile(sq, block_k, padded):
    """Far more pairs than SMs over keys that come from HBM, and some of the pairs have no second
    tile (an odd number of tiles, rows behind q_lens): the CTA that takes one goes on to a pair that has."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    b, s, h = 2, 30000, 24
    k, v = _randn((b, s, h, 128), 2), _randn((b, s, h, 128), 3)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    nq, nk = -(-sq // 256), -(-s // block_k)
    q_lens = torch.tensor([sq, sq - 450], dtype=torch.int32, device="cuda") if padded else None
    few = slice(0, 2)
    for seed in range(2):
        q = _randn((b, sq, h, 128), 10 + seed)
        indices, counts = _lists(b, h, nq, nk, 40, seed)
        kw = dict(block_q=256, block_k=block_k, q_lens=q_lens)
        first, lse = block_sparse_attention(q, k, v, indices, counts, return_lse=True, **kw)
        for _ in range(20):
            flush.zero_()
            assert torch.equal(first, block_sparse_attention(q, k, v, indices, counts, **kw))
        _check(first[:, :, few], lse[:, few], q[:, :, few], k[:, :, few], v[:, :, few], indices[:, few], counts[:, few], **kw)


@pytest.mark.parametrize("block_k", [64, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_padded_batch_with_nan(d, block_k):
    """What lies behind q_lens and k_lens is NaN and inf; rows there get zeros."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention, select_key_blocks

    b, s, h = 5, 600, 2
    q, k, v = (_randn((b, s, h, d), i) for i in (1, 2, 3))
    q_lens = torch.tensor([600, 0, 1, 300, 257], dtype=torch.int32, device="cuda")
    k_lens = torch.tensor([513, 600, 0, 1, 127], dtype=torch.int32, device="cuda")
    for i in range(b):
        q[i, int(q_lens[i]):] = float("nan")
        k[i, int(k_lens[i]):] = float("inf")
        v[i, int(k_lens[i]):] = float("nan")
    nk = -(-s // block_k)
    indices = torch.arange(nk, dtype=torch.int32, device="cuda").expand(b, h, -(-s // 128), nk).contiguous()
    kw = dict(block_k=block_k, q_lens=q_lens, k_lens=k_lens)
    out, lse = block_sparse_attention(q, k, v, indices, return_lse=True, **kw)
    _check(out, lse, q, k, v, indices, None, **kw)
    for i in range(b):
        assert (out[i, int(q_lens[i]):] == 0).all()
    got, n = select_key_blocks(q, k, 3, **kw)
    ref, ref_n = sparse_ref.select(q, k, 3, **kw)
    assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)
    _check(block_sparse_attention(q, k, v, got, n, **kw), None, q, k, v, got, n, **kw)


@pytest.mark.parametrize("sq", [1, 100, 129, 300, 385, 640])
def test_lists_per_256_rows_with_odd_tiles(sq):
    """A list that serves one tile only (the other lies behind the rows), whole and split; a
    padded batch on top."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention, select_key_blocks

    b, sk, h = 3, 1100, 2
    q, k, v = _randn((b, sq, h, 128), 1), _randn((b, sk, h, 128), 2), _randn((b, sk, h, 128), 3)
    q_lens = torch.tensor([sq, max(0, sq - 130), sq // 2], dtype=torch.int32, device="cuda")
    k_lens = torch.tensor([sk, 700, 1000], dtype=torch.int32, device="cuda")
    for block_k in (64, 128):
        indices, counts = _lists(b, h, -(-sq // 256), -(-sk // block_k), 7, 4)
        kw = dict(block_q=256, block_k=block_k)
        out, lse = block_sparse_attention(q, k, v, indices, counts, return_lse=True, **kw)
        _check(out, lse, q, k, v, indices, counts, **kw)
        out, lse = block_sparse_attention(q, k, v, indices, counts, q_lens=q_lens, k_lens=k_lens, return_lse=True, **kw)
        _check(out, lse, q, k, v, indices, counts, q_lens=q_lens, k_lens=k_lens, **kw)
        got, n = select_key_blocks(q, k, 5, q_lens=q_lens, k_lens=k_lens, **kw)
        ref, ref_n = sparse_ref.select(q, k, 5, q_lens=q_lens, k_lens=k_lens, **kw)
        assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


@pytest.mark.parametrize("sq", [1, 200, 700])
def test_without_a_workspace(sq):
    """A caller of the C entry point that gives none: every list whole, the same result."""

    from h3_flash_b200 import _lib

    h, sk, n = 3, 2000, 12
    q, k, v = _randn((1, sq, h, 128), 1), _randn((1, sk, h, 128), 2), _randn((1, sk, h, 128), 3)
    indices, _ = _lists(1, h, -(-sq // 128), -(-sk // 128), n, 4)
    for missing in (True, False):
        out, lse = torch.empty_like(q), torch.empty(1, h, sq, device="cuda")
        ws = torch.empty(64, dtype=torch.uint8, device="cuda")  # too short
        _lib.call("h3b_block_sparse_attention", out.data_ptr(), lse.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  indices.data_ptr(), None, n, 1, sq, sk, h, h, 128, 128, 128, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                  *out.stride()[:3], None, None, 128**-0.5, 0, None if missing else ws.data_ptr(), 0 if missing else 64,
                  torch.cuda.current_stream().cuda_stream)
        _check(out, lse, q, k, v, indices, None)


def test_large_batch_of_single_rows():
    """More items than SMs, each one query row: halves of a list on the two tiles of an item."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    b, h, hk, sk = 40, 8, 2, 520
    q, k, v = _randn((b, 1, h, 64), 1), _randn((b, sk, hk, 64), 2), _randn((b, sk, hk, 64), 3)
    indices, counts = _lists(b, h, 1, 9, 9, 4)
    k_lens = torch.randint(0, sk + 1, (b,), device="cuda", generator=torch.Generator("cuda").manual_seed(5)).int()
    out, lse = block_sparse_attention(q, k, v, indices, counts, block_k=64, k_lens=k_lens, return_lse=True)
    _check(out, lse, q, k, v, indices, counts, block_k=64, k_lens=k_lens)


def test_two_streams_at_once():
    """Calls that overlap on two streams do not share scratch."""

    from h3_flash_b200.runtime.attention.sparse import sparse_attention

    sets = [tuple(_randn((1, 3000, 4, 128), 10 * i + j) for j in range(3)) for i in range(2)]
    want = [sparse_attention(*s, 5) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (stream, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                got[i].append(sparse_attention(*s, 5))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_entries_outside_and_twice():
    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    q, k, v = (_randn((1, 256, 2, 128), i) for i in (1, 2, 3))
    lists = torch.tensor([[-1, 0, 7], [1, 1, 0], [-5, 2**30, -2**31], [2**31 - 1, 1, -1]], dtype=torch.int32,
                         device="cuda").view(1, 2, 2, 3).contiguous()
    out, lse = block_sparse_attention(q, k, v, lists, return_lse=True)
    _check(out, lse, q, k, v, lists, None)
    counts = torch.tensor([[[9, -3], [0, 2]]], dtype=torch.int32, device="cuda")  # held to 0..3
    out, lse = block_sparse_attention(q, k, v, lists, counts, return_lse=True)
    _check(out, lse, q, k, v, lists, counts)


def test_growing_scores_rescale():
    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    s = 1024
    ramp = torch.linspace(0.2, 2.0, s, device="cuda")[None, :, None, None]
    for dtype in (torch.bfloat16, torch.float16):
        q, v = _randn((1, s, 2, 128), 4, dtype, 3.0), _randn((1, s, 2, 128), 6, dtype)
        k = (_randn((1, s, 2, 128), 5, torch.float32, 3.0) * ramp).to(dtype)
        for flip in (False, True):
            order = torch.arange(8, dtype=torch.int32, device="cuda")
            indices = (order.flip(0) if flip else order).expand(1, 2, 8, 8).contiguous()
            out, lse = block_sparse_attention(q, k, v, indices, return_lse=True)
            _check(out, lse, q, k, v, indices, None)


def test_strided_views_out_and_scale():
    """Views into one packed buffer, heads before rows, an output inside a larger tensor."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    packed = _randn((2, 500, 3, 3 * 128), 1)
    q, k, v = (packed[..., i * 128:(i + 1) * 128] for i in range(3))
    indices, counts = _lists(2, 3, 4, 4, 3, 2)
    whole = torch.full((2, 500, 5, 136), 7.0, device="cuda", dtype=torch.bfloat16)
    out = whole[:, :, 1:4, :128]
    got, lse = block_sparse_attention(q, k, v, indices, counts, softmax_scale=0.3, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    _check(out, lse, q, k, v, indices, counts, scale=0.3)
    assert (whole[:, :, 0] == 7).all() and (whole[:, :, 4] == 7).all() and (whole[..., 128:] == 7).all()
    qt, kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    again = block_sparse_attention(qt, kt, vt, indices, counts, softmax_scale=0.3)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,block_q,block_k,sq,sk,h,hk", [(128, 128, 128, 1000, 1300, 4, 2), (64, 256, 64, 900, 2049, 3, 3),
                                                         (128, 256, 64, 1, 777, 8, 1), (64, 128, 128, 4000, 130, 1, 1)])
def test_select(dtype, d, block_q, block_k, sq, sk, h, hk):
    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    q, k = _randn((2, sq, h, d), 1, dtype), _randn((2, sk, hk, d), 2, dtype)
    nk = -(-sk // block_k)
    for top_k in (1, max(1, nk // 3), nk, nk + 5):
        got, n = select_key_blocks(q, k, top_k, block_q=block_q, block_k=block_k)
        ref, ref_n = sparse_ref.select(q, k, top_k, block_q=block_q, block_k=block_k)
        assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


def test_select_ties_kept_blocks_and_nan():
    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    # whole-number means: exact scores, many of them equal
    g = torch.Generator().manual_seed(3)
    blocks = torch.randint(-1, 2, (1, 40, 2, 128), generator=g).to(torch.bfloat16)
    k = blocks.repeat_interleave(128, 1).cuda()
    q = torch.randint(-1, 2, (1, 9, 2, 128), generator=g).to(torch.bfloat16).repeat_interleave(128, 1).cuda()
    q[:, :128] = 0.0  # every score 0: the lowest indices
    q[:, 128:256] = -0.0
    keep = torch.zeros(40, dtype=torch.bool, device="cuda")
    keep[[37, 39]] = True
    for mask in (None, keep):
        for top_k in (1, 2, 7, 39):
            got, n = select_key_blocks(q, k, top_k, keep=mask)
            ref, ref_n = sparse_ref.select(q, k, top_k, keep=mask)
            assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)
    k[:, 5 * 128 + 3, 0] = float("nan")
    k[:, 6 * 128 + 3, 1] = float("inf")
    got, n = select_key_blocks(q, k, 39)
    ref, ref_n = sparse_ref.select(q, k, 39)
    assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


@pytest.mark.parametrize("q_scale,k_scale", [(1e-32, 1.0), (1e-36, 1e30), (1e18, 1e19), (1e-20, 1e-19), (0.0, 1.0), (3e38, 1.0)])
def test_select_extreme_scales(q_scale, k_scale):
    """Means whose products leave fp32's range, or too small for their digits: fp64 decides."""

    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    q, k = _randn((1, 300, 2, 64), 1, torch.float32), _randn((1, 5000, 2, 64), 2, torch.float32)
    q = (q.clamp(-1, 1) * q_scale).to(torch.bfloat16)
    k = (k.clamp(-1, 1) * k_scale).to(torch.bfloat16)
    got, n = select_key_blocks(q, k, 11)
    ref, ref_n = sparse_ref.select(q, k, 11)
    assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


@pytest.mark.parametrize("sk", [1500, 2048, 5000, 64 * 4200])
@pytest.mark.parametrize("q_scale,k_scale", [(1e20, 1e20), (1e24, 1e17), (1e37, 3e3), (1e21, 1e20)])
def test_select_scores_beyond_fp32(q_scale, k_scale, sk):
    """Products of norms from 1e36 to 1e42: fp32 sums overflow on the way to scores that fp64 holds."""

    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    q, k = _randn((1, 900, 2, 64), 1, torch.float32), _randn((1, sk, 2, 64), 2, torch.float32)
    # (block sizes over three decades: in a row, some sums overflow and others do not)
    size = 10.0 ** -(3 * torch.rand(1, -(-sk // 64), 1, 1, device="cuda", generator=torch.Generator("cuda").manual_seed(3)))
    k = k * size.repeat_interleave(64, 1)[:, :sk]
    q = (q.clamp(-3, 3) * q_scale).to(torch.bfloat16)
    k = (k.clamp(-3, 3) * k_scale).to(torch.bfloat16)
    assert torch.isfinite(q).all() and torch.isfinite(k).all()
    blocks = -(-sk // 64)
    for top_k in (3, blocks // 4, blocks // 2):
        got, n = select_key_blocks(q, k, top_k, block_k=64)
        ref, ref_n = sparse_ref.select(q, k, top_k, block_k=64)
        assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


@pytest.mark.parametrize("dtype,low,high", [(torch.float16, -24, 15), (torch.bfloat16, -20, 17)])
def test_lists_do_not_depend_on_the_batch(dtype, low, high):
    """Columns that mix magnitudes as far apart as fp64 sums hold exactly, and cancel: an entry alone (means
    of few blocks, four warps each) chooses like the same entry in a large batch (a warp each)."""

    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    g = torch.Generator(device="cuda").manual_seed(7)
    b, s, h, d = 12, 1600, 8, 64

    def mixed(seq):
        sign = torch.randint(0, 2, (b, seq, h, d), generator=g, device="cuda") * 2 - 1
        x = sign * 2.0 ** torch.randint(low, high + 1, (b, seq, h, d), generator=g, device="cuda").float()
        x[:, 1::2] = torch.where(torch.rand(b, seq // 2, h, d, generator=g, device="cuda") < 0.9, -x[:, 0::2], x[:, 1::2])
        return x.to(dtype)

    q, k = mixed(s), mixed(s)
    assert b * h * (-(-s // 128) + -(-s // 64)) > 148 * 16 > h * (-(-s // 128) + -(-s // 64))
    got, _ = select_key_blocks(q, k, 5, block_k=64)
    for i in range(b):
        alone, _ = select_key_blocks(q[i : i + 1], k[i : i + 1], 5, block_k=64)
        assert torch.equal(alone[0], got[i])
    ref, _ = sparse_ref.select(q[:1], k[:1], 5, block_k=64)
    assert torch.equal(got[:1].cpu(), ref)


def test_select_close_scores():
    """Blocks that differ in the last bits of their means only, in groups of more and fewer than a warp."""

    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    g = torch.Generator().manual_seed(5)
    for groups in (40, 3):
        base = torch.randn(1, groups, 1, 128, generator=g).repeat_interleave(120 // groups, 1)
        k = base.repeat_interleave(64, 1).to(torch.bfloat16)
        k[:, ::64, 0, :4] += torch.randint(-1, 2, (1, 120, 4), generator=g).to(torch.bfloat16) * 2.0**-7
        q = torch.randn(1, 640, 1, 128, generator=g).to(torch.bfloat16)
        for top_k in (1, 17, 50, 119):
            got, n = select_key_blocks(q.cuda(), k.cuda(), top_k, block_k=64)
            ref, ref_n = sparse_ref.select(q, k, top_k, block_k=64)
            assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


def test_select_long_rows():
    """More key blocks than a warp keeps in registers."""

    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    for sk in (128 * 1700, 64 * 6500 + 1):
        q, k = _randn((1, 520, 1, 64), 1), _randn((1, sk, 1, 64), 2)
        for block_k in (64, 128):
            got, n = select_key_blocks(q, k, 50, block_k=block_k)
            ref, ref_n = sparse_ref.select(q, k, 50, block_k=block_k)
            assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


@pytest.mark.parametrize("nk,top_k", [(200, 20), (256, 255), (257, 26), (500, 90), (513, 1), (800, 80), (1025, 300), (2036, 204), (2049, 64), (3900, 390)])
def test_select_row_lengths(nk, top_k):
    """Rows of every size that a lane's registers come in, with kept blocks, a padded batch and
    heads that share keys."""

    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    sk = nk * 64 - 5
    q, k = _randn((2, 300, 4, 64), 1), _randn((2, sk, 2, 64), 2)
    k_lens = torch.tensor([sk, sk // 3], dtype=torch.int32, device="cuda")
    keep = torch.zeros(nk, dtype=torch.bool, device="cuda")
    keep[[0, nk // 5, nk - 1]] = True
    for mask in (None, keep):
        got, n = select_key_blocks(q, k, top_k, block_k=64, k_lens=k_lens, keep=mask)
        ref, ref_n = sparse_ref.select(q, k, top_k, block_k=64, k_lens=k_lens, keep=mask)
        assert torch.equal(got.cpu(), ref) and torch.equal(n.cpu(), ref_n)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,sq,sk,h,hk", [(2, 700, 9000, 40, 40), (3, 500, 17000, 36, 12), (1, 17000, 300, 96, 96)])
def test_select_many_heads(d, b, sq, sk, h, hk):
    """More tiles of scores than SMs, ragged in both directions; heads that share keys cross tiles."""

    from h3_flash_b200.runtime.attention.sparse import select_key_blocks

    q, k = _randn((b, sq, h, d), 1), _randn((b, sk, hk, d), 2)
    top_k = max(1, sk // 64 // 9)
    got, n = select_key_blocks(q, k, top_k, block_k=64)
    # (the oracle walks head by head: a few of them, with their own keys)
    for head in (0, h // 2 + 1, h - 1):
        kv = head // (h // hk)
        ref, ref_n = sparse_ref.select(q[:, :, head : head + 1], k[:, :, kv : kv + 1], top_k, block_k=64)
        assert torch.equal(got[:, head : head + 1].cpu(), ref) and torch.equal(n[:, head : head + 1].cpu(), ref_n)


def test_offsets_past_32_bits():
    """A key tensor of more than 2^32 bytes and 2^31 elements: the last blocks are read where they are."""

    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention, select_key_blocks

    s, h = 1100000, 16
    k = torch.zeros((1, s, h, 128), device="cuda", dtype=torch.bfloat16)
    assert k.numel() > 2**31
    k[:, -300:] = _randn((1, 300, h, 128), 1)
    q, tail = _randn((1, 5, h, 128), 2), s // 128 - 2
    nk = -(-s // 128)
    indices = torch.tensor([nk - 1, nk - 3], dtype=torch.int32, device="cuda").expand(1, h, 1, 2).contiguous()
    out, lse = block_sparse_attention(q, k, k, indices, return_lse=True)
    lo = (nk - 3) * 128
    part = k[:, lo:].contiguous()
    moved = (indices - (nk - 3)).contiguous()
    _check(out, lse, q, part, part, moved, None)
    got, _ = select_key_blocks(q[:, :, :1], k[:, :, :1], 2)
    ref, _ = sparse_ref.select(q[:, :, :1], k[:, :, :1], 2)
    assert torch.equal(got.cpu(), ref) and tail > 0


def test_all_blocks_equal_dense_attention():
    """With every block listed in order the result is the dense op's within one rounding."""

    from h3_flash_b200.runtime.attention.dense import attention_bshd
    from h3_flash_b200.runtime.attention.sparse import sparse_attention

    q, k, v = (_randn((1, 1000, 3, 128), i) for i in (1, 2, 3))
    out = sparse_attention(q, k, v, 1000)
    assert (out.float() - attention_bshd(q, k, v).float()).abs().max() <= 2 * _half_step(torch.bfloat16) * 4


def test_packed_run_select_then_attend():
    from h3_flash_b200.runtime.attention.sparse import packed_sparse_attention

    packed = _randn((1400, 3, 384), 1)
    keep = torch.arange(11, device="cuda") == 10
    out, lse = packed_sparse_attention(packed, 4, keep=keep, return_lse=True)
    q, k, v = (packed[None, ..., i * 128:(i + 1) * 128] for i in range(3))
    indices, counts = sparse_ref.select(q, k, 4, keep=keep)
    assert (indices == 10).any(-1).all()
    _check(out[None], lse[None], q, k, v, indices, counts)


def test_graph_capture_and_second_stream():
    """Captured once, replayed on new inputs; two captured calls keep their own workspaces."""

    from h3_flash_b200.runtime.attention.sparse import sparse_attention

    q, k, v = (_randn((1, 300, 2, 128), i) for i in (1, 2, 3))
    q1 = _randn((1, 1, 2, 128), 9)
    sparse_attention(q, k, v, 2), sparse_attention(q1, k, v, 3)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, n in ((q, 2), (q1, 3)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sparse_attention(x, k, v, n))
        graphs.append(g)
    for t, seed in ((q, 11), (k, 12), (v, 13), (q1, 14)):
        t.copy_(_randn(t.shape, seed))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for x, n, out in ((q, 2, outs[0]), (q1, 3, outs[1])):
        assert torch.equal(out, sparse_attention(x, k, v, n))
        indices, counts = sparse_ref.select(x, k, n)
        _check(out, None, x, k, v, indices, counts)


def test_same_bits_every_time():
    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention

    q, k, v = (_randn((1, 1000, 4, 128), i) for i in (1, 2, 3))
    indices, counts = _lists(1, 4, 8, 8, 6, 4)
    first = block_sparse_attention(q, k, v, indices, counts)
    for _ in range(5):
        assert torch.equal(first, block_sparse_attention(q, k, v, indices, counts))


def test_refusals():
    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention, packed_sparse_attention, select_key_blocks

    q, k, v = (_randn((1, 256, 2, 128), i) for i in (1, 2, 3))
    idx = torch.zeros(1, 2, 2, 1, dtype=torch.int32, device="cuda")
    for bad, error in (
        (lambda: block_sparse_attention(q.float(), k.float(), v.float(), idx), TypeError),
        (lambda: block_sparse_attention(q, k.half(), v, idx), TypeError),
        (lambda: block_sparse_attention(q, k, v[:, :100], idx), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx.long()), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx[:, :1]), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx, torch.ones(1, 2, 3, dtype=torch.int32, device="cuda")), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx, block_q=64), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx, block_k=32), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx, softmax_scale=0.0), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx, softmax_scale=float("nan")), ValueError),
        (lambda: block_sparse_attention(q[..., :96], k[..., :96], v[..., :96], idx), RuntimeError),
        (lambda: block_sparse_attention(q[..., 1:65], k[..., :64], v[..., :64], idx), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx, out=q[:, :100]), ValueError),
        (lambda: block_sparse_attention(q, k, v, idx.cpu()), RuntimeError),
        (lambda: block_sparse_attention(q.clone().requires_grad_(), k, v, idx), RuntimeError),
        (lambda: select_key_blocks(q, k, 0), ValueError),
        (lambda: select_key_blocks(q, k[:, :, :1].expand(-1, -1, 3, -1), 1), ValueError),
        (lambda: select_key_blocks(q, k, 1, keep=torch.ones(3, dtype=torch.bool, device="cuda")), ValueError),
        (lambda: select_key_blocks(q, k[:, :0], 1), ValueError),
        (lambda: packed_sparse_attention(q[0], 1), ValueError),
    ):
        with pytest.raises(error):
            bad()
    with torch.no_grad():
        block_sparse_attention(q.clone().requires_grad_(), k, v, idx)


def test_empty_calls():
    from h3_flash_b200.runtime.attention.sparse import block_sparse_attention, select_key_blocks

    q, k, v = (_randn((1, 256, 2, 128), i) for i in (1, 2, 3))
    none = torch.zeros(1, 2, 2, 0, dtype=torch.int32, device="cuda")
    out, lse = block_sparse_attention(q, k, v, none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = block_sparse_attention(q, k[:, :0], v[:, :0], torch.zeros(1, 2, 2, 1, dtype=torch.int32, device="cuda"),
                                      return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert block_sparse_attention(q[:, :0], k, v, none[:, :, :0]).shape == (1, 0, 2, 128)
    assert select_key_blocks(q[:, :0], k, 1)[0].shape == (1, 2, 0, 1)
