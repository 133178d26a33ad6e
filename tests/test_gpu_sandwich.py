"""The sandwich-norm ops against fp64.

Bounds: each output is rounded once (u = eps/2). fp32 leaves, in a sum of squares over a
row of at most 2^14 values, at most 2^-17 relative (64 sequential additions per thread and a
tree), half of that in its root, and a few 2^-24 per product: 2^-17 of the terms' sizes.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(rows, cols, dtype, table=3, seed=0, lead=(1,)):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    return dict(residual=t(*lead, rows, cols), branch=t(*lead, rows, cols, std=3.0), post_weight=t(cols, std=0.1, mean=1.0),
                weight=t(cols, std=0.1, mean=1.0), tables=t(table, 3 * cols, std=0.3),
                index=torch.randint(0, table, (rows,), generator=g, device="cuda"))


def _check(got, s, post_eps, eps, scale_by, index=None):
    hidden, normed = got
    cols = s["residual"].shape[-1]
    u = torch.finfo(s["residual"].dtype).eps / 2
    idx = s["index"] if index is None else index
    gate, scale, shift = (t.double()[idx] for t in s["tables"].chunk(3, -1))
    b = s["branch"].double()
    b = b * torch.rsqrt(b.square().mean(-1, keepdim=True) + post_eps) * s["post_weight"].double()
    h = scale_by * s["residual"].double() + gate * b
    size = (scale_by * s["residual"].double()).abs() + (gate * b).abs()
    tiny = 2.0**-24 if s["residual"].dtype == torch.float16 else 2.0**-120  # half a subnormal step
    bound = u * h.abs() * (1 + 2.0**-6) + 2.0**-17 * size + tiny
    assert ((hidden.double() - h).abs() <= bound).all()
    if normed is None:
        return
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
    factor = rstd * s["weight"].double() * (1 + scale)
    n = h * factor + shift
    # an error of 2^-17 of the row's sizes in h moves its root mean square by as much
    size_n = size * factor.abs() + shift.abs() + h.abs() * factor.abs() * rstd * size.square().mean(-1, keepdim=True).sqrt()
    bound = u * n.abs() * (1 + 2.0**-6) + 2.0**-17 * size_n + tiny
    assert ((normed.double() - n).abs() <= bound).all()
    assert hidden.shape[-1] == cols


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (5, 64), (2, 1000), (7, 1001), (33, 1536), (64, 3072), (9, 4096),
                                       (4, 5376), (3, 8192), (2, 16384), (2, 16392)])
@pytest.mark.parametrize("scale_by", [1.0, 0.75])
def test_sandwich(dtype, rows, cols, scale_by):
    from h3_flash_b200.runtime.kernels.fusions import fused_sandwich_residual, fused_sandwich_residual_rmsnorm_modulate

    s = _inputs(rows, cols, dtype)
    gate, scale, shift = s["tables"].chunk(3, -1)
    got = fused_sandwich_residual_rmsnorm_modulate(s["residual"], s["branch"], s["post_weight"], gate, s["weight"], scale, shift,
                                                   s["index"], 1e-6, 1e-5, residual_scale=scale_by)
    _check(got, s, 1e-6, 1e-5, scale_by)
    closing = fused_sandwich_residual(s["residual"], s["branch"], s["post_weight"], gate, s["index"], 1e-6, residual_scale=scale_by)
    _check((closing, None), s, 1e-6, 1e-5, scale_by)
    assert torch.equal(closing, got[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_short_index(dtype):
    """Rows inside a wider tensor, at an odd offset, a one-row table and an index that repeats."""

    from h3_flash_b200.runtime.kernels.fusions import fused_sandwich_residual_rmsnorm_modulate as op

    s = _inputs(12, 640, dtype, table=4)
    gate, scale, shift = s["tables"].chunk(3, -1)
    wide = torch.zeros(12, 700, dtype=dtype, device="cuda")
    for offset in (0, 8, 3):
        wide[:, offset:offset + 640] = s["branch"][0]
        branch = wide[:, offset:offset + 640].unsqueeze(0)
        _check(op(s["residual"], branch, s["post_weight"], gate, s["weight"], scale, shift, s["index"], 1e-6, 1e-5), s, 1e-6, 1e-5, 1.0)
    index = torch.tensor([2, 0, 3, 1], device="cuda")
    _check(op(s["residual"], s["branch"], s["post_weight"], gate, s["weight"], scale, shift, index, 1e-6, 1e-5), s, 1e-6, 1e-5, 1.0,
           index.repeat(3))
    one = dict(s, tables=s["tables"][:1])
    _check(op(s["residual"], s["branch"], s["post_weight"], gate[0], s["weight"], scale[0], shift[0], None, 1e-6, 1e-5), one, 1e-6,
           1e-5, 1.0, torch.zeros(12, dtype=torch.int64, device="cuda"))
    outside = torch.tensor([-1, 0, 4, 2**40], device="cuda")  # the nearest rows
    _check(op(s["residual"], s["branch"], s["post_weight"], gate, s["weight"], scale, shift, outside, 1e-6, 1e-5), s, 1e-6, 1e-5, 1.0,
           torch.tensor([0, 0, 3, 3], device="cuda").repeat(3))


def test_zero_and_extreme_rows():
    """An all-zero branch gives the scaled residual; large and tiny branches are normalised alike."""

    from h3_flash_b200.runtime.kernels.fusions import fused_sandwich_residual_rmsnorm_modulate as op

    s = _inputs(4, 1024, torch.bfloat16)
    s["branch"][:, 0] = 0.0
    s["branch"][:, 1] *= 1e15
    s["branch"][:, 2] *= 1e-3
    s["residual"][:, 3] = 0.0
    gate, scale, shift = s["tables"].chunk(3, -1)
    got = op(s["residual"], s["branch"], s["post_weight"], gate, s["weight"], scale, shift, s["index"], 1e-6, 1e-5)
    _check(got, s, 1e-6, 1e-5, 1.0)
    assert torch.equal(got[0][:, 0], s["residual"][:, 0])


def test_graph_capture():
    from h3_flash_b200.runtime.kernels.fusions import fused_sandwich_residual_rmsnorm_modulate as op

    s = _inputs(40, 512, torch.bfloat16)
    gate, scale, shift = s["tables"].chunk(3, -1)
    args = (s["residual"], s["branch"], s["post_weight"], gate, s["weight"], scale, shift, s["index"], 1e-6, 1e-5)
    op(*args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = op(*args)
    new = _inputs(40, 512, torch.bfloat16, seed=5)
    for name, t in new.items():
        s[name].copy_(t)
    g.replay()
    torch.cuda.synchronize()
    _check(got, s, 1e-6, 1e-5, 1.0)


def test_refusals():
    from h3_flash_b200.runtime.kernels.fusions import fused_sandwich_residual as op

    s = _inputs(4, 64, torch.bfloat16)
    gate = s["tables"][:, :64]
    for args, error in (
        ((s["residual"].float(), s["branch"], s["post_weight"], gate, None, 1e-6), TypeError),
        ((s["residual"].double(), s["branch"].double(), s["post_weight"].double(), gate.double(), None, 1e-6), TypeError),
        ((s["residual"], s["branch"][:, :3], s["post_weight"], gate, None, 1e-6), ValueError),
        ((s["residual"], s["branch"], s["post_weight"][:32], gate, None, 1e-6), ValueError),
        ((s["residual"], s["branch"], s["post_weight"], gate[:, :32], None, 1e-6), ValueError),
        ((s["residual"], s["branch"], s["post_weight"], gate, s["index"][:0], 1e-6), ValueError),
        ((s["residual"], s["branch"], s["post_weight"].cpu(), gate, None, 1e-6), RuntimeError),
        ((s["residual"], s["branch"].clone().requires_grad_(), s["post_weight"], gate, None, 1e-6), RuntimeError),
    ):
        with pytest.raises(error):
            op(*args)
    assert op(s["residual"][:, :0], s["branch"][:, :0], s["post_weight"], gate, None, 1e-6).shape == (1, 0, 64)
