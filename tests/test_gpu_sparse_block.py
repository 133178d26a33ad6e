"""Blocks that run sparse attention and sandwich norms together, as they are installed.

Bars as for the dense block: max-abs 2e-2 above half a bf16 spacing of the element, cosine 0.9999.
"""

from __future__ import annotations

import pytest
import torch

from oracle import sparse_ref

pytestmark = pytest.mark.gpu


def _setup(rows, dim, heads, activation="gelu-tanh", blocks=1, seed=0, **kw):
    from h3_flash_b200.runtime.h3_block import H3BlockStack, H3TransformerBlock
    from h3_flash_b200.workloads import init_block_, rope_tables

    stack = H3BlockStack([init_block_(H3TransformerBlock(dim=dim, heads=heads, head_dim=128, ffn_inner=4 * dim,
                                                         activation=activation, **kw), seed=seed + i) for i in range(blocks)])
    stack = stack.to(device="cuda", dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(seed + 1)
    hidden = torch.randn(1, rows, dim, generator=g).to(torch.bfloat16).cuda()
    idx = torch.randint(0, 3, (rows,), generator=g).cuda()
    pos = torch.stack([torch.arange(rows) // 64, (torch.arange(rows) // 8) % 8, torch.arange(rows) % 8], -1)
    cos, sin = rope_tables(pos, 96)
    return stack, hidden, idx, (cos.cuda(), sin.cuda())


def _attention_reference(attention, x, rope, runtime):
    """The module's own projections and norms in fp64, then the reference's selection and attention."""

    a, rows = attention, x.shape[1]

    def project(layer, norm):
        t = (x[0].double() @ layer.weight.double().T + layer.bias.double()).view(rows, a.heads, 128)
        if norm is not None:
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
            cos, sin = (c.double()[:, None] for c in rope)
            r = t[..., :96]
            t = torch.cat([r * cos + torch.cat([-r[..., 48:], r[..., :48]], -1) * sin, t[..., 96:]], -1)
        return t[None].cpu()

    q, k, v = project(a.to_q, a.norm_q), project(a.to_k, a.norm_k), project(a.to_v, None)
    keep = runtime._keep_mask(rows, x.device)
    q16, k16 = q.to(torch.bfloat16), k.to(torch.bfloat16)
    indices, counts = sparse_ref.select(q16, k16, runtime.list_length(rows), block_q=runtime.block_q, block_k=runtime.block_k,
                                        keep=keep.cpu() if keep is not None else None)
    out = sparse_ref.attend(q, k, v, indices, counts, block_q=runtime.block_q, block_k=runtime.block_k)[0]
    o = a.to_out[0]
    return out[0].reshape(rows, -1).cuda() @ o.weight.double().T + o.bias.double(), (indices, counts)


def _check(got, ref):
    got, ref = got.double().flatten(), ref.double().flatten()
    assert torch.isfinite(got).all()
    spacing = 2.0 ** torch.floor(torch.log2(ref.abs().clamp_min(2.0**-20))) * 2.0**-8
    assert ((got - ref).abs() - spacing).max() <= 2e-2
    assert torch.nn.functional.cosine_similarity(got, ref, dim=0) >= 0.9999


@pytest.mark.parametrize("block_q,block_k,keep", [(128, 128, 0), (256, 64, 70)])
def test_attention_module_is_sparse(block_q, block_k, keep):
    from h3_flash_b200.runtime.attention import install_sparse_attention, remove_sparse_attention
    from h3_flash_b200.runtime.kernels import install_transformer_fusions

    stack, hidden, idx, rope = _setup(1300, 256, 2)
    attention = stack.transformer_blocks[0].attn
    install_transformer_fusions(stack)
    x = torch.randn(1, 1300, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(torch.bfloat16)
    with torch.no_grad():
        dense = attention.forward(x, rope)
        meta = install_sparse_attention(stack, density=0.3, block_q=block_q, block_k=block_k, keep_last_rows=keep)
        sparse = attention.forward(x, rope)
        ref, (indices, counts) = _attention_reference(attention, x, rope, meta["runtime"])
        assert meta["runtime"].calls == 1
        # A block whose score the bf16 projections put on the other side of the border gives other
        # rows: of the lists, at most a few differ; the rest is held to the bar.
        from h3_flash_b200.runtime.attention.sparse import select_key_blocks
        from h3_flash_b200.runtime.kernels.fusions import fused_qkv_gemm_pack
        from h3_flash_b200.runtime.parallel.packed_ulysses import qkv_weights

        w, b = qkv_weights(attention)
        packed = fused_qkv_gemm_pack(x, w, b, attention.norm_q.weight, attention.norm_k.weight, *rope, 2, 1, attention.norm_q.eps,
                                     attention.norm_k.eps)[0]
        got, n = select_key_blocks(packed[None, ..., :128], packed[None, ..., 128:256], meta["runtime"].list_length(1300),
                                   block_q=block_q, block_k=block_k, keep=meta["runtime"]._keep_mask(1300, x.device))
        same = (got.cpu() == indices).all(-1).all(1)[0]  # per query block, all heads
        assert same.float().mean() >= 0.7
        rows = same.repeat_interleave(block_q)[:1300].cuda()
        _check(sparse[0][rows], ref[rows])
        remove_sparse_attention(stack)
        assert torch.equal(attention.forward(x, rope), dense)


def _sandwich_reference(block, hidden, idx, attention_output):
    """The block after attention, in fp64."""

    norm = lambda t, m: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + m.eps) * m.weight.double()  # noqa: E731
    _, _, gate1, shift2, scale2, gate2 = (t.double()[idx] for t in block.adaln_proj())
    h = block.residual_scale * hidden.double() + gate1 * norm(attention_output.double(), block.norm1_post)
    n = norm(h, block.norm2) * (1 + scale2) + shift2
    act, _, out = block.ff.net
    y = n @ act.proj.weight.double().T + act.proj.bias.double()
    if hasattr(act, "approximate"):
        y = torch.nn.functional.gelu(y, approximate="tanh")
    else:
        value, gate = y.chunk(2, -1)
        y = value * torch.nn.functional.silu(gate)
    f = y @ out.weight.double().T + out.bias.double()
    return block.residual_scale * h + gate2 * norm(f, block.norm2_post)


@pytest.mark.parametrize("rows,dim,heads,activation,scale", [(300, 384, 3, "gelu-tanh", 1.0), (1000, 256, 2, "swiglu", 0.75)])
def test_sandwich_block(rows, dim, heads, activation, scale):
    from h3_flash_b200.runtime.kernels import install_transformer_fusions

    stack, hidden, idx, rope = _setup(rows, dim, heads, activation, sandwich_norm=True, residual_scale=scale)
    block = stack.transformer_blocks[0]
    seen = {}
    with torch.no_grad():
        eager = stack(hidden, None, idx, rope)
        runtime = install_transformer_fusions(stack)
        forward = block.attn.forward
        block.attn.forward = lambda *a, **k: seen.setdefault("out", forward(*a, **k))
        out = stack(hidden, None, idx, rope)
        ref = _sandwich_reference(block, hidden, idx, seen["out"])
    _check(out, ref)
    assert (out.double() - ref).abs().mean() <= (eager.double() - ref).abs().mean()
    assert {"sandwich_output", "sandwich_chain", "rmsnorm_modulate"} <= set(runtime["gate"])
    assert runtime["gate"]["sandwich_chain"]["cosine"] > 0.9999
    # without the fused AdaLN ops the same math runs eagerly
    with torch.no_grad():
        del block.attn.forward
        plain, _, _, _ = _setup(rows, dim, heads, activation, sandwich_norm=True, residual_scale=scale)
        install_transformer_fusions(plain, modulate=False)
        _check(plain(hidden, None, idx, rope), ref)


def test_the_first_call_compares_every_sandwich_step():
    from h3_flash_b200.runtime.kernels import install_transformer_fusions, transformer

    stack, hidden, idx, rope = _setup(300, 256, 2, sandwich_norm=True, residual_scale=0.5)
    runtime = install_transformer_fusions(stack)
    with torch.no_grad():
        first = stack(hidden, None, idx, rope)
        assert {"sandwich_output", "sandwich_chain", "sandwich_closing"} <= set(runtime["gate"])
        assert runtime["gate"]["sandwich_closing"]["cosine"] > 0.9999
        seen = dict(runtime["gate"])
        assert torch.equal(stack(hidden, None, idx, rope), first) and runtime["gate"] == seen
        # a closing step that is off shows
        other, _, _, _ = _setup(300, 256, 2, sandwich_norm=True, residual_scale=0.5)
        runtime = install_transformer_fusions(other)
        right = transformer.fused_sandwich_residual
        transformer.fused_sandwich_residual = lambda *a, residual_scale: right(*a, residual_scale=1.0)
        try:
            other(hidden, None, idx, rope)
        finally:
            transformer.fused_sandwich_residual = right
    assert runtime["gate"]["sandwich_closing"]["relative_l2"] > 0.1


def test_sparse_sandwich_stack_runs_captured_like_eagerly():
    """Two blocks with everything installed: selection, sparse attention, sandwich norms, GEMMs;
    replayed from a graph on new rows it gives the bits of the eager run."""

    from h3_flash_b200 import _lib
    from h3_flash_b200.runtime.attention import install_sparse_attention
    from h3_flash_b200.runtime.kernels import install_transformer_fusions

    stack, hidden, idx, rope = _setup(900, 256, 2, blocks=2, sandwich_norm=True)
    install_transformer_fusions(stack)
    meta = install_sparse_attention(stack, density=0.4, keep_last_rows=100)
    with torch.no_grad():
        for _ in range(2):
            stack(hidden, None, idx, rope)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = stack(hidden, None, idx, rope)
        assert meta["runtime"].calls == 6
        hidden.copy_(torch.randn(hidden.shape, device="cuda").to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, stack(hidden, None, idx, rope))
    assert torch.isfinite(replayed).all() and _lib.device_status() == 0


def _packed(rows, seed):
    return torch.randn(rows, 2, 384, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(torch.bfloat16)


def test_captured_kept_blocks_outlive_other_lengths():
    """Captured at one length after a warm-up, then run at others: replays still keep their blocks."""

    from h3_flash_b200.runtime.attention.sparse import SparseAttention

    runtime = SparseAttention(0.1, keep_last_rows=300)
    packed = _packed(2000, 1)
    runtime.attend(packed, 128)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = runtime.attend(packed, 128)
    for i in range(20):
        runtime.attend(_packed(900 + 128 * i, 2), 128)
        full = [torch.full((512,), 255, dtype=torch.uint8, device="cuda") for _ in range(50)]
    packed.copy_(_packed(2000, 3))
    graph.replay()
    torch.cuda.synchronize()
    q, k, v = (packed[None, ..., i * 128:(i + 1) * 128] for i in range(3))
    keep = torch.arange(16) >= 13  # rows 1700 to 1999 lie in blocks 13 to 15
    indices, counts = sparse_ref.select(q, k, runtime.list_length(2000), keep=keep)
    _check(out, sparse_ref.attend(q, k, v, indices, counts)[0][0].cuda())
    assert torch.equal(out, runtime.attend(packed, 128)) and full


@pytest.mark.parametrize("rows", [0, 1, 127, 129])
def test_shortest_sequences(rows):
    """None to a few rows: what the dense op answers (all blocks are kept, or there is one)."""

    from h3_flash_b200.runtime.attention.dense import packed_attention
    from h3_flash_b200.runtime.attention.sparse import SparseAttention

    packed = _packed(rows, 5)
    out = SparseAttention(0.1, keep_first_rows=100, keep_last_rows=3).attend(packed, 128)
    dense = packed_attention(packed)
    assert out.shape == dense.shape == (rows, 2, 128) and torch.isfinite(out).all()
    if rows:
        _check(out, dense)


def test_two_lengths_on_two_streams():
    from h3_flash_b200.runtime.attention.sparse import SparseAttention

    runtime = SparseAttention(0.2, block_k=64, keep_last_rows=100)
    sets = [_packed(3000, 1), _packed(2100, 2)]
    want = [runtime.attend(p, 128) for p in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (stream, p) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                got[i].append(runtime.attend(p, 128))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def _record(runtime):
    """What the runtime's attention calls get and give, in order."""

    calls, attend = [], runtime.attend
    runtime.attend = lambda packed, head_dim: calls.append((packed.clone(), attend(packed, head_dim))) or calls[-1][1]
    return calls


def _check_call(packed, out, runtime, keep):
    """Every row of one packed attention call, against the lists that the oracle chooses from the same rows.

    The bound: weights rounded once (half a step each), the output once, and what fp32 leaves of scores
    and exponentials (128 products that truncate, 2^-18)."""

    q, k, v = (packed[None, ..., i * 128:(i + 1) * 128] for i in range(3))
    kw = dict(block_q=runtime.block_q, block_k=runtime.block_k)
    indices, counts = sparse_ref.select(q, k, runtime.list_length(packed.shape[0]), keep=keep, **kw)
    ref, _, weight_abs, score_abs = sparse_ref.attend(q, k, v, indices, counts, **kw)
    u = torch.finfo(packed.dtype).eps / 2
    slack = 128 * 2.0**-23 * score_abs + 2.0**-18
    bound = (u + 2 * slack.transpose(1, 2)[..., None]) * weight_abs + u * ref.abs() * (1 + 2.0**-6) + 2.0**-24
    assert ((out[None].double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("block_q,block_k,first,last", [(128, 128, 0, 0), (256, 64, 0, 70), (128, 64, 130, 0), (256, 128, 1, 300)])
def test_every_row_of_the_module_follows_its_list(block_q, block_k, first, last):
    from h3_flash_b200.runtime.attention import install_sparse_attention
    from h3_flash_b200.runtime.kernels import install_transformer_fusions

    rows = 1300
    stack, hidden, idx, rope = _setup(rows, 256, 2)
    attention = stack.transformer_blocks[0].attn
    install_transformer_fusions(stack)
    runtime = install_sparse_attention(stack, density=0.3, block_q=block_q, block_k=block_k, keep_first_rows=first,
                                       keep_last_rows=last)["runtime"]
    calls = _record(runtime)
    x = torch.randn(1, rows, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(torch.bfloat16)
    with torch.no_grad():
        got = attention.forward(x, rope)
    starts = torch.arange(0, rows, block_k)
    keep = (starts < first) | ((starts + block_k).clamp(max=rows) > rows - last)
    (packed, out), = calls
    _check_call(packed, out, runtime, keep)
    o = attention.to_out[0]
    _check(got[0], out.reshape(rows, -1).double() @ o.weight.double().T + o.bias.double())


def test_transformer_keeps_its_text_and_audio():
    """A whole transformer: text first, then video, then audio; text and audio are attended to by all rows."""

    from h3_flash_b200.runtime.attention import install_sparse_attention
    from h3_flash_b200.runtime.h3_model import H3Transformer, make_inputs
    from h3_flash_b200.runtime.kernels import install_transformer_fusions

    torch.manual_seed(0)
    model = H3Transformer(256, 2, 128, 512, 2, text_dim=64, video_channels=32, audio_channels=16, freq_dim=64, freqs_per_axis=16)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if "norm" in name and name.endswith("weight") and p.dim() == 1:
                p.copy_(1.0 + 0.02 * torch.randn_like(p))
            else:
                p.normal_(0.0, 0.05)
    model = model.to("cuda", torch.bfloat16).eval()
    n_text, n_video, n_audio = 77, 6 * 12 * 16, 30
    inputs = make_inputs(model, n_text=n_text, n_video=n_video, n_audio=n_audio, text_dim=64, grid=(6, 12, 16), device="cuda",
                         dtype=torch.bfloat16)
    install_transformer_fusions(model)
    with torch.no_grad():
        dense = model(**inputs)
        runtime = install_sparse_attention(model, density=0.25, block_k=64, keep_first_rows=n_text,
                                           keep_last_rows=n_audio)["runtime"]
        calls = _record(runtime)
        sparse = model(**inputs)
    rows = n_text + n_video + n_audio
    starts = torch.arange(0, rows, 64)
    keep = (starts < n_text) | ((starts + 64).clamp(max=rows) > n_text + n_video)
    assert keep.tolist() == [True] * 2 + [False] * (len(keep) - 3) + [True] and runtime.list_length(rows) == 5
    assert len(calls) == 2
    for packed, out in calls:
        _check_call(packed, out, runtime, keep)
    assert torch.isfinite(sparse.sample).all() and not torch.equal(sparse.sample, dense.sample)
    with torch.no_grad():
        runtime.density = 1.0
        _check(model(**inputs).sample, dense.sample)


def test_full_density_is_dense_attention():
    from h3_flash_b200.runtime.attention import install_sparse_attention
    from h3_flash_b200.runtime.kernels import install_transformer_fusions

    stack, hidden, idx, rope = _setup(700, 256, 2)
    install_transformer_fusions(stack)
    with torch.no_grad():
        dense = stack(hidden, None, idx, rope)
        install_sparse_attention(stack, density=1.0)
        _check(stack(hidden, None, idx, rope), dense)
