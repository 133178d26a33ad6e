"""Cases, plain forms and exact values of the sparse-attention and sandwich-norm operators.

Four operators and one composition are covered:

- ``select``    which key blocks each block of queries attends to: the mean query and the
                mean key of every block, their products, the ``top_k`` best
                (``runtime.attention.sparse.select_key_blocks``)
- ``attend``    softmax attention of every block of queries over its own list of key blocks
                (``runtime.attention.sparse.block_sparse_attention``)
- ``sparse``    both in one call, on the packed [S, heads, 3 * head_dim] buffer of the
                attention path (``runtime.attention.sparse.packed_sparse_attention``)
- ``sandwich``  RMSNorm after a branch, its gate, the scaled residual, RMSNorm before the next
                branch and its modulation (``runtime.kernels.fusions.
                fused_sandwich_residual_rmsnorm_modulate``)
- ``closing``   the same without the norm before the next branch
                (``fused_sandwich_residual``)

A block is 128 or 256 queries and 64 or 128 keys. Rows past a batch entry's length hold
whatever a padded batch holds there (NaN here) and must not reach any result.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------

def _attention_case(op, *, batch=1, sq, sk, heads, kv_heads=None, dim=128, block_q=128, block_k=128, top_k, dtype="bf16",
                    ragged=False, kept=0):
    return {"op": op, "batch": batch, "sq": sq, "sk": sk, "heads": heads, "kv_heads": kv_heads or heads, "dim": dim,
            "block_q": block_q, "block_k": block_k, "top_k": top_k, "dtype": dtype, "ragged": ragged, "kept": kept}


def _norm_case(op, *, rows, cols, dtype="bf16", table=3, residual_scale=1.0):
    return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "table": table, "residual_scale": residual_scale}


def listed():
    return [
        # All 24 heads of the 480p-5s sequence (51,200 rows) on one GPU, lists of 64-key blocks.
        dict(_attention_case("select", sq=51200, sk=51200, heads=24, block_k=64, top_k=80), name="select-480p5s-24h"),
        # One query row per sequence against four long padded caches, keys shared by groups of heads.
        dict(_attention_case("select", batch=4, sq=1, sk=130304, heads=24, kv_heads=3, top_k=102, dtype="fp16", ragged=True),
             name="select-one-query"),
        # The three heads that one of eight ranks holds of the 480p-5s sequence; a tenth of the keys.
        dict(_attention_case("attend", sq=51200, sk=51200, heads=3, top_k=40), name="attend-480p5s-3h"),
        # The same share of the 768p-5s sequence, a twentieth of the keys, lists per 256 queries.
        dict(_attention_case("attend", sq=130304, sk=130304, heads=3, block_q=256, top_k=51), name="attend-768p5s-3h"),
        # A padded batch of odd lengths, one of them empty: 64-wide heads in fp16, 64-key blocks, grouped heads.
        dict(_attention_case("attend", batch=4, sq=4097, sk=4351, heads=6, kv_heads=2, dim=64, block_k=64, top_k=12, dtype="fp16",
                             ragged=True), name="attend-ragged-fp16"),
        # One query row over a tenth of the 768p-5s keys: latency and key bandwidth.
        dict(_attention_case("attend", sq=1, sk=130304, heads=24, top_k=102), name="attend-one-query"),
        # Selection and attention of one layer on the packed buffer of one rank of eight; the
        # audio rows behind the video (10 blocks) are always attended to.
        dict(_attention_case("sparse", sq=51200, sk=51200, heads=3, top_k=40, kept=10), name="sparse-480p5s-3h"),
        # The smallest configured sequence (4 x 32 x 32 patches and 256 audio rows).
        dict(_attention_case("sparse", sq=4352, sk=4352, heads=3, top_k=6, kept=2), name="sparse-small"),
        # Between the branches of a block, at the width and rows of one GPU's 480p-5s step.
        dict(_norm_case("sandwich", rows=51200, cols=3072), name="sandwich-480p5s"),
        # A single row at an odd width.
        dict(_norm_case("sandwich", rows=1, cols=1001, dtype="fp32", residual_scale=0.5), name="sandwich-one-row"),
        # The end of a block: one rank's rows of eight at the wide model width, fp16.
        dict(_norm_case("closing", rows=6400, cols=5376, dtype="fp16", residual_scale=0.75), name="closing-5376-fp16"),
        # The end of a block, all rows of one GPU.
        dict(_norm_case("closing", rows=51200, cols=3072), name="closing-480p5s"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["select", "attend", "attend", "sparse", "sandwich", "closing"])
    if op in ("sandwich", "closing"):
        cols = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            cols = -(-cols // 8) * 8
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return _norm_case(op, rows=min(_log_int(rng, 1, 51200), 314_000_000 // (cols * _TYPES[dtype].itemsize)), cols=cols, dtype=dtype,
                          table=rng.randint(1, 6), residual_scale=rng.choice([1.0, 0.5, 1.25]))
    block_q, block_k = rng.choice([128, 256]), rng.choice([64, 128])
    if op == "sparse":
        s, heads = _log_int(rng, 1, 51200), rng.randint(1, 4)
        blocks = -(-s // block_k)
        top_k = max(1, min(blocks, int(blocks * rng.uniform(0.05, 0.3))))
        dim, limit = 128, 51200 * 40 * 128 * 3
        top_k = max(1, min(top_k, limit // (s * block_k * heads)))
        return _attention_case(op, sq=s, sk=s, heads=heads, dim=dim, block_q=block_q, block_k=block_k, top_k=top_k,
                               dtype=rng.choice(["bf16", "fp16"]), kept=rng.choice([0, min(2, top_k)]))
    batch, kv_heads = rng.randint(1, 3), rng.randint(1, 4)
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    sq = 1 if rng.random() < 0.25 else _log_int(rng, 1, 32000)
    sk = _log_int(rng, 1, 100000)
    blocks = -(-sk // block_k)
    top_k = max(1, min(blocks, int(blocks * rng.uniform(0.05, 0.3))))
    limit = 130304 * 51 * 128 * 3
    while batch * heads * sq * top_k * block_k > limit and top_k > 1:
        top_k -= 1
    while batch * heads * sq * top_k * block_k > limit:
        sq = (sq + 1) // 2
    return _attention_case(op, batch=batch, sq=sq, sk=sk, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]), block_q=block_q,
                           block_k=block_k, top_k=top_k, dtype=rng.choice(["bf16", "fp16"]), ragged=rng.random() < 0.5)


def _lens(case, length, seed):
    """Row counts of a padded batch: the whole length, none, and odd ones between."""

    if not case["ragged"]:
        return None
    rng = np.random.RandomState(seed % (1 << 31))
    lens = [length, 0] + [int(x) for x in rng.randint(length // 2, length + 1, max(0, case["batch"] - 2))]
    return (lens if case["batch"] > 1 else [max(1, length - length // 3)])[:case["batch"]]


def work(case):
    if case["op"] in ("sandwich", "closing"):
        size = _TYPES[case["dtype"]].itemsize
        cells = case["rows"] * case["cols"]
        tables, streams = (4, 4) if case["op"] == "sandwich" else (2, 3)
        return {"bytes": cells * streams * size + tables * case["cols"] * size + case["rows"] * 8, "flops": cells * (14 if case["op"] == "sandwich" else 7)}
    b, h, hk, d, bq, bk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "block_q", "block_k"))
    nq, nk, top = -(-case["sq"] // bq), -(-case["sk"] // bk), case["top_k"]
    q_bytes, kv_bytes, list_bytes = 2 * b * case["sq"] * h * d, 2 * b * case["sk"] * hk * d, 4 * b * h * nq * (top + 1)
    select_flops = b * h * (case["sq"] + case["sk"]) * d + 2 * b * h * nq * nk * d
    if case["op"] == "select":
        return {"bytes": q_bytes + kv_bytes + list_bytes, "flops": select_flops}
    attend_flops = 4 * b * h * case["sq"] * min(case["sk"], top * bk) * d
    read = min(kv_bytes, 2 * b * h * nq * top * bk * d)  # few lists do not touch every key
    if case["op"] == "attend":
        return {"bytes": 2 * q_bytes + 2 * read + list_bytes + 4 * b * h * case["sq"], "flops": attend_flops}
    return {"bytes": 2 * q_bytes + 2 * kv_bytes + 4 * b * h * case["sq"], "flops": select_flops + attend_flops}


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------

def _normed_rows(g, batch, seq, heads, dim, dtype):
    """Rows as QK-norm leaves them: neighbours alike (a direction per 64 rows, drifting), RMS about one."""

    anchors = torch.randn(batch, -(-seq // 64) + 2, heads, dim, generator=g, device="cuda")
    anchors = anchors[:, :-2] + anchors[:, 1:-1] + anchors[:, 2:]
    x = torch.randn(batch, seq, heads, dim, generator=g, device="cuda") + 0.5 * anchors.repeat_interleave(64, 1)[:, :seq]
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True))).to(dtype)


def _random_lists(g, case, nq, nk):
    """Distinct blocks per list, near ones preferred, ascending: what a selection hands over."""

    shape = (case["batch"], case["heads"], nq, nk)
    at = torch.arange(nq, device="cuda")[:, None] / max(1, nq) - torch.arange(nk, device="cuda")[None, :] / max(1, nk)
    score = torch.rand(shape, generator=g, device="cuda") - at.abs()
    return torch.sort(torch.topk(score, min(case["top_k"], nk), dim=-1).indices, dim=-1).values.to(torch.int32)


def prepare(case, seed):
    dtype = _TYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] in ("sandwich", "closing"):
        rows, cols, table = case["rows"], case["cols"], case["table"]

        def tensor(*shape, std=1.0, mean=0.0):
            return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

        state.update(residual=tensor(1, rows, cols), branch=tensor(1, rows, cols, std=3.0), post_weight=tensor(cols, std=0.02, mean=1.0),
                     weight=tensor(cols, std=0.02, mean=1.0), tables=tensor(table, 3 * cols, std=0.1),
                     index=torch.randint(0, table, (rows,), generator=g, device="cuda"))
        return state
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    nq, nk = -(-case["sq"] // case["block_q"]), -(-case["sk"] // case["block_k"])
    q = _normed_rows(g, b, case["sq"], h, d, dtype)
    k = _normed_rows(g, b, case["sk"], hk, d, dtype)
    v = torch.randn(b, case["sk"], hk, d, generator=g, device="cuda").to(dtype) if case["op"] != "select" else None
    if case["op"] == "sparse":
        state["packed"] = torch.cat([q, k, v], dim=-1)[0].contiguous()  # [S, heads, 3 * dim]
        state["keep"] = torch.arange(nk, device="cuda") >= nk - case["kept"] if case["kept"] else None
        return state
    state.update(q=q, k=k, v=v, q_lens=None, k_lens=None)
    q_lens, k_lens = (_lens(case, case["sq"], seed) if case["sq"] > 1 else None), _lens(case, case["sk"], seed + 1)
    for name, lens, tensors in (("q_lens", q_lens, (q,)), ("k_lens", k_lens, (k, v))):
        if lens is None:
            continue
        state[name] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for i, n in enumerate(lens):
            for t in tensors:
                if t is not None:
                    t[i, n:] = float("nan")
    if case["op"] == "attend":
        state["indices"] = _random_lists(g, case, nq, nk)
        state["counts"] = torch.full((b, h, nq), state["indices"].shape[-1], dtype=torch.int32, device="cuda")
        if case["ragged"]:  # lists of differing lengths, some empty
            state["counts"] = torch.randint(0, state["indices"].shape[-1] + 1, (b, h, nq), generator=g, device="cuda").to(torch.int32)
    return state


# ---------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------

def _valid_rows(lens, batch, seq, device):
    """[B, seq] truth values: which rows exist."""

    rows = torch.arange(seq, device=device)[None]
    return rows < lens[:, None] if lens is not None else (rows < seq).expand(batch, seq)


def _blocks(x, size):
    """[B, S, ...] -> [B, blocks, size, ...], filled up with zeros."""

    pad = -x.shape[1] % size
    x = torch.cat([x, x.new_zeros(x.shape[0], pad, *x.shape[2:])], 1) if pad else x
    return x.unflatten(1, (-1, size))


def _means(x, valid, size):
    """Mean row of every block, summed in 64 bits, held in 32: [B, H, blocks, D], and which blocks have rows."""

    total = _blocks(torch.where(valid[:, :, None, None], x, torch.zeros_like(x)).double(), size).sum(2)
    count = _blocks(valid.to(torch.float64), size).sum(2)
    mean = (total / count.clamp_min(1)[:, :, None, None]).float()
    return mean.transpose(1, 2), count > 0


def _plain_select(q, k, top_k, block_q, block_k, q_lens=None, k_lens=None, keep=None):
    batch, _, heads, _ = q.shape
    q_mean, q_there = _means(q, _valid_rows(q_lens, batch, q.shape[1], q.device), block_q)
    k_mean, k_there = _means(k, _valid_rows(k_lens, batch, k.shape[1], k.device), block_k)
    k_mean = k_mean.repeat_interleave(heads // k.shape[2], 1)
    score = q_mean.double() @ k_mean.double().transpose(-1, -2)  # in 64 bits: choices next to a border
    score = torch.where(torch.isnan(score), torch.full_like(score, -math.inf), score)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    rank = torch.ones_like(k_there, dtype=torch.int8) if keep is None else torch.where(keep, 2, 1).to(torch.int8).expand_as(k_there)
    rank = torch.where(k_there, rank, torch.zeros_like(rank))[:, None, None].expand(score.shape)
    best = torch.sort(rank.gather(-1, order), dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, best)[..., :top_k]
    there = (rank.gather(-1, order) > 0) & q_there[:, None, :, None]
    missing = score.shape[-1]
    order = torch.sort(torch.where(there, order, torch.full_like(order, missing)), dim=-1).values
    return torch.where(order < missing, order, torch.full_like(order, -1)).int(), there.sum(-1).int()


def _plain_attend(q, k, v, indices, counts, block_q, block_k, q_lens=None, k_lens=None):
    batch, sq, heads, dim = q.shape
    group, top = heads // k.shape[2], indices.shape[-1]
    k_valid = _valid_rows(k_lens, batch, k.shape[1], q.device)
    k_blocks = _blocks(k, block_k)
    v_blocks = _blocks(torch.where(k_valid[:, :, None, None], v, torch.zeros_like(v)), block_k)
    valid_blocks = _blocks(k_valid, block_k)
    at_b = torch.arange(batch, device=q.device)[:, None, None, None]
    at_h = (torch.arange(heads, device=q.device) // group)[None, :, None, None]
    listed_ = torch.arange(top, device=q.device) < counts[..., None]
    at = torch.where(listed_, indices, torch.zeros_like(indices)).long()
    keys = k_blocks[at_b, at, :, at_h].flatten(3, 4).float()  # [B, H, nq, top * block_k, D]
    there = (valid_blocks[at_b, at] & listed_[..., None]).flatten(3, 4)
    rows = _blocks(q, block_q).permute(0, 3, 1, 2, 4).float()  # [B, H, nq, block_q, D]
    score = (rows @ keys.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    del keys
    score = score.masked_fill(~there[:, :, :, None], -math.inf)
    top_score = score.amax(-1, keepdim=True)
    base = torch.where(top_score == -math.inf, torch.zeros_like(top_score), top_score)
    p = score.sub_(base).exp_()
    total = p.sum(-1, keepdim=True)
    values = v_blocks[at_b, at, :, at_h].flatten(3, 4).float()
    out = p @ values / torch.where(total > 0, total, torch.ones_like(total))
    lse = (base + total.log())[..., 0]
    out = out.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :sq]
    lse = lse.flatten(2, 3)[:, :, :sq]
    q_valid = _valid_rows(q_lens, batch, sq, q.device)
    out = torch.where(q_valid[:, :, None, None], out, torch.zeros_like(out))
    lse = torch.where(q_valid[:, None], lse, torch.full_like(lse, -math.inf))
    return out.to(q.dtype), lse


def _plain_sandwich(s, closing):
    case = s["case"]
    gate, scale, shift = (t.float()[s["index"]] for t in s["tables"].chunk(3, -1))
    branch, residual = s["branch"].float(), s["residual"].float()
    normed = branch * torch.rsqrt(branch.square().mean(-1, keepdim=True) + 1e-6) * s["post_weight"].float()
    hidden = case["residual_scale"] * residual + gate * normed
    if closing:
        return hidden.to(s["branch"].dtype)
    normed = hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + 1e-5) * s["weight"].float()
    return hidden.to(s["branch"].dtype), (normed * (1 + scale) + shift).to(s["branch"].dtype)


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------

def _run_own(s):
    case = s["case"]
    if case["op"] in ("sandwich", "closing"):
        from h3_flash_b200.runtime.kernels.fusions import fused_sandwich_residual, fused_sandwich_residual_rmsnorm_modulate

        gate, scale, shift = s["tables"].chunk(3, -1)
        if case["op"] == "closing":
            return fused_sandwich_residual(s["residual"], s["branch"], s["post_weight"], gate, s["index"], 1e-6,
                                           residual_scale=case["residual_scale"])
        return fused_sandwich_residual_rmsnorm_modulate(s["residual"], s["branch"], s["post_weight"], gate, s["weight"], scale, shift,
                                                        s["index"], 1e-6, 1e-5, residual_scale=case["residual_scale"])
    from h3_flash_b200.runtime.attention import sparse

    blocks = {"block_q": case["block_q"], "block_k": case["block_k"]}
    if case["op"] == "select":
        return sparse.select_key_blocks(s["q"], s["k"], case["top_k"], q_lens=s["q_lens"], k_lens=s["k_lens"], **blocks)
    if case["op"] == "attend":
        return sparse.block_sparse_attention(s["q"], s["k"], s["v"], s["indices"], s["counts"], q_lens=s["q_lens"], k_lens=s["k_lens"],
                                             return_lse=True, **blocks)
    return sparse.packed_sparse_attention(s["packed"], case["top_k"], case["dim"], keep=s["keep"], return_lse=True, **blocks)


def run(state):
    if own:
        return _run_own(state)
    s, case = state, state["case"]
    if case["op"] in ("sandwich", "closing"):
        return _plain_sandwich(s, case["op"] == "closing")
    sizes = (case["block_q"], case["block_k"])
    if case["op"] == "select":
        return _plain_select(s["q"], s["k"], case["top_k"], *sizes, s["q_lens"], s["k_lens"])
    if case["op"] == "attend":
        return _plain_attend(s["q"], s["k"], s["v"], s["indices"], s["counts"], *sizes, s["q_lens"], s["k_lens"])
    q, k, v = (x[None] for x in s["packed"].chunk(3, -1))
    indices, counts = _plain_select(q, k, case["top_k"], *sizes, keep=s["keep"])
    out, lse = _plain_attend(q, k, v, indices, counts, *sizes)
    return out[0], lse[0]


# ---------------------------------------------------------------------------------------
# Exact values, in 64 bits
# ---------------------------------------------------------------------------------------

def _exact_lists(q, k, case, keep):
    """The chosen blocks of one sequence from the definition, block by block: {(head, query block): [key blocks]}."""

    bq, bk = case["block_q"], case["block_k"]
    means = [[x[i:i + size].double().mean(0).float().double() for i in range(0, x.shape[0], size)] for x, size in ((q, bq), (k, bk))]
    q_mean, k_mean = (torch.stack(m).cpu().numpy() for m in means)  # [blocks, H, D]
    first = set(np.nonzero(keep.cpu().numpy())[0].tolist()) if keep is not None else set()
    chosen = {}
    for head in range(q.shape[1]):
        score = np.einsum("id,jd->ij", q_mean[:, head], k_mean[:, head])
        for i in range(score.shape[0]):
            ranked = sorted(range(score.shape[1]), key=lambda j: (j not in first, -score[i, j], j))
            chosen[head, i] = sorted(ranked[:case["top_k"]])
    return chosen


def exact(case, seed):
    if case["op"] == "select":
        return None  # whole numbers: compared as such
    s = prepare(case, seed)
    if case["op"] in ("sandwich", "closing"):
        index = s["index"].cpu()
        table = s["tables"].double().cpu()
        gate, scale, shift = (table[:, i * case["cols"]:(i + 1) * case["cols"]] for i in range(3))
        hidden, normed = [], []
        for part in torch.split(torch.arange(case["rows"]), 4096):
            at = index[part].to("cuda")
            x = s["branch"][0, part].double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["cols"] + 1e-6)
            y = s["residual"][0, part].double() * case["residual_scale"] + x * s["post_weight"].double() * gate.to("cuda")[at]
            hidden.append(y)
            if case["op"] == "sandwich":
                z = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["cols"] + 1e-5) * s["weight"].double()
                normed.append(z + z * scale.to("cuda")[at] + shift.to("cuda")[at])
        whole = [torch.cat(x)[None] for x in (hidden, normed) if x]
        return whole[0] if case["op"] == "closing" else tuple(whole)
    if case["op"] == "sparse":
        d = case["dim"]
        q, k, v = (s["packed"][None, :, :, i * d:(i + 1) * d] for i in range(3))
        lists = [_exact_lists(q[0], k[0], case, s["keep"])]
        q_lens = k_lens = None
    else:
        q, k, v = s["q"], s["k"], s["v"]
        indices, counts = s["indices"].cpu().numpy(), s["counts"].cpu().numpy()
        lists = [{(h, i): indices[b, h, i, :counts[b, h, i]].tolist() for h in range(case["heads"]) for i in range(indices.shape[2])}
                 for b in range(case["batch"])]
        q_lens, k_lens = (x.tolist() if x is not None else None for x in (s["q_lens"], s["k_lens"]))
    batch, sq, heads, dim = q.shape
    bq, bk, group = case["block_q"], case["block_k"], heads // k.shape[2]
    out = torch.zeros(batch, sq, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, heads, sq), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(batch):
        rows_end = sq if q_lens is None else q_lens[b]
        keys_end = k.shape[1] if k_lens is None else k_lens[b]
        for (h, i), blocks in lists[b].items():
            lo, hi = i * bq, min((i + 1) * bq, rows_end)
            keys = np.concatenate([np.arange(j * bk, min((j + 1) * bk, keys_end)) for j in blocks] + [np.arange(0)])
            if lo >= hi or not keys.size:
                continue
            at = torch.from_numpy(keys.astype(np.int64)).to("cuda")
            t = q[b, lo:hi, h].double() @ k[b, :, h // group][at].double().T / math.sqrt(dim)
            lse[b, h, lo:hi] = torch.logsumexp(t, -1)
            out[b, lo:hi, h] = torch.softmax(t, -1) @ v[b, :, h // group][at].double()
    return (out[0], lse[0]) if case["op"] == "sparse" else (out, lse)
