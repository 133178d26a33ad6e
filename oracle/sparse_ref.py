"""Block selection and block-sparse attention in fp64, block by block, from their definitions."""

from __future__ import annotations

import math

import torch


def _rows(lens, b: int, seq: int) -> int:
    return seq if lens is None else max(0, min(seq, int(lens[b])))


def block_means(x: torch.Tensor, lens, block: int) -> list[torch.Tensor]:
    """Per batch entry: the mean rows of the blocks that have rows, fp64 sums held in fp32,
    as fp64 [blocks, H, D]."""

    means = []
    for b in range(x.shape[0]):
        n = _rows(lens, b, x.shape[1])
        rows = [x[b, i : min(i + block, n)].double().mean(0).float().double() for i in range(0, n, block)]
        means.append(torch.stack(rows) if rows else torch.zeros(0, *x.shape[2:], dtype=torch.float64))
    return means


def select(q, k, top_k, *, block_q=128, block_k=128, q_lens=None, k_lens=None, keep=None):
    """indices int32 [B, H, nq, top_k] (ascending, -1 behind the last) and counts int32 [B, H, nq]."""

    q, k = q.cpu(), k.cpu()
    b_, sq, h_, _ = q.shape
    nq, nk, group = -(-sq // block_q), -(-k.shape[1] // block_k), h_ // k.shape[2]
    top_k = min(top_k, nk)
    indices = torch.full((b_, h_, nq, top_k), -1, dtype=torch.int32)
    counts = torch.zeros((b_, h_, nq), dtype=torch.int32)
    q_mean, k_mean = block_means(q, q_lens, block_q), block_means(k, k_lens, block_k)
    for b in range(b_):
        for h in range(h_):
            score = q_mean[b][:, h] @ k_mean[b][:, h // group].T
            for i in range(score.shape[0]):
                def rank(j, i=i):
                    s = float(score[i, j])
                    return (keep is None or not bool(keep[j]), math.inf if math.isnan(s) else -s, j)

                best = sorted(sorted(range(score.shape[1]), key=rank)[:top_k])
                indices[b, h, i, : len(best)] = torch.tensor(best, dtype=torch.int32)
                counts[b, h, i] = len(best)
    return indices, counts


def attend(q, k, v, indices, counts=None, *, block_q=128, block_k=128, scale=None, q_lens=None, k_lens=None):
    """(out [B, Sq, H, D], lse [B, H, Sq], weight_abs, score_abs) in fp64: weight_abs is
    softmax(s) |v|, the size of what rounded weights can be off by; score_abs [B, H, Sq] the
    largest scale * |q| . |k| of a row. A key listed twice counts twice."""

    q, k, v, indices = (t.cpu() for t in (q, k, v, indices))
    b_, sq, h_, d = q.shape
    group, nk = h_ // k.shape[2], -(-k.shape[1] // block_k)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(b_, sq, h_, d, dtype=torch.float64)
    weight_abs = torch.zeros_like(out)
    lse = torch.full((b_, h_, sq), -math.inf, dtype=torch.float64)
    score_abs = torch.zeros_like(lse)
    for b in range(b_):
        n_q, n_k = _rows(q_lens, b, sq), _rows(k_lens, b, k.shape[1])
        for h in range(h_):
            for i in range(indices.shape[2]):
                lo, hi = i * block_q, min((i + 1) * block_q, n_q)
                n = indices.shape[3] if counts is None else max(0, min(indices.shape[3], int(counts[b, h, i])))
                keys = [c for j in indices[b, h, i, :n].tolist() if 0 <= j < nk
                        for c in range(j * block_k, min((j + 1) * block_k, n_k))]
                if lo >= hi or not keys:
                    continue
                rows, at = q[b, lo:hi, h].double(), k[b, keys, h // group].double()
                values = v[b, keys, h // group].double()
                s = rows @ at.T * scale
                p = torch.softmax(s, -1)
                out[b, lo:hi, h] = p @ values
                weight_abs[b, lo:hi, h] = p @ values.abs()
                lse[b, h, lo:hi] = torch.logsumexp(s, -1)
                score_abs[b, h, lo:hi] = (rows.abs() @ at.abs().T).amax(-1) * scale
    return out, lse, weight_abs, score_abs
