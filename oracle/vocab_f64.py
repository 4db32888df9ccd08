"""The operators at the vocabulary from their definitions, in float64 on the CPU (test
infrastructure).  Inputs are float arrays holding exactly the values the kernels see (16-bit
tensors widened), indices integer arrays."""
from __future__ import annotations

import numpy as np


def embedding(x, ids, scale=1.0, first_row=0):
    x = np.asarray(x, np.float64)
    ids = np.asarray(ids).astype(object) - first_row  # no overflow at the ends of int64
    out = np.zeros(ids.shape + (x.shape[1],))
    for at in np.ndindex(ids.shape):
        if 0 <= ids[at] < x.shape[0]:
            out[at] = float(scale) * x[ids[at]]
    return out


def embedding_dx(dy, ids, num_weight, scale=1.0, padding_idx=None, first_row=0):
    """(gradient, sum of the magnitudes that were added, number of them), each by rows."""
    width = dy.shape[-1]
    dy = np.asarray(dy, np.float64).reshape(-1, width)
    dx = np.zeros((num_weight, width))
    size = np.zeros((num_weight, width))
    count = np.zeros(num_weight, np.int64)
    for t, i in enumerate(np.asarray(ids).reshape(-1).tolist()):
        r = i - first_row
        if 0 <= r < num_weight and (padding_idx is None or i != padding_idx):
            dx[r] += dy[t]
            size[r] += np.abs(dy[t])
            count[r] += 1
    return float(scale) * dx, abs(float(scale)) * size, count


def topk_distill(z, indices, teacher, temperature=1.0, soft_weight=1.0, labels=None, hard_weight=0.0, dloss=None):
    """Dictionary of loss, stats, dlogits (for dloss) and, for error bounds, per row and column the
    parts that cancel: ``soft`` and ``p`` (both times |dloss| soft T), ``hard`` (times |dloss hard|)."""
    z = np.asarray(z, np.float64)
    teacher = np.asarray(teacher, np.float64)
    n, v = z.shape
    t = float(temperature)
    dloss = np.ones(n) if dloss is None else np.broadcast_to(np.asarray(dloss, np.float64), (n,))
    loss, stats, grad = np.zeros(n), np.zeros((n, 3)), np.zeros((n, v))
    soft_part, p_part, hard_part, cross = np.zeros((n, v)), np.zeros((n, v)), np.zeros((n, v)), np.zeros(n)
    with np.errstate(all="ignore"):
        for i in range(n):
            idx = np.asarray(indices[i]).tolist()
            there = [j for j, c in enumerate(idx) if 0 <= c < v and teacher[i, j] != -np.inf] if soft_weight != 0 else []
            label = -1 if labels is None or hard_weight == 0 else int(labels[i])
            has_label = 0 <= label < v
            if not there and not has_label:
                continue
            m = np.max(z[i]) if v else -np.inf
            stats[i, 0] = m
            if there:
                a = teacher[i, there] / t
                logp = a - np.max(a) - np.log(np.sum(np.exp(a - np.max(a))))
                p = np.exp(logp)
                stats[i, 1] = np.log(np.sum(np.exp((z[i] - m) / t)))
                logq = (z[i] - m) / t - stats[i, 1]
                terms = [pj * (lp - logq[idx[j]]) for pj, lp, j in zip(p, logp, there) if pj != 0]
                cross[i] = sum(abs(pj * ((teacher[i, j] - np.max(teacher[i, there])) - (z[i, idx[j]] - m)) / t)
                               for pj, j in zip(p, there) if pj != 0)
                loss[i] += soft_weight * t * t * np.sum(terms)
                soft_part[i] = np.exp(logq)
                for pj, j in zip(p, there):
                    p_part[i, idx[j]] += pj
                grad[i] += dloss[i] * soft_weight * t * (soft_part[i] - p_part[i])
            if has_label:
                stats[i, 2] = np.log(np.sum(np.exp(z[i] - m)))
                logq = z[i] - m - stats[i, 2]
                loss[i] += hard_weight * -logq[label]
                hot = np.zeros(v)
                hot[label] = 1.0
                grad[i] += dloss[i] * hard_weight * (np.exp(logq) - hot)
                hard_part[i] = (np.exp(logq) + hot) * abs(dloss[i] * hard_weight)
            soft_part[i] *= abs(dloss[i] * soft_weight) * t
            p_part[i] *= abs(dloss[i] * soft_weight) * t
    return {"loss": loss, "stats": stats, "dlogits": grad, "soft": soft_part, "p": p_part, "hard": hard_part, "cross": cross}
