"""Plain statements in 64 bits of decoding over a paged key / value cache (tests only): appending with rotation,
attention of new tokens over the cache, drawing a token. Loops over sequences, heads and rows; CPU tensors."""
import math

import numpy as np
import torch


def spans(B, N, kv_len, cu_q, cap):
    """(first row, end, keys) per sequence, as the library reads them."""
    out = []
    for b in range(B):
        first, end = (b, b + 1) if cu_q is None else (max(int(cu_q[b]), 0), min(int(cu_q[b + 1]), N))
        out.append((first, end, min(max(int(kv_len[b]), 0), cap)))
    return out


def rotate(x, pos, inv_freq, interleaved):
    """x [..., D] f64 at one position."""
    half = len(inv_freq)
    a = float(pos) * inv_freq.double()
    c, s = torch.cos(a), torch.sin(a)
    y = x.clone()
    if interleaved:
        x1, x2 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def append(k, v, kp, vp, table, kv_len, cu_q=None, q=None, inv_freq=None, interleaved=False, pos=None, q_out=None):
    """-> (q_out, kp, vp) in f64; rows without a sequence keep q_out's values."""
    B, W = table.shape
    P, page = kp.shape[:2]
    kp, vp = kp.double().clone(), vp.double().clone()
    qo = None if q is None else q_out.double().clone()
    turn = (lambda x, p: rotate(x.double(), p, inv_freq, interleaved)) if inv_freq is not None else (lambda x, p: x.double())
    for b, (first, end, n) in enumerate(spans(B, k.shape[0], kv_len, cu_q, W * page)):
        for i in range(first, end):
            at = n - (end - first) + i - first
            p = at if pos is None else int(pos[i])
            if q is not None:
                qo[i] = turn(q[i], p)
            pg = int(table[b, at // page]) if 0 <= at < n else -1
            if 0 <= pg < P:
                kp[pg, at % page] = turn(k[i], p)
                vp[pg, at % page] = v[i].double()
    return qo, kp, vp


def attend(q, kp, vp, table, kv_len, cu_q=None, scale=None, causal=True, window=0, out=None):
    """-> (out f64, bound): bound [N, Hq, D] = sum_j p_j |v_j|, what relative errors of the probabilities act on, and
    spread [N, Hq] = scale max_j sum_d |q_d k_jd|, what errors of the scores are relative to."""
    N, Hq, D = q.shape
    B, W = table.shape
    P, page, Hk = kp.shape[:3]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(N, Hq, D, dtype=torch.float64) if out is None else out.double().clone()
    bound, spread = torch.zeros(N, Hq, D, dtype=torch.float64), torch.zeros(N, Hq, dtype=torch.float64)
    q = q.double()
    for b, (first, end, n) in enumerate(spans(B, N, kv_len, cu_q, W * page)):
        if end <= first:
            continue
        j = torch.arange(n)
        pg = table[b, (j // page).long()].long() if n else torch.zeros(0, dtype=torch.long)
        real = (pg >= 0) & (pg < P)
        j, pg = j[real], pg[real]
        K, V = kp[pg, j % page].double(), vp[pg, j % page].double()
        for i in range(first, end):
            p = n - (end - first) + i - first
            see = torch.ones(len(j), dtype=torch.bool)
            if causal:
                see &= j <= p
            if window:
                see &= j > p - window
            for h in range(Hq):
                Kh, Vh = K[see, h // (Hq // Hk)], V[see, h // (Hq // Hk)]
                x = (Kh * q[i, h]).sum(-1) * scale
                if not len(x) or x.max() == -math.inf:
                    out[i, h] = 0
                    continue
                w = torch.exp(x - x.max())
                w = w / w.sum()
                out[i, h] = (w[:, None] * Vh).sum(0)
                bound[i, h] = (w[:, None] * Vh.abs()).sum(0)
                spread[i, h] = abs(scale) * (Kh * q[i, h]).abs().sum(-1).max()
    return out, bound, spread


def sample(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """-> (tokens, probs) lists; x [B, V] of any float type."""
    tokens, probs = [], []
    for b in range(x.shape[0]):
        row = x[b].double().numpy().copy()
        row[np.isnan(row)] = -np.inf
        get = lambda t, off: off if t is None else float(t[b])  # noqa: E731
        T, k, tp, mp = get(temperature, 1.0), int(get(top_k, 0)), get(top_p, 1.0), get(min_p, 0.0)
        if row.max() == -np.inf:
            tokens.append(-1)
            probs.append(0.0)
            continue
        if not T > 0:
            tokens.append(int(np.argmax(row)))
            probs.append(1.0)
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            p = np.where(row == row.max(), 1.0, np.exp((row - row.max()) / min(T, 1e30)))
        order = np.argsort(-row, kind="stable")
        order = order[p[order] > 0]
        if k > 0:
            order = order[:k]
        if tp < 1:
            s = np.cumsum(p[order])
            order = order[np.concatenate([[True], s[:-1] < max(tp, 0.0) * s[-1]])]
        if mp > 0:
            order = order[p[order] >= min(mp, 1.0)]
        kept = np.sort(order)
        s = np.cumsum(p[kept])
        at = min(int(np.searchsorted(s, max(float(u[b]), 0.0) * s[-1], side="right")), len(kept) - 1)
        tokens.append(int(kept[at]))
        probs.append(p[kept[at]] / s[-1])
    return tokens, probs
