"""64-bit reference forms of the serving-step operators (squish_b200.ops.step), on the CPU."""
import math

import numpy as np
import torch

PAD_Q0 = 1 << 30


def layout_ref(ctx, q, table, free, ps, tile, cap, tile_cap):
    """Lists in, dict of int lists out; the table is changed in place."""
    out = dict(q_start=[0], kv_len=[], positions=[], slots=[], token_seq=[], last_row=[], tile_seq=[], tile_q0=[])
    used = 0
    for b, (c, n) in enumerate(zip(ctx, q)):
        for i in range(-(-c // ps), -(-(c + n) // ps)):
            table[b][i] = free[used]
            used += 1
        for p in range(c, c + n):
            page = table[b][p // ps]
            out["positions"].append(p)
            out["slots"].append(page * ps + p % ps if page >= 0 else -1)
            out["token_seq"].append(b)
        out["q_start"].append(out["q_start"][-1] + n)
        out["kv_len"].append(c + n)
        out["last_row"].append(out["q_start"][-1] - 1 if n else -1)
        for s in range(0, n, tile):
            out["tile_seq"].append(b)
            out["tile_q0"].append(s)
    out["totals"] = [len(out["positions"]), used, len(out["tile_seq"])]
    for k, v in (("positions", 0), ("slots", -1), ("token_seq", -1)):
        out[k] += [v] * (cap - len(out[k]))
    for k, v in (("tile_seq", 0), ("tile_q0", PAD_Q0)):
        out[k] += [v] * (tile_cap - len(out[k]))
    return out


def sample_ref(row, u, temp, top_p=1.0, top_k=0, min_p=0.0, allow=None):
    """(token, log-probability) of one row (float64 numpy values of the bf16 logits)."""
    x = np.asarray(row, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if allow is not None:
        x[~allow] = -np.inf
    if not (x > -np.inf).any():
        return -1, -np.inf
    if not temp > 0:
        return int(np.argmax(x)), 0.0
    idx = np.lexsort((np.arange(len(x)), -x))
    idx = idx[x[idx] > -np.inf]
    v = x[idx]
    with np.errstate(invalid="ignore"):
        z = np.where(v == v[0], 0.0, (v - v[0]) / float(np.float32(temp)))
    w = np.exp(z)
    n = len(w)
    if top_k > 0:
        n = min(n, top_k)
    n = min(n, max(1, int((w >= float(np.float32(min_p))).sum())))
    cum = np.cumsum(w)
    tp = float(np.float32(top_p))
    if tp < 1.0:
        n = min(n, max(1, int((cum < tp * cum[-1]).sum()) + 1))
    total = cum[n - 1]
    at = min(int((cum[:n] <= float(np.float32(u)) * total).sum()), n - 1)
    return int(idx[at]), float(z[at] - math.log(total))


def route_ref(logits, k, score="softmax", bias=None, groups=1, top_groups=None, group_score="max", renorm=True,
              scale=1.0):
    """(ids [T, k] int64, weights [T, k] float64)."""
    x = logits.double().cpu().numpy().copy()
    x[np.isnan(x)] = -np.inf
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        if score == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-x))
        else:
            m = x.max(-1, keepdims=True)
            e = np.where(x == m, 1.0, np.exp(x - m))
            e = np.where(x == -np.inf, 0.0, e)
            z = e.sum(-1, keepdims=True)
            s = np.where(z > 0, e / np.where(z > 0, z, 1.0), 0.0)
    # without a bias both scores order the experts as the logits do
    c = x.copy() if bias is None else s + bias.double().cpu().numpy()
    c[np.isnan(c)] = -np.inf
    T, E = x.shape
    gs = E // groups
    top_groups = groups if top_groups is None else top_groups
    ids = np.zeros((T, k), dtype=np.int64)
    w = np.zeros((T, k))
    for t in range(T):
        open_ = set(range(groups))
        if groups > 1:
            gsc = []
            for g in range(groups):
                if group_score == "max" or gs == 1:
                    gsc.append(c[t, g * gs:(g + 1) * gs].max())
                else:
                    v = s[t] if bias is None else c[t]
                    gsc.append(np.sort(v[g * gs:(g + 1) * gs])[-2:].sum())
            open_ = set(sorted(range(groups), key=lambda g: (-gsc[g], g))[:top_groups])
        cand = [e for e in range(E) if e // gs in open_]
        pick = sorted(cand, key=lambda e: (-c[t, e], e))[:k]
        ids[t] = pick
        v = s[t, pick]
        if renorm:
            v = v / v.sum() if v.sum() > 0 else np.zeros(k)
        w[t] = v * scale
    return ids, w


def lora_ref(x, y, rows, adapters, silu=False):
    """(out, bound) in float64: the exact result and the error that fp32 sums over K terms, h held
    as two bf16 (2^-16 of it), a sum that starts from y (at most 16 steps of 16 ranks, each off by up
    to 2^-23 of y: 2^-19 |y|) and one rounding to bf16 (half a step: 2^-8 relative) may reach.
    ``adapters``: {slot: (A, B, scale)}."""
    x64, out = x.double().cpu(), y.double().cpu().clone()
    K = x.shape[1]
    slack = out.abs() * 2.0**-19
    for s, (a, b, sc) in adapters.items():
        sel = (rows.cpu() == s).nonzero().flatten()
        if not sel.numel():
            continue
        a, b, sc = a.double().cpu(), b.double().cpu(), float(np.float32(sc))
        out[sel] += (x64[sel] @ a.T) @ b.T * sc
        mass = (x64[sel].abs() @ a.abs().T) @ b.abs().T * abs(sc)
        slack[sel] += mass * (2.0**-16 + (K + 128) * 2.0**-23)
    if silu:
        m, n = out.shape
        g, u = out.view(m, n // 128, 2, 64).unbind(2)
        dg, du = slack.view(m, n // 128, 2, 64).unbind(2)
        sg = g * torch.sigmoid(g)
        # |silu'| <= 1.1; the exponential's argument rounds by 2^-24 |g| log2 e and the exponential and
        # reciprocal by 3 ulp: together below 2^-18 of the result for |g| <= 40; results below
        # 1.1e-36 |u| may be flushed
        slack = 1.1 * dg * u.abs() + sg.abs() * du + dg * du + (sg * u).abs() * 2.0**-18 + 1.1e-36 * u.abs()
        out, slack = (sg * u).reshape(m, n // 2), slack.reshape(m, n // 2)
    return out, out.abs() * 2.0**-8 + slack + 2.0**-126
