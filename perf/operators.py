"""Measured cases of the serving-step operators.

* ``layout``  -- block tables, slot map and attention tiles of a step from the request lengths
* ``adapter`` -- low-rank adapters of many requests at once beside a shared projection
* ``route``   -- expert routing: softmax or sigmoid scores, balance bias, groups, top-k
* ``sample``  -- temperature / min-p / top-k / top-p sampling from given uniform numbers

``run`` computes them in elementary torch operations, or, where ``own`` is true, through the
package's operators. ``exact`` computes the same from the definitions in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TILE = 32  # queries of one attention tile
PAD_Q0 = 1 << 30  # first query of a padding tile: past every sequence's end


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # decode step of 64 running requests (the benchmark's concurrency), 16-token pages
        dict(name="layout-decode-64", op="layout", seqs=64, kind="decode", max_ctx=2304, chunk=1, budget=64, page=16,
             width=160),
        # chunked prefill riding with decodes: 256 requests, a 4096-token budget
        dict(name="layout-mixed-256", op="layout", seqs=256, kind="mixed", max_ctx=4096, chunk=512, budget=4096, page=16,
             width=288),
        # long-context prefill of a large batch: about a quarter of a million tokens, odd page size
        dict(name="layout-prefill-1000", op="layout", seqs=1000, kind="prefill", max_ctx=32768, chunk=520, budget=250000,
             page=24, width=1400),
        # one decoding request with an adapter on the attention output projection of a 7B model
        dict(name="adapter-o-1", op="adapter", rows=1, k=3584, n=3584, rank=16, slots=8, used=1, bare=0.0,
             layout="scattered", silu=False),
        # 64 decoding requests over 32 adapters, fused qkv of a 7B model, some rows without an adapter
        dict(name="adapter-qkv-64", op="adapter", rows=64, k=3584, n=4608, rank=16, slots=32, used=32, bare=0.1,
             layout="scattered", silu=False),
        # prefill chunks of several requests through gate/up with the SiLU*up epilogue
        dict(name="adapter-gateup-2048", op="adapter", rows=2048, k=3584, n=37888, rank=32, slots=16, used=5, bare=0.2,
             layout="runs", silu=True),
        # long prefill of an 8B model's qkv, large rank, a row count that fills no tile
        dict(name="adapter-qkv-8185", op="adapter", rows=8185, k=4096, n=6144, rank=64, slots=16, used=7, bare=0.1,
             layout="runs", silu=False),
        # decode step of 64 tokens: 256 experts in 8 groups, sigmoid scores with a balance bias
        dict(name="route-sigmoid-64", op="route", tokens=64, experts=256, top_k=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, group_score="top2", renorm=True, scale=2.5, dtype="bf16"),
        # prefill of 16384 tokens through the same router
        dict(name="route-sigmoid-16384", op="route", tokens=16384, experts=256, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, group_score="top2", renorm=True, scale=2.5, dtype="bf16"),
        # softmax scores in fp32 without renormalisation, groups ranked by their best expert, odd sizes
        dict(name="route-softmax-4099", op="route", tokens=4099, experts=160, top_k=6, score="softmax", bias=False,
             groups=8, top_groups=3, group_score="max", renorm=False, scale=16.0, dtype="fp32"),
        # one request, large vocabulary, every filter on
        dict(name="sample-1", op="sample", rows=1, vocab=152064, filters="all", mask=False),
        # a full batch with mixed per-request parameters and a grammar mask
        dict(name="sample-256", op="sample", rows=256, vocab=152064, filters="mixed", mask=True),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layout", "adapter", "route", "sample"])
    if op == "layout":
        kind = rng.choice(["decode", "mixed", "prefill"])
        seqs = _logint(rng, 1, 1000)
        chunk = 1 if kind == "decode" else _logint(rng, 16, 520)
        page = rng.choice([8, 16, 24, 32, 64])
        max_ctx = _logint(rng, 64, 32768)
        budget = seqs if kind == "decode" else min(250000, max(seqs, _logint(rng, 16, seqs * chunk + 16)))
        return dict(op=op, seqs=seqs, kind=kind, max_ctx=max_ctx, chunk=chunk, budget=budget, page=page,
                    width=(max_ctx + 2 * chunk) // page + 2)
    if op == "adapter":
        silu = rng.random() < 0.3
        k = 8 * _logint(rng, 32, 2368)
        n = 128 * _logint(rng, 2, 296) if silu else 8 * _logint(rng, 32, 2368)
        rows = max(1, min(_logint(rng, 1, 8185), int(1.2e8 / (k + 2 * n))))
        slots = rng.choice([1, 4, 16, 32, 48])
        return dict(op=op, rows=rows, k=k, n=n, rank=rng.choice([4, 8, 16, 24, 32, 64]), slots=slots,
                    used=rng.randint(1, min(slots, rows)), bare=rng.choice([0.0, 0.1, 0.5]),
                    layout=rng.choice(["scattered", "runs"]), silu=silu)
    if op == "route":
        experts, groups = rng.choice([(16, 1), (60, 1), (72, 6), (128, 1), (160, 8), (256, 8), (256, 1), (384, 1),
                                      (512, 16)])
        score = rng.choice(["sigmoid", "softmax"])
        bias = rng.random() < 0.6
        top_groups = groups if groups == 1 else rng.randint(max(1, groups // 4), groups)
        return dict(op=op, tokens=_logint(rng, 1, 16384), experts=experts,
                    top_k=rng.randint(1, min(10, experts // groups * top_groups)), score=score, bias=bias, groups=groups,
                    top_groups=top_groups, group_score=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["bf16", "fp32"]))
    return dict(op="sample", rows=_logint(rng, 1, 256), vocab=_logint(rng, 1000, 152064),
                filters=rng.choice(["all", "mixed", "temperature"]), mask=rng.random() < 0.4)


# ----------------------------------------------------------------------------- inputs
def _gen(seed, device=DEV):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    return g


def _layout_inputs(c, seed):
    """Lengths as the scheduler hands them over, a table whose rows hold the cached pages, and
    the free list (the pages of the pool in a shuffled order)."""
    g = _gen(seed, "cpu")
    b, ps = c["seqs"], c["page"]
    ctx = torch.randint(0, c["max_ctx"], (b,), generator=g)
    if c["kind"] == "decode":
        q = torch.ones(b, dtype=torch.int64)
        ctx = ctx.clamp(min=1)
    else:
        q = torch.randint(1, c["chunk"] + 1, (b,), generator=g)
        if c["kind"] == "mixed":  # most requests decode, an eighth prefills a chunk, a few rest
            u = torch.rand(b, generator=g)
            q = torch.where(u < 0.8, torch.ones_like(q), torch.where(u < 0.86, torch.zeros_like(q), q))
    # the scheduler stops at the step's token budget: the rest gets a shorter chunk, then none
    end = torch.cumsum(q, 0).clamp(max=c["budget"])
    q = torch.diff(end, prepend=torch.zeros(1, dtype=torch.int64))
    have = (ctx + ps - 1) // ps
    need = (ctx + q + ps - 1) // ps - have
    pool = torch.randperm(int(have.sum() + need.sum()) + 64, generator=g).to(torch.int32)
    w = c["width"]
    col = torch.arange(w)[None, :]
    table = torch.zeros(b, w, dtype=torch.int32)
    m = col < have[:, None]
    table[m] = pool[: int(m.sum())]
    free = pool[int(m.sum()):]
    to = lambda t: t.to(torch.int32).to(DEV)  # noqa: E731
    return dict(ctx=to(ctx), q=to(q), table=to(table), free=to(free), page=ps, cap=c["budget"],
                tile_cap=c["budget"] // TILE + b)


def _adapter_inputs(c, seed):
    g, h = _gen(seed), _gen(seed + 1, "cpu")
    m, k, n, r, s = c["rows"], c["k"], c["n"], c["rank"], c["slots"]
    bf = torch.bfloat16
    x = torch.randn(m, k, generator=g, device=DEV).to(bf)
    y = torch.randn(m, n, generator=g, device=DEV).to(bf)
    a = (torch.randn(s, r, k, generator=g, device=DEV) / math.sqrt(k)).to(bf)
    b = (torch.randn(s, n, r, generator=g, device=DEV) * 0.1).to(bf)
    # adapters trained at different ranks, up to the pool's
    ranks = [max(1, r // (1 << int(e))) for e in torch.randint(0, 2, (s,), generator=h)]
    scales = [float(v) for v in 0.5 + 1.5 * torch.rand(s, generator=h)]
    pick = torch.randperm(s, generator=h)[: c["used"]]
    if c["layout"] == "scattered":
        rows = pick[torch.randint(0, c["used"], (m,), generator=h)]
        rows = torch.where(torch.rand(m, generator=h) < c["bare"], torch.full_like(rows, -1), rows)
    else:  # requests' chunks one after another
        cuts = max(1, min(m, 2 * c["used"]))
        edge = torch.sort(torch.randint(0, m + 1, (cuts - 1,), generator=h)).values
        seg = torch.bucketize(torch.arange(m), edge, right=True)
        of = pick[torch.arange(cuts) % c["used"]]
        of = torch.where(torch.rand(cuts, generator=h) < c["bare"], torch.full_like(of, -1), of)
        rows = of[seg]
    return dict(x=x, y=y, a=a, b=b, ranks=ranks, scales=scales, rows=rows.to(torch.int32).to(DEV), host_rows=rows,
                silu=c["silu"])


def _route_inputs(c, seed):
    g = _gen(seed)
    t, e = c["tokens"], c["experts"]
    skew = torch.randn(e, generator=g, device=DEV) * 0.5  # some experts are liked more
    logits = torch.randn(t, e, generator=g, device=DEV) * 1.5 + skew
    logits = logits.to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float32)
    bias = (torch.randn(e, generator=g, device=DEV) * 0.05 - 0.1 * skew) if c["bias"] else None
    return dict(logits=logits, bias=bias)


def _sample_inputs(c, seed):
    g = _gen(seed)
    b, v = c["rows"], c["vocab"]
    logits = torch.randn(b, v, generator=g, device=DEV) * 2.0
    # a language model's rows: a few likely tokens above a wide floor, sharper in some rows
    n_top = min(24, v)
    where = torch.randint(0, v, (b, n_top), generator=g, device=DEV)
    lift = 6.0 + 8.0 * torch.rand(b, n_top, generator=g, device=DEV)
    logits.scatter_add_(1, where, lift * torch.rand(b, 1, generator=g, device=DEV))
    logits = logits.to(torch.bfloat16)
    uni = torch.rand(b, generator=g, device=DEV)
    temp = 0.5 + torch.rand(b, generator=g, device=DEV)
    one, zero = torch.ones(b, device=DEV), torch.zeros(b, device=DEV)
    if c["filters"] == "all":
        top_p = 0.8 + 0.19 * torch.rand(b, generator=g, device=DEV)
        min_p = 0.05 * torch.rand(b, generator=g, device=DEV)
        top_k = torch.randint(20, 200, (b,), generator=g, device=DEV)
    elif c["filters"] == "temperature":
        top_p, min_p, top_k = one, zero, zero.long()
    else:  # each request its own: greedy, plain temperature, nucleus, top-k, min-p, all of them
        kind = torch.randint(0, 6, (b,), generator=g, device=DEV)
        temp = torch.where(kind == 0, zero, temp)
        top_p = torch.where((kind == 2) | (kind == 5), 0.7 + 0.29 * torch.rand(b, generator=g, device=DEV), one)
        min_p = torch.where((kind == 4) | (kind == 5), 0.1 * torch.rand(b, generator=g, device=DEV), zero)
        top_k = torch.where((kind == 3) | (kind == 5), torch.randint(1, 500, (b,), generator=g, device=DEV),
                            torch.zeros(b, dtype=torch.int64, device=DEV))
    mask = None
    if c["mask"]:  # a grammar allows half of the vocabulary in every third row, all of it elsewhere
        words = (v + 31) // 32
        mask = torch.randint(-2**31, 2**31, (b, words), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
        free = (torch.arange(b, device=DEV) % 3 != 0)[:, None]
        mask = torch.where(free, torch.full_like(mask, -1), mask)
    return dict(logits=logits, u=uni, temp=temp, top_p=top_p, top_k=top_k.to(torch.int32), min_p=min_p, mask=mask)


_INPUTS = dict(layout=_layout_inputs, adapter=_adapter_inputs, route=_route_inputs, sample=_sample_inputs)


def prepare(case, seed):
    st = _INPUTS[case["op"]](case, seed)
    st["case"] = case
    op = case["op"]
    if op == "adapter":
        rows = st.pop("host_rows")
        # the rows of each adapter, which the plain form works through one after another
        st["groups"] = [(s, torch.nonzero(rows == s).flatten().to(DEV)) for s in sorted(set(rows.tolist())) if s >= 0]
        m, n = st["y"].shape
        st["out"] = torch.empty(m, n // 2 if st["silu"] else n, dtype=torch.bfloat16, device=DEV)
    if not own:
        return st
    from squish_b200 import ops

    if op == "layout":
        st["out"] = ops.StepLayout(case["seqs"], st["cap"], st["tile_cap"], DEV)
    elif op == "adapter":
        a, b = st["a"], st["b"]
        pool = ops.LoraPool(case["slots"], case["k"], case["n"], case["rank"], DEV)
        for s in range(case["slots"]):
            r = st["ranks"][s]
            pool.load(s, a[s, :r], b[s, :, :r], st["scales"][s])
        st["pool"] = pool
        st["plan"] = ops.lora_plan(st["rows"], case["slots"])  # once per step, shared by every projection
    elif op == "route":
        n = case["tokens"] * case["top_k"]
        st["ids"] = torch.empty(n, dtype=torch.int32, device=DEV)
        st["w"] = torch.empty(n, dtype=torch.float32, device=DEV)
    else:
        b = case["rows"]
        st["tok"] = torch.empty(b, dtype=torch.int32, device=DEV)
        st["lp"] = torch.empty(b, dtype=torch.float32, device=DEV)
    return st


# ----------------------------------------------------------------------------- plain forms
def _layout_plain(st):
    ctx, q, table, free, ps = st["ctx"].long(), st["q"].long(), st["table"], st["free"], st["page"]
    b, w = table.shape
    end = torch.cumsum(q, 0)
    start = end - q
    kv = ctx + q
    have = (ctx + ps - 1) // ps
    need = (kv + ps - 1) // ps - have
    pend = torch.cumsum(need, 0)
    col = torch.arange(w, device=DEV)[None, :]
    new = (col >= have[:, None]) & (col < (have + need)[:, None])
    src = ((pend - need)[:, None] + col - have[:, None]).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(new, free[src], table))
    t = torch.arange(st["cap"], device=DEV)
    seq = torch.searchsorted(end, t, right=True)
    live = seq < b
    s = seq.clamp(max=b - 1)
    pos = torch.where(live, ctx[s] + t - start[s], torch.zeros_like(t))
    slot = torch.where(live, table[s, pos // ps].long() * ps + pos % ps, torch.full_like(t, -1))
    seq = torch.where(live, seq, torch.full_like(t, -1))
    tiles = (q + TILE - 1) // TILE
    tend = torch.cumsum(tiles, 0)
    i = torch.arange(st["tile_cap"], device=DEV)
    ts = torch.searchsorted(tend, i, right=True)
    tlive = ts < b
    tc = ts.clamp(max=b - 1)
    tq0 = torch.where(tlive, (i - (tend - tiles)[tc]) * TILE, torch.full_like(i, PAD_Q0))
    tseq = torch.where(tlive, ts, torch.zeros_like(ts))
    last = torch.where(q > 0, end - 1, torch.full_like(end, -1))
    q_start = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), end])
    totals = torch.stack([end[-1], pend[-1], tend[-1]])
    return (table,) + tuple(v.to(torch.int32) for v in (q_start, kv, pos, slot, seq, last, tseq, tq0, totals))


def _adapter_plain(st):
    x, y = st["x"], st["y"]
    acc = y.float()
    for s, rows in st["groups"]:
        r = st["ranks"][s]
        h = x[rows].float() @ st["a"][s, :r].float().T
        acc[rows] += (h * st["scales"][s]) @ st["b"][s, :, :r].float().T
    if st["silu"]:
        m, n = acc.shape
        g, u = acc.view(m, n // 128, 2, 64).unbind(2)
        acc = (g / (1.0 + torch.exp(-g)) * u).reshape(m, n // 2)
    return acc.to(torch.bfloat16)


def _rank_first(v, k):
    """Indices of the k largest of each row, the lower index first among equals."""
    return torch.sort(v, dim=-1, descending=True, stable=True).indices[:, :k]


def _route_plain(st):
    c = st["case"]
    x = st["logits"].double()
    t, e = x.shape
    if c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        w = torch.exp(x - x.max(-1, keepdim=True).values)
        s = w / w.sum(-1, keepdim=True)
    choice = s if st["bias"] is None else s + st["bias"].double()
    if c["groups"] > 1:
        grp = choice.view(t, c["groups"], -1)
        rank = torch.sort(grp, dim=-1, descending=True).values
        gs = rank[..., 0] if c["group_score"] == "max" else rank[..., :2].sum(-1)
        keep = torch.zeros(t, c["groups"], dtype=torch.bool, device=x.device)
        keep.scatter_(1, _rank_first(gs, c["top_groups"]), True)
        choice = torch.where(keep.repeat_interleave(e // c["groups"], dim=1), choice,
                             torch.full_like(choice, float("-inf")))
    ids = _rank_first(choice, c["top_k"])
    w = torch.gather(s, 1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return ids.to(torch.int32).flatten(), (w * c["scale"]).float().flatten()


def _sample_plain(st):
    x = st["logits"].double()
    b, v = x.shape
    if st["mask"] is not None:
        bit = torch.arange(v, device=DEV)
        ok = (st["mask"][:, bit // 32] >> (bit % 32)) & 1
        x = torch.where(ok == 1, x, torch.full_like(x, float("-inf")))
    greedy = ~(st["temp"] > 0)
    t = torch.where(greedy, torch.ones_like(st["temp"]), st["temp"]).double()[:, None]
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    z = (x - x[:, :1]) / t
    w = torch.exp(z)
    n = torch.arange(v, device=DEV)[None, :]
    keep = w >= st["min_p"].double()[:, None]
    keep &= (st["top_k"][:, None] <= 0) | (n < st["top_k"][:, None])
    cum = torch.cumsum(w, -1)
    top_p = st["top_p"].double()[:, None]
    keep &= (top_p >= 1) | (cum - w < top_p * w.sum(-1, keepdim=True))
    keep |= n == 0
    w = torch.where(keep, w, torch.zeros_like(w))
    cum = torch.cumsum(w, -1)
    total = cum[:, -1:]
    at = torch.sum(cum <= st["u"].double()[:, None] * total, -1, keepdim=True)
    at = torch.minimum(at, keep.sum(-1, keepdim=True) - 1)
    at = torch.where(greedy[:, None], torch.zeros_like(at), at)
    lp = torch.gather(z, 1, at) - torch.log(total)
    lp = torch.where(greedy[:, None], torch.zeros_like(lp), lp)
    return torch.gather(order, 1, at)[:, 0].to(torch.int32), lp[:, 0].float()


_PLAIN = dict(layout=_layout_plain, adapter=_adapter_plain, route=_route_plain, sample=_sample_plain)


def run(st):
    c = st["case"]
    op = c["op"]
    if not own:
        return _PLAIN[op](st)
    from squish_b200 import ops

    if op == "layout":
        o = ops.step_layout(st["ctx"], st["q"], st["table"], st["free"], st["page"], st["out"])
        return (st["table"], o.q_start, o.kv_len, o.positions, o.slots, o.token_seq, o.last_row, o.tile_seq, o.tile_q0,
                o.totals)
    if op == "adapter":
        return ops.lora_add(st["x"], st["pool"], st["plan"], st["y"], out=st["out"], silu_mul=st["silu"])
    if op == "route":
        ops.moe_route_scored(st["logits"], c["top_k"], st["ids"], st["w"], score=c["score"], bias=st["bias"],
                             groups=c["groups"], top_groups=c["top_groups"], group_score=c["group_score"],
                             renorm=c["renorm"], scale=c["scale"])
        return st["ids"], st["w"]
    ops.sample_uniform(st["logits"], st["u"], st["tok"], temperature=st["temp"], top_p=st["top_p"], top_k=st["top_k"],
                       min_p=st["min_p"], allow_mask=st["mask"], out_logprob=st["lp"])
    return st["tok"], st["lp"]


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, op = case, case["op"]
    if op == "layout":
        # lengths in, start / kv length / last row out; 12 bytes a token; a new page read and
        # entered; 8 bytes a tile
        return {"bytes": int(c["seqs"] * 28 + c["budget"] * (12 + 8 / c["page"] + 8 / TILE)), "flops": 0}
    if op == "adapter":
        m, k, n = c["rows"], c["k"], c["n"]
        r = 0.75 * c["rank"]
        act = m * (1.0 - c["bare"])
        used = min(c["used"], m)
        out = n // 2 if c["silu"] else n
        return {"bytes": int(2 * (act * k + used * r * (k + n) + m * n + m * out)),
                "flops": int(2 * act * r * (k + n))}
    if op == "route":
        size = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": c["tokens"] * (c["experts"] * size + c["top_k"] * 8) + 4 * c["experts"],
                "flops": 4 * c["tokens"] * c["experts"]}
    b, v = c["rows"], c["vocab"]
    return {"bytes": 2 * b * v + (b * v // 8 if c["mask"] else 0) + 28 * b, "flops": 4 * b * v}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _layout_exact(st):
    """One sequence after another on the host, as the definition reads."""
    ctx, q, table, free = st["ctx"].tolist(), st["q"].tolist(), st["table"].cpu().clone(), st["free"].tolist()
    ps = st["page"]
    start, pos, slot, seq, last, tseq, tq0, kv = [0], [], [], [], [], [], [], []
    used = 0
    for b, (c, n) in enumerate(zip(ctx, q)):
        row = table[b].tolist()
        lo, hi = -(-c // ps), -(-(c + n) // ps)
        row[lo:hi] = free[used:used + hi - lo]
        used += hi - lo
        table[b] = torch.tensor(row, dtype=torch.int32)
        p = range(c, c + n)
        pos += p
        slot += [row[i // ps] * ps + i % ps for i in p]
        seq += [b] * n
        start.append(start[-1] + n)
        kv.append(c + n)
        last.append(start[-1] - 1 if n else -1)
        tq0 += range(0, n, TILE)
        tseq += [b] * len(range(0, n, TILE))
    totals = [start[-1], used, len(tq0)]
    pad, tpad = st["cap"] - len(pos), st["tile_cap"] - len(tq0)
    pos, slot, seq = pos + [0] * pad, slot + [-1] * pad, seq + [-1] * pad
    tseq, tq0 = tseq + [0] * tpad, tq0 + [PAD_Q0] * tpad
    return (table.to(DEV),) + tuple(torch.tensor(v, dtype=torch.int32, device=DEV)
                                    for v in (start, kv, pos, slot, seq, last, tseq, tq0, totals))


def _adapter_exact(st):
    x, out = st["x"].double(), st["y"].double()
    rows = st["rows"].long()
    for s in range(st["a"].shape[0]):
        sel = (rows == s).double()[:, None]
        if not bool(sel.any()):
            continue
        r = st["ranks"][s]
        h = torch.matmul(x * sel, st["a"][s, :r].double().transpose(0, 1))
        out.addmm_(h, st["b"][s, :, :r].double().transpose(0, 1), alpha=float(torch.tensor(st["scales"][s])))
    if st["silu"]:
        m, n = out.shape
        out = out.reshape(m, n // 128, 128)
        out = (out[..., :64] * torch.special.expit(out[..., :64]) * out[..., 64:]).reshape(m, n // 2)
    return out


def _route_exact(st):
    c = st["case"]
    x = st["logits"].double()
    s = torch.special.expit(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
    v = s.clone() if st["bias"] is None else s + st["bias"].double()
    t, e = v.shape
    ninf = float("-inf")
    if c["groups"] > 1:
        size = e // c["groups"]
        best = torch.topk(v.view(t, c["groups"], size), 1 if c["group_score"] == "max" else min(2, size), dim=-1)
        gs = best.values.sum(-1)
        open_ = torch.zeros_like(gs)
        for _ in range(c["top_groups"]):  # one group after another, the first of the largest
            i = torch.argmax((gs == gs.max(-1, keepdim=True).values).to(torch.int8), -1, keepdim=True)
            open_.scatter_(1, i, 1.0)
            gs.scatter_(1, i, ninf)
        v[(open_ == 0).repeat_interleave(size, dim=1)] = ninf
    ids = []
    for _ in range(c["top_k"]):
        i = torch.argmax((v == v.max(-1, keepdim=True).values).to(torch.int8), -1, keepdim=True)
        ids.append(i)
        v.scatter_(1, i, ninf)
    ids = torch.cat(ids, 1)
    w = s.gather(1, ids)
    if c["renorm"]:
        w /= w.sum(-1, keepdim=True)
    return ids.to(torch.int32).flatten(), (w * c["scale"]).flatten()


def _sample_exact(st):
    toks, lps = [], []
    for i in range(st["logits"].shape[0]):
        x = st["logits"][i].double()
        v = x.shape[0]
        if st["mask"] is not None:
            bits = (st["mask"][i].long()[:, None] >> torch.arange(32, device=DEV)) & 1
            x[bits.flatten()[:v] == 0] = float("-inf")
        temp = float(st["temp"][i])
        if not temp > 0:
            toks.append(int(torch.nonzero(x == x.max())[0]))
            lps.append(0.0)
            continue
        p = torch.softmax(x / temp, -1)
        idx = torch.argsort(p, descending=True, stable=True)
        # (equal logits only: softmax keeps their order, and distinct logits stay distinct here)
        idx = idx[torch.argsort(x[idx], descending=True, stable=True)]
        p = p[idx]
        n = v
        k = int(st["top_k"][i])
        if k > 0:
            n = min(n, k)
        n = min(n, max(1, int((p >= float(st["min_p"][i]) * p[0] * (1 - 1e-15)).sum())))
        tp = float(st["top_p"][i])
        cum = torch.cumsum(p, 0)
        if tp < 1:
            n = min(n, int(torch.searchsorted(cum, torch.tensor([tp], dtype=torch.float64, device=DEV))) + 1)
        n = max(1, n)
        at = int(torch.searchsorted(cum[:n].contiguous(), (cum[n - 1] * float(st["u"][i])).reshape(1), right=True))
        at = min(at, n - 1)
        toks.append(int(idx[at]))
        lps.append(math.log(float(p[at])) - math.log(float(cum[n - 1])))
    return torch.tensor(toks, dtype=torch.int32, device=DEV), torch.tensor(lps, dtype=torch.float64, device=DEV)


_EXACT = dict(layout=_layout_exact, adapter=_adapter_exact, route=_route_exact, sample=_sample_exact)


def exact(case, seed):
    st = _INPUTS[case["op"]](case, seed)
    st["case"] = case
    return _EXACT[case["op"]](st)
