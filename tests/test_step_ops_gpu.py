"""Serving-step operators (squish_b200.ops.step) on the GPU against 64-bit reference forms.

Integer outputs (layout, tokens, expert ids) must be equal. Router weights are fp32 with an accurate
exponential and divide: 2^-18 of the value covers the exponent's rounding (|x| <= 30 times 2^-24), the
exponential (2 ulp), a sum of at most 32 and a divide. Log-probabilities are computed in fp64 and
rounded once to fp32. Adapter outputs have the bound that _step_refs.lora_ref derives."""
import math
import random

import numpy as np
import pytest
import torch

from squish_b200 import ops
from squish_b200._ext import native
from squish_b200.ops import kernels as K

from ._step_refs import PAD_Q0, layout_ref, lora_ref, route_ref, sample_ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def status(cuda):
    ws = ops.workspace(cuda)
    code = int(ws.status.item())
    ws.status.zero_()
    return code


# ----------------------------------------------------------------------------- layout
def run_layout(cuda, ctx, q, ps, cap=None, tile_cap=None, width=None, free_extra=3, seed=0):
    rng = random.Random(seed)
    B = len(ctx)
    have = [-(-c // ps) for c in ctx]
    need = [-(-(c + n) // ps) - h for c, n, h in zip(ctx, q, have)]
    pages = list(range(sum(have) + sum(need) + free_extra))
    rng.shuffle(pages)
    width = width or max(1, max(h + n for h, n in zip(have, need)))
    table = [[-7] * width for _ in range(B)]
    for b in range(B):
        for i in range(have[b]):
            table[b][i] = pages.pop()
    cap = sum(q) + 5 if cap is None else cap
    lay = ops.StepLayout(B, max(cap, 1), tile_cap, cuda)
    tab = i32(table, cuda)
    got = ops.step_layout(i32(ctx, cuda), i32(q, cuda), tab, i32(pages, cuda), ps, lay)
    want = layout_ref(ctx, q, table, pages, ps, 32, lay.positions.numel(), lay.tile_seq.numel())
    assert tab.tolist() == table
    for k, v in want.items():
        assert getattr(got, k).tolist() == v, k
    assert status(cuda) == 0
    return got


@pytest.mark.parametrize("ctx,q,ps", [
    ([0], [1], 16),
    ([15], [1], 16),                       # the last slot of a page
    ([16], [1], 16),                       # the first of a new one
    ([0, 5, 16, 31, 0], [0, 0, 1, 2, 0], 16),
    ([0], [100], 1),                       # a page per token
    ([7, 0, 1000], [1, 64, 33], 24),       # a page size that is no power of two
    ([0, 0, 0], [0, 0, 0], 8),             # nothing to do
    ([3], [5000], 64),
])
def test_layout_small(cuda, ctx, q, ps):
    run_layout(cuda, ctx, q, ps)


@pytest.mark.parametrize("B,maxq,maxc,ps", [(64, 1, 2000, 16), (257, 40, 300, 16), (400, 800, 90, 16), (1000, 3, 5000, 32), (8192, 2, 40, 8),
                                            (300, 700, 90, 24)])
def test_layout_random(cuda, B, maxq, maxc, ps):
    rng = random.Random(B)
    ctx = [rng.randrange(maxc) for _ in range(B)]
    q = [rng.choice([0, 1, rng.randint(0, maxq)]) for _ in range(B)]
    run_layout(cuda, ctx, q, ps, seed=B)


def test_layout_strided_table_keeps_the_rest(cuda):
    big = torch.full((3, 12), -5, dtype=torch.int32, device=cuda)
    tab = big[:2, 4:9]
    tab[0, 0] = 3
    lay = ops.StepLayout(4, 16, device=cuda)  # buffers of a larger step
    ops.step_layout(i32([4, 0], cuda), i32([1, 5], cuda), tab, i32([8, 6, 1], cuda), 4, lay)
    assert lay.slots.tolist()[:6] == [8 * 4, 6 * 4, 6 * 4 + 1, 6 * 4 + 2, 6 * 4 + 3, 4]
    want = torch.full((3, 12), -5, dtype=torch.int32)
    want[0, 4:6] = torch.tensor([3, 8])
    want[1, 4:6] = torch.tensor([6, 1])
    assert torch.equal(big.cpu(), want) and lay.totals.tolist() == [6, 3, 2]
    assert lay.kv_len.tolist() == [5, 5] and lay._kv_len.tolist() == [5, 5, 0, 0]


def test_layout_what_does_not_fit(cuda):
    # (free list of one page, three needed): the first page goes out, later tokens have no slot
    lay = ops.StepLayout(2, 16, device=cuda)
    tab = torch.full((2, 2), -9, dtype=torch.int32, device=cuda)
    ops.step_layout(i32([0, 0], cuda), i32([4, 8], cuda), tab, i32([5], cuda), 4, lay)
    assert tab.tolist() == [[5, -9], [-9, -9]]
    assert lay.slots.tolist()[:12] == [20, 21, 22, 23] + [-1] * 8 and lay.totals.tolist() == [12, 3, 2]
    assert status(cuda) == 6
    # a row narrower than the sequence
    tab = torch.full((1, 1), -9, dtype=torch.int32, device=cuda)
    lay = ops.StepLayout(1, 16, device=cuda)
    ops.step_layout(i32([0], cuda), i32([6], cuda), tab, i32([2, 3], cuda), 4, lay)
    assert tab.tolist() == [[2]] and lay.slots.tolist()[:6] == [8, 9, 10, 11, -1, -1] and status(cuda) == 6
    # more tokens than rows
    lay = ops.StepLayout(2, 4, device=cuda)
    tab = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    ops.step_layout(i32([0, 0], cuda), i32([3, 3], cuda), tab, i32([1, 2], cuda), 4, lay)
    assert lay.positions.tolist() == [0, 1, 2, 0] and lay.last_row.tolist() == [2, -1] and status(cuda) == 6
    # lengths that are none: the sequence rests
    lay = ops.StepLayout(3, 4, device=cuda)
    tab = torch.zeros(3, 4, dtype=torch.int32, device=cuda)
    ops.step_layout(i32([-1, 2**31 - 1, 4], cuda), i32([1, 1, -3], cuda), tab, i32([1, 2], cuda), 4, lay)
    assert lay.totals.tolist() == [0, 0, 0] and lay.slots.tolist() == [-1] * 4 and status(cuda) == 6
    # sums past 32 bits saturate and are reported
    lay = ops.StepLayout(4, 4, device=cuda)
    tab = torch.zeros(4, 1, dtype=torch.int32, device=cuda)
    ops.step_layout(i32([0] * 4, cuda), i32([2**30] * 4, cuda), tab, i32([1], cuda), 4, lay)
    assert lay.totals.tolist()[0] == 2**30 and status(cuda) == 6
    # a page given back: its tokens are not stored, which is no error
    lay = ops.StepLayout(1, 4, device=cuda)
    tab = torch.full((1, 4), -1, dtype=torch.int32, device=cuda)
    ops.step_layout(i32([2], cuda), i32([3], cuda), tab, i32([6], cuda), 4, lay)
    assert lay.slots.tolist() == [-1, -1, 24, -1] and status(cuda) == 0


def test_layout_refusals(cuda):
    lay = ops.StepLayout(2, 8, device=cuda)
    good = dict(c=i32([0, 0], cuda), q=i32([1, 1], cuda), t=torch.zeros(2, 4, dtype=torch.int32, device=cuda),
                f=i32([1, 2, 3], cuda), ps=4)

    def call(**kw):
        a = {**good, **kw}
        ops.step_layout(a["c"], a["q"], a["t"], a["f"], a["ps"], lay)

    call()
    for kw, msg in [(dict(q=i32([1], cuda)), "q_len"), (dict(ps=0), "page_size"),
                    (dict(c=good["c"].long()), "ctx_len must be"), (dict(f=good["f"].cpu()), "free_pages must be a CUDA"),
                    (dict(t=good["t"].t()), "block_tables"), (dict(t=good["t"][:1].expand(2, 4)), "block_tables"),
                    (dict(c=i32([0, 9, 0, 9], cuda)[::2]), "contiguous")]:
        with pytest.raises(RuntimeError, match=msg):
            call(**kw)
    with pytest.raises(ValueError, match="sequences in a layout"):
        call(c=i32([0] * 3, cuda))
    with pytest.raises(RuntimeError, match="ctx_len is part of the step layout"):
        call(c=lay.kv_len)
    with pytest.raises(RuntimeError, match="q_len is part of the step layout"):
        call(q=lay.positions[:2])
    call(c=lay.kv_len.clone())
    none = ops.StepLayout(2, 8, 0, cuda)  # no tiles wanted, no pages left, a table without columns
    ops.step_layout(good["c"], i32([0, 0], cuda), good["t"][:, :0], good["f"][:0], 4, none)
    assert none.totals.tolist() == [0, 0, 0] and status(cuda) == 0


# ----------------------------------------------------------------------------- routing
ROUTES = [
    dict(T=1, E=128, k=8),
    dict(T=33, E=128, k=8, renorm=False, scale=2.0),
    dict(T=7, E=16, k=4, score="sigmoid"),
    dict(T=65, E=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, group_score="top2", scale=2.5),
    dict(T=65, E=256, k=8, score="sigmoid", groups=8, top_groups=3, group_score="top2"),
    dict(T=20, E=256, k=8, score="softmax", bias=True, groups=8, top_groups=4, group_score="max", renorm=False),
    dict(T=20, E=160, k=6, score="softmax", groups=8, top_groups=3, renorm=False, scale=16.0),
    dict(T=9, E=160, k=6, score="softmax", groups=8, top_groups=3, group_score="top2"),
    dict(T=9, E=72, k=5, score="sigmoid", bias=True, groups=6, top_groups=2, group_score="top2"),
    dict(T=9, E=66, k=5, score="sigmoid", bias=True, groups=6, top_groups=2, group_score="top2"),  # 11 per group
    dict(T=9, E=66, k=11, score="softmax", groups=6, top_groups=1),  # every open expert
    dict(T=5, E=1, k=1),
    dict(T=5, E=60, k=4, bias=True),
    dict(T=5, E=97, k=32, score="sigmoid", bias=True),
    dict(T=5, E=384, k=8, score="sigmoid", bias=True),
    dict(T=5, E=512, k=10, score="sigmoid", bias=True, groups=16, top_groups=5, group_score="top2"),
    dict(T=5, E=32, k=32, groups=32, top_groups=32, group_score="top2"),  # one expert per group
    dict(T=4, E=500, k=3, groups=4, top_groups=1),
]


def run_route(cuda, logits, k, bias=None, **kw):
    T = logits.shape[0]
    ids = torch.full((T * k + 4,), -3, dtype=torch.int32, device=cuda)
    w = torch.full((T * k + 4,), -3.0, device=cuda)
    ops.moe_route_scored(logits, k, ids, w, bias=bias, **kw)
    assert ids[T * k:].tolist() == [-3] * 4 and w[T * k:].tolist() == [-3.0] * 4
    want_i, want_w = route_ref(logits, k, bias=bias, **kw)
    assert np.array_equal(ids[:T * k].view(T, k).cpu().numpy(), want_i)
    got = w[:T * k].view(T, k).double().cpu().numpy()
    assert (np.abs(got - want_w) <= 2.0**-18 * np.abs(want_w) + 2.0**-140).all(), np.abs(got - want_w).max()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("case", range(len(ROUTES)))
def test_route(cuda, case, dtype):
    c = dict(ROUTES[case])
    g = torch.Generator().manual_seed(case)
    T, E, k = c.pop("T"), c.pop("E"), c.pop("k")
    logits = (torch.randn(T, E, generator=g) * 1.5).to(dtype).to(cuda)
    bias = (torch.randn(E, generator=g) * 0.1).to(cuda) if c.pop("bias", False) else None
    run_route(cuda, logits, k, bias=bias, **c)


@pytest.mark.parametrize("kw", [
    dict(score="sigmoid"), dict(score="sigmoid", bias=True), dict(score="softmax", bias=True, renorm=False),
    dict(score="sigmoid", bias=True, groups=8, top_groups=2, group_score="top2"),
    dict(score="sigmoid", groups=8, top_groups=2, group_score="top2"), dict(score="softmax", groups=8, top_groups=2),
])
def test_route_ties_go_to_the_lower_index(cuda, kw):
    g = torch.Generator().manual_seed(5)
    kw = dict(kw)
    logits = torch.randint(-2, 3, (40, 64), generator=g).float()  # many equal values
    logits[0] = 0.0
    logits[1, ::2] = -0.0
    logits[2] = 30.0  # sigmoid saturates
    bias = torch.randint(0, 2, (64,), generator=g).float().mul(0.25).to(cuda) if kw.pop("bias", False) else None
    run_route(cuda, logits.to(cuda), 8, bias=bias, **kw)


def test_route_close_scores_are_ordered_exactly(cuda):
    """Scores that differ by far less than fp32 resolves: the choice is that of the exact scores."""
    E = 64
    base = torch.linspace(-1, 1, E, dtype=torch.float64)
    logits = base.float()[None].repeat(16, 1)
    s = torch.sigmoid(logits[0].double())
    bias = (0.7 - s).float()  # every s + bias is 0.7 up to the bias' rounding
    run_route(cuda, logits.to(cuda), 16, bias=bias.to(cuda), score="sigmoid")
    run_route(cuda, logits.to(cuda), 4, bias=bias.to(cuda), score="sigmoid", groups=8, top_groups=3, group_score="top2")
    sm = torch.softmax(logits[0].double(), -1)
    run_route(cuda, logits.to(cuda), 16, bias=(0.7 - sm).float().to(cuda), score="softmax", renorm=False)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_infinities_and_nan(cuda, score, groups):
    inf, nan = math.inf, math.nan
    x = torch.randn(8, 32, generator=torch.Generator().manual_seed(1))
    x[0, 5] = inf
    x[1, [3, 9]] = inf
    x[2] = -inf
    x[3, ::2] = -inf
    x[4, 7] = nan
    x[5] = nan
    x[6] = -inf
    x[6, 30] = 1.0
    x[7] = inf
    for bias in (None, torch.linspace(-0.5, 0.5, 32).to(cuda)):
        run_route(cuda, x.to(cuda), 4, bias=bias, score=score, groups=groups, top_groups=min(groups, 2),
                  group_score="top2")


@pytest.mark.parametrize("k", [4, 20])
def test_route_infinite_bias(cuda, k):
    """A bias of +inf puts experts first, of -inf last, however many."""
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(6, 64, generator=g).to(cuda)
    for n in (1, k, 30):
        bias = torch.randn(64, generator=g) * 0.1
        bias[torch.randperm(64, generator=g)[:n]] = math.inf
        bias[torch.randperm(64, generator=g)[:3]] = -math.inf
        for kw in (dict(), dict(groups=8, top_groups=4), dict(groups=8, top_groups=4, group_score="top2")):
            run_route(cuda, logits, k, bias=bias.to(cuda), score="sigmoid", **kw)
            run_route(cuda, logits, k, bias=bias.to(cuda), score="softmax", **kw)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("shift", [-25.0, -35.0, -100.0, -300.0])
def test_route_small_sigmoids_are_renormalised(cuda, shift, bias):
    """Scores below what fp32 holds still give weights that sum to 1."""
    g = torch.Generator().manual_seed(9)
    logits = (torch.randn(6, 64, generator=g) * 2 + shift).to(cuda)
    logits[1, 5:] = -math.inf
    b = (torch.randn(64, generator=g) * 0.1).to(cuda) if bias else None
    run_route(cuda, logits, 8, bias=b, score="sigmoid")


def test_route_strides(cuda):
    g = torch.Generator().manual_seed(3)
    big = torch.randn(9, 300, generator=g).to(BF).to(cuda)
    run_route(cuda, big[:, 3:259], 8, score="sigmoid")      # rows off the 16-byte border
    run_route(cuda, big[::2, 8:264], 8, score="softmax")
    run_route(cuda, big[:1, :128].expand(5, 128), 8)        # one row for all tokens
    run_route(cuda, big[:0, :128], 8)


def test_route_refusals(cuda):
    x = torch.zeros(2, 16, device=cuda)
    ids, w = torch.zeros(8, dtype=torch.int32, device=cuda), torch.zeros(8, device=cuda)
    for kw, msg in [(dict(top_k=17), "top_k"), (dict(groups=3), "groups"), (dict(groups=4, top_groups=5), "top_groups"),
                    (dict(groups=4, top_groups=1, top_k=5), "top_k"), (dict(top_k=5), "ids needs 10"),
                    (dict(bias=torch.zeros(15, device=cuda)), "bias needs 16"),
                    (dict(bias=torch.zeros(16, device=cuda, dtype=BF)), "bias must be"),
                    (dict(logits=x.half()), "bf16 or float32"), (dict(logits=torch.zeros(2, 513, device=cuda)), "experts")]:
        a = dict(logits=x, top_k=4)
        a.update(kw)
        with pytest.raises(RuntimeError, match=msg):
            ops.moe_route_scored(a.pop("logits"), a.pop("top_k"), ids, w, **a)


# ----------------------------------------------------------------------------- sampling
def run_sample(cuda, logits, u, temp, top_p=None, top_k=None, min_p=None, mask=None):
    B, V = logits.shape
    f = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32, device=cuda)  # noqa: E731
    tok = torch.full((B + 2,), -9, dtype=torch.int32, device=cuda)
    lp = torch.full((B + 2,), -9.0, device=cuda)
    m = allow = None
    if mask is not None:
        words = (V + 31) // 32
        bits = np.zeros((B, words * 32), dtype=np.uint8)
        bits[:, :V] = mask.numpy()
        bits[:, V:] = 1  # bits behind the vocabulary are never read as tokens
        m = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).to(cuda)
        allow = mask.numpy()
    ops.sample_uniform(logits, f(u), tok[:B], temperature=f(temp), top_p=f(top_p),
                       top_k=None if top_k is None else i32(top_k, cuda), min_p=f(min_p), allow_mask=m,
                       out_logprob=lp[:B])
    assert tok[B:].tolist() == [-9, -9] and lp[B:].tolist() == [-9.0, -9.0]
    host = logits.float().cpu().numpy()
    for b in range(B):
        want, wlp = sample_ref(host[b], u[b], 0.0 if temp is None else temp[b], 1.0 if top_p is None else top_p[b],
                               0 if top_k is None else top_k[b], 0.0 if min_p is None else min_p[b],
                               None if allow is None else allow[b])
        assert int(tok[b]) == want, (b, int(tok[b]), want)
        got = float(lp[b])
        assert got == wlp or abs(got - wlp) <= 2.0**-24 * abs(wlp) + 1e-9, (b, got, wlp)


def rand_params(rng, B):
    u = [rng.random() for _ in range(B)]
    temp = [rng.choice([0.0, 0.3, 0.7, 1.0, 2.5]) for _ in range(B)]
    top_p = [rng.choice([1.0, 1.0, 0.05, 0.6, 0.95, 0.999]) for _ in range(B)]
    top_k = [rng.choice([0, 0, 1, 3, 40, 5000]) for _ in range(B)]
    min_p = [rng.choice([0.0, 0.0, 0.02, 0.5, 1.0]) for _ in range(B)]
    return u, temp, top_p, top_k, min_p


@pytest.mark.parametrize("B,V", [(1, 152064), (3, 50001), (5, 32000), (9, 4099), (40, 1000), (2, 1), (7, 2), (6, 7),
                                 (5, 31), (4, 8192), (20, 16389), (80, 9001), (150, 4500), (300, 777)])
@pytest.mark.parametrize("masked", [False, True])
def test_sample(cuda, B, V, masked):
    g = torch.Generator().manual_seed(B * V)
    rng = random.Random(B + V)
    logits = (torch.randn(B, V, generator=g) * 2.5).to(BF).to(cuda)
    mask = None
    if masked:
        mask = torch.rand(B, V, generator=g) < 0.5
        if B > 1:
            mask[1] = False        # nothing allowed
            mask[0] = False
            mask[0, V - 1] = True  # one token allowed
    run_sample(cuda, logits, *rand_params(rng, B), mask=mask)


def test_sample_walks_the_whole_range_of_u(cuda):
    """Equal and distinct logits; u on, just below and just above the borders between tokens."""
    row = torch.tensor([0.0, 2.0, 0.0, 2.0, -1.0, 0.0, -0.0]).to(BF)
    us = [0.0, 1e-7, 0.25, 0.4999, 0.5, 0.73, 0.9, 0.99, 1.0 - 2.0**-24, 1.0, 2.0, -1.0, math.nan]
    n = len(us)
    ref_u = [min(max(v, 0.0), 1.0) if v == v else 0.0 for v in us]
    tok = torch.empty(n, dtype=torch.int32, device=cuda)
    for kw in ({}, dict(top_k=3), dict(top_k=1), dict(top_p=0.5), dict(top_p=0.9), dict(min_p=0.2), dict(top_p=0.0)):
        dev = {k: torch.full((n,), v, device=cuda, dtype=torch.int32 if k == "top_k" else torch.float32)
               for k, v in kw.items()}
        ops.sample_uniform(row[None].expand(n, 7).to(cuda), torch.tensor(us, device=cuda), tok,
                           temperature=torch.ones(n, device=cuda), **dev)
        want = [sample_ref(row.float().numpy(), v, 1.0, **kw)[0] for v in ref_u]
        assert tok.tolist() == want, kw


@pytest.mark.parametrize("C_rows", [1, 200])
def test_sample_unusual_values(cuda, C_rows):
    """Constant rows, zeros of both signs, infinities, NaN, and magnitudes outside the main bins."""
    V = 9000
    g = torch.Generator().manual_seed(0)
    rows = [torch.zeros(V), torch.full((V,), 3.0), torch.randn(V, generator=g) * 1e-12, torch.randn(V, generator=g) * 1e20,
            torch.randn(V, generator=g), torch.randn(V, generator=g), torch.full((V,), -math.inf), torch.full((V,), math.nan),
            torch.randn(V, generator=g), torch.randn(V, generator=g).abs() * 1e-38]
    rows[0][::2] = -0.0
    rows[4][7] = math.inf
    rows[5][::3] = math.nan
    rows[5][1::3] = -math.inf
    rows[8][100:103] = torch.tensor([1e-20, -1e-20, 1e-11])
    logits = torch.stack(rows).to(BF).to(cuda)
    reps = -(-C_rows // len(rows))
    logits = logits.repeat(reps, 1)
    B = logits.shape[0]
    rng = random.Random(7)
    for temps in ([1.0] * B, [0.0] * B, [rng.choice([0.1, 1e-3, 50.0]) for _ in range(B)]):
        u, _, top_p, top_k, min_p = rand_params(rng, B)
        run_sample(cuda, logits, u, temps)
        run_sample(cuda, logits, u, temps, top_p, top_k, min_p)


@pytest.mark.parametrize("V", [9000, 70001])
def test_sample_masked_unusual_values(cuda, V):
    """Infinities, NaN and values outside the main bins in masked places do not count."""
    g = torch.Generator().manual_seed(1)
    B = 6
    logits = torch.randn(B, V, generator=g) * 2
    mask = torch.rand(B, V, generator=g) < 0.7
    mask[:, 17] = True
    bad = torch.tensor([math.inf, math.nan, 1e20, -math.inf, 1e-20, -1e-30])
    for b in range(B):
        where = torch.nonzero(~mask[b]).flatten()[::5]
        logits[b, where] = bad[torch.arange(len(where)) % len(bad)]
    rng = random.Random(3)
    lg = logits.to(BF).to(cuda)
    run_sample(cuda, lg, *rand_params(rng, B), mask=mask)
    run_sample(cuda, lg, [rng.random() for _ in range(B)], [1.0] * B, mask=mask)
    run_sample(cuda, lg, [0.5] * B, [0.0] * B, mask=mask)


@pytest.mark.parametrize("B,V", [(1, 65537), (9, 70000), (18, 66001), (40, 80003), (74, 65600), (75, 65600)])
def test_sample_rows_shared_by_ctas(cuda, B, V):
    """Each number of CTAs per row, at its borders, with some rows greedy and some without a token."""
    g = torch.Generator().manual_seed(V)
    rng = random.Random(B)
    logits = (torch.randn(B, V, generator=g) * 3).to(BF)
    if B > 1:
        logits[B // 2] = -math.inf
        logits[B - 1] = 0.0
        logits[0, 1234] = 1e-12  # outside the main bins: one CTA does the row
    u, temp, top_p, top_k, min_p = rand_params(rng, B)
    run_sample(cuda, logits.to(cuda), u, temp, top_p, top_k, min_p)


@pytest.mark.parametrize("V", [1, 4099, 70001])
def test_sample_extreme_parameters(cuda, V):
    """The ends of each parameter's range, and what lies behind them."""
    cases = [(t, p, k, m) for t in (1e-40, 1e-6, 1e30, math.inf)
             for p, k, m in ((1.0, 0, 0.0), (0.0, 0, 0.0), (-1.0, 0, 0.0), (2.0, 2**31 - 1, -1.0), (0.5, -5, 0.0),
                             (1.0, 0, 1.0), (1.0, 0, 2.0), (1e-30, 7, 1e-30), (1.0 - 2.0**-24, 0, 0.0))]
    B = len(cases)
    logits = (torch.randn(B, V, generator=torch.Generator().manual_seed(V)) * 2).to(BF).to(cuda)
    for u in (0.0, 2.0**-24, 0.37, 1.0 - 2.0**-24):
        run_sample(cuda, logits, [u] * B, *map(list, zip(*cases)))


@pytest.mark.parametrize("B", [2, 12, 30, 80])
def test_sample_greedy_zeros_of_both_signs(cuda, B):
    """-0 and +0 are equal: the lower index wins, whichever CTA of the row holds it."""
    V = 70001
    logits = torch.full((B, V), -1.0)
    logits[:, 11] = -0.0
    logits[:, V - 2] = 0.0
    logits[1, 11], logits[1, V - 2] = 0.0, -0.0
    tok = torch.empty(B, dtype=torch.int32, device=cuda)
    ops.sample_uniform(logits.to(BF).to(cuda), torch.full((B,), 0.5, device=cuda), tok)
    assert tok.tolist() == [11] * B


def test_sample_strides_and_optional_parameters(cuda):
    g = torch.Generator().manual_seed(2)
    big = (torch.randn(7, 5003, generator=g) * 2).to(BF).to(cuda)
    for lg in (big[:, 1:4999], big[::3], big[1:2].expand(4, 5003), big[:0]):
        B = lg.shape[0]
        run_sample(cuda, lg, [0.37] * B, [0.9] * B)
        run_sample(cuda, lg, [0.37] * B, None)
    tok = torch.empty(7, dtype=torch.int32, device=cuda)
    assert ops.sample_uniform(big, torch.zeros(7, device=cuda), tok) is tok
    assert torch.equal(tok.long(), big.float().argmax(-1))


def test_sample_distribution(cuda):
    """Tokens drawn with evenly spaced u appear in proportion to their weights."""
    n = 40000
    row = torch.tensor([0.0, 1.0, -2.0, 3.0, 0.5]).to(BF)
    p = torch.softmax(row.double() / 1.25, -1)
    tok = torch.empty(n, dtype=torch.int32, device=cuda)
    ops.sample_uniform(row[None].expand(n, 5).to(cuda), (torch.arange(n, device=cuda) + 0.5) / n, tok,
                       temperature=torch.full((n,), 1.25, device=cuda))
    f = torch.bincount(tok.long().cpu(), minlength=5).double() / n
    assert (f - p).abs().max() <= 1.0 / n + 1e-6  # evenly spaced: off by at most one draw


def test_sample_refusals(cuda):
    lg = torch.zeros(2, 40, dtype=BF, device=cuda)
    u, tok = torch.zeros(2, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    for a, kw, msg in [((lg.float(), u, tok), {}, "logits must be"), ((lg.t(), u, tok), {}, "unit column"),
                       ((lg, u[:1], tok), {}, "uniforms needs 2"), ((lg, u, tok.long()), {}, "out_tokens must be"),
                       ((lg, u, tok), dict(top_k=u), "top_k must be"), ((lg, u.cpu(), tok), {}, "CUDA tensor"),
                       ((lg, u, tok), dict(allow_mask=tok[:, None].contiguous()), "allow_mask must be"),
                       ((lg[:, :0], u, tok), {}, "vocab")]:
        with pytest.raises(RuntimeError, match=msg):
            ops.sample_uniform(*a, **kw)


# ----------------------------------------------------------------------------- adapters
def make_adapters(cuda, slots, k, n, rank, seed=0, ranks=None):
    g = torch.Generator().manual_seed(seed)
    pool = ops.LoraPool(slots, k, n, rank, cuda)
    ads = {}
    for s in range(slots):
        r = ranks[s] if ranks else max(1, rank - s)
        a = (torch.randn(r, k, generator=g) / math.sqrt(k)).to(BF)
        b = (torch.randn(n, r, generator=g) * 0.3).to(BF)
        sc = 0.25 + s
        pool.load(s, a, b, sc)
        ads[s] = (a, b, sc)
    return pool, ads


def check_lora(cuda, m, k, n, rank, slots, rows=None, silu=False, seed=0, ranks=None):
    g = torch.Generator().manual_seed(seed + 1)
    pool, ads = make_adapters(cuda, slots, k, n, rank, seed, ranks)
    if rows is None:
        rows = torch.randint(-1, slots, (m,), generator=g)
    x = torch.randn(m, k, generator=g).to(BF)
    y = torch.randn(m, n, generator=g).to(BF)
    rs = rows.to(torch.int32).to(cuda)
    plan = ops.lora_plan(rs, slots)
    order = plan.order.cpu().long()
    key = torch.where(rows < 0, torch.full_like(rows, slots), rows)
    assert torch.equal(order, torch.sort(key, stable=True).indices)  # stable, rows without an adapter last
    xd, yd = x.to(cuda), y.to(cuda)
    out = ops.lora_add(xd, pool, plan, yd, silu_mul=silu)
    want, tol = lora_ref(x, y, rows, ads, silu)
    err = (out.double().cpu() - want).abs()
    assert (err <= tol).all(), ((err / tol).max(), (err > tol).sum())
    assert torch.equal(yd.cpu(), y) and torch.equal(xd.cpu(), x)
    assert torch.equal(out, ops.lora_add(xd, pool, plan, yd, silu_mul=silu))  # the same bits again
    if not silu:
        assert ops.lora_add(xd, pool, plan, yd, out=yd) is yd and torch.equal(yd, out)  # in place
    assert status(cuda) == 0


@pytest.mark.parametrize("m,k,n,rank,slots", [
    (1, 8, 8, 1, 1), (1, 256, 128, 16, 1), (3, 64, 40, 4, 2), (16, 1000, 264, 16, 1), (17, 264, 1000, 9, 3),
    (64, 3584, 512, 16, 32), (100, 520, 136, 33, 5), (128, 256, 256, 64, 7), (130, 136, 72, 128, 3),
    (512, 128, 64, 8, 512), (513, 320, 200, 16, 4), (700, 968, 328, 64, 9), (1030, 128, 520, 100, 2),
    (2100, 64, 96, 24, 3), (5, 18944, 48, 64, 2), (600, 40, 4104, 32, 1024),
])
def test_lora_add(cuda, m, k, n, rank, slots):
    check_lora(cuda, m, k, n, rank, slots, seed=m + n, ranks=[max(1, rank - s % 5) for s in range(slots)])


@pytest.mark.parametrize("m,k,n,rank,slots", [(1, 64, 128, 4, 1), (40, 256, 1280, 16, 5), (600, 200, 384, 40, 3),
                                              (520, 136, 256, 128, 2), (9, 3584, 37888, 16, 4)])
def test_lora_add_silu_mul(cuda, m, k, n, rank, slots):
    check_lora(cuda, m, k, n, rank, slots, silu=True, seed=m)


@pytest.mark.parametrize("m", [1, 48, 700])
def test_lora_row_patterns(cuda, m):
    for rows in (torch.full((m,), -1), torch.zeros(m, dtype=torch.int64), torch.arange(m) % 3,
                 (torch.arange(m) * 3 // m), torch.full((m,), 2)):
        check_lora(cuda, m, 72, 104, 16, 3, rows=rows)
    check_lora(cuda, m, 72, 128, 16, 3, rows=torch.full((m,), -1), silu=True)


def test_lora_strides_and_neighbours(cuda):
    m, k, n = 70, 136, 104
    pool, ads = make_adapters(cuda, 2, k, n, 8)
    rows = torch.arange(m) % 3 - 1
    plan = ops.lora_plan(rows.to(torch.int32).to(cuda), 2)
    g = torch.Generator().manual_seed(1)
    xb = torch.randn(m, k + 24, generator=g).to(BF).to(cuda)
    yb = torch.randn(2 * m, n + 16, generator=g).to(BF).to(cuda)
    ob = torch.full((m, n + 32), 7.0, dtype=BF, device=cuda)
    x, y, o = xb[:, 8:8 + k], yb[::2, 8:8 + n], ob[:, 16:16 + n]
    ops.lora_add(x, pool, plan, y, out=o)
    want, tol = lora_ref(x, y, rows, ads)
    assert ((o.double().cpu() - want).abs() <= tol).all()
    assert (ob[:, :16] == 7).all() and (ob[:, 16 + n:] == 7).all()
    xe = xb[:1, :k].expand(m, k)  # one activation row for all
    want, tol = lora_ref(xe, y, rows, ads)
    assert ((ops.lora_add(xe, pool, plan, y).double().cpu() - want).abs() <= tol).all()


def test_lora_special_values_stay_in_their_rows(cuda):
    m, k, n = 20, 64, 64
    pool, ads = make_adapters(cuda, 2, k, n, 8)
    pool.clear(1)
    rows = torch.tensor([0, 1, -1, 0] * 5)
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn(m, k, generator=g).to(BF), torch.randn(m, n, generator=g).to(BF)
    x[2], x[1], x[3] = math.nan, math.inf, math.nan  # rows without an adapter, with a cleared one, with one
    y[4, 5] = math.inf
    plan = ops.lora_plan(rows.to(torch.int32).to(cuda), 2)
    out = ops.lora_add(x.to(cuda), pool, plan, y.to(cuda)).cpu()
    assert torch.equal(out[2], y[2]) and torch.equal(out[1], y[1]) and out[3].isnan().all() and out[4, 5] == math.inf
    keep = torch.ones(m, dtype=torch.bool)
    keep[3] = False
    x[1:4] = 0.0
    want, tol = lora_ref(x, y, rows, {0: ads[0]})
    ok = ((out.double() - want).abs() <= tol) | (out.double() == want)
    assert ok[keep].all()


@pytest.mark.parametrize("n,rank", [(128, 16), (2176, 16), (2176, 64), (640, 128)])
@pytest.mark.parametrize("silu", [False, True])
def test_lora_empty_slots_between_full_ones(cuda, n, rank, silu):
    """Large steps: tiles that are left as they are, first, between others and last, in place and not."""
    m, k, slots = 900, 72, 6
    pool, ads = make_adapters(cuda, slots, k, n, rank)
    for s in (0, 2, 3):
        pool.clear(s)
        ads.pop(s, None)
    g = torch.Generator().manual_seed(n + rank)
    rows = torch.randint(-1, slots, (m,), generator=g)
    x, y = torch.randn(m, k, generator=g).to(BF), torch.randn(m, n, generator=g).to(BF)
    for r in (rows, torch.full_like(rows, 2), torch.full_like(rows, -1), torch.where(rows < 4, -1, rows)):
        plan = ops.lora_plan(r.to(torch.int32).to(cuda), slots)
        yc = y.to(cuda)
        out = ops.lora_add(x.to(cuda), pool, plan, yc, out=None if silu else yc, silu_mul=silu)
        want, tol = lora_ref(x, y, r, ads, silu)
        assert ((out.double().cpu() - want).abs() <= tol).all()


def test_lora_plan_reports_bad_slots(cuda):
    rows = i32([0, 5, -2, 1, 2**31 - 1, -1], cuda)
    plan = ops.lora_plan(rows, 2)
    assert status(cuda) == 6
    assert plan.order.tolist() == [0, 3, 1, 2, 4, 5]
    n = int(plan.num_tiles)
    assert plan.tiles[:n].tolist() == [[0, 0, 1, 0], [1, 1, 1, 0], [-1, 2, 4, 0]]
    empty = ops.lora_plan(rows[:0], 2)
    pool, _ = make_adapters(cuda, 2, 8, 8, 4)
    z = torch.zeros(0, 8, dtype=BF, device=cuda)
    assert ops.lora_add(z, pool, empty, z).shape == (0, 8)


def test_lora_refusals(cuda):
    pool, _ = make_adapters(cuda, 2, 64, 128, 8)
    plan = ops.lora_plan(i32([0, 1, -1], cuda), 2)
    x, y = torch.zeros(3, 64, dtype=BF, device=cuda), torch.zeros(3, 128, dtype=BF, device=cuda)
    big = torch.zeros(4, 192, dtype=BF, device=cuda)
    other = ops.lora_plan(i32([0, 1, -1], cuda), 3)
    for a, kw, msg in [((x[:2], pool, plan, y), {}, "x must be"), ((x.float(), pool, plan, y), {}, "x must be"),
                       ((x, pool, other, y), {}, "the plan is for 3"), ((x, pool, plan, y.t()), {}, "y must be"),
                       ((x, pool, plan, y), dict(out=y[:, :64]), "out must be"),
                       ((x, pool, plan, y), dict(out=y[:, :64], silu_mul=True), "overlaps y"),
                       ((big[:3, 64:128], pool, plan, y), dict(out=big[:3, 64:]), "overlaps x"),
                       ((x, pool, plan, big[:3, :128]), dict(out=big[1:4, :128]), "overlaps y"),
                       ((big[:3, 1:65], pool, plan, y), {}, "16-byte aligned"),
                       ((x, pool, plan, y), dict(out=y[:1].expand(3, 128)), "overlap")]:
        with pytest.raises(RuntimeError, match=msg):
            ops.lora_add(*a, **kw)
    narrow, _ = make_adapters(cuda, 2, 64, 64, 8)
    with pytest.raises(RuntimeError, match="multiple of 128"):
        ops.lora_add(x, narrow, plan, torch.zeros(3, 64, dtype=BF, device=cuda), silu_mul=True)


@pytest.mark.parametrize("m", [5, 600])
def test_lora_linear(cuda, m):
    """The quantized projection with adapters: what w4a16_linear gives, plus the exact adapter term."""
    k, n = 256, 384
    g = torch.Generator().manual_seed(m)
    C = native()
    packed, scales, offsets = C.cpu.quantize_int4_asym(torch.randn(n, k, generator=g) * 0.05, 64)
    w = ops.prepare_int4_weight(packed, scales, offsets, k, 64, cuda)
    pool, ads = make_adapters(cuda, 3, k, n, 8)
    rows = torch.randint(-1, 3, (m,), generator=g)
    plan = ops.lora_plan(rows.to(torch.int32).to(cuda), 3)
    x = torch.randn(m, k, generator=g).to(BF).to(cuda)
    h = torch.randn(m, n, generator=g).to(BF).to(cuda)
    base = ops.w4a16_linear(x, w)
    want, tol = lora_ref(x, base, rows, ads)
    assert ((ops.lora_linear(x, w, pool, plan).double().cpu() - want).abs() <= tol).all()
    want, tol = lora_ref(x, base, rows, ads, silu=True)
    assert ((ops.lora_linear(x, w, pool, plan, silu_mul=True).double().cpu() - want).abs() <= tol).all()
    base = ops.w4a16_linear(x, w, residual=h)
    want, tol = lora_ref(x, base, rows, ads)
    got = ops.lora_linear(x, w, pool, plan, out=h, residual=h)
    assert got is h and ((h.double().cpu() - want).abs() <= tol).all()
    with pytest.raises(ValueError, match="residual"):
        ops.lora_linear(x, w, pool, plan, residual=h, silu_mul=True)
    ops.workspace(cuda).check()


# ----------------------------------------------------------------------------- streams, graphs, the run together
def test_two_streams_at_once(cuda):
    """Every operator on two streams at the same time gives what it gives alone."""
    g = torch.Generator().manual_seed(0)
    work = []
    for i in range(2):
        lg = (torch.randn(9, 40000, generator=g) * 2).to(BF).to(cuda)
        rl = torch.randn(500, 128, generator=g).to(cuda)
        pool, _ = make_adapters(cuda, 2, 512, 512, 16, seed=i)
        m = (300, 900)[i]  # (both tile sizes)
        plan = ops.lora_plan((torch.arange(m) % 3 - 1).to(torch.int32).to(cuda), 2)
        x, y = torch.randn(m, 512, generator=g).to(BF).to(cuda), torch.randn(m, 512, generator=g).to(BF).to(cuda)
        u, t = torch.rand(9, generator=g).to(cuda), torch.full((9,), 0.8, device=cuda)
        work.append((lg, u, t, rl, pool, plan, x, y))

    def go(lg, u, t, rl, pool, plan, x, y):
        tok = torch.empty(9, dtype=torch.int32, device=cuda)
        ids, w = torch.empty(500 * 8, dtype=torch.int32, device=cuda), torch.empty(500 * 8, device=cuda)
        ops.sample_uniform(lg, u, tok, temperature=t)
        ops.moe_route_scored(rl, 8, ids, w, score="sigmoid", groups=8, top_groups=4, group_score="top2")
        return tok, ids, w, ops.lora_add(x, pool, plan, y)

    want = [go(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(5):
        for i, (s, w) in enumerate(zip(streams, work)):
            with torch.cuda.stream(s):
                got[i].append(go(*w))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_step_in_a_graph_with_new_lengths(cuda):
    """Layout, adapter plan, adapters, routing and the draw captured once and replayed for steps of
    other lengths, slots and numbers, two graphs alive at the same time."""
    B, ps, cap, k, n, V, E = 6, 16, 96, 64, 128, 3000, 64
    g = torch.Generator().manual_seed(0)
    pool, ads = make_adapters(cuda, 3, k, n, 8)
    free = torch.arange(100, 160, dtype=torch.int32, device=cuda)
    xs = torch.randn(cap, k, generator=g).to(BF).to(cuda)
    ys = torch.randn(cap, n, generator=g).to(BF).to(cuda)
    lg = (torch.randn(B, V, generator=g) * 2).to(BF).to(cuda)
    rl = torch.randn(cap, E, generator=g).to(cuda)

    def make():
        st = dict(ctx=i32([0] * B, cuda), q=i32([1] * B, cuda), tab=torch.zeros(B, 8, dtype=torch.int32, device=cuda),
                  lay=ops.StepLayout(B, cap, device=cuda), slot=i32([-1] * cap, cuda), plan=ops.LoraPlan(cap, 3, cuda),
                  u=torch.zeros(B, device=cuda), t=torch.ones(B, device=cuda),
                  tok=torch.zeros(B, dtype=torch.int32, device=cuda), out=torch.zeros(cap, n, dtype=BF, device=cuda),
                  ids=torch.zeros(cap * 4, dtype=torch.int32, device=cuda), w=torch.zeros(cap * 4, device=cuda))

        def step():
            ops.step_layout(st["ctx"], st["q"], st["tab"], free, ps, st["lay"])
            ops.lora_plan(st["slot"], 3, out=st["plan"])
            ops.lora_add(xs, pool, st["plan"], ys, out=st["out"])
            ops.moe_route_scored(rl, 4, st["ids"], st["w"], score="sigmoid")
            ops.sample_uniform(lg, st["u"], st["tok"], temperature=st["t"])

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step()
        return st, gr

    rng = random.Random(1)
    pair = [make(), make()]
    want_ids, _ = route_ref(rl, 4, score="sigmoid")
    for _ in range(3):
        for st, gr in pair:
            ctx = [rng.randrange(60) for _ in range(B)]
            q = [rng.choice([0, 1, 20]) for _ in range(B)]
            while sum(q) > cap:
                q[rng.randrange(B)] = 0
            table = [[50 + 8 * b + i if i < -(-c // ps) else 0 for i in range(8)] for b, c in enumerate(ctx)]
            rows = torch.tensor([rng.randrange(-1, 3) for _ in range(cap)])
            u = [rng.random() for _ in range(B)]
            st["ctx"].copy_(i32(ctx, cuda))
            st["q"].copy_(i32(q, cuda))
            st["tab"].copy_(i32(table, cuda))
            st["slot"].copy_(rows)
            st["u"].copy_(torch.tensor(u))
            gr.replay()
            want = layout_ref(ctx, q, table, free.tolist(), ps, 32, cap, st["lay"].tile_seq.numel())
            for name, v in want.items():
                assert getattr(st["lay"], name).tolist() == v, name
            assert st["tab"].tolist() == table
            ref, tol = lora_ref(xs, ys, rows, ads)
            assert ((st["out"].double().cpu() - ref).abs() <= tol).all()
            host = lg.float().cpu().numpy()
            assert st["tok"].tolist() == [sample_ref(host[b], u[b], 1.0)[0] for b in range(B)]
            assert np.array_equal(st["ids"].view(cap, 4).cpu().numpy(), want_ids)
    assert status(cuda) == 0


@pytest.mark.parametrize("m", [40, 700])
@pytest.mark.parametrize("silu", [False, True])
def test_lora_in_two_graphs(cuda, m, silu):
    """Two captured graphs of one plan and pool, replayed in turn and next to eager calls, with new rows
    and a new adapter between replays."""
    k, n = 264, 256
    g = torch.Generator().manual_seed(m)
    pool, ads = make_adapters(cuda, 3, k, n, 16)
    slot = torch.full((m,), -1, dtype=torch.int32, device=cuda)
    plan = ops.LoraPlan(m, 3, cuda)
    pairs = []
    for _ in range(2):
        x, y = torch.randn(m, k, generator=g).to(BF).to(cuda), torch.randn(m, n, generator=g).to(BF).to(cuda)
        out = torch.zeros(m, n // 2 if silu else n, dtype=BF, device=cuda)
        ops.lora_plan(slot, 3, out=plan)
        ops.lora_add(x, pool, plan, y, out=out, silu_mul=silu)  # warm up
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            ops.lora_plan(slot, 3, out=plan)
            ops.lora_add(x, pool, plan, y, out=out, silu_mul=silu)
        pairs.append((gr, x, y, out))
    for it in range(3):
        rows = torch.randint(-1, 3, (m,), generator=g)
        slot.copy_(rows)
        a, b = (torch.randn(5, k, generator=g) / 16).to(BF), (torch.randn(n, 5, generator=g) * 0.3).to(BF)
        pool.load(it, a, b, 1.5)
        ads[it] = (a, b, 1.5)
        for gr, *_ in pairs:
            gr.replay()
        for _, x, y, out in pairs:
            want, tol = lora_ref(x, y, rows, ads, silu)
            assert ((out.double().cpu() - want).abs() <= tol).all()
            eager = ops.lora_add(x, pool, ops.lora_plan(slot, 3), y, silu_mul=silu)
            assert torch.equal(eager, out)
    assert status(cuda) == 0


def test_lora_column_ranges_of_one_buffer(cuda):
    """x, y and out as column ranges of the same rows."""
    m, k, n = 33, 64, 128
    pool, ads = make_adapters(cuda, 2, k, n, 8)
    rows = torch.arange(m) % 3 - 1
    plan = ops.lora_plan(rows.to(torch.int32).to(cuda), 2)
    buf = torch.randn(m, 400, generator=torch.Generator().manual_seed(0)).to(BF).to(cuda)
    keep = buf.clone()
    x, y, out = buf[:, 8:72], buf[:, 72:200], buf[:, 200:328]
    ops.lora_add(x, pool, plan, y, out=out)
    want, tol = lora_ref(keep[:, 8:72], keep[:, 72:200], rows, ads)
    assert ((out.double().cpu() - want).abs() <= tol).all()
    assert torch.equal(buf[:, :200], keep[:, :200]) and torch.equal(buf[:, 328:], keep[:, 328:])
    ops.lora_add(x, pool, plan, y, out=y)  # in place, next to its input
    assert torch.equal(y, out)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.lora_add(x, pool, plan, y, out=buf[:, 64:192])


@pytest.mark.parametrize("pad_tiles", [0, 7])
def test_layout_drives_the_paged_attention(cuda, pad_tiles):
    """The arrays of step_layout go straight into the KV write and both attention kernels: adapters on
    qkv, cache write, prefill attention over padded tiles, and decode attention of the next step,
    against the same numbers computed densely."""
    hq, hkv, d, ps, grp = 8, 2, 64, 16, 32
    N, Kd = (hq + 2 * hkv) * d, 128
    g = torch.Generator().manual_seed(0)
    fk, fv = K.KV_FORMATS["bf16"]
    lens = [5, 40, 0, 33]
    B, T, pages = len(lens), sum(lens), 16
    kc, vc = (torch.zeros(pages, hkv, ps, d * 2, dtype=torch.uint8, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros(pages, hkv, ps, 1, dtype=torch.float16, device=cuda) for _ in range(2))
    cos_sin = torch.cat([torch.ones(128, d // 2), torch.zeros(128, d // 2)], 1).to(cuda)  # no rotation
    pool, ads = make_adapters(cuda, 2, Kd, N, 8)
    tab = torch.full((B, 4), -1, dtype=torch.int32, device=cuda)
    free = torch.randperm(pages, generator=g).to(torch.int32).to(cuda)
    hist = [torch.zeros(0, N, dtype=torch.float64) for _ in range(B)]
    lay = ops.StepLayout(B, T + 11, T // 32 + B + pad_tiles, cuda)  # padded rows and tiles
    ctx = [0] * B
    used = 0
    for step, q in enumerate((lens, [1, 1, 1, 1])):
        n = sum(q)
        ops.step_layout(i32(ctx, cuda), i32(q, cuda), tab, free[used:], ps, lay)
        used += int(lay.totals[1])
        cap = lay.slots.numel()
        x = torch.randn(cap, Kd, generator=g).to(BF).to(cuda)
        y = torch.randn(cap, N, generator=g).to(BF).to(cuda)
        rows = torch.where(lay.token_seq >= 0, lay.token_seq % 3 - 1, torch.full_like(lay.token_seq, -1))
        plan = ops.lora_plan(rows, 2)
        qkv = ops.lora_add(x, pool, plan, y)
        ref, tol = lora_ref(x, y, rows.cpu().long(), ads)
        assert ((qkv.double().cpu() - ref).abs() <= tol).all()
        qo = torch.empty(cap, hq * d, dtype=BF, device=cuda)
        ops.rope_kv_write(qkv, lay.positions, cos_sin, qo, lay.slots, kc, ks, vc, vs, hq, hkv, d, ps, grp, fk, fv)
        out = torch.full((cap, hq * d), 3.0, dtype=BF, device=cuda)
        if step == 0:
            ops.paged_prefill_attention(qo, kc, ks, vc, vs, tab, lay.tile_seq, lay.tile_q0, lay.q_start[:B],
                                        i32(q, cuda), lay.kv_len, lay.tile_seq.numel(), out, hq, hkv, d, ps, grp, fk,
                                        fv, 1 / math.sqrt(d))
        else:
            ops.paged_decode_attention(qo[:B], kc, ks, vc, vs, tab, lay.kv_len, out[:B], hq, hkv, d, ps, grp, fk, fv,
                                       1 / math.sqrt(d), 64)
        assert (out[n:] == 3).all()  # rows behind the last sequence stay as they were
        v = qkv.double().cpu()
        r0 = 0
        for b in range(B):
            hist[b] = torch.cat([hist[b], v[r0:r0 + q[b]]])
            for i in range(q[b]):
                p = ctx[b] + i
                qq = v[r0 + i, :hq * d].view(hq, d)
                kk = hist[b][:p + 1, hq * d:(hq + hkv) * d].view(-1, hkv, d).repeat_interleave(hq // hkv, 1)
                vv = hist[b][:p + 1, (hq + hkv) * d:].view(-1, hkv, d).repeat_interleave(hq // hkv, 1)
                pr = torch.softmax(torch.einsum("hd,khd->hk", qq, kk) / math.sqrt(d), -1)
                want = torch.einsum("hk,khd->hd", pr, vv).reshape(-1)
                got = out[r0 + i].double().cpu()
                assert (got - want).abs().max() <= 2e-2 * want.abs().max() + 1e-3  # (bf16 probabilities)
            r0 += q[b]
        ctx = [c + n_ for c, n_ in zip(ctx, q)]
    ops.workspace(cuda).check()
    assert lay.tile_q0.tolist().count(PAD_Q0) >= pad_tiles


# ----------------------------------------------------------------------------- in the model
def test_scored_router_model_matches_the_cpu_model(cuda):
    """A MoE model with sigmoid scores, a choice bias, expert groups and a weight scale: the layer's
    routing is the exact one, and the engine (eager and in decode graphs) follows the CPU model."""
    from squish_b200.engine.engine import EngineConfig, LLMEngine
    from squish_b200.engine.sampling import SamplingParams
    from squish_b200.models.moe import MoELayer
    from squish_b200.models.reference import ReferenceModel

    from .test_step_ops_cpu import _scored_moe

    cfg, _, ck = _scored_moe()
    layer = MoELayer.from_checkpoint(ck, 0, cuda)
    x = torch.randn(70, cfg.hidden_size, generator=torch.Generator().manual_seed(2)).to(BF)
    h = torch.zeros(70, cfg.hidden_size, dtype=BF, device=cuda)
    layer.forward(x.to(cuda), h)
    logits = torch.mm(x.to(cuda), layer.gate_w.t())
    n, k = 70 * cfg.num_experts_per_tok, cfg.num_experts_per_tok
    ids, w = route_ref(logits, k, "sigmoid", layer.gate_bias.cpu(), 4, 2, "top2", cfg.norm_topk_prob, 2.5)
    assert np.array_equal(layer.scratch.ids[:n].view(70, k).cpu().numpy(), ids)
    np.testing.assert_allclose(layer.scratch.w[:n].view(70, k).cpu().numpy(), w, rtol=2.0**-18)
    assert h.abs().max() > 0

    ref = ReferenceModel(ck)
    prompt = np.random.default_rng(5).integers(0, cfg.vocab_size, 40).tolist()
    ref_logits = ref.forward(prompt, ref.new_cache(), 0)[-1]
    eng = LLMEngine.from_checkpoint(_scored_moe()[2], cuda, EngineConfig(max_num_seqs=4, max_num_batched_tokens=64,
                                                                         max_model_len=256, num_pages=64))
    eng.add_request(prompt, SamplingParams(max_tokens=1, ignore_eos=True))
    eng.step()
    cos = torch.nn.functional.cosine_similarity(eng.runner.logits[0].float().cpu(), ref_logits, dim=0)
    assert cos > 0.99, cos
    outs = eng.generate([prompt, prompt[:17]], SamplingParams(max_tokens=6, ignore_eos=True))
    assert [len(o) for o in outs] == [6, 6]
    eng.runner.ws.check()
