"""Edges of the serving-step operators (squish_b200.ops.step) on the GPU: each test is a call that the
documentation allows, or a refusal, next to the limits of an operator."""
import math
import subprocess
import sys

import numpy as np
import pytest
import torch

from squish_b200 import ops
from squish_b200.ops import kernels as K

from ._step_refs import PAD_Q0, route_ref
from .test_step_ops_gpu import BF, i32, status

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- routing
def opposite_biases(B, score, groups, gsize, T, seed):
    """Logits and a bias with which every group's two best choice values are near +B and -B and the
    groups' exact sums lie a few fp32 rounding steps of B apart (rows with an exact tie are dropped)."""
    g = torch.Generator().manual_seed(seed)
    E = groups * gsize
    s1 = 0.05 + 0.6 * torch.rand(T, groups, generator=g, dtype=torch.float64)
    total = 0.765 + (2 * torch.rand(T, groups, generator=g, dtype=torch.float64) - 1) * B * 2.0**-22
    s = torch.full((T, groups, gsize), 0.01, dtype=torch.float64)
    s[..., 0], s[..., 1] = s1, total - s1
    s = s.view(T, E)
    x = torch.log(s / (1 - s)) if score == "sigmoid" else torch.log(s)
    bias = torch.full((groups, gsize), -2.0 * B)
    bias[:, 0], bias[:, 1] = B, -B
    x, bias = x.float(), bias.view(E).float()
    exact = torch.sigmoid(x.double()) if score == "sigmoid" else torch.softmax(x.double(), -1)
    sums = (exact + bias.double()).view(T, groups, gsize)[..., :2].sum(-1).sort(-1).values
    keep = (sums[:, 1:] - sums[:, :-1]).amin(-1) > B * 2.0**-44  # (64-bit sums resolve 2^-52 B)
    return x[keep], bias


@pytest.mark.parametrize("B", [16.0, 100.0, 1e4])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,gsize", [(8, 8), (6, 11), (4, 2)])
def test_group_sums_of_opposite_biases_are_ranked_exactly(cuda, B, score, groups, gsize):
    x, bias = opposite_biases(B, score, groups, gsize, 2000, int(B) + groups)
    assert x.shape[0] > 1500
    T, k = x.shape[0], groups // 2
    ids = torch.empty(T * k, dtype=torch.int32, device=cuda)
    w = torch.empty(T * k, device=cuda)
    kw = dict(score=score, groups=groups, top_groups=groups // 2, group_score="top2")
    ops.moe_route_scored(x.to(cuda), k, ids, w, bias=bias.to(cuda), **kw)
    want, _ = route_ref(x, k, bias=bias, **kw)
    assert np.array_equal(ids.view(T, k).cpu().numpy(), want)


# ----------------------------------------------------------------------------- layout
@pytest.mark.parametrize("B", [3065, 3066, 3069, 3071, 3073])
def test_layout_sizes_around_48_kb_of_shared_memory(cuda, B):
    """The first launch of a process (a larger step before it would raise the kernel's limit)."""
    code = f"""
import torch
from squish_b200 import ops
from tests._step_refs import layout_ref
B = {B}
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
lay = ops.StepLayout(B, B, 2 * B)
table = [[b] for b in range(B)]
tab = i32(table)
ops.step_layout(i32([1] * B), i32([1] * B), tab, i32([]), 4, lay)
want = layout_ref([1] * B, [1] * B, table, [], 4, 32, B, 2 * B)
for k, v in want.items():
    assert getattr(lay, k).tolist() == v, k
ops.workspace(torch.device("cuda", 0)).check()
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_layout_sequences_that_do_not_fit_keep_their_length(cuda):
    """Without pages, table columns or rows for all of its tokens a sequence rests: kv_len is that of the
    pages it has, last_row -1, its attention tiles padding; the others are as without it."""
    def run(ctx, q, tab, free, cap=32, width=2):
        lay = ops.StepLayout(len(ctx), cap, device=cuda)
        ops.step_layout(i32(ctx, cuda), i32(q, cuda), tab, i32(free, cuda), 4, lay)
        n = lay.totals.tolist()[2]
        return lay, list(zip(lay.tile_seq.tolist(), lay.tile_q0.tolist()))[:n]

    full = lambda b, w=2: torch.full((b, w), -9, dtype=torch.int32, device=cuda)  # noqa: E731
    # one page left, the first sequence takes it; the second, with 3 tokens cached, needs two more
    tab = full(3, 3)
    tab[1, 0], tab[2, 0] = 7, 8
    lay, tiles = run([0, 3, 1], [4, 8, 2], tab, [5])
    assert lay.kv_len.tolist() == [4, 3, 3] and lay.last_row.tolist() == [3, -1, 13] and status(cuda) == 6
    assert tiles == [(0, 0), (0, PAD_Q0), (2, 0)] and tab.tolist()[0][0] == 5 and tab.tolist()[1] == [7, -9, -9]
    # a table row too narrow for the new tokens
    lay, tiles = run([3, 1], [6, 1], torch.tensor([[1, -9], [2, -9]], dtype=torch.int32, device=cuda), [4, 3])
    assert lay.kv_len.tolist() == [3, 2] and lay.last_row.tolist() == [-1, 6] and status(cuda) == 6
    assert tiles == [(0, PAD_Q0), (1, 0)]
    # a resting sequence whose context its table row cannot hold: no more than the row's pages
    lay, _ = run([100, 8], [0, 0], full(2), [])
    assert lay.kv_len.tolist() == [8, 8] and lay.last_row.tolist() == [-1, -1] and status(cuda) == 6
    lay, _ = run([8, 8], [0, 0], full(2), [])
    assert lay.kv_len.tolist() == [8, 8] and status(cuda) == 0
    # more tokens than rows: sequences past the buffers rest, q_start tells the rows that were asked for
    lay, tiles = run([0, 2, 1], [3, 3, 2], torch.ones(3, 2, dtype=torch.int32, device=cuda), [1, 2, 3], cap=4)
    assert lay.kv_len.tolist() == [3, 2, 1] and lay.last_row.tolist() == [2, -1, -1] and status(cuda) == 6
    assert tiles == [(0, 0), (0, PAD_Q0), (0, PAD_Q0)]
    # sums past 32 bits
    lay, _ = run([2] * 4, [2**30] * 4, full(4), [1], cap=4)
    assert lay.kv_len.tolist() == [2] * 4 and lay.last_row.tolist() == [-1] * 4 and status(cuda) == 6


def test_layout_inputs_inside_the_tables_are_refused(cuda):
    """(other blocks write the tables while the lengths and the free list are read)"""
    lay = ops.StepLayout(2, 8, device=cuda)
    tab = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    ok = dict(c=i32([0, 0], cuda), q=i32([1, 1], cuda), f=i32([1, 2, 3], cuda))
    for k, name in (("c", "ctx_len"), ("q", "q_len"), ("f", "free_pages")):
        a = {**ok, k: tab[1, 1:3]}
        with pytest.raises(RuntimeError, match=name + " is part of block_tables"):
            ops.step_layout(a["c"], a["q"], tab, a["f"], 4, lay)
    with pytest.raises(RuntimeError, match="block_tables is part of the step layout"):
        ops.step_layout(ok["c"], ok["q"], lay.buf[:8].view(2, 4), ok["f"], 4, lay)
    arena = torch.zeros(16, dtype=torch.int32, device=cuda)  # neighbours in one buffer are allowed
    arena[10:12] = 1
    ops.step_layout(arena[8:10], arena[10:12], arena[:8].view(2, 4), arena[12:16], 4, lay)
    assert lay.kv_len.tolist() == [1, 1] and status(cuda) == 0


def paged(cuda, pages, hkv, ps, d, seed):
    """bf16 KV pages with values, and [pages * ps, hkv, d] views of keys and values."""
    g = torch.Generator().manual_seed(seed)
    kv = [torch.randn(pages, hkv, ps, d, generator=g).to(BF).to(cuda) for _ in range(2)]
    codes = [t.view(torch.uint8).view(pages, hkv, ps, 2 * d) for t in kv]
    scales = [torch.zeros(pages, hkv, ps, 1, dtype=torch.float16, device=cuda) for _ in range(2)]
    return (codes[0], scales[0], codes[1], scales[1]), kv


def attend(q, k, v, n):
    """Rows of one query [hq * d] over the first n keys and values [*, hkv, d], in 64 bits, and the error of
    probabilities in bf16 (2^-8 of the mass of |v|, its sums far below) and of the output in bf16."""
    d = k.shape[-1]
    q = q.double().cpu().view(-1, d)
    kk, vv = (t[:n].double().cpu().repeat_interleave(q.shape[0] // t.shape[1], 1) for t in (k, v))
    p = torch.softmax(torch.einsum("hd,khd->hk", q, kk) / math.sqrt(d), -1)
    out = torch.einsum("hk,khd->hd", p, vv).reshape(-1)
    return out, 2.0**-7 * torch.einsum("hk,khd->hd", p, vv.abs()).reshape(-1) + 2.0**-8 * out.abs() + 2.0**-12


def test_attention_reads_no_page_that_a_sequence_did_not_get(cuda):
    """The free list runs out: the table entries behind a sequence's pages still name pages that belong to
    others, and neither attention kernel looks at them."""
    hq, hkv, d, ps, pages = 4, 2, 64, 16, 6
    cache, kv = paged(cuda, pages, hkv, ps, d, 3)
    fk, fv = K.KV_FORMATS["bf16"]
    x = torch.randn(64, hq * d, generator=torch.Generator().manual_seed(4)).to(BF).to(cuda)
    # (sequence 0 has pages 0 and 1; sequence 1 has page 2 for its 16 tokens, then a stale entry, page 1)
    tab = torch.tensor([[0, 1, -1], [2, 1, 0]], dtype=torch.int32, device=cuda)
    rows = [t[[2]].transpose(1, 2).reshape(ps, hkv, d) for t in kv]
    lay = ops.StepLayout(2, 64, device=cuda)
    ops.step_layout(i32([31, 16], cuda), i32([1, 1], cuda), tab, i32([], cuda), ps, lay)
    assert status(cuda) == 6 and lay.kv_len.tolist() == [32, 16] and lay.last_row.tolist() == [0, -1]
    out = torch.zeros(2, hq * d, dtype=BF, device=cuda)
    ops.paged_decode_attention(x[:2], *cache, tab, lay.kv_len, out, hq, hkv, d, ps, 32, fk, fv, 1 / math.sqrt(d), 64)
    want, tol = attend(x[1], *rows, 16)
    assert ((out[1].double().cpu() - want).abs() <= tol).all()
    q = i32([1, 20], cuda)
    ops.step_layout(i32([31, 16], cuda), q, tab, i32([], cuda), ps, lay)
    out = torch.full((64, hq * d), 3.0, dtype=BF, device=cuda)
    ops.paged_prefill_attention(x, *cache, tab, lay.tile_seq, lay.tile_q0, lay.q_start[:2], q, lay.kv_len,
                                lay.tile_seq.numel(), out, hq, hkv, d, ps, 32, fk, fv, 1 / math.sqrt(d))
    assert (out[1:] == 3).all() and not (out[0] == 3).all()
    assert status(cuda) == 6


def test_padding_tiles_do_not_read_the_cache(cuda):
    """A padding tile names sequence 0: whatever that sequence's table holds, it is not looked at (bf16 KV,
    which the tensor-core kernel does not serve)."""
    hq, hkv, d, ps, pages = 4, 2, 64, 16, 4
    cache, kv = paged(cuda, pages, hkv, ps, d, 0)
    ops.workspace(cuda).status.zero_()
    fk, fv = K.KV_FORMATS["bf16"]
    lay = ops.StepLayout(2, 40, device=cuda)
    # sequence 0 rests; its entries were given to nobody (10^6 lies outside the pool)
    tab = torch.tensor([[10**6, 10**6, 10**6], [2, 1, 3]], dtype=torch.int32, device=cuda)
    ops.step_layout(i32([40, 13], cuda), i32([0, 20], cuda), tab, i32([1, 3, 0], cuda), ps, lay)
    assert lay.tile_q0.tolist().count(PAD_Q0) == 2 and lay.tile_seq.tolist()[1:] == [0, 0]
    x = torch.randn(40, hq * d, generator=torch.Generator().manual_seed(1)).to(BF).to(cuda)
    out = torch.full((40, hq * d), 3.0, dtype=BF, device=cuda)
    ops.paged_prefill_attention(x, *cache, tab, lay.tile_seq, lay.tile_q0, lay.q_start[:2], i32([0, 20], cuda),
                                lay.kv_len, lay.tile_seq.numel(), out, hq, hkv, d, ps, 32, fk, fv, 1 / math.sqrt(d))
    assert status(cuda) == 0
    assert (out[20:] == 3).all()
    rows = [t[[2, 1, 3]].transpose(1, 2).reshape(3 * ps, hkv, d) for t in kv]
    for i in range(20):
        want, tol = attend(x[i], *rows, 13 + i + 1)
        assert ((out[i].double().cpu() - want).abs() <= tol).all()


# ----------------------------------------------------------------------------- in the model
@pytest.mark.parametrize("graphs", [False, True])
def test_scored_router_decode_steps_follow_the_cpu_model(cuda, graphs):
    """Each decode step's logits, launched eagerly and from captured graphs, against the CPU model fed the
    tokens that the engine drew."""
    from squish_b200.engine.engine import EngineConfig, LLMEngine
    from squish_b200.engine.sampling import SamplingParams
    from squish_b200.models.reference import ReferenceModel

    from .test_step_ops_cpu import _scored_moe

    cfg, _, ck = _scored_moe()
    ref = ReferenceModel(ck)
    prompt = np.random.default_rng(7).integers(0, cfg.vocab_size, 21).tolist()
    eng = LLMEngine.from_checkpoint(ck, cuda, EngineConfig(max_num_seqs=4, max_num_batched_tokens=64,
                                                           max_model_len=256, num_pages=64, cuda_graphs=graphs))
    rid = eng.add_request(prompt, SamplingParams(max_tokens=6, ignore_eos=True))
    cache = ref.new_cache()
    want = ref.forward(prompt, cache, 0)[-1]
    n = 0
    while eng.has_unfinished():
        eng.step()
        out = eng.requests[rid].output
        assert len(out) == n + 1
        got = eng.runner.logits[0].float().cpu()
        assert torch.nn.functional.cosine_similarity(got, want, dim=0) > 0.99, n
        n += 1
        want = ref.forward([out[-1]], cache, len(prompt) + n - 1)[-1]
    assert n == 6
    eng.runner.ws.check()
