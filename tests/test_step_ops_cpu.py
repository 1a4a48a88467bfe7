"""Serving-step operators without a GPU: refusals, fused adapter factors, the reference forms."""
import numpy as np
import pytest
import torch

from squish_b200 import ops
from squish_b200._ext import native

from ._step_refs import layout_ref, route_ref, sample_ref


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    f = torch.zeros(2)
    C = native()
    with pytest.raises(RuntimeError, match="ctx_len must be a CUDA tensor"):
        C.step_layout(i32(2), i32(2), i32(2, 4), i32(8), 16, 32, i32(64), 2, 4, 4, i32(1))
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        ops.sample_uniform(x, f, i32(2))
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        ops.moe_route_scored(x, 2, i32(4), torch.zeros(4))
    with pytest.raises(RuntimeError, match="row_slots must be a CUDA tensor"):
        C.lora_plan(i32(2), 1, 16, i32(2), i32(3, 4), i32(1), i32(1))
    pool = ops.LoraPool(1, 8, 8, 4, "cpu")
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        ops.lora_add(x, pool, ops.LoraPlan(2, 1, "cpu"), x)


@pytest.mark.parametrize("kw,msg", [
    (dict(score="tanh"), "score must be"),
    (dict(group_score="mean"), "group_score must be"),
])
def test_route_names(kw, msg):
    with pytest.raises(ValueError, match=msg):
        ops.moe_route_scored(torch.zeros(1, 8), 1, i32(1), torch.zeros(1), **kw)


def test_layout_buffers():
    lay = ops.StepLayout(4, 70, device="cpu")
    assert lay.tile_seq.numel() == 70 // 32 + 4  # a tile per sequence and one per further 32 tokens
    lay._narrow(2)
    assert lay.q_start.numel() == 3 and lay.kv_len.numel() == 2
    with pytest.raises(ValueError, match="5 sequences in a layout of 4"):
        lay._narrow(5)
    with pytest.raises(ValueError):
        ops.StepLayout(0, 4, device="cpu")


def test_pool_checks_and_padding():
    with pytest.raises(ValueError, match="multiples of 8"):
        ops.LoraPool(1, 12, 8, 4, "cpu")
    with pytest.raises(ValueError, match="rank must be"):
        ops.LoraPool(1, 8, 8, 129, "cpu")
    with pytest.raises(ValueError, match="slots"):
        ops.LoraPool(0, 8, 8, 4, "cpu")
    p = ops.LoraPool(2, 8, 16, 20, "cpu")
    assert p.a.shape == (2, 32, 8) and p.b.shape == (2, 16, 32)
    p.load(1, torch.ones(20, 8), torch.ones(16, 20), 0.5)
    p.load(1, torch.full((3, 8), 2.0), torch.full((16, 3), 2.0), 0.25)  # a smaller rank leaves nothing behind
    assert p.rank.tolist() == [0, 3] and p.scale.tolist() == [0.0, 0.25]
    assert p.a[1].sum() == 48 and p.b[1].sum() == 96
    for bad in [(2, torch.ones(3, 8), torch.ones(16, 3)), (0, torch.ones(21, 8), torch.ones(16, 21)),
                (0, torch.ones(3, 8), torch.ones(16, 4)), (0, torch.ones(3, 9), torch.ones(16, 3))]:
        with pytest.raises(ValueError):
            p.load(*bad)
    p.clear(1)
    assert p.rank.tolist() == [0, 0]
    with pytest.raises(ValueError):
        p.clear(-1)
    with pytest.raises(ValueError, match="a plan for"):
        ops.lora_plan(i32(3), 2, out=ops.LoraPlan(4, 2, "cpu"))


def test_plan_tiles_cover_the_worst_case():
    for m in (1, 16, 17, 512, 513, 4000):
        for s in (1, 5, 64):
            p = ops.LoraPlan(m, s, "cpu")
            groups = min(s + 1, m)  # every group but one holds a single row
            worst = (groups - 1) + -(-(m - groups + 1) // p.tile_rows)
            assert worst <= p.max_tiles


def test_fuse_lora():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 24, generator=g, dtype=torch.float64)
    parts = [(torch.randn(r, 24, generator=g, dtype=torch.float64), torch.randn(n, r, generator=g, dtype=torch.float64))
             for r, n in ((2, 16), (5, 8))]
    a, b = ops.fuse_lora([parts[0], None, parts[1]], [16, 8, 8])
    want = torch.cat([x @ parts[0][0].T @ parts[0][1].T, torch.zeros(3, 8, dtype=torch.float64),
                      x @ parts[1][0].T @ parts[1][1].T], 1)
    torch.testing.assert_close(x @ a.T @ b.T, want)
    gu = [(torch.randn(r, 24, generator=g, dtype=torch.float64), torch.randn(100, r, generator=g, dtype=torch.float64))
          for r in (3, 4)]
    a, b = ops.fuse_lora(gu, [100, 100], interleave=True)
    y = (x @ a.T @ b.T).view(3, 2, 2, 64)
    for i in range(2):
        full = y[:, :, i].reshape(3, 128)
        torch.testing.assert_close(full[:, :100], x @ gu[i][0].T @ gu[i][1].T)
        assert (full[:, 100:] == 0).all()
    a, b = ops.fuse_lora([None, None], [8, 8], k=24)
    assert a.shape == (0, 24) and b.shape == (16, 0)
    for bad in [([None], [8]), ([parts[0]], [8]), ([parts[0], parts[1]], [16])]:
        with pytest.raises(ValueError):
            ops.fuse_lora(*bad)
    with pytest.raises(ValueError, match="equal sizes"):
        ops.fuse_lora(parts, [16, 8], interleave=True)


def test_reference_forms():
    """The 64-bit forms the GPU tests compare with, on cases worked out by hand."""
    t = [[7, -1, -1], [3, 4, -1]]
    r = layout_ref([2, 8], [3, 1], t, [9, 5, 6], 4, 2, 6, 4)
    assert t == [[7, 9, -1], [3, 4, 5]]
    assert r["positions"] == [2, 3, 4, 8, 0, 0] and r["slots"] == [30, 31, 36, 20, -1, -1]
    assert r["tile_seq"] == [0, 0, 1, 0] and r["totals"] == [4, 2, 3] and r["last_row"] == [2, 3]
    # weights 4 : 2 : 2 : 1 in the order 3, 0, 2, 1
    x = np.log(np.array([2.0, 1.0, 2.0, 4.0]))
    assert [sample_ref(x, u, 1.0)[0] for u in (0.0, 0.4, 0.5, 0.7, 0.95)] == [3, 3, 0, 2, 1]
    assert [sample_ref(x, u, 1.0, top_k=2)[0] for u in (0.6, 0.7, 0.999)] == [3, 0, 0]  # 4 : 2
    assert sample_ref(x, 0.999, 1.0, top_p=0.6)[0] == 0 and sample_ref(x, 0.999, 1.0, min_p=0.6)[0] == 3
    assert sample_ref(np.full(3, -np.inf), 0.5, 1.0)[0] == -1 and sample_ref(x, 0.5, 0.0) == (3, 0.0)
    ids, w = route_ref(torch.tensor([[0.0, 1.0, 1.0, -1.0]]), 2, "sigmoid", torch.tensor([2.0, 0.0, 0.0, 0.0]))
    assert ids.tolist() == [[0, 1]]
    s = 1 / (1 + np.exp(-np.array([0.0, 1.0])))
    np.testing.assert_allclose(w[0], s / s.sum())
    ids, _ = route_ref(torch.tensor([[0.0, 3.0, 2.0, 2.0]]), 2, "sigmoid", groups=2, top_groups=1, group_score="top2")
    assert ids.tolist() == [[2, 3]]


def _scored_moe():
    import dataclasses

    from squish_b200.models.config import get_preset
    from squish_b200.models.weights import QTensor, random_checkpoint

    cfg, q = get_preset("tiny-moe")
    cfg = dataclasses.replace(cfg, router_score="sigmoid", router_groups=4, router_top_groups=2,
                              router_group_score="top2", router_scale=2.5)
    ck = random_checkpoint(cfg, q, seed=3)
    g = torch.Generator().manual_seed(5)
    for i in range(cfg.num_layers):
        ck.tensors[f"model.layers.{i}.mlp.gate.bias"] = QTensor(
            "dense", (cfg.num_experts,), data=torch.randn(cfg.num_experts, generator=g) * 0.05)
    return cfg, q, ck


def test_scored_router_in_the_reference_model():
    """The CPU model's router against the 64-bit form, and through the layers."""
    from squish_b200.models.reference import ReferenceModel

    cfg, _, ck = _scored_moe()
    ref = ReferenceModel(ck)
    x = torch.randn(9, cfg.hidden_size, generator=torch.Generator().manual_seed(1))
    p = "model.layers.0."
    w, ids = ref.route(p, x)
    want_i, want_w = route_ref(x @ ref.w[p + "mlp.gate.weight"].T, cfg.num_experts_per_tok, "sigmoid",
                               ref.w[p + "mlp.gate.bias"], 4, 2, "top2", cfg.norm_topk_prob, 2.5)
    assert np.array_equal(ids.numpy(), want_i)
    np.testing.assert_allclose(w.numpy(), want_w, rtol=1e-5)
    assert torch.isfinite(ref.forward([1, 2, 3], ref.new_cache(), 0)).all()


def test_router_config_round_trip(tmp_path):
    import json

    from squish_b200.models.config import from_hf_config, get_preset, to_hf_config

    cfg, _, _ = _scored_moe()
    (tmp_path / "config.json").write_text(json.dumps(to_hf_config(cfg)))
    back = from_hf_config(str(tmp_path))
    for f in ("router_score", "router_groups", "router_top_groups", "router_group_score", "router_scale"):
        assert getattr(back, f) == getattr(cfg, f), f
    assert not back.plain_router
    plain, _ = get_preset("tiny-moe")
    assert plain.plain_router and "scoring_func" not in to_hf_config(plain)


def test_shards_keep_the_router_bias():
    from squish_b200.parallel.shard import shard_checkpoint

    cfg, _, ck = _scored_moe()
    for r in range(2):
        sh = shard_checkpoint(ck, r, 2)
        assert sh.config.router_score == "sigmoid" and "model.layers.1.mlp.gate.bias" in sh.tensors
