"""Edges of the scored router in the models, without a GPU."""
import dataclasses
import json

import numpy as np
import pytest
import torch

from squish_b200.models.config import from_hf_config, get_preset, to_hf_config
from squish_b200.models.reference import ReferenceModel

from ._step_refs import route_ref
from .test_step_ops_cpu import _scored_moe

P = "model.layers.0.mlp."


def read_config(tmp_path, **fields):
    d = to_hf_config(get_preset("tiny-moe")[0])
    d.update(fields)
    (tmp_path / "config.json").write_text(json.dumps(d))
    return from_hf_config(str(tmp_path))


def rename(ck, new):
    """The checkpoint with its router biases under another name (None: without them)."""
    for i in range(ck.config.num_layers):
        t = ck.tensors.pop(f"model.layers.{i}.mlp.gate.bias")
        if new:
            ck.tensors[f"model.layers.{i}.mlp.{new}"] = t
    return ck


# ----------------------------------------------------------------------------- config and tensor names
def test_published_router_fields(tmp_path):
    c = read_config(tmp_path, scoring_func="sigmoid", n_group=4, topk_group=2, topk_method="noaux_tc",
                    routed_scaling_factor=2.5)
    assert (c.router_score, c.router_groups, c.router_top_groups, c.router_group_score, c.router_scale,
            c.router_bias) == ("sigmoid", 4, 2, "top2", 2.5, True)
    c = read_config(tmp_path, n_group=4, topk_group=2, topk_method="group_limited_greedy")
    assert (c.router_groups, c.router_top_groups, c.router_group_score, c.router_bias) == (4, 2, "max", False)
    # greedy: the best of all experts, whatever the groups say
    c = read_config(tmp_path, n_group=4, topk_group=2, topk_method="greedy")
    assert c.router_groups == 1 and c.plain_router
    for bad, msg in [(dict(topk_method="hash"), "topk_method 'hash'"), (dict(scoring_func="relu"), "router scores"),
                     (dict(n_group=3), "do not split"), (dict(n_group=4, topk_group=5), "do not split"),
                     (dict(n_group=8, topk_group=1), "4 picks from 2 open"),
                     (dict(n_group=4, router_group_score="mean"), "group score")]:
        with pytest.raises(ValueError, match=msg):
            read_config(tmp_path, **bad)


@pytest.mark.parametrize("kw", [dict(router_group_score="top2", router_groups=4), dict(router_bias=True),
                                dict(router_score="sigmoid", router_bias=True, router_groups=2)])
def test_router_fields_survive_a_config_file(tmp_path, kw):
    cfg = dataclasses.replace(get_preset("tiny-moe")[0], **kw)
    (tmp_path / "config.json").write_text(json.dumps(to_hf_config(cfg)))
    back = from_hf_config(str(tmp_path))
    for f in ("router_score", "router_groups", "router_group_score", "router_scale", "router_bias"):
        assert getattr(back, f) == getattr(cfg, f), f


def test_router_bias_under_its_published_name():
    from squish_b200.parallel.shard import shard_checkpoint

    x = torch.randn(9, 256, generator=torch.Generator().manual_seed(1))
    want = ReferenceModel(_scored_moe()[2]).route("model.layers.0.", x)
    none = ReferenceModel(rename(_scored_moe()[2], None)).route("model.layers.0.", x)
    assert not torch.equal(none[1], want[1])  # (the bias matters)
    ck = rename(_scored_moe()[2], "gate.e_score_correction_bias")
    got = ReferenceModel(ck).route("model.layers.0.", x)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert P + "gate.e_score_correction_bias" in shard_checkpoint(ck, 1, 2).tensors


def test_a_missing_router_bias_is_refused():
    from squish_b200.models.moe import MoELayer
    from squish_b200.parallel.shard import shard_checkpoint

    ck = rename(_scored_moe()[2], None)
    ck.config = dataclasses.replace(ck.config, router_bias=True)
    for load in (ReferenceModel, lambda c: shard_checkpoint(c, 0, 2), lambda c: MoELayer.from_checkpoint(c, 0, "cpu")):
        with pytest.raises(ValueError, match="no model.layers.0.mlp.gate.e_score_correction_bias"):
            load(ck)


def test_a_router_bias_of_another_length_is_refused():
    ck = _scored_moe()[2]
    ck.tensors[P + "gate.bias"] = dataclasses.replace(ck.tensors[P + "gate.bias"], shape=(3,), data=torch.zeros(3))
    with pytest.raises(ValueError, match="one value for each of 16 experts"):
        ReferenceModel(ck)


@pytest.mark.parametrize("name", ["gate.bias", "gate.e_score_correction_bias"])
@pytest.mark.parametrize("df11", [False, True])
def test_router_bias_keeps_its_bits_through_compress(tmp_path, name, df11):
    """A choice bias near 8 whose values differ by less than a float16 step there."""
    from safetensors.torch import save_file

    from squish_b200.io.convert import compress, load_checkpoint

    ck = rename(_scored_moe()[2], name)
    cfg = ck.config
    src, out = tmp_path / "src", tmp_path / "out"
    src.mkdir()
    (src / "config.json").write_text(json.dumps(to_hf_config(cfg)))
    bias = 8.0 + torch.randperm(cfg.num_experts, generator=torch.Generator().manual_seed(0)).float() * 2.0**-16
    tensors = {k: v.dequantize().to(torch.bfloat16).contiguous() for k, v in ck.tensors.items()}
    for i in range(cfg.num_layers):
        tensors[f"model.layers.{i}.mlp.{name}"] = bias.clone()
    save_file(tensors, str(src / "model.safetensors"))
    compress(str(src), str(out), device="cpu", df11=df11, log=lambda *_: None)
    back = load_checkpoint(str(out), "cpu")[0]
    for i in range(cfg.num_layers):
        assert torch.equal(back[f"model.layers.{i}.mlp.{name}"].data.float(), bias)


# ----------------------------------------------------------------------------- the CPU model's choice
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("kw", [
    dict(router_score="sigmoid", router_groups=1, router_top_groups=0, router_group_score="max"),
    dict(router_score="sigmoid", router_groups=4, router_top_groups=2, router_group_score="top2"),
    dict(router_score="softmax", router_groups=4, router_top_groups=2, router_group_score="max"),
    dict(router_score="softmax", router_groups=8, router_top_groups=5, router_group_score="top2"),
    dict(router_score="softmax", router_groups=2, router_top_groups=1, norm_topk_prob=False),
])
def test_cpu_router_decides_like_the_kernel(kw, biased):
    """Equal scores go to the lower index, saturated ones are told apart, masked experts in an open group
    come before closed ones: the rules of ops.moe_route_scored."""
    ck = _scored_moe()[2]
    ck.config = c = dataclasses.replace(ck.config, **kw)
    ref = ReferenceModel(ck)
    E = c.num_experts
    g = torch.Generator().manual_seed(3)
    ref.w.pop(P + "gate.bias")
    if biased:
        b = torch.randint(0, 2, (E,), generator=g).float() * 0.25
        b[8:] = -float("inf")
        b[12] = 0.0  # the last groups: one expert left, or none
        ref.w[P + "gate.bias"] = b
    ref.w[P + "gate.weight"] = torch.eye(E, c.hidden_size)
    x = torch.zeros(40, c.hidden_size)
    x[:, :E] = torch.randint(-2, 3, (40, E), generator=g).float()
    x[0, :E] = 0.0
    x[1, :E] = torch.linspace(18, 30, E)     # 1 in 32 bits
    x[2, :E] = torch.linspace(-150, -120, E)  # 0 in 32 bits
    w, ids = ref.route("model.layers.0.", x)
    want_i, want_w = route_ref(x[:, :E], c.num_experts_per_tok, c.router_score, ref.w.get(P + "gate.bias"),
                               c.router_groups, c.router_top_groups or None, c.router_group_score, c.norm_topk_prob,
                               c.router_scale)
    assert np.array_equal(ids.numpy(), want_i)
    # (64-bit weights, rounded to 32 bits once)
    np.testing.assert_allclose(w.double().numpy(), want_w, rtol=2.0**-23, atol=2.0**-149)
