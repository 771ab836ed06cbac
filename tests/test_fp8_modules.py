"""Modules held in block-scaled e4m3 beside product-quantised ones: the config key, the method's parameters and loaders, the
quantise command, and (gpu) a checkpoint with both formats through the layers."""
import json
import os

import pytest
import torch

from vllm_pq_amd import BlockFP8LinearMethod, PQConfig, PQLinearMethod
from vllm_pq_amd.fp8 import fp8_quantize_weight, fp8_reconstruct, is_fp8_module
from vllm_pq_amd.host import parallel_state
from vllm_pq_amd.host.linear import (ColumnParallelLinear, MergedColumnParallelLinear, QKVParallelLinear, RowParallelLinear)

F8 = torch.float8_e4m3fn
BF16 = torch.bfloat16
DEV = "cuda:0"


def _dense(seed, n, k):
    return (torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) / k ** 0.5).to(BF16)


def _with_rank(monkeypatch, rank, size):
    monkeypatch.setattr(parallel_state, "_TP_RANK", rank)
    monkeypatch.setattr(parallel_state, "_TP_SIZE", size)


def test_config_key_and_method_choice():
    cfg = PQConfig.from_config({"in_group_size": 8, "nbits_per_codebook": 8, "fp8_modules": ["down_proj", r"layers\.0\.self_attn"]})
    assert cfg.fp8_modules == ["down_proj", r"layers\.0\.self_attn"]
    pick = lambda p: type(ColumnParallelLinear(256, 128, bias=False, params_dtype=BF16, quant_config=cfg, prefix=p).quant_method)  # noqa: E731
    assert pick("model.layers.3.mlp.down_proj") is BlockFP8LinearMethod
    assert pick("model.layers.0.self_attn.qkv_proj") is BlockFP8LinearMethod
    assert pick("model.layers.1.self_attn.qkv_proj") is PQLinearMethod and pick("") is PQLinearMethod
    assert PQConfig().fp8_modules == []
    # a fused layer goes by the names of what it stacks, all of them or none
    assert is_fp8_module("a.mlp.gate_up_proj", ["gate_proj", "up_proj"]) and is_fp8_module("a.mlp.gate_up_proj", ["gate_up"])
    assert not is_fp8_module("a.mlp.gate_up_proj", ["down_proj"]) and not is_fp8_module("qkv_proj", ["o_proj$"])
    with pytest.raises(ValueError, match="only a part"):
        is_fp8_module("a.self_attn.qkv_proj", ["v_proj"])


def test_one_expression_in_place_of_a_list_is_refused():
    from vllm_pq_amd.quantize import quantization_config, quantize_state_dict
    for call in (lambda: PQConfig(fp8_modules="down_proj"), lambda: quantization_config(8, 8, 1, "down_proj"),
                 lambda: PQConfig.from_config({"in_group_size": 8, "nbits_per_codebook": 8, "fp8_modules": "down_proj"}),
                 lambda: quantize_state_dict({}, fp8_modules="down_proj")):
        with pytest.raises(ValueError, match="list of regular expressions"):
            call()


def test_create_weights_shapes_and_refusals(monkeypatch):
    cfg = PQConfig(fp8_modules=["."])
    layer = RowParallelLinear(300, 200, bias=False, params_dtype=BF16, quant_config=cfg, prefix="x")
    assert layer.weight.shape == (200, 300) and layer.weight.dtype == F8
    assert layer.weight_scale_inv.shape == (2, 3) and layer.weight_scale_inv.dtype == torch.float32
    with pytest.raises(ValueError, match="half and bfloat16"):
        ColumnParallelLinear(256, 256, bias=False, params_dtype=torch.float32, quant_config=cfg, prefix="x")
    with pytest.raises(ValueError, match="scale block"):
        MergedColumnParallelLinear(256, [192, 192], bias=False, params_dtype=BF16, quant_config=cfg, prefix="x")
    _with_rank(monkeypatch, 0, 2)
    with pytest.raises(ValueError, match="scale block"):
        RowParallelLinear(384, 128, bias=False, params_dtype=BF16, quant_config=cfg, prefix="x")
    with pytest.raises(ValueError, match="scale block"):
        ColumnParallelLinear(256, 384, bias=False, params_dtype=BF16, quant_config=cfg, prefix="x")


@pytest.mark.parametrize("tp", [1, 2])
def test_loaders_shard_weight_and_scales_alike(monkeypatch, tp):
    cfg = PQConfig(fp8_modules=["."])
    mats = {n: fp8_quantize_weight(_dense(i, rows, 512)) for i, (n, rows) in
            enumerate({"q": 512, "k": 256, "v": 256, "gate": 512, "up": 512, "down": 384}.items())}
    got = {n: [] for n in mats}
    for rank in range(tp):
        _with_rank(monkeypatch, rank, tp)
        qkv = QKVParallelLinear(512, 128, 4, 2, bias=False, params_dtype=BF16, quant_config=cfg, prefix="qkv_proj")
        gu = MergedColumnParallelLinear(512, [512, 512], bias=False, params_dtype=BF16, quant_config=cfg, prefix="gate_up_proj")
        down = RowParallelLinear(512, 384, bias=False, params_dtype=BF16, quant_config=cfg, prefix="down_proj")
        for layer, ids in ((qkv, ("q", "k", "v")), (gu, ("gate", "up")), (down, ("down",))):
            for i, n in enumerate(ids):
                for p, t in zip((layer.weight, layer.weight_scale_inv), mats[n]):
                    args = () if n == "down" else (n,) if layer is qkv else (i,)
                    p.weight_loader(p, t, *args)
            layer.quant_method.process_weights_after_loading(layer)
            dense = fp8_reconstruct(layer.weight.data, layer.weight_scale_inv.data)
            rows = [mats[n][0].shape[0] // (1 if n == "down" else tp) for n in ids]
            for n, part in zip(ids, dense.split(rows)):
                got[n].append(part)
    for n, (w, s) in mats.items():
        assert torch.equal(torch.cat(got[n], 1 if n == "down" else 0), fp8_reconstruct(w, s))


@pytest.mark.parametrize("n,k", [(128, 128), (300, 200), (1, 5), (257, 129)])
def test_weight_quantisation(n, k):
    w = _dense(n + k, n, k)
    q, s = fp8_quantize_weight(w)
    assert q.shape == (n, k) and q.dtype == F8 and s.shape == ((n + 127) // 128, (k + 127) // 128)
    sd = s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k].double()
    # half a step: 2^-4 of the value, or half the smallest step, 2^-10 of the scale; the quotient's fp32 rounding on top
    err = (q.double() * sd - w.double()).abs()
    assert (err <= torch.maximum(2.0 ** -4 * w.double().abs(), 2.0 ** -10 * sd) * (1 + 2.0 ** -20)).all()
    z, zs = fp8_quantize_weight(torch.zeros(3, 4))
    assert not z.float().any() and torch.isfinite(zs).all() and (zs > 0).all()
    with pytest.raises(ValueError):
        fp8_quantize_weight(torch.zeros(3))


def _checkpoint(tmp_path, H=256, inter=512):
    from safetensors.torch import save_file
    state = {f"model.layers.0.mlp.{n}.weight": _dense(i, r, c) for i, (n, r, c) in
             enumerate((("gate_proj", inter, H), ("up_proj", inter, H), ("down_proj", H, inter)))}
    state["model.norm.weight"] = torch.ones(H, dtype=BF16)
    os.makedirs(tmp_path / "in")
    save_file(state, str(tmp_path / "in" / "model.safetensors"))
    (tmp_path / "in" / "config.json").write_text(json.dumps({"hidden_size": H}))
    return state


def test_quantise_command_writes_both_formats(tmp_path, capsys):
    from safetensors.torch import load_file
    from vllm_pq_amd.quantize import _main
    state = _checkpoint(tmp_path)
    assert _main([str(tmp_path / "in"), str(tmp_path / "out"), "--iters", "2", "--device", "cpu", "--fp8", "down_proj"]) == 0
    assert capsys.readouterr().out.count("relative error") == 3
    disk = load_file(str(tmp_path / "out" / "model.safetensors"))
    name = "model.layers.0.mlp.down_proj.weight"
    assert disk[name].dtype == F8 and disk[name + "_scale_inv"].dtype == torch.float32
    assert "model.layers.0.mlp.gate_proj.codes" in disk and "model.layers.0.mlp.down_proj.codes" not in disk
    assert "model.layers.0.mlp.gate_proj.weight" not in disk and "model.norm.weight" in disk
    rel = (fp8_reconstruct(disk[name], disk[name + "_scale_inv"]) - state[name].float()).norm() / state[name].float().norm()
    assert rel < 2.0 ** -4
    cfg = PQConfig.from_config(json.loads((tmp_path / "out" / "config.json").read_text())["quantization_config"])
    assert cfg.fp8_modules == ["down_proj"]


def _attention_state(head="model.layers.0."):
    names = [f"{head}self_attn.{n}_proj" for n in "qkvo"] + [f"{head}mlp.{n}_proj" for n in ("gate", "up", "down")]
    return {n + ".weight": _dense(i, 128, 128) for i, n in enumerate(names)}


@pytest.mark.parametrize("fp8", [["qkv_proj"], ["gate_up_proj"], ["gate_up"], ["self_attn"], ["[qkv]_proj"], ["o_proj", "qkv_proj$"], [r"\.0\.mlp"],
                                 ["."], ["q_proj", "k_proj", "v_proj", "down_proj"]])
def test_quantiser_and_loader_choose_alike(fp8):
    """Whatever the expressions, a layer that the config makes an e4m3 one finds e4m3 tensors, and the others find codes."""
    from vllm_pq_amd.quantize import quantization_config, quantize_state_dict
    state = _attention_state()
    out = quantize_state_dict(state, iters=1, fp8_modules=fp8)
    cfg = PQConfig.from_config(quantization_config(8, 8, 1, fp8))
    kinds = set()
    for layer, parts in (("self_attn.qkv_proj", ("q_proj", "k_proj", "v_proj")), ("self_attn.o_proj", ("o_proj",)),
                         ("mlp.gate_up_proj", ("gate_proj", "up_proj")), ("mlp.down_proj", ("down_proj",))):
        prefix = "model.layers.0." + layer
        method = type(ColumnParallelLinear(128, 128, bias=False, params_dtype=BF16, quant_config=cfg, prefix=prefix).quant_method)
        kinds.add(method)
        for n in parts:
            base = prefix.rpartition(".")[0] + "." + n
            has = {k for k in ("weight", "weight_scale_inv", "codes", "codebooks", "scales") if f"{base}.{k}" in out}
            assert has == ({"weight", "weight_scale_inv"} if method is BlockFP8LinearMethod else {"codes", "codebooks", "scales"})
    assert BlockFP8LinearMethod in kinds


def test_quantiser_refuses_what_the_loader_would():
    from vllm_pq_amd.quantize import quantize_state_dict
    state = _attention_state()
    for fp8 in (["v_proj"], ["up_proj"], ["down_proj", "gate_proj"], ["q_proj", "k_proj"]):
        with pytest.raises(ValueError, match="only a part"):
            quantize_state_dict(state, iters=1, fp8_modules=fp8)
    # a q_proj that nothing is stacked with goes by its own name, as the layer of that name does
    alone = {"m.q_proj.weight": state["model.layers.0.self_attn.q_proj.weight"]}
    assert "m.q_proj.weight_scale_inv" in quantize_state_dict(alone, fp8_modules=["q_proj"])
    # and a matrix that is stacked on disk already by the stacked layer's
    stacked = {"m.qkv_proj.weight": _dense(0, 384, 128)}
    assert "m.qkv_proj.weight_scale_inv" in quantize_state_dict(stacked, fp8_modules=["qkv_proj"])
    with pytest.raises(ValueError, match="only a part"):
        quantize_state_dict(stacked, fp8_modules=["v_proj"])


def test_quantiser_refuses_an_expression_that_names_nothing(tmp_path):
    from vllm_pq_amd.quantize import _main, quantize_state_dict
    state = _attention_state()
    for fp8, lost in ((["dwon_proj"], "dwon_proj"), (["down_proj", r"layers\.7\."], "layers"), (["norm"], "norm")):
        with pytest.raises(ValueError, match=lost):
            quantize_state_dict({**state, "model.norm.weight": torch.ones(128)}, iters=1, fp8_modules=fp8)
    _checkpoint(tmp_path)
    with pytest.raises(ValueError, match="o_proj"):
        _main([str(tmp_path / "in"), str(tmp_path / "out"), "--iters", "1", "--device", "cpu", "--fp8", "o_proj"])
    assert not (tmp_path / "out").exists()


def test_quantiser_refuses_stacked_matrices_of_odd_size():
    from vllm_pq_amd.quantize import quantize_state_dict
    state = {f"mlp.{n}.weight": _dense(i, 192, 128) for i, n in enumerate(("gate_proj", "up_proj"))}
    with pytest.raises(ValueError, match="scale block"):
        quantize_state_dict(state, fp8_modules=["gate_up_proj"])
    alone = quantize_state_dict({"mlp.down_proj.weight": _dense(0, 192, 100)}, fp8_modules=["down_proj"])
    assert alone["mlp.down_proj.weight_scale_inv"].shape == (2, 1)


def test_method_raises_on_cpu():
    layer = ColumnParallelLinear(256, 128, bias=False, params_dtype=BF16, quant_config=PQConfig(fp8_modules=["."]), prefix="x")
    m, x = layer.quant_method, torch.zeros(2, 256, dtype=BF16)
    for call in (lambda: layer(x), lambda: m.apply_after_norm(layer, x, None, x[0], 1e-5), lambda: m.apply_silu_and_mul(layer, x),
                 lambda: m.apply_after_silu_and_mul(layer, torch.zeros(2, 512, dtype=BF16))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 90])
def test_gpu_layers_of_both_formats(tmp_path, T):
    """A quantised checkpoint through the layers: gate_up_proj product-quantised, down_proj in e4m3, and the other way round."""
    from safetensors.torch import load_file
    from vllm_pq_amd.host.layers import RMSNorm, SiluAndMul
    from vllm_pq_amd.quantize import _main
    H, inter = 256, 512
    state = _checkpoint(tmp_path, H, inter)
    gen = torch.Generator().manual_seed(T)
    x, res = (torch.randn(T, H, generator=gen).to(BF16).to(DEV) for _ in range(2))
    norm = RMSNorm(H, eps=1e-5).to(DEV).to(BF16)
    for fp8 in (["down_proj"], ["gate_proj", "up_proj"]):
        out = str(tmp_path / ("out" + fp8[0]))
        assert _main([str(tmp_path / "in"), out, "--iters", "2", "--device", "cpu"] + [a for f in fp8 for a in ("--fp8", f)]) == 0
        disk = load_file(os.path.join(out, "model.safetensors"))
        with open(os.path.join(out, "config.json")) as f:
            cfg = PQConfig.from_config(json.load(f)["quantization_config"])
        gu = MergedColumnParallelLinear(H, [inter, inter], bias=False, params_dtype=BF16, quant_config=cfg, prefix="model.layers.0.mlp.gate_up_proj")
        down = RowParallelLinear(inter, H, bias=False, params_dtype=BF16, quant_config=cfg, prefix="model.layers.0.mlp.down_proj")
        for layer, names in ((gu, ("gate_proj", "up_proj")), (down, ("down_proj",))):
            for i, n in enumerate(names):
                for pname, p in layer.named_parameters():
                    t = disk[f"model.layers.0.mlp.{n}.{pname}"]
                    p.weight_loader(p, t, i) if len(names) > 1 else p.weight_loader(p, t)
            layer.to(DEV)
            layer.quant_method.process_weights_after_loading(layer)
        gm, dm = gu.quant_method, down.quant_method
        act = gm.apply_silu_and_mul(gu, norm(x))
        y, _ = down(act)
        if isinstance(dm, BlockFP8LinearMethod):
            gate_up, _ = gu(norm(x))
            want = fp8_reconstruct(down.weight.data, down.weight_scale_inv.data)
            z = dm.apply_after_silu_and_mul(down, gate_up)
            # both against the product in 64 bits: 8-bit activations are off by at most 2^-4 of themselves, about 2^-5.5 rms, and
            # the errors of one sum's 512 terms are independent: the results' norm is off by about as much
            exact = SiluAndMul()(gate_up).double() @ want.double().t()
            for got in (y, z):
                assert (got.double() - exact).norm() / exact.norm() < 2.0 ** -4
        else:
            want = fp8_reconstruct(gu.weight.data, gu.weight_scale_inv.data)
            r1, r2 = res.clone(), res.clone()
            got = gm.apply_after_norm(gu, x, r1, norm.weight.data, 1e-5)
            h, _ = norm(x.clone(), r2)
            assert torch.equal(r1, r2)
            exact = h.double() @ want.double().t()
            assert (got.double() - exact).norm() / exact.norm() < 2.0 ** -4
            assert (gu(h)[0].double() - exact).norm() / exact.norm() < 2.0 ** -4
            assert (gm.apply_after_norm(gu, x, None, norm.weight.data, 1e-5).double() - norm(x).double() @ want.double().t()).norm() \
                < 2.0 ** -4 * (norm(x).double() @ want.double().t()).norm()
        assert y.shape == (T, H) and torch.isfinite(y.float()).all()
