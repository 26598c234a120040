"""Checkpoints with matrices in 8 bits: reading, writing, checking and random weights (no GPU needed)."""

import json

import pytest
import torch

import tiny
from bitwise_amd.config.llama import ConfigError, LlamaConfig
from bitwise_amd.model import describe, write_random_model
from bitwise_amd.parts.base import TensorSpec
from bitwise_amd.weights import block_scaled, loader, safetensors_io
from bitwise_amd.weights.block_scaled import BlockScaled


def matrix(n, k, seed=0):
    return block_scaled.quantize(torch.randn(n, k, generator=torch.Generator().manual_seed(seed)))


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 300), (257, 64)])
def test_quantized_matrices(n, k):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(1))
    codes, scales = block_scaled.quantize(w)
    assert codes.shape == (n, k) and scales.shape == (-(-n // 128), -(-k // 128))
    back = BlockScaled([(codes, scales)], k).widened()
    spread = scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    # half a step of a normal number, half the least step of a small one, and the roundings of scale, quotient and product
    assert ((back - w).abs() <= torch.maximum(w.abs() * 2.0 ** -4, spread * 2.0 ** -10) + 4 * 2.0 ** -24 * w.abs()).all()
    zeros, s = block_scaled.quantize(torch.zeros(3, 5))
    assert (zeros.float() == 0).all() and (s == 2.0 ** -126).all()


def test_codes_survive_a_file(tmp_path):
    codes, scales = matrix(40, 200)
    safetensors_io.write_file(tmp_path / "x.safetensors", [("w", codes), ("w_scale_inv", scales), ("b", torch.ones(3).bfloat16())])
    back = safetensors_io.read_file(tmp_path / "x.safetensors")
    assert back["w"].dtype == torch.float8_e4m3fn and torch.equal(back["w"].view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(back["w_scale_inv"], scales)


def test_stacks_keep_their_blocks():
    a, b = (BlockScaled([matrix(n, 200, n)], 200) for n in (130, 60))
    both = block_scaled.stacked([a, b])
    assert both.shape == (190, 200) and both.dtype == torch.float8_e4m3fn and len(both.parts) == 2
    assert torch.equal(both.widened(), torch.cat([a.widened(), b.widened()]))
    on = both.on("cpu")
    assert on.codes.shape == (190, 256) and on.scales.shape == (3, 2) and len(on.parts) == 2
    assert torch.equal(on.widened(), both.widened()) and not on.codes[:, 200:].view(torch.uint8).any()
    whole = block_scaled.stacked([BlockScaled([matrix(256, 200)], 200), b]).on("cpu")
    assert len(whole.parts) == 1 and whole.parts[0][0].shape == (316, 256)


SPECS = {"m": TensorSpec((130, 200), block_scaled=True), "plain": TensorSpec((4, 4))}


def found(**more):
    codes, scales = matrix(130, 200)
    return {"m": codes, "m_scale_inv": scales, "plain": torch.zeros(4, 4), **more}


def test_a_checkpoint_in_8_bits_is_taken():
    out = loader.check_and_convert(SPECS, found())
    assert isinstance(out["m"], BlockScaled) and out["m"].shape == (130, 200) and set(out) == {"m", "plain"}
    wide = loader.check_and_convert(SPECS, found(m_scale_inv=torch.ones(2, 2).bfloat16()))
    assert wide["m"].parts[0][1].dtype == torch.float32


@pytest.mark.parametrize("change,says", [
    ({"m_scale_inv": None}, "m_scale_inv"),
    ({"m_scale_inv": torch.ones(2, 1)}, "scale for each block"),
    ({"m_scale_inv": torch.ones(2, 2, dtype=torch.int32)}, "scale for each block"),
    ({"m_scale_inv": torch.full((2, 2), float("nan"))}, "no finite"),
    ({"plain": torch.zeros(4, 4).to(torch.float8_e4m3fn), "plain_scale_inv": torch.ones(1, 1)}, "unsupported dtype"),
    ({"m": torch.zeros(130, 200)}, "unexpected"),
])
def test_what_does_not_fit_is_named(change, says):
    tensors = {n: t for n, t in found(**change).items() if t is not None}
    with pytest.raises(loader.WeightError, match=says):
        loader.check_and_convert(SPECS, tensors)


def test_random_models_in_8_bits(tmp_path):
    cfg = tiny.CONFIGS["B"][0]
    folder = write_random_model(tmp_path, cfg, 3, 0.05, "float8")
    tensors = safetensors_io.read_folder(folder)
    specs = describe(json.loads((folder / "config.json").read_text()))
    for name, spec in specs.items():
        assert tensors[name].dtype == (torch.float8_e4m3fn if spec.block_scaled else torch.bfloat16)
    assert sum(s.block_scaled for s in specs.values()) == 7 * cfg["num_hidden_layers"]
    assert isinstance(loader.load_folder(folder, specs)["model.layers.0.mlp.up_proj.weight"], BlockScaled)


def test_a_config_of_other_blocks_is_refused():
    cfg = dict(tiny.CONFIGS["A"][0])
    LlamaConfig.from_dict(dict(cfg, quantization_config={"quant_method": "fp8", "fmt": "e4m3", "weight_block_size": [128, 128]}))
    for other in ("fp8", {"quant_method": "gptq"}, {"quant_method": "fp8", "weight_block_size": [64, 64]}, {"quant_method": "fp8"},
                  {"quant_method": "fp8", "fmt": "e5m2", "weight_block_size": [128, 128]},
                  {"quant_method": "fp8", "weight_block_size": [128, 128], "activation_scheme": "static"}):
        with pytest.raises(ConfigError, match="quantization_config"):
            LlamaConfig.from_dict(dict(cfg, quantization_config=other))


def test_the_command_line_writes_a_folder_in_8_bits(tmp_path):
    from bitwise_amd.cli import main

    config = tmp_path / "config.json"
    config.write_text(json.dumps(tiny.CONFIGS["A"][0]))
    assert main(["random", "--config", str(config), "--seed", "3", "--weight-dtype", "float8", "--out", str(tmp_path / "m")]) == 0
    tensors = safetensors_io.read_folder(tmp_path / "m")
    assert tensors["model.layers.0.self_attn.q_proj.weight"].dtype == torch.float8_e4m3fn
    assert tensors["model.layers.0.self_attn.q_proj.weight_scale_inv"].dtype == torch.float32
    assert tensors["model.norm.weight"].dtype == torch.bfloat16
