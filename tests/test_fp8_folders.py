"""What a model folder's config.json says of quantized tensors, beside how its tensors are stored (no GPU needed)."""

import json

import pytest
import torch

import tiny
from bitwise_amd import registry
from bitwise_amd.config.llama import ConfigError, LlamaConfig
from bitwise_amd.model import describe, model_spec, write_random_model
from bitwise_amd.weights import loader, safetensors_io

FOREIGN = [{"quant_method": "gptq", "bits": 4}, {"quant_method": "fp8"}, {"quant_method": "fp8", "weight_block_size": [64, 64]}, "fp8"]


def folder_of(tmp_path, weight_dtype, quantization):
    folder = write_random_model(tmp_path / weight_dtype, tiny.CONFIGS["A"][0], 3, 0.05, weight_dtype)
    config = json.loads((folder / "config.json").read_text())
    (folder / "config.json").write_text(json.dumps(dict(config, quantization_config=quantization)))
    return folder


@pytest.mark.parametrize("quantization", FOREIGN, ids=str)
@pytest.mark.parametrize("weight_dtype", ["bfloat16", "float32", "float16"])
def test_a_folder_without_quantized_tensors_is_read_whatever_its_config_says(tmp_path, weight_dtype, quantization):
    folder = folder_of(tmp_path, weight_dtype, quantization)
    raw = registry.read_model_config(folder)
    assert LlamaConfig.from_dict(raw) == LlamaConfig.from_dict(tiny.CONFIGS["A"][0])
    assert loader.load_folder(folder, describe(raw))


@pytest.mark.parametrize("quantization", FOREIGN, ids=str)
def test_a_folder_with_tensors_in_8_bits_is_held_to_its_config(tmp_path, quantization):
    raw = registry.read_model_config(folder_of(tmp_path, "float8", quantization))
    with pytest.raises(ConfigError, match="quantization_config"):
        LlamaConfig.from_dict(raw)


def test_a_folder_with_packed_tensors_is_held_to_its_config(tmp_path):
    folder = folder_of(tmp_path, "bfloat16", FOREIGN[0])
    safetensors_io.write_file(folder / "more.safetensors", [("packed", torch.zeros(4, dtype=torch.int32))])
    with pytest.raises(ConfigError, match="quantization_config"):
        LlamaConfig.from_dict(registry.read_model_config(folder))


@pytest.mark.parametrize("quantization", FOREIGN, ids=str)
def test_random_weights_are_stored_as_asked_whatever_the_config_says(tmp_path, quantization):
    config = dict(tiny.CONFIGS["A"][0], quantization_config=quantization)
    assert describe(config) == describe(tiny.CONFIGS["A"][0]) and model_spec(config) == model_spec(tiny.CONFIGS["A"][0])
    folder = write_random_model(tmp_path, config, 3, 0.05)
    assert "quantization_config" not in json.loads((folder / "config.json").read_text())


@pytest.mark.parametrize("blocks", [128, "128", None, {}, [128], [128, 128, 128], [[128, 128]]])
def test_sizes_of_blocks_that_are_no_pair_are_refused(blocks):
    with pytest.raises(ConfigError, match="quantization_config"):
        LlamaConfig.from_dict(dict(tiny.CONFIGS["A"][0], quantization_config={"quant_method": "fp8", "weight_block_size": blocks}))


@pytest.mark.parametrize("name", ["LlamaForCausalLM", "Kuponex", "Sepedra"])
@pytest.mark.parametrize("weight_dtype", ["float8", "bfloat16"])
def test_a_written_folder_says_whether_its_tensors_are_in_8_bits(tmp_path, name, weight_dtype):
    folder = write_random_model(tmp_path, dict(registry.ARCHITECTURES[name].tiny_config), 3, 0.05, weight_dtype)
    said = json.loads((folder / "config.json").read_text()).get("quantization_config")
    stored = any(t.dtype == torch.float8_e4m3fn for t in safetensors_io.read_folder(folder).values())
    assert stored == (weight_dtype == "float8" and name != "Sepedra")                   # (its parts take no matrix so)
    assert said == ({"quant_method": "fp8", "fmt": "e4m3", "activation_scheme": "dynamic", "weight_block_size": [128, 128]} if stored else None)
    raw = registry.read_model_config(folder)
    assert loader.load_folder(folder, describe(raw)).keys() == describe(raw).keys()
    registry.ARCHITECTURES[name].config_from_dict(raw)
