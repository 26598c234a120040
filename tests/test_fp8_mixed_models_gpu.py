"""Layers some of whose matrices are in 8 bits, against the float64 decoder with the inputs of just those products in 8 bits."""

import json

import pytest
import torch

import plain_llama as pl
import tiny
from bitwise_amd.csrc import ops
from bitwise_amd.weights import block_scaled, loader, safetensors_io
from replay_util import check_against_plain, requests_for
from test_fp8_models_gpu import quantized_rows, widened

pytestmark = pytest.mark.gpu

STORED = {"gate_up": ("gate_proj", "up_proj"), "down": ("down_proj",), "qkv": ("q_proj", "k_proj", "v_proj"), "o": ("o_proj",),
          "mlp": ("gate_proj", "up_proj", "down_proj"), "attention": ("q_proj", "k_proj", "v_proj", "o_proj")}


def normed_codes(x, weight, eps):
    """What the normed rows in front of q|k|v stand for in 8 bits, as the operator leaves them: the codes of the definition but where the quotient
    lies at the border between two (the norm's 32-bit steps, sixteen half steps at most in rows of 96, put it on either side: x w of bfloat16
    numbers is often exactly there).  Such a code is taken over, because keys and values carry it into every later position."""
    rows, dim = x.shape
    codes = torch.zeros(rows, ops.fp8_width(dim), dtype=torch.uint8, device="cuda").view(ops.FP8)
    scales = torch.zeros(codes.shape[1] // 128, rows, device="cuda")
    ops.norm_add_norm(x.float().cuda(), None, weight.float().cuda(), codes, rows, eps, scales=scales)
    got, xn = codes.cpu()[:, :dim].double(), pl.rmsnorm(x, weight, eps)
    quotient = 448.0 * xn / xn.abs().amax(dim=1, keepdim=True)
    near = [(quotient * (1.0 + off * 2.0 ** -24)).float().to(torch.float8_e4m3fn).double() for off in (-16.0, 16.0)]
    assert ((got == near[0]) | (got == near[1])).all()
    return (codes.cpu().double() * scales.cpu().double().t())[:, :dim]


def plain(config, w, tokens, stored):
    """``plain_llama.forward`` as bfloat16 mode has it, but for the inputs of the products whose matrices are in 8 bits: q|k|v's behind its norm
    from the unrounded rows; gate|up's and down's from unrounded rows where all three are in 8 bits, else from bfloat16 ones."""
    c, positions = pl.read_config(config), list(range(len(tokens)))
    has = lambda n: n in STORED[stored]
    inv = pl.rope_inv_freq(c["theta"], c["head_dim"])
    x, T = pl.embed(tokens, w["model.embed_tokens.weight"]), len(tokens)
    for layer in range(c["layers"]):
        pre = f"model.layers.{layer}."
        xn = pl.rmsnorm(x, w[pre + "input_layernorm.weight"], c["eps"])
        xn = normed_codes(x, w[pre + "input_layernorm.weight"], c["eps"]) if has("q_proj") else pl.round_bf16(xn)
        q, k, v = (pl.linear(xn, w[pre + f"self_attn.{n}_proj.weight"]).view(T, -1, c["head_dim"]) for n in "qkv")
        q, k, v = pl.round_bf16(pl.rope(q, positions, inv)), pl.round_bf16(pl.rope(k, positions, inv)), pl.round_bf16(v)
        a = pl.round_bf16(pl.attention(q, k, v, pl.round_bf16, None, 64)).reshape(T, -1)
        x = x + pl.linear(quantized_rows(a) if has("o_proj") else a, w[pre + "self_attn.o_proj.weight"])
        xn, through = pl.rmsnorm(x, w[pre + "post_attention_layernorm.weight"], c["eps"]), has("gate_proj") and has("down_proj")
        xn = xn if through else pl.round_bf16(xn)
        xn = quantized_rows(xn) if has("gate_proj") else xn
        h = pl.swiglu(pl.linear(xn, w[pre + "mlp.gate_proj.weight"]), pl.linear(xn, w[pre + "mlp.up_proj.weight"]))
        h = h if through else pl.round_bf16(h)
        x = x + pl.linear(quantized_rows(h) if has("down_proj") else h, w[pre + "mlp.down_proj.weight"])
    return pl.linear(pl.round_bf16(pl.rmsnorm(x, w["model.norm.weight"], c["eps"])),
                     w["model.embed_tokens.weight"] if c["tied"] else w["lm_head.weight"])


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("stored", STORED)
def test_some_matrices_in_8_bits_against_the_plain_decoder(gpu, tmp_path, stored, name):
    from bitwise_amd.model import Model, describe

    cfg, seed, sigma, page = tiny.CONFIGS[name]
    cfg = dict(cfg, num_hidden_layers=1)
    tensors = []
    for n, t in loader.random_tensors(describe(cfg), seed, sigma, torch.float32):
        if any(part in n for part in STORED[stored]):
            codes, scales = block_scaled.quantize(t)
            tensors += [(n, codes), (n + block_scaled.SCALE_SUFFIX, scales)]
        else:
            tensors.append((n, t.bfloat16()))
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    safetensors_io.write_file(tmp_path / "model.safetensors", tensors)
    model, w = Model.load(tmp_path, "bfloat16"), {n: t.double() for n, t in widened(tmp_path).items()}
    for rid, toks in requests_for(cfg["vocab_size"], 21, [90, 33]).items():
        # (a code that a last bit in front of it moves changes one element of a product's input by an eighth of itself at most)
        check_against_plain(model.logits(toks, block_size=page), plain(cfg, w, toks, stored).numpy(), "bfloat16", f"{name}, {stored} in 8 bits, {rid}",
                            max_tol=2.0 ** -3, median=True)
