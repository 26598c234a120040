"""Models whose attention and feed-forward matrices are stored in 8 bits (e4m3 codes, a scale for each block of 128 x 128).

bfloat16 mode runs them in 8 bits, against the float64 decoder with the same roundings, and the cuttings give the same bits;
the 32-bit mode widens them, to the bits of a checkpoint that stores the widened values."""

import json

import numpy as np
import pytest
import torch

import plain_llama as pl
import tiny
from bitwise_amd.weights import block_scaled, loader, safetensors_io
from replay_util import check_against_plain, mixed_steps, portion_steps, requests_for, run_steps, tail_steps, whole_steps

pytestmark = pytest.mark.gpu


def quantized_rows(x):
    """What a product's input stands for: scales and quotients 32-bit, codes rounded to nearest even."""
    x32 = x.to(torch.float32)
    kb = -(-x32.shape[1] // 128)
    b = torch.nn.functional.pad(x32, (0, kb * 128 - x32.shape[1])).view(x32.shape[0], kb, 128)
    most = b.abs().amax(2, keepdim=True).clamp_min(448.0 * 2.0 ** -126)
    return ((448.0 * b.double() / most.double()).float().to(torch.float8_e4m3fn).double() * (most / 448.0).double()).view(x32.shape[0], -1)[:, :x32.shape[1]]


def plain_8bit(config, w, tokens):
    """``plain_llama.forward`` with the inputs of the layers' products in 8 bits: the normed rows and SwiGLU's from their unrounded
    values, the attention's output from its bfloat16 ones; everything else as bfloat16 mode has it."""
    c, positions = pl.read_config(config), list(range(len(tokens)))
    inv = pl.rope_inv_freq(c["theta"], c["head_dim"])
    x, T = pl.embed(tokens, w["model.embed_tokens.weight"]), len(tokens)
    for layer in range(c["layers"]):
        pre = f"model.layers.{layer}."
        xn = quantized_rows(pl.rmsnorm(x, w[pre + "input_layernorm.weight"], c["eps"]))
        q, k, v = (pl.linear(xn, w[pre + f"self_attn.{n}_proj.weight"]).view(T, -1, c["head_dim"]) for n in "qkv")
        q, k, v = pl.round_bf16(pl.rope(q, positions, inv)), pl.round_bf16(pl.rope(k, positions, inv)), pl.round_bf16(v)
        a = pl.round_bf16(pl.attention(q, k, v, pl.round_bf16, None, 64)).reshape(T, -1)
        x = x + pl.linear(quantized_rows(a), w[pre + "self_attn.o_proj.weight"])
        xn = quantized_rows(pl.rmsnorm(x, w[pre + "post_attention_layernorm.weight"], c["eps"]))
        h = pl.swiglu(pl.linear(xn, w[pre + "mlp.gate_proj.weight"]), pl.linear(xn, w[pre + "mlp.up_proj.weight"]))
        x = x + pl.linear(quantized_rows(h), w[pre + "mlp.down_proj.weight"])
    return pl.linear(pl.round_bf16(pl.rmsnorm(x, w["model.norm.weight"], c["eps"])),
                     w["model.embed_tokens.weight"] if c["tied"] else w["lm_head.weight"])


def widened(folder):
    """The folder's tensors, matrices in 8 bits as 32-bit ones."""
    found = safetensors_io.read_folder(folder)
    out = {}
    for n, t in found.items():
        if t.dtype == block_scaled.DTYPE:
            out[n] = block_scaled.BlockScaled([(t, found[n + block_scaled.SCALE_SUFFIX])], t.shape[1]).widened()
        elif not n.endswith(block_scaled.SCALE_SUFFIX):
            out[n] = t
    return out


def make(tmp, name, layers=0):
    from bitwise_amd.model import write_random_model

    cfg, seed, sigma, _ = tiny.CONFIGS[name]
    folder = tmp / f"{name}_{layers}"
    return write_random_model(folder, dict(cfg, num_hidden_layers=layers) if layers else cfg, seed, sigma, "float8")


@pytest.mark.parametrize("name", ["A", "B", "LONG"])
def test_a_model_in_8_bits(gpu, tmp_path, name):
    from bitwise_amd.model import Model
    from bitwise_amd.replay import Replayer

    cfg, page = tiny.CONFIGS[name][0], tiny.CONFIGS[name][3]
    folder = make(tmp_path, name)
    model = Model.load(folder, "bfloat16")
    block = model.assembled.layers[0]
    assert block.mixer.qkv.fp8 and block.mixer.o.fp8 and block.feed_forward.in_codes
    assert model.weight_bytes < Model.load(tiny.make_folder(tmp_path, name), "bfloat16").weight_bytes
    reqs = requests_for(cfg["vocab_size"], 17, [70, 41, 20])
    one = make(tmp_path, name, 1)
    model1, w1 = Model.load(one, "bfloat16"), {n: t.double() for n, t in widened(one).items()}
    for rid, toks in reqs.items():
        # (a code that a last bit in front of it moves changes one element of a product's input by an eighth of itself at most)
        check_against_plain(model1.logits(toks, block_size=page), plain_8bit(tiny.read_config(one), w1, toks).numpy(), "bfloat16",
                            f"{name} in 8 bits {rid}, one layer", max_tol=2.0 ** -3, median=True)

    def replayer(max_tokens, **kw):
        return Replayer("", "bfloat16", max_tokens, block_size=page, model=model, **kw)

    whole = {rid: run_steps(replayer(128), whole_steps(rid, toks))[rid] for rid, toks in reqs.items()}
    for rid, toks in reqs.items():
        for use_graphs in (True, False):
            got = run_steps(replayer(128, use_graphs=use_graphs), tail_steps(rid, toks))
            assert np.array_equal(got[rid], whole[rid]), f"{rid}: decoding differs from the whole prompt (graphs={use_graphs})"
        got = run_steps(replayer(128), portion_steps(rid, toks, seed=len(toks)))
        assert np.array_equal(got[rid], whole[rid]), f"{rid}: portions differ from the whole prompt"
    steps, most = mixed_steps(reqs, seed=5, page=page, max_live=2)
    rp = replayer(most, poison_freed_pages=True)
    got = run_steps(rp, steps)
    for rid in reqs:
        assert np.array_equal(got[rid], whole[rid]), f"{rid}: the mixed trace differs from the whole prompt"


@pytest.mark.parametrize("name", ["A", "B"])
def test_the_32_bit_mode_widens(gpu, tmp_path, name):
    from bitwise_amd.model import Model

    folder = make(tmp_path, name)
    wide = tmp_path / "wide"
    wide.mkdir()
    (wide / "config.json").write_text((folder / "config.json").read_text())
    safetensors_io.write_file(wide / "model.safetensors", widened(folder).items())
    toks = requests_for(tiny.CONFIGS[name][0]["vocab_size"], 3, [33])
    (toks,) = toks.values()
    assert np.array_equal(Model.load(folder, "float32").logits(toks), Model.load(wide, "float32").logits(toks))


def test_an_engine_serves_a_model_in_8_bits(gpu, tmp_path):
    """Crowded or alone, through captured steps and launched ahead: the same tokens and fingerprints."""
    import bitwise_amd as bw

    folder = make(tmp_path, "LONG")
    model = bw.Model.load(folder)
    prompts = list(requests_for(320, 9, [65, 8, 33, 120, 17]).values())
    sp = bw.SamplingParams(max_new_tokens=12, ignore_eos=True)
    cfg = lambda **kw: bw.EngineConfig(num_blocks=64, max_batched_tokens=48, **kw)
    together = bw.generate(model, prompts, sp, cfg())
    for prompt, got in zip(prompts, together):
        (alone,) = bw.generate(model, [prompt], sp, cfg(use_graphs=False))
        assert alone.tokens == got.tokens and alone.logits_fingerprint == got.logits_fingerprint


@pytest.mark.parametrize("stored", ["gate_up", "down", "qkv"])
def test_matrices_in_8_bits_beside_others(gpu, tmp_path, stored):
    """Only some of a layer's matrices are in 8 bits: the others run as they would, and every cutting gives the same bits."""
    from bitwise_amd.model import Model, describe

    cfg, seed, sigma, page = tiny.CONFIGS["B"]
    names = {"gate_up": ("gate_proj", "up_proj"), "down": ("down_proj",), "qkv": ("q_proj", "k_proj", "v_proj")}[stored]
    tensors = []
    for n, t in loader.random_tensors(describe(cfg), seed, sigma, torch.float32):
        if any(part in n for part in names):
            codes, scales = block_scaled.quantize(t)
            tensors += [(n, codes), (n + block_scaled.SCALE_SUFFIX, scales)]
        else:
            tensors.append((n, t.bfloat16()))
    folder = tmp_path / stored
    folder.mkdir()
    (folder / "config.json").write_text(json.dumps(cfg))
    safetensors_io.write_file(folder / "model.safetensors", tensors)
    model = Model.load(folder, "bfloat16")
    (toks,) = requests_for(cfg["vocab_size"], 21, [90]).values()
    whole = model.logits(toks, block_size=page)
    assert np.isfinite(whole).all()
    for chunk in (1, 17, 64):
        assert np.array_equal(model.logits(toks, chunk=chunk, block_size=page), whole), chunk
