"""Parts whose matrices are in 8 bits, in arrangements that the Llama models do not have."""

import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import fp8_stand_ins as stand_ins
from bitwise_amd.csrc import ops
from bitwise_amd.parts.mlp import ClampedGLU, GeGLU, SwiGLU
from bitwise_amd.parts.norm import RMSNorm
from bitwise_amd.runtime import Runtime, Workspace
from bitwise_amd.weights import block_scaled
from bitwise_amd.weights.block_scaled import BlockScaled
from replay_util import MEDIAN_TOL, mixed_steps, portion_steps, requests_for, run_steps, tail_steps, whole_steps

pytestmark = pytest.mark.gpu


def bound(part, seed=0):
    tensors = {}
    for i, (n, s) in enumerate(part.tensors().items()):
        w = torch.randn(*s.shape, generator=torch.Generator().manual_seed(seed + i)) * 0.1
        tensors[n] = BlockScaled([block_scaled.quantize(w)], s.shape[1]) if s.block_scaled else 1.0 + w
    part.bind(tensors)
    return part


@pytest.mark.parametrize("rows", [1, 20, 64, 65, 200])
def test_a_feed_forward_of_normed_rows_is_the_one_behind_its_norm(gpu, rows):
    """The norm's 32-bit rows quantized are the codes that the norm leaves: the same bits from both ways into the feed-forward, added to the
    stream or stored."""
    rt = Runtime("bfloat16")
    part, norm = bound(SwiGLU({"width": 328, "inter": 200}, rt)), bound(RMSNorm({"width": 328, "eps": 1e-6}, rt), 5)
    x = torch.randn(rows + 1, 328, generator=torch.Generator().manual_seed(rows)).to(gpu)
    ctx = SimpleNamespace(ws=Workspace(gpu, rows + 1, 16), rows=rows)
    behind = x.clone()
    assert part.forward_with_norm(ctx, behind, norm, behind)
    h = torch.empty_like(x)
    ops.norm_add_norm(x, None, norm.weight, h, rows, norm.eps)
    normed = x.clone()
    part.forward(ctx, h, normed)
    assert torch.equal(normed, behind) and torch.equal(normed[rows], x[rows])
    out = torch.full_like(x, 9.0)
    part.forward_out(ctx, h, out)
    again = torch.zeros_like(x)
    part.forward(ctx, h, again)
    assert torch.equal(out[:rows], again[:rows]) and (out[rows] == 9.0).all() and out[:rows].any()


ACTS = {
    "swiglu": (SwiGLU, {}, lambda g, u: g * torch.sigmoid(g) * u),
    "geglu": (GeGLU, {}, lambda g, u: 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))) * u),
    "clamped_glu": (ClampedGLU, {"limit": 1.5, "alpha": 1.702},
                    lambda g, u: (c := g.clamp(max=1.5)) * torch.sigmoid(1.702 * c) * (u.clamp(-1.5, 1.5) + 1.0)),
}


@pytest.mark.parametrize("inter", [200, 256])
@pytest.mark.parametrize("rows", [20, 64, 65, 200])
@pytest.mark.parametrize("kind", ACTS)
def test_gated_feed_forwards_against_their_formulas(gpu, kind, rows, inter):
    """Every gated feed-forward with its three matrices in 8 bits: the products' inputs are quantized, SwiGLU's between them from the 32-bit
    values, the others' from the activation's bfloat16 ones.  A code on the border between two may fall the other way and changes one
    element of the down projection's input by an eighth of itself at most; most rows have none."""
    cls, params, act = ACTS[kind]
    part = bound(cls(dict(params, width=328, inter=inter, names=("gate", "up", "down")), Runtime("bfloat16")), seed=rows)
    wide = [stand_ins.matrix_values(*block_scaled.quantize(torch.randn(*s.shape, generator=torch.Generator().manual_seed(rows + i)) * 0.1))
            for i, s in enumerate(part.tensors().values())]
    g = torch.Generator().manual_seed(inter)
    h, x = torch.randn(rows + 1, 328, generator=g).bfloat16(), torch.randn(rows + 1, 328, generator=g)
    got = x.to(gpu)
    part.forward(SimpleNamespace(ws=Workspace(gpu, rows + 1, 16), rows=rows), h.to(gpu), got)
    assert torch.equal(got[rows].cpu(), x[rows])
    rows_in = lambda t: stand_ins.values(*stand_ins.quantized(t))[:, :t.shape[1]]
    xq = rows_in(h[:rows])
    a = act(xq @ wide[0].t(), xq @ wide[1].t()).float()
    want = x[:rows].double() + rows_in(a if kind == "swiglu" else a.bfloat16()) @ wide[2].t()
    worst = 2.0 ** -3 * (a.double().abs() @ wide[2].abs().t()) + 1e-5
    off = (got[:rows].cpu().double() - want).abs()
    assert (off <= worst).all()
    assert off.amax(dim=1).median() <= MEDIAN_TOL["bfloat16"] * want.abs().max()


@pytest.mark.parametrize("name", ["Kuponex", "Kikarax"])
def test_models_whose_feed_forwards_alone_are_in_8_bits(gpu, tmp_path, name):
    """Their dense gated feed-forwards take matrices in 8 bits: every cutting gives the same bits, and the logits are those of the same
    model with the widened matrices in 32 bits but for the rounding of the products' inputs."""
    from bitwise_amd.model import Model, write_random_model
    from bitwise_amd.registry import ARCHITECTURES
    from bitwise_amd.replay import Replayer

    cfg = dict(ARCHITECTURES[name].tiny_config)
    folder = write_random_model(tmp_path, cfg, 7, 0.15, "float8")
    model = Model.load(folder)
    assert any(getattr(getattr(l.feed_forward, "gate_up", None), "fp8", False) for l in model.assembled.layers if l.feed_forward is not None)
    reqs = requests_for(cfg["vocab"], 17, [70, 41, 20])

    def replayer(max_tokens, **kw):
        return Replayer("", "bfloat16", max_tokens, block_size=16, model=model, **kw)

    whole = {rid: run_steps(replayer(128), whole_steps(rid, toks))[rid] for rid, toks in reqs.items()}
    for rid, toks in reqs.items():
        for use_graphs in (True, False):
            assert np.array_equal(run_steps(replayer(128, use_graphs=use_graphs), tail_steps(rid, toks))[rid], whole[rid])
        assert np.array_equal(run_steps(replayer(128), portion_steps(rid, toks, seed=len(toks)))[rid], whole[rid])
    steps, most = mixed_steps(reqs, seed=5, page=16, max_live=2)
    got = run_steps(replayer(most, poison_freed_pages=True), steps)
    assert all(np.array_equal(got[rid], whole[rid]) for rid in reqs)
    wide = Model.load(folder, "float32")
    for rid, toks in reqs.items():
        want = wide.logits(toks)
        # (a code is off by 2^-4 of its value at most, their errors do not all point one way, and the stream carries most of a logit)
        assert np.linalg.norm(whole[rid] - want) <= 2.0 ** -3 * np.linalg.norm(want)


@pytest.mark.parametrize("name", ["LONG", "B"])
def test_an_engine_whose_captured_steps_hold_products_back(gpu, tmp_path, name):
    """8-bit operators among products that captured steps send as phases of a few launches (the head's, and the matrices that are not in 8
    bits): each comes behind what was held back, and the tokens and fingerprints are the ones of eager steps."""
    import json

    import bitwise_amd as bw
    import tiny
    from bitwise_amd.model import describe
    from bitwise_amd.weights import loader, safetensors_io

    cfg, seed, sigma, page = tiny.CONFIGS[name]
    for stored in (("proj",), ("down_proj",), ("q_proj", "k_proj", "v_proj"), ("gate_proj", "up_proj")):
        tensors = []
        for n, t in loader.random_tensors(describe(cfg), seed, sigma, torch.float32):
            tensors += list(loader.stored_as(n, describe(cfg)[n], t, block_scaled.DTYPE if any(s in n for s in stored) else torch.bfloat16))
        folder = tmp_path / stored[0]
        folder.mkdir()
        (folder / "config.json").write_text(json.dumps(cfg))
        safetensors_io.write_file(folder / "model.safetensors", tensors)
        model = bw.Model.load(folder)
        prompts = list(requests_for(cfg["vocab_size"], 9, [33, 8, 21, 5]).values())
        sp = bw.SamplingParams(max_new_tokens=10, ignore_eos=True)
        runs = [bw.generate(model, prompts, sp, bw.EngineConfig(num_blocks=64, block_size=page, max_batched_tokens=48, **kw))
                for kw in (dict(decode_phases=True), dict(decode_phases=False), dict(use_graphs=False))]
        for other in runs[1:]:
            assert [r.tokens for r in runs[0]] == [r.tokens for r in other]
            assert [r.logits_fingerprint for r in runs[0]] == [r.logits_fingerprint for r in other]
