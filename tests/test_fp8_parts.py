"""Which operators the parts call for matrices in 8 bits, with stand-ins for the kernels (no GPU needed)."""

from types import SimpleNamespace

import pytest
import torch

import fp8_stand_ins as stand_ins
from bitwise_amd.parts.mlp import SwiGLU
from bitwise_amd.runtime import Workspace
from bitwise_amd.weights import block_scaled
from bitwise_amd.weights.block_scaled import BlockScaled

ON_CPU = SimpleNamespace(bf16=True, device=torch.device("cpu"), act_dtype=torch.bfloat16)


def matrix(n, k, seed):
    return BlockScaled([block_scaled.quantize(torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) * 0.1)], k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("stored", [False, True])
def test_a_feed_forward_in_8_bits_takes_rows_that_are_normed_already(monkeypatch, stored, dtype):
    """As every block gives them whose norm is not the plain one in front of it."""
    calls = []
    stand_ins.put(calls, monkeypatch)
    part = SwiGLU({"width": 200, "inter": 130}, ON_CPU)
    tensors = {n: matrix(*s.shape, i) for i, (n, s) in enumerate(part.tensors().items())}
    part.bind(tensors)
    assert part.in_codes
    g = torch.Generator().manual_seed(9)
    h, residual = torch.randn(5, 200, generator=g).to(dtype), torch.randn(5, 200, generator=g)
    ctx = SimpleNamespace(ws=Workspace(ON_CPU.device, 5, 16), rows=4)
    before = residual.clone()
    (part.forward_out if stored else part.forward)(ctx, h, residual)
    assert calls == ["quantize_fp8", "gemm_fp8_swiglu", "gemm_fp8"]
    wide = [stand_ins.matrix_values(*tensors[n].parts[0]) for n in part.names]
    x = stand_ins.values(*stand_ins.quantized(h[:4]))[:, :200]
    gate, up = x @ wide[0].t(), x @ wide[1].t()
    act = stand_ins.values(*stand_ins.quantized((gate * torch.sigmoid(gate) * up).float()))[:, :130]
    want = act @ wide[2].t() + (0.0 if stored else before[:4].double())
    assert (residual[:4].double() - want).abs().max() <= 2.0 ** -23 * want.abs().max()           # (one rounding, and sums in another order)
    assert torch.equal(residual[4], before[4])
