"""Parts whose matrices are in 8 bits, in arrangements that the Llama models do not have."""

from types import SimpleNamespace

import pytest
import torch

from bitwise_amd.csrc import ops
from bitwise_amd.parts.mlp import SwiGLU
from bitwise_amd.parts.norm import RMSNorm
from bitwise_amd.runtime import Runtime, Workspace
from bitwise_amd.weights import block_scaled
from bitwise_amd.weights.block_scaled import BlockScaled

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
