"""Gates over the whole range of their numbers, infinities among them: the norm's sigmoid, and silu behind a gated product, against their
definitions in 64 bits."""

import pytest
import torch

from bitwise_amd.csrc import ops

pytestmark = pytest.mark.gpu
F8, U, LEAST = torch.float8_e4m3fn, 2.0 ** -24, 2.0 ** -149       # U: half a step of a 32-bit number, relative; LEAST: the least of them
INF, NAN = float("inf"), float("nan")

GATES = [0.0, -0.0, 1e-30, -1e-30, 1.0, -1.0, 16.0, -16.0, 63.5, -63.5, 64.0, -64.0, 64.5, -64.5, 80.0, -80.0, 86.5, -86.5, 87.0, -87.0, 87.5, -87.5,
         88.0, -88.0, 88.5, -88.5, 89.0, -89.0, 95.0, -95.0, 100.0, -100.0, 103.0, -103.0, 104.0, -104.0, 112.0, -112.0, 120.0, -120.0, 1e3, -1e3, 1e20, -1e20,
         2.2e38, -2.2e38, 2.4e38, -2.4e38, 3.3e38, -3.3e38, INF, -INF]


@pytest.mark.parametrize("size", [1.0, 1e30])
@pytest.mark.parametrize("vector", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_sigmoid_gate_of_any_number(gpu, dtype, vector, size):
    """The sigmoid is within four half steps, or, under the normal numbers, within the least number and half of it (two roundings there); the
    product with y and the addition to zero round once each."""
    gate = torch.tensor(GATES).to(dtype)
    dim, g = gate.numel(), torch.Generator().manual_seed(3)
    y = torch.randn(3, dim, generator=g).clamp_min(0.1) * size
    x, w = torch.zeros(3, dim, device=gpu), torch.ones(dim, device=gpu)
    stream, out = torch.full((3, dim), 9.0, device=gpu), torch.empty(3, dim, device=gpu)
    ops.norm_add_norm(x, y.to(gpu), w, out, 3, 1e-6, gate=(gate if vector else gate.expand(3, dim).contiguous()).to(gpu), gate_sigmoid=True, stream=stream)
    want = y.double() * torch.sigmoid(gate.double())
    allowed = 5 * U * want.abs() + 1.5 * LEAST * y.double() + LEAST
    off = (stream.cpu().double() - want).abs()
    assert (off <= allowed).all(), (gate[(~(off <= allowed)).any(0)], stream.cpu()[:, (~(off <= allowed)).any(0)])


def test_a_gate_that_is_no_number_stays_in_its_row(gpu):
    gate = torch.randn(4, 256, generator=torch.Generator().manual_seed(4))
    gate[2, 17] = NAN
    gate[3, :2] = torch.tensor([INF, -INF])
    x, y, w = torch.zeros(4, 256, device=gpu), torch.ones(4, 256, device=gpu), torch.ones(256, device=gpu)
    stream, out = torch.empty_like(x), torch.empty_like(x)
    ops.norm_add_norm(x, y, w, out, 4, 1e-6, gate=gate.to(gpu), gate_sigmoid=True, stream=stream)
    assert stream[2].isnan().sum() == 1 and out[2].isnan().all()
    assert stream[[0, 1, 3]].isfinite().all() and out[[0, 1, 3]].isfinite().all()
    assert stream[3, 0] == 1.0 and stream[3, 1] == 0.0


# (size of g, size of u, rows): a row's gate comes from its first block of K, its up value from the second, each with a scale of its own
SPANS = [(1.0, 1.0), (0.25, 1e30), (2.0 ** 119, 0.01), (2.0 ** 119, 2.0 ** -119), (2.0 ** 119, 1e-30), (2.0 ** 60, 2.0 ** 50)]


@pytest.mark.parametrize("rows", [3, 40, 70])
@pytest.mark.parametrize("span", SPANS, ids=lambda s: f"{s[0]:.0e},{s[1]:.0e}")
def test_silu_of_any_number(gpu, rows, span):
    """g is one product of a code and its scales, u another: both are exact in 32 bits.  Behind them: the sigmoid (four half steps, or the least
    number and half of it under the normal ones), two products, then the definition of the codes."""
    inter = 256
    codes = torch.arange(256, dtype=torch.uint8)
    codes = torch.where((codes & 0x7f) == 0x7f, torch.zeros_like(codes), codes)                       # (no NaN)
    w = torch.zeros(2 * inter, 256, dtype=torch.uint8)
    w[:inter, 0] = codes
    w[inter:, 128] = codes.roll(77)
    ws = torch.ones(2 * inter // 128, 2)
    x = torch.zeros(rows, 256, dtype=torch.uint8)
    x[:, 0] = x[:, 128] = 0x38                                                                        # 1.0
    xs = torch.tensor(span).view(2, 1).expand(2, rows).contiguous()
    out, scales = torch.zeros(rows, inter, dtype=torch.uint8, device=gpu).view(F8), torch.zeros(inter // 128, rows, device=gpu)
    ops.gemm_fp8_swiglu(x.to(gpu).view(F8), xs.to(gpu), w.to(gpu).view(F8), ws.to(gpu), out, scales, rows, sums=torch.empty(64, inter, device=gpu))
    value = codes.view(F8).double()
    g, u = (value * xs[0, 0].double()).float().double(), (value.roll(77) * xs[1, 0].double()).float().double()
    s = g * torch.sigmoid(g)
    want = s * u
    assert want.abs().max() < 3e38 and g.abs().max() < 3.4e38
    near = 7 * U * want.abs() + 1.5 * LEAST * (g * u).abs() + LEAST * (u.abs() + 1.0)                 # (g's product with the sigmoid can lie under the normal ones too)
    scale = scales.cpu().double()
    got = out.cpu().double() * scale.t().repeat_interleave(128, 1)
    spread = scale.t().repeat_interleave(128, 1)
    allowed = near * (1 + 2.0 ** -4) + torch.maximum(want.abs() * 2.0 ** -4, spread * 2.0 ** -10) + 4 * U * want.abs()
    off = (got - want).abs()
    assert (off <= allowed).all(), (g[(~(off <= allowed)).any(0)], u[(~(off <= allowed)).any(0)], got[0][(~(off <= allowed)).any(0)])
    most, slack = want.abs().view(2, 128).amax(1), near.view(2, 128).amax(1)
    assert ((scale - (most / 448.0).clamp_min(2.0 ** -126)[:, None]).abs() <= ((slack + 2 * U * most) / 448.0)[:, None]).all()
