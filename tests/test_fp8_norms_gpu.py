"""The norm in front of a product in 8 bits, without a sublayer's output: the form that models run, at the widths, strides and alignments
where it takes another way, against its definition in 64 bits."""

import pytest
import torch

from bitwise_amd.csrc import ops

pytestmark = pytest.mark.gpu
F8, U = torch.float8_e4m3fn, 2.0 ** -24                # U: half a step of a 32-bit number, relative


def norm_bound(dim):
    """Relative error of v / sqrt(mean(v^2) + eps) * weight: a thread's chain of eight squares (rows over 8,192: for each pass of 1,024 threads),
    six joins of a wave's lanes, one for each further wave of up to 16; half of that behind the root, then mean, eps, root, reciprocal and
    the two products."""
    waves = min(16, -(-dim // 512))
    return ((8 * -(-dim // 8192) + 6 + waves - 1) / 2 + 6) * U


def wide_rows(rows, dim, offset, gpu, seed):
    """Rows of ``dim`` columns that start ``offset`` elements into rows of a wider matrix (offset 0: of a matrix of their own)."""
    x = torch.randn(rows + 1, dim, generator=torch.Generator().manual_seed(seed)) * 3
    wide = torch.full((rows + 1, dim + 2 * offset), 7.0)
    wide[:, offset:offset + dim] = x
    return x, wide.to(gpu)[:, offset:offset + dim]


@pytest.mark.parametrize("weight_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (2, 129), (17, 576), (5, 2049), (4, 4096), (3, 8191), (2, 8192), (2, 8193), (3, 9000), (2, 16392), (1, 28672)])
def test_a_norm_without_a_sublayer(gpu, rows, dim, offset, weight_dtype):
    x, on_gpu = wide_rows(rows, dim, offset, gpu, dim)
    weight = (1.0 + 0.1 * torch.randn(dim + 1, generator=torch.Generator().manual_seed(1))).to(weight_dtype)
    w = weight.to(gpu)[offset % 2:][:dim]                                                  # (odd offsets: a weight that starts anywhere)
    eps, x64 = 1e-5, x[:rows].double()
    want = x64 / (x64.square().mean(1, keepdim=True) + eps).sqrt() * weight[offset % 2:][:dim].double()
    plain = torch.full((rows + 1, dim), 9.0, device=gpu)
    ops.norm_add_norm(on_gpu, None, w, plain, rows, eps)
    assert ((plain[:rows].cpu().double() - want).abs() <= norm_bound(dim) * want.abs()).all() and (plain[rows] == 9.0).all()
    rounded = torch.full((rows + 1, dim), 9.0, device=gpu, dtype=torch.bfloat16)
    ops.norm_add_norm(on_gpu, None, w, rounded, rows, eps)
    assert torch.equal(rounded[:rows], plain[:rows].bfloat16()) and (rounded[rows] == 9.0).all()
    kp = ops.fp8_width(dim)
    codes, scales = torch.full((rows + 1, kp), 0x2a, dtype=torch.uint8, device=gpu).view(F8), torch.full((kp // 128, rows + 1), 7.0, device=gpu)
    ops.norm_add_norm(on_gpu, None, w, codes, rows, eps, scales=scales)
    assert (codes[rows].view(torch.uint8) == 0x2a).all() and (scales[:, rows] == 7.0).all()
    assert not codes[:rows, dim:].view(torch.uint8).any()
    # against the definition: the scale is the largest magnitude's, a code off by half a step of a normal number or of the least one
    full = torch.nn.functional.pad(want, (0, kp - dim)).view(rows, -1, 128)
    most, scale = full.abs().amax(dim=2), scales[:, :rows].cpu().double().t()
    assert ((scale - (most / 448.0).clamp_min(2.0 ** -126)).abs() <= (norm_bound(dim) + 2 * U) * scale).all()
    got = codes[:rows].cpu().double() * scale.repeat_interleave(128, 1)
    spread = scale.repeat_interleave(128, 1)[:, :dim]
    off = norm_bound(dim) + 4 * U
    assert ((got[:, :dim] - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, spread * 2.0 ** -10) * (1 + off) + off * want.abs()).all()
    # and the bits of the 32-bit rows quantized
    again, again_s = torch.zeros_like(codes), torch.zeros_like(scales)
    ops.quantize_fp8(plain, again, again_s, rows)
    assert torch.equal(again[:rows].view(torch.uint8), codes[:rows].view(torch.uint8)) and torch.equal(again_s[:, :rows], scales[:, :rows])
    assert torch.equal(on_gpu.cpu(), x)


def test_codes_that_start_between_16_bytes_are_refused(gpu):
    """Views of whole blocks whose rows start elsewhere, or lie an odd number of bytes apart."""
    x = torch.randn(4, 256, device=gpu)
    wide, s = torch.zeros(4, 528, dtype=torch.uint8, device=gpu).view(F8), torch.ones(2, 4, device=gpu)
    odd = torch.zeros(4 * 264, dtype=torch.uint8, device=gpu).view(F8).as_strided((4, 256), (264, 1))
    w, ws, out = torch.zeros(8, 256, dtype=torch.uint8, device=gpu).view(F8), torch.ones(1, 2, device=gpu), torch.full((4, 8), 9.0, device=gpu)
    good, s2, sums = wide[:, 16:272], torch.ones(2, 4, device=gpu), torch.empty(4, 256, device=gpu)
    up, ups = torch.zeros(512, 256, dtype=torch.uint8, device=gpu).view(F8), torch.ones(4, 2, device=gpu)
    for bad in (wide[:, 8:264], wide[:, 1:257], odd):
        for call in (lambda: ops.quantize_fp8(x, bad, s, 4), lambda: ops.norm_add_norm(x, None, x[0].clone(), bad, 4, 1e-6, scales=s),
                     lambda: ops.gemm_fp8(bad, s, w, ws, out, 4), lambda: ops.gemm_fp8_swiglu(good, s, up, ups, bad, s2, 4, sums=sums)):
            with pytest.raises(ValueError, match="multiples of 16 bytes"):
                call()
    ops.gemm_fp8(good, s, w, ws, out, 4)
    assert not out.any() and not wide.view(torch.uint8).any()


def test_results_in_the_place_of_what_is_read(gpu):
    """Element for element they may lie there, and beside it as columns of one matrix; the bits are those of memory of its own."""
    for dim in (256, 9000):
        g = torch.Generator().manual_seed(dim)
        x, y, gate = (torch.randn(5, dim, generator=g).to(gpu) for _ in range(3))
        w = torch.ones(dim, device=gpu)
        stream, out = torch.empty_like(x), torch.empty_like(x)
        ops.norm_add_norm(x, y, w, out, 5, 1e-6, post_weight=w, gate=gate, scale=0.5, stream=stream)
        for where_s, where_o in (("x", None), ("y", None), ("gate", None), (None, "x"), (None, "y"), (None, "gate"), ("y", "x"), ("x", "gate")):
            t = {"x": x.clone(), "y": y.clone(), "gate": gate.clone(), None: torch.empty_like(x)}
            s, o = t[where_s], t[where_o] if where_o else torch.empty_like(x)
            ops.norm_add_norm(t["x"], t["y"], w, o, 5, 1e-6, post_weight=w, gate=t["gate"], scale=0.5, stream=s)
            assert torch.equal(s, stream) and torch.equal(o, out), (where_s, where_o)
        half = y.bfloat16()
        rounded = torch.empty_like(half)
        ops.norm_add_norm(x, half, w, rounded, 5, 1e-6, stream=stream)
        ops.norm_add_norm(x, half, w, half, 5, 1e-6, stream=stream)
        assert torch.equal(half, rounded)
        wide = torch.cat([x, y, gate, x], dim=1)
        part = [wide[:, i * dim:(i + 1) * dim] for i in range(4)]
        ops.norm_add_norm(x, y, w, out, 5, 1e-6, gate=gate, stream=stream)
        ops.norm_add_norm(part[0], part[1], w, part[3], 5, 1e-6, gate=part[2], stream=part[0])
        assert torch.equal(part[0], stream) and torch.equal(part[3], out) and torch.equal(part[1], y) and torch.equal(part[2], gate)
        alone, again = x.clone(), torch.empty_like(x)
        ops.norm_add_norm(x, None, w, again, 5, 1e-6)
        ops.norm_add_norm(alone, None, w, alone, 5, 1e-6)
        assert torch.equal(alone, again)
        with pytest.raises(RuntimeError, match="norm_add_norm"):
            ops.norm_add_norm(x, None, w, x.view(torch.bfloat16)[:, :dim], 5, 1e-6)
        assert torch.equal(part[1], y)
