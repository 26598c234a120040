"""Strides and widths that pass 31 bits: refused, not cut."""

import pytest
import torch

from bitwise_amd.csrc import ops

pytestmark = pytest.mark.gpu
F8, FAR = torch.float8_e4m3fn, 2 ** 32 + 512          # (its low 32 bits are a stride that would do)


def test_strides_and_widths_past_31_bits_are_refused(gpu):
    room = torch.zeros(2 * FAR + 8192, dtype=torch.uint8, device=gpu)
    halves, bytes8 = room.view(torch.bfloat16), room.view(F8)
    far16, far8 = halves.as_strided((2, 256), (FAR, 1)), bytes8.as_strided((2, 256), (FAR, 1))
    x, w, out = torch.randn(2, 256, device=gpu), torch.ones(256, device=gpu), torch.empty(2, 256, device=gpu)
    codes, scales = torch.zeros(2, 256, dtype=torch.uint8, device=gpu).view(F8), torch.ones(2, 2, device=gpu)
    m, ms = torch.zeros(256, 256, dtype=torch.uint8, device=gpu).view(F8), torch.ones(2, 2, device=gpu)
    up, ups, sums = torch.zeros(512, 256, dtype=torch.uint8, device=gpu).view(F8), torch.ones(4, 2, device=gpu), torch.empty(2, 256, device=gpu)
    wide8, wide_scales = bytes8[:FAR].view(1, FAR), torch.ones(FAR // 128, 1, device=gpu)
    for call in (lambda: ops.quantize_fp8(far16, codes, scales, 2), lambda: ops.quantize_fp8(x, far8, scales, 2),
                 lambda: ops.quantize_fp8(halves[:FAR].view(1, FAR), wide8, wide_scales, 1),
                 lambda: ops.norm_add_norm(x, far16, w, out, 2, 1e-6), lambda: ops.norm_add_norm(x, x, w, far16, 2, 1e-6, stream=out),
                 lambda: ops.norm_add_norm(x, x, w, out, 2, 1e-6, gate=far16), lambda: ops.norm_add_norm(x, None, w, far8, 2, 1e-6, scales=scales),
                 lambda: ops.gemm_fp8(far8, scales, m, ms, out, 2), lambda: ops.gemm_fp8(codes, scales, m, ms, far16, 2),
                 lambda: ops.gemm_fp8(wide8, wide_scales, wide8, wide_scales.view(1, -1), out[:1, :1], 1),
                 lambda: ops.gemm_fp8_swiglu(codes, scales, up, ups, far8, scales.clone(), 2, sums=sums)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    assert not room[:8192].any() and not room[FAR:FAR + 8192].any()
