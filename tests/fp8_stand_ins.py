"""The 8-bit operators on the CPU, in 64 bits between their roundings: stand-ins for the kernels where a test looks at which of them a part
calls, and with what."""

import torch

from bitwise_amd.csrc import ops


def quantized(x):
    """Codes [rows, whole blocks] and scales [blocks, rows] of 32-bit rows."""
    x = x.float()
    kp = ops.fp8_width(x.shape[1])
    b = torch.nn.functional.pad(x, (0, kp - x.shape[1])).view(x.shape[0], kp // 128, 128)
    most = b.abs().amax(dim=2).clamp_min(448.0 * 2.0 ** -126)
    return (448.0 * b.double() / most.double()[:, :, None]).float().view(x.shape[0], kp).to(ops.FP8), (most / 448.0).t().contiguous()


def values(codes, scales):
    return codes.double() * scales.double().t().repeat_interleave(128, 1)


def matrix_values(w, scales, halves=1):
    n, nb, k = w.shape[0] // halves, scales.shape[0] // halves, w.shape[1]
    return torch.cat([w[h * n:(h + 1) * n].double() * scales[h * nb:(h + 1) * nb].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
                      for h in range(halves)])


def put(on, monkeypatch):
    """The stand-ins in the place of ``ops``' functions; ``on`` gets their names as they are called."""
    def quantize_fp8(x, codes, scales, rows):
        on.append("quantize_fp8")
        c, s = quantized(x[:rows])
        codes[:rows], scales[:, :rows] = c, s

    def gemm_fp8(x, xs, w, ws, out, rows, residual=None):
        on.append("gemm_fp8")
        y = values(x[:rows], xs[:, :rows]) @ matrix_values(w, ws).t()
        out[:rows] = (y if residual is None else residual[:rows].double() + y).to(out.dtype)

    def gemm_fp8_swiglu(x, xs, w, ws, codes, scales, rows, sums=None):
        on.append("gemm_fp8_swiglu")
        g, u = (values(x[:rows], xs[:, :rows]) @ matrix_values(w, ws, 2).t()).chunk(2, dim=1)
        c, s = quantized((g * torch.sigmoid(g) * u).float())
        codes[:rows], scales[:, :rows] = c, s

    def norm_add_norm(x, y, weight, out, rows, eps, scales=None):
        on.append("norm_add_norm")
        h = x[:rows].double()
        c, s = quantized((h / (h.square().mean(1, keepdim=True) + eps).sqrt() * weight.double()).float())
        out[:rows], scales[:, :rows] = c, s

    for f in (quantize_fp8, gemm_fp8, gemm_fp8_swiglu, norm_add_norm):
        monkeypatch.setattr(ops, f.__name__, f)
