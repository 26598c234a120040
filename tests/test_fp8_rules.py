"""What the 8-bit entry points refuse, before anything is launched: no GPU is needed."""

import pytest
import torch

from bitwise_amd.csrc import build, ops

if build._find_current() is None and build._hipcc() is None:
    pytest.skip("the kernel library is neither built nor buildable", allow_module_level=True)

P = 1 << 20          # a pointer that a refused call never follows


def quantize(x=P, ldx=256, codes=2 * P, ldq=256, scales=P, lds=4, rows=4, width=256):
    return ops._fn("bw_quantize_fp8")(x, 0, ldx, codes, ldq, scales, lds, rows, width, None)


def test_quantization_refuses():
    assert quantize(rows=0) == 0
    assert quantize(width=0) == -2 and quantize(ldx=255) == -2 and quantize(ldq=128) == -2 and quantize(lds=3) == -2
    assert quantize(codes=P + 8) == -3 and quantize(ldq=264) == -3
    assert quantize(rows=2 ** 21, lds=2 ** 21) == -2
    assert quantize(x=P, codes=P) == -2                                               # rows written over while they are read


def norm(x=P, y=P, post=None, gate=None, ldg=0, vec=None, stream=P, out=2 * P, kind=0, ldo=256, scales=None, lds=0, rows=4, dim=256, ldx=256, ldy=256, ldst=256):
    return ops._fn("bw_norm_add_norm")(x, ldx, y, 0, ldy, post, 0, 1e-6, gate, 0, ldg, 0, vec, 0, 1.0, stream, ldst, P, 0, 1e-6, out, kind, ldo, scales, lds,
                                       rows, dim, None)


def test_norm_refuses():
    assert norm(rows=0) == 0
    assert norm(dim=0) == -2 and norm(kind=3) == -2 and norm(stream=None) == -2
    assert norm(out=P) == -2                                                          # both results in one place
    assert norm(kind=2) == -2 and norm(kind=2, scales=P, lds=3) == -2                 # codes without scales, or with too few
    assert norm(kind=2, scales=P, lds=4, out=2 * P + 4) == -3 and norm(kind=2, scales=P, lds=4, ldo=260) == -3
    assert norm(ldx=255) == -2 and norm(ldy=255) == -2 and norm(ldst=255) == -2 and norm(ldo=255) == -2 and norm(gate=P, ldg=255) == -2
    assert norm(dim=(1 << 30) + 1) == -2                                              # (an index of eights would pass 32 bits)
    for given in ("post", "gate", "vec"):
        assert norm(y=None, **{given: P}) == -2                                       # nothing to norm, gate or scale


def product(x=P, ldx=256, ldxs=4, w=P, residual=None, ldr=64, ldo=64, bf16=0, rows=4, n=64, k=256, out=2 * P):
    return ops._fn("bw_gemm_fp8")(x, ldx, P, ldxs, w, P, residual, ldr, out, ldo, bf16, rows, n, k, None)


def test_products_refuse():
    assert product(rows=0) == 0
    assert product(k=200) == -2 and product(k=0) == -2 and product(n=0) == -2 and product(ldx=128) == -2 and product(ldxs=3) == -2
    assert product(ldo=63) == -2 and product(residual=P, ldr=63) == -2 and product(residual=P, bf16=1) == -2
    assert product(x=P + 1) == -3 and product(w=P + 4) == -3 and product(ldx=264) == -3
    assert product(ldx=1 << 24) == -2
    assert product(out=P) == -2                                                       # (x itself)


def gated(x=P, ldx=256, ldxs=4, sums=P, ldsums=64, codes=2 * P, ldq=128, lds=4, rows=4, n=64, k=256, scales=3 * P):
    return ops._fn("bw_gemm_fp8_swiglu")(x, ldx, P, ldxs, P, P, sums, ldsums, codes, ldq, scales, lds, rows, n, k, None)


def test_gated_products_refuse():
    assert gated(rows=0) == 0
    assert gated(sums=None) == -2 and gated(ldsums=63) == -2 and gated(ldq=112) == -2 and gated(lds=3) == -2 and gated(k=100) == -2
    assert gated(codes=P + 8) == -3 and gated(ldq=136) == -3
    assert gated(codes=P) == -2 and gated(scales=P) == -2                             # (x itself, its scales)


def test_wrappers_refuse_tensors_off_the_gpu():
    x, c, s = torch.zeros(2, 256), torch.zeros(2, 256).to(torch.float8_e4m3fn), torch.zeros(2, 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.quantize_fp8(x, c, s, 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.norm_add_norm(x, None, torch.ones(256), x, 2, 1e-6)
    with pytest.raises(ValueError, match="GPU"):
        ops.gemm_fp8(c, s, c, s, x, 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.gemm_fp8_swiglu(c, s, c, s, c, s, 2)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        ops.quantize_fp8(x.half(), c, s, 2)


def test_width_of_rows_of_codes():
    assert [ops.fp8_width(n) for n in (1, 127, 128, 129, 2000)] == [128, 128, 128, 256, 2048]


def test_the_gpu_tests_sizes_reach_every_kernel():
    import test_fp8_gpu as sizes

    stored = [ops.gemm_fp8_choice(rows, n, ops.fp8_width(k)) for rows, n, k in sizes.STORED]
    assert {c[0] for c in stored} - {-1} == {*range(4), 100} and {c[1] for c in stored if c[0] < 0 and not c[2]} == set(range(4))
    assert len({c[1] for c in stored if c[2]}) >= 3
    long = [ops.gemm_fp8_choice(rows, n, ops.fp8_width(k)) for rows, n, k in sizes.STORED if k > 512]
    assert {c[1] for c in long if c[0] < 0} == set(range(4))
    gated = [ops.gemm_fp8_choice(rows, n, ops.fp8_width(k), gated=True) for rows, n, k in sizes.GATED]
    assert {c[0] for c in gated} - {-1} == {*range(4), 100} and {c[1] for c in gated if c[0] < 0} == set(range(4))
    long = [ops.gemm_fp8_choice(rows, n, ops.fp8_width(k), gated=True) for rows, n, k in sizes.GATED if k > 512]
    assert {c[1] for c in long if c[0] < 0} == set(range(4))
    for n, k in ((2048, 2048), (2048, 8192), (4096, 4096), (6144, 4096)):
        assert ops.gemm_fp8_choice(16, n, k)[0] == 100 and ops.gemm_fp8_choice(17, n, k)[0] != 100
    with pytest.raises(RuntimeError):
        ops.gemm_fp8_choice(0, 64, 128)
