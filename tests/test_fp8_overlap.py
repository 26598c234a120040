"""Results in memory that a call still reads are refused before anything is launched: no GPU is needed."""

import pytest

from bitwise_amd.csrc import build, ops

if build._find_current() is None and build._hipcc() is None:
    pytest.skip("the kernel library is neither built nor buildable", allow_module_level=True)

M = 1 << 20          # pointers a megabyte apart, that a refused call never follows


def at(n, offset=0):
    return (n + 1) * M + offset


def quantize(x=at(0), codes=at(1), scales=at(2), bf16=0, ldx=256, ldq=256, rows=4, width=256, lds=4):
    return ops._fn("bw_quantize_fp8")(x, bf16, ldx, codes, ldq, scales, lds, rows, width, None)


@pytest.mark.parametrize("call", [
    dict(codes=at(0)), dict(codes=at(0, 1024)), dict(codes=at(0, 4 * 1024 - 16)), dict(codes=at(0, -4 * 256 + 16)),
    dict(scales=at(0, 64)), dict(scales=at(1, 1020)), dict(scales=at(1, -28)),
    dict(x=at(0), codes=at(0, 256), ldx=512, ldq=1024),                                   # the same rows' columns, but where they end
    dict(codes=at(0, 16), bf16=1, rows=1),
], ids=str)
def test_quantization(call):
    assert quantize(**call) == -2


def norm(x=at(0), ldx=256, y=at(1), y_bf16=0, ldy=256, post=0, gate=0, gate_bf16=0, ldg=0, vec=0, stream=at(2), ldst=256, weight=at(3), out=at(4),
         kind=0, ldo=256, scales=0, lds=4, rows=4, dim=256):
    return ops._fn("bw_norm_add_norm")(x, ldx, y, y_bf16, ldy, post, 0, 1e-6, gate, gate_bf16, ldg, 0, vec, 0, 1.0, stream, ldst, weight, 0, 1e-6, out, kind,
                                       ldo, scales, lds, rows, dim, None)


ALONE = dict(y=0, stream=0)


@pytest.mark.parametrize("call", [
    dict(ALONE, out=at(0), kind=1), dict(ALONE, out=at(0), kind=2, scales=at(5)),         # narrower rows in x's place: others' rows lie there
    dict(ALONE, out=at(0), ldx=512), dict(ALONE, out=at(0, 1024)), dict(ALONE, out=at(0, 16)), dict(ALONE, out=at(0, -4096 + 16)),
    dict(ALONE, out=at(0), kind=1, ldo=512, ldx=512), dict(ALONE, out=at(3, 512)), dict(ALONE, out=at(4), kind=2, scales=at(0, 8)),
    dict(ALONE, out=at(4), kind=2, scales=at(4, 16)), dict(ALONE, out=at(4), kind=2, scales=at(3)),
    dict(out=at(1), kind=1), dict(out=at(1), y_bf16=1), dict(out=at(1), ldy=512), dict(stream=at(1), y_bf16=1), dict(stream=at(0), ldst=512),
    dict(stream=at(1, 1024)), dict(stream=at(3)), dict(stream=at(2), out=at(2, 2048)), dict(out=at(2)), dict(out=at(2), kind=1),
    dict(gate=at(5), ldg=256, out=at(5), gate_bf16=1), dict(gate=at(5), ldg=256, stream=at(5, 4)), dict(gate=at(5), stream=at(5)), dict(gate=at(5), out=at(5, 1020)),
    dict(vec=at(5), out=at(5)), dict(post=at(5), stream=at(5)),
], ids=str)
def test_norms(call):
    assert norm(**call) == -2



@pytest.mark.parametrize("rows", [1, 4, 100])
@pytest.mark.parametrize("call", [
    dict(out=at(0)), dict(out=at(0, 128)), dict(out=at(1)), dict(out=at(2)), dict(out=at(2, 64 * 256 - 4)), dict(out=at(3, 4)),
    dict(out=at(4), residual=at(4, 4)), dict(out=at(4), residual=at(4), ldr=128, rows=4), dict(out=at(4), residual=at(4, 256), rows=100),
], ids=str)
def test_products(call, rows):
    call = dict(dict(rows=rows), **call)
    assert ops._fn("bw_gemm_fp8")(call.get("x", at(0)), 256, call.get("xs", at(1)), 128, at(2), at(3), call.get("residual", 0), call.get("ldr", 64),
                                  call["out"], 64, 0, call["rows"], 64, 256, None) == -2


@pytest.mark.parametrize("rows", [4, 100])
@pytest.mark.parametrize("call", [
    dict(codes=at(0)), dict(codes=at(0, 256)), dict(codes=at(1)), dict(codes=at(2, 4096)), dict(codes=at(3)), dict(scales=at(0, 64)), dict(scales=at(1)),
    dict(scales=at(2, 4)), dict(scales=at(3, 4)), dict(scales=at(4, 16)),
], ids=str)
def test_gated_products(call, rows):
    c = dict(dict(codes=at(4), scales=at(5)), **call)
    assert ops._fn("bw_gemm_fp8_swiglu")(at(0), 256, at(1), 128, at(2), at(3), at(6), 64, c["codes"], 128, c["scales"], 128, rows, 64, 256, None) == -2


@pytest.mark.parametrize("sums", [at(0), at(1), at(2), at(3), at(4, 64), at(5, 8)])
def test_sums_of_gated_products(sums):
    assert ops._fn("bw_gemm_fp8_swiglu")(at(0), 256, at(1), 128, at(2), at(3), sums, 64, at(4), 128, at(5), 128, 4, 64, 256, None) == -2
