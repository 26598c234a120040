"""Rows and matrices of e4m3 codes with a scale for each block of 128: quantization, the norms around a sublayer, and the products,
against their definitions in 64 bits (or, where the definition is a sequence of single 32-bit operations, to the bit)."""

import pytest
import torch

from bitwise_amd.csrc import ops

pytestmark = pytest.mark.gpu
F8, U = torch.float8_e4m3fn, 2.0 ** -24                # U: half a step of a 32-bit number, relative
TINY = 2.0 ** -126


def gen(seed):
    return torch.Generator().manual_seed(seed)


def codes_like(rows, width, gpu, more=0, fill=0x2a):
    """Buffers for codes and scales of ``rows`` rows and ``more`` rows behind them, all filled with something."""
    kp = ops.fp8_width(width)
    c = torch.full((rows + more, kp), fill, dtype=torch.uint8, device=gpu).view(F8)
    return c, torch.full((kp // 128, rows + more), 7.0, device=gpu)


def quantized(x):
    """The definition on the CPU, scales and quotients rounded to 32 bits once: codes [rows, whole blocks] and scales [blocks, rows]."""
    x = x.float()
    kp = ops.fp8_width(x.shape[1])
    b = torch.nn.functional.pad(x, (0, kp - x.shape[1])).view(x.shape[0], kp // 128, 128)
    amax = b.abs().amax(dim=2)
    most = torch.where(amax < 448.0 * TINY, torch.tensor(448.0 * TINY), amax)
    return (448.0 * b.double() / most.double()[:, :, None]).float().view(x.shape[0], kp).to(F8), (most / 448.0).t().contiguous()


def values(codes, scales):
    """What codes stand for, in 64 bits."""
    return codes.cpu().double() * scales.cpu().double().t().repeat_interleave(128, 1)


def matrix(n, k, seed, gpu, halves=1, size=1.0):
    """Codes and scales of a random [halves * n, k] matrix, each half with scale blocks of its own, and its values in 64 bits."""
    kb, nb = ops.fp8_width(k) // 128, -(-n // 128)
    g, out = gen(seed), []
    for _ in range(halves):
        c = torch.zeros(n, kb * 128)
        c[:, :k] = torch.randn(n, k, generator=g) * 60
        out.append((c.to(F8), (torch.rand(nb, kb, generator=g) * 1e-3 + 1e-4) * size))
    codes = torch.cat([c.view(torch.uint8) for c, _ in out]).view(F8)
    w64 = torch.cat([c.double() * s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1) for c, s in out])
    return codes.to(gpu), torch.cat([s for _, s in out]).to(gpu), w64


def rows_of_codes(rows, k, seed, gpu):
    c, s = quantized(torch.randn(rows, k, generator=gen(seed)) * torch.exp(torch.randn(rows, 1, generator=gen(seed + 1))))
    return c.to(gpu), s.to(gpu), values(c, s)


def same_bits(a, b):
    return torch.equal(a.view(torch.uint8).cpu(), b.view(torch.uint8).cpu()) if a.dtype == F8 else torch.equal(a.cpu(), b.cpu())


# ------------------------------------------------------------------------------ quantization

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (3, 129), (16, 127), (17, 1000), (130, 2048), (33, 8)])
def test_quantization_is_the_definition_to_the_bit(gpu, rows, width, dtype):
    x = (torch.randn(rows, width, generator=gen(rows)) * torch.exp(3 * torch.randn(rows, 1, generator=gen(width)))).to(dtype)
    x[0, : width // 2] = 0.0
    codes, scales = codes_like(rows, width, gpu, more=2)
    ops.quantize_fp8(x.to(gpu), codes, scales, rows)
    want_c, want_s = quantized(x)
    assert same_bits(codes[:rows], want_c) and same_bits(scales[:, :rows].contiguous(), want_s)
    assert (codes[rows:].view(torch.uint8) == 0x2a).all() and (scales[:, rows:] == 7.0).all()      # rows behind are left as they were


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,width,stride", [(0, 256, 300), (1, 200, 333), (8, 264, 512), (3, 128, 131)])
def test_quantization_of_columns_of_a_wider_matrix(gpu, offset, width, stride, dtype):
    wide = torch.randn(19, stride, generator=gen(offset)).to(dtype).to(gpu)
    x = wide[:, offset:offset + width] if offset + width <= stride else wide[:, :width]
    codes = torch.zeros(19, ops.fp8_width(width) + 48, dtype=torch.uint8, device=gpu).view(F8)
    scales = torch.zeros(ops.fp8_width(width) // 128, 40, device=gpu)
    ops.quantize_fp8(x, codes[:, 16:16 + ops.fp8_width(width)], scales, 19)
    want_c, want_s = quantized(x.cpu())
    assert same_bits(codes[:, 16:16 + ops.fp8_width(width)].contiguous(), want_c) and same_bits(scales[:, :19].contiguous(), want_s)
    assert not codes[:, :16].view(torch.uint8).any() and not codes[:, 16 + ops.fp8_width(width):].view(torch.uint8).any() and not scales[:, 19:].any()


def test_quantization_of_numbers_at_the_ends_of_the_range(gpu):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(8, 256)
    x[0, 0] = 1e-45                     # the least number: beside it a scale of 448 * 2^-126 / 448
    x[1, :] = 448.0 * TINY
    x[2, 3], x[2, 200] = 3.4e38, -1e-30
    x[3, 5] = inf
    x[4, 7], x[4, 8] = nan, 5.0
    x[5, :128] = torch.linspace(-464.0, 464.0, 128)
    x[6, 0], x[6, 1:9] = 448.0, torch.tensor([2.0 ** -10, 1.5 * 2.0 ** -9, 2.0 ** -11, 17.0, 18.0, 19.0, 432.0, 440.0])   # ties
    x[7, 130] = -inf
    codes, scales = codes_like(8, 256, gpu)
    ops.quantize_fp8(x.to(gpu), codes, scales, 8)
    want_c, want_s = quantized(x)
    finite = torch.tensor([0, 1, 2, 5, 6])
    assert same_bits(codes[finite].contiguous(), want_c[finite]) and same_bits(scales[:, finite].contiguous(), want_s[:, finite])
    v = values(codes, scales)
    for row, first in ((3, True), (4, True), (7, False)):         # the block with an infinity or NaN is NaN throughout, the other is not
        bad, good = (v[row, :128], v[row, 128:]) if first else (v[row, 128:], v[row, :128])
        assert bad.isnan().all() and (good == 0).all()


# ------------------------------------------------------------------------------ the norms around a sublayer

def norm_bound(dim):
    """Relative error of v / sqrt(mean(v^2) + eps): a thread's chain of 8 ceil(dim / 2048) squares, ten joins, division, root,
    reciprocal and product; half of what the sum is off by shows behind the root."""
    return (4 * -(-dim // 2048) + 5 + 4) * U


CASES = [   # rows, dim, y's type, post norm, gate, sigmoid, scale vector, weights' type
    (1, 64, torch.float32, True, None, False, False, torch.float32),
    (5, 2048, torch.bfloat16, True, "row", True, False, torch.bfloat16),
    (3, 2049, torch.float32, True, "channel", False, True, torch.float32),
    (17, 576, torch.bfloat16, False, "row", False, True, torch.bfloat16),
    (2, 4096, torch.float32, False, None, False, False, torch.float32),
    (4, 5120, torch.bfloat16, True, "channel", True, True, torch.float32),
    (3, 8192, torch.float32, True, "row", True, False, torch.bfloat16),
    (2, 12288, torch.bfloat16, True, "row", False, True, torch.float32),
    (2, 9001, torch.float32, True, "row", True, True, torch.bfloat16),
    (6, 100, torch.bfloat16, True, "channel", False, False, torch.bfloat16),
    (1, 1, torch.float32, True, None, False, False, torch.float32),
]


def norm_inputs(case, gpu):
    rows, dim, yt, post, gate, sigmoid, vector, wt = case
    g = gen(rows * 10007 + dim)
    rnd = lambda *s: torch.randn(*s, generator=g)
    x, y = rnd(rows + 1, dim), (rnd(rows + 1, dim) * 3).to(yt)
    weight, post_weight = (1 + 0.1 * rnd(dim)).to(wt), (1 + 0.1 * rnd(dim)).to(wt) if post else None
    gt = None if gate is None else (rnd(rows + 1, dim) * 2).to(torch.bfloat16) if gate == "row" else rnd(dim)
    scale = torch.rand(dim, generator=g).to(wt) if vector else 0.35
    put = lambda t: t.to(gpu) if isinstance(t, torch.Tensor) else t
    return x, y, weight, post_weight, gt, scale, put


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, F8])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}")
def test_norms_around_a_sublayer(gpu, case, out_dtype):
    rows, dim, sigmoid, eps = case[0], case[1], case[5], 1e-5
    x, y, weight, post_weight, gt, scale, put = norm_inputs(case, gpu)
    z, bound = y.double(), 0.0
    if post_weight is not None:
        z, bound = z / (z.square().mean(1, keepdim=True) + 1e-3).sqrt() * post_weight.double(), norm_bound(dim) + U
    if gt is not None:
        z, bound = z * (torch.sigmoid(gt.double()) if sigmoid else gt.double()), bound + (5 * U if sigmoid else U)
    z = z * (scale.double() if isinstance(scale, torch.Tensor) else torch.tensor(scale, dtype=torch.float32).double())
    want = x.double() + z

    def run(out, scales=None):
        stream = torch.full((rows + 1, dim), 9.0, device=gpu)
        ops.norm_add_norm(put(x), put(y), put(weight), out, rows, eps, post_weight=put(post_weight), post_eps=1e-3, gate=put(gt), gate_sigmoid=sigmoid,
                          scale=put(scale), stream=stream, scales=scales)
        assert (stream[rows] == 9.0).all()                       # the row behind is left as it was
        return stream[:rows].cpu()

    if out_dtype == F8:
        out, scales = codes_like(rows, dim, gpu, more=1)
        stream = run(out, scales)
        assert (out[rows].view(torch.uint8) == 0x2a).all() and (scales[:, rows] == 7.0).all()
        plain = torch.empty(rows, dim, device=gpu)
        run(plain)
        again_c, again_s = codes_like(rows, dim, gpu)
        ops.quantize_fp8(plain, again_c, again_s, rows)           # the bits of the 32-bit rows quantized
        assert same_bits(out[:rows], again_c) and same_bits(scales[:, :rows].contiguous(), again_s)
    else:
        out = torch.full((rows + 1, dim), 9.0, device=gpu, dtype=out_dtype)
        stream = run(out)
        h = stream.double() / (stream.double().square().mean(1, keepdim=True) + eps).sqrt() * weight.double()
        off = (out[:rows].cpu().double() - h).abs()
        allowed = (norm_bound(dim) + U + (2.0 ** -8 if out_dtype == torch.bfloat16 else 0.0)) * h.abs() + 1e-40
        assert (off <= allowed).all(), (off / allowed).max()
        assert (out[rows] == 9.0).all()
    allowed = bound * z.abs() + U * want.abs() + 1e-40
    off = (stream.double() - want[:rows]).abs()
    assert (off <= allowed[:rows]).all(), (off / allowed[:rows]).max()


def test_norm_without_a_sublayer_and_in_place(gpu):
    x = torch.randn(7, 768, generator=gen(1)).to(gpu)
    w = (1 + 0.1 * torch.randn(768, generator=gen(2))).to(gpu)
    codes, scales = codes_like(7, 768, gpu)
    ops.norm_add_norm(x, None, w, codes, 7, 1e-6, scales=scales)
    plain = torch.empty(7, 768, device=gpu)
    ops.norm_add_norm(x, None, w, plain, 7, 1e-6)
    again = codes_like(7, 768, gpu)
    ops.quantize_fp8(plain, *again, 7)
    assert same_bits(codes, again[0]) and same_bits(scales, again[1])
    y = torch.randn(7, 768, generator=gen(3)).to(gpu)
    apart, out, out2 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ops.norm_add_norm(x, y, w, out, 7, 1e-6, scale=0.5, stream=apart)
    inplace = x.clone()
    ops.norm_add_norm(inplace, y, w, out2, 7, 1e-6, scale=0.5)
    assert same_bits(apart, inplace) and same_bits(out, out2)


@pytest.mark.parametrize("dim", [512, 500, 9000])
def test_norm_of_columns_of_wider_matrices(gpu, dim):
    """Rows a stride apart, starting anywhere: the bits of contiguous rows."""
    g = gen(dim)
    wide = {n: torch.randn(5, dim + 37, generator=g).to(gpu) for n in ("x", "y", "gate", "stream", "out")}
    part = {n: t[:, 5:5 + dim] for n, t in wide.items()}
    w = torch.randn(dim + 3, generator=g).to(gpu)
    stream, out = torch.empty(5, dim, device=gpu), torch.empty(5, dim, device=gpu)
    ops.norm_add_norm(part["x"].contiguous(), part["y"].contiguous(), w[3:].clone(), out, 5, 1e-6, post_weight=w[:dim].clone(),
                      gate=part["gate"].contiguous(), gate_sigmoid=True, scale=0.7, stream=stream)
    before = wide["out"].clone()
    ops.norm_add_norm(part["x"], part["y"], w[3:], part["out"], 5, 1e-6, post_weight=w[:dim], gate=part["gate"], gate_sigmoid=True, scale=0.7,
                      stream=part["stream"])
    assert same_bits(part["stream"].contiguous(), stream) and same_bits(part["out"].contiguous(), out)
    assert same_bits(wide["out"][:, :5].contiguous(), before[:, :5].contiguous()) and same_bits(wide["out"][:, 5 + dim:].contiguous(), before[:, 5 + dim:].contiguous())


def test_norm_of_rows_of_zeros_and_of_nan(gpu):
    x, y = torch.zeros(4, 256, device=gpu), torch.zeros(4, 256, device=gpu)
    y[1, 7], x[2, 200], y[3, 0] = float("nan"), float("inf"), 1e30           # (1e30 squared is past the range: the branch is normed to 0)
    w = torch.ones(256, device=gpu)
    codes, scales = codes_like(4, 256, gpu)
    stream = torch.empty_like(x)
    ops.norm_add_norm(x, y, w, codes, 4, 1e-6, post_weight=w, stream=stream, scales=scales)
    v = values(codes, scales)
    assert (v[0] == 0).all() and (scales[:, 0] == TINY).all()
    assert v[1].isnan().all() and stream[1].isnan().all()
    assert v[2, 128:].isnan().all() and (v[2, :128] == 0).all()
    assert (v[3] == 0).all() and (stream[3] == 0).all()


# ------------------------------------------------------------------------------ products

def product_bound(x64, w64, k):
    """What a product may be off by: each block's sum of 128 exact products in 32 bits, then a chain of one multiply-add a block."""
    return (128 + 2 * ops.fp8_width(k) // 128 + 2) * U * (x64.abs() @ w64.abs().t()) + 1e-40


SIZES = [(1, 1, 128), (1, 300, 2000), (2, 16, 256), (15, 130, 1152), (16, 128, 4096), (17, 100, 640), (33, 257, 1000), (48, 64, 128), (64, 272, 2176),
         (65, 5, 300), (100, 128, 128), (128, 257, 1152), (200, 640, 2048), (257, 384, 384), (300, 130, 4100), (520, 1000, 1024), (1030, 300, 256)]


@pytest.mark.parametrize("rows,n,k", SIZES, ids=lambda v: str(v))
def test_products(gpu, rows, n, k):
    x, xs, x64 = rows_of_codes(rows, k, rows, gpu)
    w, ws, w64 = matrix(n, k, n, gpu)
    want, bound = x64 @ w64.t(), product_bound(x64, w64, k)
    out = torch.full((rows + 1, n), 9.0, device=gpu)
    ops.gemm_fp8(x, xs, w, ws, out, rows)
    assert ((out[:rows].cpu().double() - want).abs() <= bound).all()
    assert (out[rows] == 9.0).all()
    rounded = torch.full((rows + 1, n), 9.0, device=gpu, dtype=torch.bfloat16)
    ops.gemm_fp8(x, xs, w, ws, rounded, rows)
    assert same_bits(rounded[:rows], out[:rows].bfloat16()) and (rounded[rows] == 9.0).all()
    residual = torch.randn(rows, n, generator=gen(5)).to(gpu) * want.abs().mean().item()
    added = torch.empty(rows, n, device=gpu)
    ops.gemm_fp8(x, xs, w, ws, added, rows, residual=residual)
    assert same_bits(added, residual + out[:rows])
    ops.gemm_fp8(x, xs, w, ws, residual, rows, residual=residual)
    assert same_bits(added, residual)


@pytest.mark.parametrize("n,k", [(272, 2176), (1030, 512), (128, 8192)])
def test_a_row_s_bits_do_not_depend_on_the_rows_beside_it(gpu, n, k):
    x, xs, _ = rows_of_codes(700, k, 3, gpu)
    w, ws, _ = matrix(n, k, 4, gpu)
    full = torch.empty(700, n, device=gpu)
    ops.gemm_fp8(x, xs, w, ws, full, 700)
    for rows, first in ((1, 0), (1, 699), (5, 3), (16, 16), (31, 600), (64, 100), (65, 101), (130, 200), (257, 300), (512, 100)):
        out = torch.empty(rows, n, device=gpu)
        ops.gemm_fp8(x[first:first + rows], xs[:, first:first + rows], w, ws, out, rows)
        assert same_bits(out, full[first:first + rows]), (rows, first)


def test_products_into_columns_of_a_wider_matrix(gpu):
    for rows in (3, 90):
        x, xs, _ = rows_of_codes(rows, 384, rows, gpu)
        w, ws, _ = matrix(150, 384, 1, gpu)
        out = torch.empty(rows, 150, device=gpu)
        ops.gemm_fp8(x, xs, w, ws, out, rows)
        for dtype in (torch.float32, torch.bfloat16):
            wide = torch.full((rows, 333), 9.0, device=gpu, dtype=dtype)
            ops.gemm_fp8(x, xs, w, ws, wide[:, 7:157], rows)
            assert same_bits(wide[:, 7:157].contiguous(), out.to(dtype)) and (wide[:, :7] == 9.0).all() and (wide[:, 157:] == 9.0).all()
        wide_x = torch.zeros(rows, 384 + 64, dtype=torch.uint8, device=gpu).view(F8)
        wide_x[:, 32:416].view(torch.uint8).copy_(x.view(torch.uint8))
        again = torch.empty(rows, 150, device=gpu)
        ops.gemm_fp8(wide_x[:, 32:416], xs, w, ws, again, rows)
        assert same_bits(again, out)


def test_nan_stays_in_its_row_and_its_column(gpu):
    for rows in (4, 80):
        x, xs, _ = rows_of_codes(rows, 256, 8, gpu)
        w, ws, _ = matrix(70, 256, 9, gpu)
        clean = torch.empty(rows, 70, device=gpu)
        ops.gemm_fp8(x, xs, w, ws, clean, rows)
        x.view(torch.uint8)[2, 130] = 0x7f
        w.view(torch.uint8)[33, 5] = 0xff
        xs[0, 1] = float("inf")
        out = torch.empty(rows, 70, device=gpu)
        ops.gemm_fp8(x, xs, w, ws, out, rows)
        keep_r, keep_c = torch.tensor([r for r in range(rows) if r not in (1, 2)]), torch.tensor([c for c in range(70) if c != 33])
        assert out[2].isnan().all() and out[:, 33].isnan().all() and not out[1].isfinite().any()
        assert same_bits(out.cpu()[keep_r][:, keep_c], clean.cpu()[keep_r][:, keep_c])


SWIGLU = [(1, 128, 128), (1, 300, 1000), (8, 1024, 512), (16, 65, 256), (40, 200, 640), (64, 272, 2176), (65, 65, 256), (70, 128, 128), (130, 300, 1000),
          (257, 520, 1152), (600, 384, 384)]


@pytest.mark.parametrize("rows,inter,k", SWIGLU, ids=lambda v: str(v))
def test_gated_products_into_codes(gpu, rows, inter, k):
    x, xs, x64 = rows_of_codes(rows, k, rows, gpu)
    w, ws, w64 = matrix(inter, k, inter, gpu, halves=2, size=0.1)
    codes, scales = codes_like(rows, inter, gpu, more=1)
    sums = torch.empty(min(rows, 64), inter, device=gpu)
    ops.gemm_fp8_swiglu(x, xs, w, ws, codes, scales, rows, sums=sums)
    assert (codes[rows].view(torch.uint8) == 0x2a).all() and (scales[:, rows] == 7.0).all()
    assert not codes[:rows, inter:].view(torch.uint8).any()
    y, off = x64 @ w64.t(), product_bound(x64, w64, k)
    g, u, dg, du = y[:, :inter], y[:, inter:], off[:, :inter], off[:, inter:]
    want = g * torch.sigmoid(g) * u
    # silu's slope is under 1.1; the 32-bit steps behind the sums: the sigmoid's four, two products
    near = 1.1 * dg * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du + 8 * U * want.abs()
    # the codes: half a step of a normal number, half the least step of a small one, and the steps of scale and quotient
    scale = scales[:, :rows].cpu().double().t().repeat_interleave(128, 1)[:, :inter]
    got = values(codes[:rows], scales[:, :rows].contiguous())[:, :inter]
    allowed = near * (1 + 2.0 ** -4) + torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -10) + 4 * U * want.abs()
    assert ((got - want).abs() <= allowed).all()
    most = torch.nn.functional.pad(want.abs(), (0, ops.fp8_width(inter) - inter)).view(rows, -1, 128).amax(dim=2)
    slack = torch.nn.functional.pad(near, (0, ops.fp8_width(inter) - inter)).view(rows, -1, 128).amax(dim=2)
    assert ((scales[:, :rows].cpu().double().t() * 448 - most).abs() <= slack + 2 * U * most + 449 * TINY).all()


def test_gated_products_give_the_same_bits_with_few_rows_and_many(gpu):
    x, xs, _ = rows_of_codes(200, 1024, 5, gpu)
    w, ws, _ = matrix(333, 1024, 6, gpu, halves=2, size=0.1)
    full, full_s = codes_like(200, 333, gpu)
    ops.gemm_fp8_swiglu(x, xs, w, ws, full, full_s, 200)
    for rows, first in ((1, 7), (16, 32), (64, 100), (65, 101), (64, 136)):
        codes, scales = codes_like(rows, 333, gpu)
        ops.gemm_fp8_swiglu(x[first:first + rows], xs[:, first:first + rows], w, ws, codes, scales, rows, sums=torch.empty(64, 333, device=gpu))
        assert same_bits(codes, full[first:first + rows]) and same_bits(scales, full_s[:, first:first + rows].contiguous()), (rows, first)


# ------------------------------------------------------------------------------ together

def feed_forward(x, y, s, rows):
    """A sublayer's output joins the stream, the normed stream goes through a gated feed-forward, all in 8 bits."""
    ops.norm_add_norm(x, y, s["norm"], s["h"], rows, 1e-6, post_weight=s["post"], scale=0.5, stream=s["stream"], scales=s["hs"])
    ops.gemm_fp8_swiglu(s["h"], s["hs"], s["up"], s["ups"], s["act"], s["acts"], rows, sums=s["sums"])
    ops.gemm_fp8(s["act"], s["acts"], s["down"], s["downs"], s["stream"], rows, residual=s["stream"])
    ops.quantize_fp8(s["stream"], s["q"], s["qs"], rows)


def feed_forward_state(rows, dim, inter, gpu):
    g = gen(rows)
    s = {"norm": torch.ones(dim, device=gpu), "post": torch.ones(dim, device=gpu), "stream": torch.zeros(rows, dim, device=gpu),
         "sums": torch.empty(64, inter, device=gpu)}
    s["h"], s["hs"] = codes_like(rows, dim, gpu)
    s["act"], s["acts"] = codes_like(rows, inter, gpu)
    s["q"], s["qs"] = codes_like(rows, dim, gpu)
    s["up"], s["ups"], _ = matrix(inter, dim, 1, gpu, halves=2, size=0.2)
    s["down"], s["downs"], _ = matrix(dim, inter, 2, gpu)
    return s, torch.randn(rows, dim, generator=g).to(gpu), torch.randn(rows, dim, generator=g).to(gpu)


@pytest.mark.parametrize("rows", [1, 9, 64, 65, 300])
def test_a_feed_forward_in_8_bits(gpu, rows):
    """The run of the operators against the same run in 64 bits: each rounding to codes is off by half a step (2^-4) of a value at
    most, three of them on the way, and they do not all point one way."""
    dim, inter = 384, 700
    s, x, y = feed_forward_state(rows, dim, inter, gpu)
    feed_forward(x, y, s, rows)
    norm = lambda t: t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt()
    spread = lambda c, sc, n: c.cpu().double() * sc.cpu().double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    stream = x.cpu().double() + 0.5 * norm(y.cpu().double())
    h = torch.nn.functional.pad(norm(stream), (0, s["up"].shape[1] - dim))
    half = s["ups"].shape[0] // 2
    g, u = h @ spread(s["up"][:inter], s["ups"][:half], inter).t(), h @ spread(s["up"][inter:], s["ups"][half:], inter).t()
    act = torch.nn.functional.pad(g * torch.sigmoid(g) * u, (0, s["down"].shape[1] - inter))
    want = stream + act @ spread(s["down"], s["downs"], dim).t()
    got = s["stream"].cpu().double()
    assert (got - want).norm() <= 3 * 2.0 ** -4 * (want - stream).norm() + 1e-5 * want.norm()
    assert (values(s["q"], s["qs"]) - got).norm() <= 2.0 ** -4 * got.norm()


def test_captured_runs_give_the_eager_bits_on_every_replay(gpu):
    for rows in (5, 80):
        s, x, y = feed_forward_state(rows, 256, 384, gpu)
        feed_forward(x, y, s, rows)
        first = [s[n].clone() for n in ("stream", "q", "qs")]
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            feed_forward(x, y, s, rows)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            feed_forward(x, y, s, rows)
        for change in (0.0, 0.25, 0.0):
            x0 = x.clone()
            x.add_(change)
            graph.replay()
            torch.cuda.synchronize()
            replayed = [s[n].clone() for n in ("stream", "q", "qs")]
            feed_forward(x, y, s, rows)
            torch.cuda.synchronize()
            assert all(same_bits(a, s[n]) for a, n in zip(replayed, ("stream", "q", "qs")))
            if not change:
                assert all(same_bits(a, b) for a, b in zip(replayed, first))
            x.copy_(x0)


def test_on_another_stream(gpu):
    s, x, y = feed_forward_state(70, 256, 384, gpu)
    feed_forward(x, y, s, 70)
    want = [s[n].clone() for n in ("stream", "q", "qs")]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for n in ("stream", "q", "qs"):
            s[n].view(torch.uint8).zero_()
        feed_forward(x, y, s, 70)
    side.synchronize()
    assert all(same_bits(a, s[n]) for a, n in zip(want, ("stream", "q", "qs")))


def test_no_rows_touch_nothing(gpu):
    s, x, y = feed_forward_state(3, 256, 384, gpu)
    before = {n: s[n].clone() for n in ("stream", "h", "act", "q")}
    feed_forward(x, y, s, 0)
    assert all(same_bits(before[n], s[n]) for n in before)


def test_offsets_past_31_bits(gpu):
    """Matrices and rows of codes of more than 2^31 bytes, outputs of more than 2^31 elements."""
    n, k = 140000, 16384
    w = torch.randint(0, 0x7e, (n, k), dtype=torch.uint8, device=gpu)
    ws = torch.full((-(-n // 128), k // 128), 1e-4, device=gpu)
    for rows in (2, 70):
        x, xs, x64 = rows_of_codes(rows, k, 1, gpu)
        out = torch.empty(rows, n, device=gpu)
        ops.gemm_fp8(x, xs, w.view(F8), ws, out, rows)
        for first in (0, 131072, n - 64):
            part = torch.empty(rows, 64, device=gpu)
            ops.gemm_fp8(x, xs, w[first:first + 64].clone().view(F8), ws[:1], part, rows)
            assert same_bits(out[:, first:first + 64].contiguous(), part)
    del w, out
    rows, width = 40000, 65536
    big = torch.empty(rows, width, dtype=torch.bfloat16, device=gpu)
    tail = torch.randn(8, width, generator=gen(4)).bfloat16()
    big[-8:] = tail.to(gpu)
    codes, scales = codes_like(rows, width, gpu)
    ops.quantize_fp8(big, codes, scales, rows)
    want_c, want_s = quantized(tail)
    assert same_bits(codes[-8:].contiguous(), want_c) and same_bits(scales[:, -8:].contiguous(), want_s)


# ------------------------------------------------------------------------------ every kernel that sizes lead to

# one block of K, and several: every strip and tile, plain and gated, and tiles with rows behind them (tests/test_fp8_rules.py checks
# that these sizes reach them all)
STORED = [(17, 68, 1792), (19, 77, 1536), (17, 70, 128), (18, 4904, 1792), (33, 6155, 1280), (34, 6328, 384), (335, 21916, 128), (199, 25401, 128),
          (3348, 261, 128), (1068, 65, 128), (400, 23971, 128), (194, 16868, 128), (1295, 1544, 1920), (960, 4391, 1280),
          (257, 22075, 640), (1001, 4090, 1152), (310, 6005, 1152), (500, 1501, 1152), (60, 6300, 1152),
          (3, 6001, 640), (9, 6001, 640), (16, 3001, 1152), (7, 500, 6144), (16, 500, 2176),
          (3, 500, 640), (12, 500, 640), (5, 4001, 2176), (60, 1990, 1300), (33, 1990, 700), (9, 4200, 4300), (2, 4200, 4300)]
GATED = [(17, 66, 640), (35, 2069, 384), (17, 67, 128), (17, 4591, 2176), (33, 6263, 384), (49, 6714, 640), (137, 27323, 128), (68, 22010, 128),
         (33, 20016, 128), (68, 65, 128), (132, 22012, 640), (67, 22083, 640), (33, 16470, 640), (200, 5003, 1152), (90, 1501, 1152),
         (3, 6001, 640), (16, 3001, 1152), (7, 500, 6144), (12, 5003, 640), (2, 9001, 640)]


def on_gpu(codes, scales, halves=1):
    """A matrix's values in 64 bits, on the GPU."""
    n, nb = codes.shape[0] // halves, scales.shape[0] // halves
    at = torch.arange(n, device=codes.device) // 128
    at = torch.cat([at + h * nb for h in range(halves)])
    return codes.double() * scales.double()[at][:, torch.arange(codes.shape[1], device=codes.device) // 128]


@pytest.mark.parametrize("rows,n,k", STORED, ids=lambda v: str(v))
def test_every_strip_and_tile(gpu, rows, n, k):
    x, xs, x64 = rows_of_codes(rows, k, rows, gpu)
    w, ws, _ = matrix(n, k, n, gpu)
    x64, w64 = x64.to(gpu), on_gpu(w, ws)
    want = torch.mm(x64, w64.t().contiguous())
    bound = (128 + 2 * k // 128 + 2) * U * torch.mm(x64.abs(), w64.abs().t().contiguous()) + 1e-40
    out = torch.full((rows + 1, n), 9.0, device=gpu)
    ops.gemm_fp8(x, xs, w, ws, out, rows)
    assert ((out[:rows].double() - want).abs() <= bound).all() and (out[rows] == 9.0).all()
    rounded = torch.full((rows + 1, n + 8), 9.0, device=gpu, dtype=torch.bfloat16)
    ops.gemm_fp8(x, xs, w, ws, rounded[:, :n], rows)
    assert same_bits(rounded[:rows, :n].contiguous(), out[:rows].bfloat16()) and (rounded[rows] == 9.0).all() and (rounded[:, n:] == 9.0).all()
    residual = torch.randn(rows, n, generator=gen(5)).to(gpu) * want.abs().mean().item()
    added = residual.clone()
    ops.gemm_fp8(x, xs, w, ws, added, rows, residual=added)
    assert same_bits(added, residual + out[:rows])
    # the bits of every row hang on the row alone: the last ones by themselves
    last = torch.empty(min(rows, 16), n, device=gpu)
    first = rows - last.shape[0]
    ops.gemm_fp8(x[first:], xs[:, first:], w, ws, last, last.shape[0])
    assert same_bits(last, out[first:rows])


@pytest.mark.parametrize("rows,inter,k", GATED, ids=lambda v: str(v))
def test_every_gated_strip_and_tile(gpu, rows, inter, k):
    x, xs, _ = rows_of_codes(rows, k, rows, gpu)
    w, ws, _ = matrix(inter, k, inter, gpu, halves=2, size=0.1)
    codes, scales = codes_like(rows, inter, gpu, more=1)
    ops.gemm_fp8_swiglu(x, xs, w, ws, codes, scales, rows, sums=torch.empty(64, inter, device=gpu))
    assert (codes[rows].view(torch.uint8) == 0x2a).all() and (scales[:, rows] == 7.0).all()
    # the two products' own sums, whose bits the tests above check: silu(g) u of them in 64 bits, then the definition of the codes
    half = ws.shape[0] // 2
    g, u = torch.empty(rows, inter, device=gpu), torch.empty(rows, inter, device=gpu)
    ops.gemm_fp8(x, xs, w[:inter].contiguous(), ws[:half].contiguous(), g, rows)
    ops.gemm_fp8(x, xs, w[inter:].contiguous(), ws[half:].contiguous(), u, rows)
    want = g.double() * torch.sigmoid(g.double()) * u.double()
    near = 8 * U * want.abs() + 1e-36                              # the sigmoid's four steps, two products
    spread = scales[:, :rows].double().t().repeat_interleave(128, 1)
    got = (codes[:rows].double() * spread)[:, :inter]
    allowed = near * (1 + 2.0 ** -4) + torch.maximum(want.abs() * 2.0 ** -4, spread[:, :inter] * 2.0 ** -10) + 4 * U * want.abs()
    assert ((got - want).abs() <= allowed).all()
    pad = lambda t: torch.nn.functional.pad(t, (0, ops.fp8_width(inter) - inter)).view(rows, -1, 128).amax(dim=2)
    assert ((scales[:, :rows].double().t() * 448 - pad(want.abs())).abs() <= pad(near) + 2 * U * pad(want.abs()) + 449 * TINY).all()
    few = min(rows, 16)
    last_c, last_s = codes_like(few, inter, gpu)
    ops.gemm_fp8_swiglu(x[rows - few:], xs[:, rows - few:], w, ws, last_c, last_s, few, sums=torch.empty(16, inter, device=gpu))
    assert same_bits(last_c, codes[rows - few:rows]) and same_bits(last_s, scales[:, rows - few:rows].contiguous())


def test_two_results_in_one_place_are_refused(gpu):
    x, y, w = torch.randn(4, 256, device=gpu), torch.randn(4, 256, device=gpu), torch.ones(256, device=gpu)
    before = x.clone()
    with pytest.raises(RuntimeError, match="norm_add_norm"):
        ops.norm_add_norm(x, y, w, x, 4, 1e-6)
    assert same_bits(x, before)


def test_wrappers_refuse_what_does_not_fit(gpu):
    x, c, s = torch.randn(4, 300, device=gpu), *codes_like(4, 300, gpu)
    w, ws, _ = matrix(70, 300, 1, gpu)
    out = torch.empty(4, 70, device=gpu)
    for call, says in (
            (lambda: ops.quantize_fp8(x, c[:, :256], s[:2], 4), "codes of rows of 300"),
            (lambda: ops.quantize_fp8(x, c, s[:, :3], 4), "do not fit"),
            (lambda: ops.quantize_fp8(x[:3], c, s, 4), "does not fit"),
            (lambda: ops.quantize_fp8(x.t(), c, s, 4), "rows are contiguous"),
            (lambda: ops.quantize_fp8(x, c.view(torch.uint8), s, 4), "float8"),
            (lambda: ops.quantize_fp8(x, c, s.double(), 4), "float32"),
            (lambda: ops.gemm_fp8(c[:, :200], s, w, ws, out, 4), "whole blocks"),
            (lambda: ops.gemm_fp8(c, s, w[:, :256].contiguous(), ws[:, :2].contiguous(), out, 4), "does not fit"),
            (lambda: ops.gemm_fp8(c, s, w, ws[:, :2], out, 4), "does not fit"),
            (lambda: ops.gemm_fp8(c, s, w, ws, out[:, :60], 4), "does not fit"),
            (lambda: ops.gemm_fp8(c, s, w, ws, out[:2], 4), "does not fit"),
            (lambda: ops.gemm_fp8(c, s, w, ws, out.bfloat16(), 4, residual=out), "stays 32-bit"),
            (lambda: ops.gemm_fp8(c, s, w, ws, out, 4, residual=out.double()), "float32"),
            (lambda: ops.gemm_fp8(c[:, 8:], s, w, ws, out, 4), "whole blocks"),
            (lambda: ops.gemm_fp8_swiglu(c, s, w, ws, *codes_like(4, 35, gpu), 4), "scales"),
            (lambda: ops.norm_add_norm(x, None, x[0], c, 4, 1e-6), "codes come with scales"),
            (lambda: ops.norm_add_norm(x, None, x[0], out, 4, 1e-6, scales=s), "codes come with scales"),
            (lambda: ops.norm_add_norm(x, None, x[0], x.clone(), 4, 1e-6, gate=x), "nothing to norm"),
            (lambda: ops.norm_add_norm(x, x[:2], x[0], x.clone(), 4, 1e-6), "does not fit"),
            (lambda: ops.norm_add_norm(x, x.half(), x[0], x.clone(), 4, 1e-6), "float32"),
            (lambda: ops.norm_add_norm(x, x, x[0, :200], x.clone(), 4, 1e-6), "vector of 300"),
            (lambda: ops.norm_add_norm(x, x, x[0], x.clone(), 4, 1e-6, gate=x[0].expand(4, 300)), "a vector"),
            (lambda: ops.norm_add_norm(x, x, x[0], x.clone(), 4, 1e-6, scale=x[:, 0]), "vector of 300")):
        with pytest.raises(ValueError, match=says):
            call()
    w2, ws2, _ = matrix(40, 300, 2, gpu, halves=2)
    with pytest.raises(ValueError, match="buffer for their sums"):
        ops.gemm_fp8_swiglu(c, s, w2, ws2, *codes_like(4, 40, gpu), 4)
