"""The operators of the 8-bit path, measured: what lies between a residual stream and its next product when weights and the
products' inputs are kept in 8 bits (e4m3) with a 32-bit scale for each block of 128.

* ``quantize``: rows to e4m3 codes and a scale for each 128 of their elements;
* ``norm``: a sublayer's output is normed, gated, scaled and added to the stream, and the stream is normed for the next
  sublayer, as e4m3 codes with their scales, in bfloat16 or in 32 bits;
* ``product``: rows of codes times a matrix of codes with a scale for each 128 x 128 block, stored in 32 bits or bfloat16 or
  added to the stream;
* ``swiglu``: the stacked gate|up product, its activation as codes with scales for the down projection.

Codes are rows padded with zeros to whole blocks; the scales of rows lie block by block, ``scales[block, row]``.  Layer sizes are
the benchmark's (the SmolLM2-1.7B and the Llama-3-8B shape) or generic.
"""

import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -126              # the least scale (the smallest normal 32-bit number): a block of zeros gets it
FEW_ROWS = 64                   # rows up to which the activation goes through a buffer of the caller's


def _quantize_case(name, rows, width, dtype):
    return {"name": name, "op": "quantize", "rows": rows, "width": width, "dtype": dtype}


def _norm_case(name, rows, width, branch, post, gate, scale, out):
    """``branch``: the type of the sublayer's output; ``post``: whether it is normed; ``gate``: "none", "row" (a bfloat16 matrix
    through a sigmoid) or "channel" (a 32-bit vector as it is); ``scale``: "one" (a number) or "channel" (a vector); ``out``: "fp8", "bfloat16", "float32"."""
    return {"name": name, "op": "norm", "rows": rows, "width": width, "branch": branch, "post": post, "gate": gate, "scale": scale, "out": out}


def _product_case(name, rows, n, k, out):
    """``out``: "bfloat16", "float32", or "add" (32-bit, added to the stream)."""
    return {"name": name, "op": "product", "rows": rows, "n": n, "k": k, "out": out}


def _swiglu_case(name, rows, inter, k):
    return {"name": name, "op": "swiglu", "rows": rows, "inter": inter, "k": k}


def listed():
    return [
        # one user's next token: a row of attention output on its way into the output projection
        _quantize_case("quantize_b1", 1, 2048, "bfloat16"),
        # a whole token budget of attention output on the larger model
        _quantize_case("quantize_2048", 2048, 4096, "bfloat16"),
        # a ragged portion, 32-bit rows of a width that is no whole number of blocks
        _quantize_case("quantize_ragged", 777, 5000, "float32"),
        # eight decoding requests between two sublayers of a layer with norms on both sides
        _norm_case("norm_b8", 8, 2048, "float32", True, "none", "one", "fp8"),
        # a budget of prompt rows with a gate of its own for each element
        _norm_case("norm_gated_2048", 2048, 4096, "bfloat16", True, "row", "one", "fp8"),
        # a ragged portion, no norm behind the sublayer but a scale for each channel, bfloat16 rows for products in 16 bits
        _norm_case("norm_scaled_517", 517, 5120, "float32", False, "channel", "channel", "bfloat16"),
        # one user's next token, the down projection added to the stream
        _product_case("product_b1", 1, 2048, 8192, "add"),
        # eight decoding requests on the larger model: q|k|v
        _product_case("product_b8", 8, 6144, 4096, "float32"),
        # a busy server: 43 decoding requests, the output projection of the larger model
        _product_case("product_b43", 43, 4096, 4096, "add"),
        # a ragged portion, an inner size of no whole blocks, an odd number of columns
        _product_case("product_ragged_777", 777, 5003, 2000, "bfloat16"),
        # eight decoding requests: the feed-forward's first half
        _swiglu_case("swiglu_b8", 8, 8192, 2048),
        # a whole token budget on the larger model: the feed-forward's first half
        _swiglu_case("swiglu_2048", 2048, 14336, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Over the logarithm of the range, any number, a multiple of 16 or a whole number of blocks."""
    n = _log(rng, lo, hi)
    step = rng.choice((1, 16, 128))
    return max(lo, n // step * step)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("quantize", "norm", "product", "product", "product", "swiglu", "swiglu"))
        rows = _log(rng, 1, 2048)
        if op == "quantize":
            c = _quantize_case("", rows, _size(rng, 64, 16384), rng.choice(("bfloat16", "float32")))
        elif op == "norm":
            c = _norm_case("", rows, _size(rng, 64, 8192), rng.choice(("bfloat16", "float32")), rng.random() < 0.6,
                           rng.choice(("none", "row", "channel")), rng.choice(("one", "channel")), rng.choice(("fp8", "fp8", "bfloat16", "float32")))
        elif op == "product":
            c = _product_case("", rows, _size(rng, 128, 28672), _size(rng, 128, 14336), rng.choice(("bfloat16", "float32", "add")))
        else:
            c = _swiglu_case("", rows, _size(rng, 128, 14336), _size(rng, 128, 8192))
        del c["name"]
        if _cost(c) <= most:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 500)


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    rows = case["rows"]
    if case["op"] == "quantize":
        k = case["width"]
        return {"bytes": rows * k * (2 if case["dtype"] == "bfloat16" else 4) + rows * _blocks(k) * (BLOCK + 4), "flops": 3 * rows * k}
    if case["op"] == "norm":
        k = case["width"]
        element = (2 if case["branch"] == "bfloat16" else 4) + 8 + (2 if case["gate"] == "row" else 0)
        vectors = 1 + int(case["post"]) + int(case["gate"] == "channel") + int(case["scale"] == "channel")
        out = rows * _blocks(k) * (BLOCK + 4) if case["out"] == "fp8" else rows * k * (2 if case["out"] == "bfloat16" else 4)
        return {"bytes": rows * k * element + 4 * k * vectors + out, "flops": 12 * rows * k}
    kb = _blocks(case["k"])
    read = rows * kb * (BLOCK + 4)
    if case["op"] == "product":
        n = case["n"]
        out = rows * n * {"bfloat16": 2, "float32": 4, "add": 8}[case["out"]]
        return {"bytes": read + n * kb * BLOCK + _blocks(n) * kb * 4 + out, "flops": 2 * rows * n * case["k"]}
    n = case["inter"]
    return {"bytes": read + 2 * n * kb * BLOCK + 2 * _blocks(n) * kb * 4 + rows * _blocks(n) * (BLOCK + 4), "flops": 4 * rows * n * case["k"]}


# ------------------------------------------------------------------------------ inputs

def _rows(gen, rows, width, dtype=torch.float32):
    """Activations: normal values, a few channels many times larger (as they are behind trained norms), row by row of another size."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    loud = torch.randint(0, width, (max(1, width // 256),), generator=gen, device="cuda")
    x[:, loud] *= 12.0
    x *= torch.exp(torch.randn(rows, 1, generator=gen, device="cuda") * 0.5)
    return x.to(dtype)


def _padded(x, rows_to=1):
    n, k = x.shape
    return torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k, 0, -(-n // rows_to) * rows_to - n))


def _weight(gen, n, k):
    """A checkpoint's matrix: codes [n, whole blocks] and a scale for each 128 x 128 block."""
    w = _padded(torch.randn(n, k, generator=gen, device="cuda") * 0.02, BLOCK)
    w4 = w.view(w.shape[0] // BLOCK, BLOCK, w.shape[1] // BLOCK, BLOCK)
    w4 = w4 * torch.exp(torch.randn(w4.shape[0], 1, w4.shape[2], 1, generator=gen, device="cuda") * 0.3)
    scales = w4.abs().amax(dim=(1, 3)).clamp_min(TINY) / E4M3_MAX
    codes = (w4 / scales[:, None, :, None]).reshape(w.shape).to(torch.float8_e4m3fn)
    return codes[:n].contiguous(), scales.contiguous()


def _codes(rows, width):
    """Where rows of codes go, and their scales."""
    kb = _blocks(width)
    return torch.zeros(rows, kb * BLOCK, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.zeros(kb, rows, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000003 * seed + 17)
    rows, op = case["rows"], case["op"]
    s = {"case": dict(case)}
    if op == "quantize":
        s["x"] = _rows(gen, rows, case["width"], getattr(torch, case["dtype"]))
        s["codes"], s["scales"] = _codes(rows, case["width"])
        return s
    if op == "norm":
        k = case["width"]
        s["x"] = _rows(gen, rows, k)
        s["y"] = _rows(gen, rows, k, getattr(torch, case["branch"]))
        s["weight"] = 1.0 + 0.1 * torch.randn(k, generator=gen, device="cuda")
        s["post"] = 1.0 + 0.1 * torch.randn(k, generator=gen, device="cuda") if case["post"] else None
        s["gate"] = (torch.randn(rows, k, generator=gen, device="cuda").bfloat16() if case["gate"] == "row" else
                     1.0 + 0.3 * torch.randn(k, generator=gen, device="cuda") if case["gate"] == "channel" else None)
        s["scale"] = torch.rand(k, generator=gen, device="cuda") if case["scale"] == "channel" else 0.25
        s["stream"] = torch.empty_like(s["x"])
        if case["out"] == "fp8":
            s["out"], s["scales"] = _codes(rows, k)
        else:
            s["out"], s["scales"] = torch.empty(rows, k, dtype=getattr(torch, case["out"]), device="cuda"), None
        return s
    x = _rows(gen, rows, case["k"])
    s["x"], s["xs"] = _quantized(x)
    if op == "product":
        n = case["n"]
        s["w"], s["ws"] = _weight(gen, n, case["k"])
        s["residual"] = torch.randn(rows, n, generator=gen, device="cuda") if case["out"] == "add" else None
        s["out"] = torch.empty(rows, n, dtype=torch.bfloat16 if case["out"] == "bfloat16" else torch.float32, device="cuda")
    else:
        n = case["inter"]
        (g, gs), (u, us) = _weight(gen, n, case["k"]), _weight(gen, n, case["k"])
        s["w"], s["ws"] = torch.cat([g.view(torch.uint8), u.view(torch.uint8)]).view(torch.float8_e4m3fn), torch.cat([gs, us])
        s["out"], s["scales"] = _codes(rows, n)
        s["sums"] = torch.empty(min(rows, FEW_ROWS), n, device="cuda")
    return s


# ------------------------------------------------------------------------------ the plain forms

def _quantized(x):
    """Codes and scales of 32-bit rows: scale = max(the block's largest magnitude, 448 * 2^-126) / 448, code = e4m3(x * (1 / scale))."""
    x = _padded(x.float())
    b = x.view(x.shape[0], -1, BLOCK)
    scale = b.abs().amax(dim=2).clamp_min(E4M3_MAX * TINY) / E4M3_MAX
    codes = (b * (1.0 / scale)[:, :, None]).view(x.shape).to(torch.float8_e4m3fn)
    return codes, scale.t().contiguous()


def _values(codes, scales):
    """What rows of codes stand for, in 32 bits."""
    rows, k = codes.shape
    return (codes.float().view(rows, -1, BLOCK) * scales.t()[:, :, None]).view(rows, k)


def _matrix(codes, scales):
    """What a matrix of codes stands for, in 32 bits."""
    n, k = codes.shape
    return codes.float() * scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)


def _normed(x, weight, eps=1e-6):
    return x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + eps) * weight


def _plain(s):
    op = s["case"]["op"]
    if op == "quantize":
        return _quantized(s["x"])
    if op == "norm":
        z = s["y"].float()
        if s["post"] is not None:
            z = _normed(z, s["post"])
        if s["gate"] is not None:
            z = z * (torch.sigmoid(s["gate"].float()) if s["gate"].dim() == 2 else s["gate"])
        stream = s["x"] + s["scale"] * z
        h = _normed(stream, s["weight"])
        return (stream, *_quantized(h)) if s["scales"] is not None else (stream, h.to(s["out"].dtype))
    x = _values(s["x"], s["xs"])
    if op == "product":
        y = x @ _matrix(s["w"], s["ws"]).t()
        return y + s["residual"] if s["residual"] is not None else y.to(s["out"].dtype)
    n, b = s["case"]["inter"], s["ws"].shape[0] // 2
    g = x @ _matrix(s["w"][:n], s["ws"][:b]).t()
    u = x @ _matrix(s["w"][n:], s["ws"][b:]).t()
    return _quantized(g / (1.0 + torch.exp(-g)) * u)


def run(s):
    if not own:
        return _plain(s)
    from bitwise_amd.csrc import ops
    case, rows, op = s["case"], s["case"]["rows"], s["case"]["op"]
    if op == "quantize":
        ops.quantize_fp8(s["x"], s["codes"], s["scales"], rows)
        return s["codes"], s["scales"]
    if op == "norm":
        ops.norm_add_norm(s["x"], s["y"], s["weight"], s["out"], rows, 1e-6, post_weight=s["post"], gate=s["gate"],
                          gate_sigmoid=case["gate"] == "row", scale=s["scale"], stream=s["stream"], scales=s["scales"])
        return (s["stream"], s["out"], s["scales"]) if s["scales"] is not None else (s["stream"], s["out"])
    if op == "product":
        ops.gemm_fp8(s["x"], s["xs"], s["w"], s["ws"], s["out"], rows, residual=s["residual"])
        return s["out"]
    ops.gemm_fp8_swiglu(s["x"], s["xs"], s["w"], s["ws"], s["out"], s["scales"], rows, sums=s["sums"])
    return s["out"], s["scales"]


# ------------------------------------------------------------------------------ the definitions in 64 bits

def _exact_codes(h):
    n, k = h.shape
    full = torch.zeros(n, _blocks(k) * BLOCK, dtype=torch.float64, device=h.device)
    full[:, :k] = h
    b = full.reshape(n, _blocks(k), BLOCK)
    scale = torch.clamp(b.abs().max(dim=2).values / 448.0, min=2.0 ** -126)
    return (b / scale[:, :, None]).reshape(n, -1).to(torch.float32).to(torch.float8_e4m3fn), scale.t().contiguous()


def _spread(scale, rows, columns):
    """A scale for each element from one for each block."""
    i = torch.arange(rows, device=scale.device) // 128
    j = torch.arange(columns, device=scale.device) // 128
    return scale.double()[i][:, j]


def exact(case, seed):
    s, op, rows = prepare(case, seed), case["op"], case["rows"]
    if op == "quantize":
        return _exact_codes(s["x"].double())
    if op == "norm":
        z = s["y"].double()
        if s["post"] is not None:
            z = z / (z.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * s["post"].double()
        if case["gate"] == "row":
            z = z / (1.0 + torch.exp(-s["gate"].double()))
        elif case["gate"] == "channel":
            z = z * s["gate"].double()
        stream = s["x"].double() + z * (s["scale"].double() if case["scale"] == "channel" else s["scale"])
        h = stream / (stream.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * s["weight"].double()
        return (stream, *_exact_codes(h)) if case["out"] == "fp8" else (stream, h)
    k = s["x"].shape[1]
    at = torch.arange(k, device="cuda") // 128
    x = s["x"].double() * s["xs"].double()[at].t()
    if op == "product":
        y = torch.mm(x, (s["w"].double() * _spread(s["ws"], case["n"], k)).t().contiguous())
        return y + s["residual"].double() if case["out"] == "add" else y
    n, half = case["inter"], s["ws"].shape[0] // 2
    g = torch.mm(x, (s["w"][:n].double() * _spread(s["ws"][:half], n, k)).t().contiguous())
    u = torch.mm(x, (s["w"][n:].double() * _spread(s["ws"][half:], n, k)).t().contiguous())
    return _exact_codes(g * u / (1.0 + torch.exp(-g)))
