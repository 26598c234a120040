"""Weights by tensor name: checking a checkpoint against a model's tensor specs, and
seeded random weights written as a model folder.

Dtype policy (the reference's converter, tools/convert.py:85-92, keeps BF16 and F32
bytes and widens F16 to F32): bfloat16 stays bfloat16, a tensor stored in 32-bit stays
32-bit, float16 is widened to float32, integer tables become int32; a matrix in 8 bits (e4m3 codes
beside a tensor of scales) stays in 8 bits where the part that owns it takes it so.  Names are the
checkpoint's own (src/model.cpp:136-171); nothing is renamed.
"""

from __future__ import annotations

import json
import warnings
from pathlib import Path
from typing import Dict, Iterator, Mapping, Sequence, Tuple

import torch

from ..parts.base import TensorSpec
from . import block_scaled, safetensors_io


class WeightError(ValueError):
    """One error for everything wrong with a checkpoint: missing, unexpected, misshapen."""


class UnusedTensorWarning(UserWarning):
    """A checkpoint tensor that the architecture knows of and this configuration does not read."""


def check_and_convert(specs: Mapping[str, TensorSpec], found: Mapping[str, torch.Tensor],
                      source: str = "checkpoint", ignored_suffixes: Sequence[str] = (),
                      unused: Sequence[str] = ()) -> Dict[str, torch.Tensor]:
    """``ignored_suffixes`` and ``unused`` come from the architecture (``ModelSpec``): tensors it
    knows to carry nothing (passed over in silence) or nothing this configuration reads (passed
    over with an ``UnusedTensorWarning``).  Any other tensor the model has no use for is an error."""
    missing = [n for n in specs if n not in found]
    ignored = tuple(ignored_suffixes)
    # (a matrix in 8 bits brings its scales under a name of their own)
    scales = {n + block_scaled.SCALE_SUFFIX for n in specs if n in found and found[n].dtype == block_scaled.DTYPE}
    extra = [n for n in found if n not in specs and n not in scales and not (ignored and n.endswith(ignored))]
    unexpected = [n for n in extra if n not in unused]
    tolerated = [n for n in extra if n in unused]
    wrong = []
    out: Dict[str, torch.Tensor] = {}
    for name, spec in specs.items():
        if name not in found:
            continue
        t = found[name]
        if tuple(t.shape) != tuple(spec.shape):
            wrong.append(f"{name}: stored {tuple(t.shape)}, the configuration needs {tuple(spec.shape)}")
            continue
        if spec.kind == "int":
            if t.dtype not in (torch.int32, torch.int64):
                wrong.append(f"{name}: stored as {t.dtype}, an integer table is needed")
                continue
            if spec.below:
                bad = int(((t < 0) | (t >= spec.below)).sum())
                if bad:
                    wrong.append(f"{name}: {bad} entries outside 0 .. {spec.below - 1}")
                    continue
                ordered = t.reshape(-1, t.shape[-1]).sort(dim=-1).values
                if bool((ordered[:, 1:] == ordered[:, :-1]).any()):
                    wrong.append(f"{name}: a row names one entry twice")
                    continue
            out[name] = t.to(torch.int32)
        elif t.dtype == torch.bfloat16 or t.dtype == torch.float32:
            out[name] = t
        elif t.dtype == torch.float16:
            out[name] = t.to(torch.float32)
        elif t.dtype == block_scaled.DTYPE and spec.block_scaled:
            s = found.get(name + block_scaled.SCALE_SUFFIX)
            want = (block_scaled.blocks(spec.shape[0]), block_scaled.blocks(spec.shape[1]))
            if s is None:
                missing.append(name + block_scaled.SCALE_SUFFIX)
            elif tuple(s.shape) != want or s.dtype not in (torch.float32, torch.bfloat16):
                wrong.append(f"{name}{block_scaled.SCALE_SUFFIX}: stored {tuple(s.shape)} {s.dtype}, a floating scale for each block of "
                             f"{block_scaled.BLOCK} x {block_scaled.BLOCK} is needed, {want}")
            elif not bool(torch.isfinite(s).all()):
                wrong.append(f"{name}{block_scaled.SCALE_SUFFIX}: scales that are no finite numbers")
            else:
                out[name] = block_scaled.BlockScaled([(t, s.float())], spec.shape[1])
        else:
            wrong.append(f"{name}: unsupported dtype {t.dtype}")
    if missing or unexpected or wrong:
        lines = [f"{source} does not fit the model:"]
        if missing:
            lines.append(f"  missing tensors ({len(missing)}): " + ", ".join(missing))
        if unexpected:
            lines.append(f"  unexpected tensors ({len(unexpected)}): " + ", ".join(unexpected))
        if wrong:
            lines.append(f"  wrong shape or dtype ({len(wrong)}):")
            lines.extend("    " + w for w in wrong)
        raise WeightError("\n".join(lines))
    if tolerated:
        warnings.warn(f"{source}: tensors stored and not used by this configuration: " + ", ".join(tolerated),
                      UnusedTensorWarning, stacklevel=2)
    return out


def load_folder(folder: str | Path, specs: Mapping[str, TensorSpec], ignored_suffixes: Sequence[str] = (),
                unused: Sequence[str] = ()) -> Dict[str, torch.Tensor]:
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")       # read-only memory maps viewed as tensors
        found = safetensors_io.read_folder(folder)
    return check_and_convert(specs, found, str(folder), ignored_suffixes, unused)


def shape_values(kind: str, z: torch.Tensor, sigma: float) -> torch.Tensor:
    """Standard normals ``z`` turned into the values of a tensor of this kind (parts.base.TensorSpec)."""
    if kind == "norm":
        return 1.0 + 0.1 * z
    if kind == "around_zero":
        return 0.1 * z
    if kind == "unit_interval":
        return torch.sigmoid(z)
    if kind == "bias":
        return z
    if kind == "small_bias":
        return 0.1 * z
    if kind == "conv":                         # taps of a short convolution: of the order of 1 / taps
        return 0.5 * z
    if kind == "router":                       # logits that spread over a few units
        return 0.3 * z
    if kind == "gate_matrix":                  # square matrices in front of a sigmoid: rows of norm about 1 for inputs of norm 1
        return z / (z.shape[-1] ** 0.5)
    return sigma * z


def random_table(spec: TensorSpec, generator: torch.Generator, device="cpu") -> torch.Tensor:
    """An integer table's random entries: uniform in [0, 2**15), or, bounded, the first of a random order of 0 .. below - 1."""
    if not spec.below:
        return torch.randint(0, 2 ** 15, spec.shape, generator=generator, dtype=torch.int32, device=device)
    *rows, n = spec.shape
    if n > spec.below:
        raise ValueError(f"{n} different entries out of {spec.below}")
    order = torch.rand((*rows, spec.below), generator=generator, device=device).argsort(dim=-1)
    return order[..., :n].to(torch.int32).contiguous()


def stored_as(name: str, spec: TensorSpec, values: torch.Tensor, dtype: torch.dtype) -> Iterator[Tuple[str, torch.Tensor]]:
    """The tensor or tensors that hold these values in a dtype.  8 bits: codes and scales where the part takes them, bfloat16
    elsewhere."""
    if dtype != block_scaled.DTYPE:
        yield name, values.to(dtype)
    elif spec.block_scaled:
        codes, scales = block_scaled.quantize(values)
        yield name, codes
        yield name + block_scaled.SCALE_SUFFIX, scales
    else:
        yield name, values.to(torch.bfloat16)


def random_tensors(specs: Mapping[str, TensorSpec], seed: int, sigma: float = 0.02,
                   dtype: torch.dtype = torch.bfloat16) -> Iterator[Tuple[str, torch.Tensor]]:
    """Seeded random weights, one tensor after the other in the order of ``specs``.

    All draws come from one ``torch.Generator`` (CPU, ``manual_seed(seed)``) as float32
    standard normals in tensor order: linear and embedding weights are ``sigma * z``,
    norm weights ``1 + 0.1 * z``, integer tables as ``random_table`` draws them.  Values are then
    rounded to ``dtype`` (round to nearest even for bfloat16; float8_e4m3fn: matrices of parts that take them so in 8 bits, the
    rest in bfloat16).
    """
    g = torch.Generator(device="cpu")
    g.manual_seed(int(seed))
    for name, spec in specs.items():
        if spec.kind == "int":
            yield name, random_table(spec, g)
            continue
        z = torch.randn(spec.shape, generator=g, dtype=torch.float32)
        yield from stored_as(name, spec, shape_values(spec.kind, z, sigma), dtype)


def write_model_folder(folder: str | Path, config: Mapping[str, object], specs: Mapping[str, TensorSpec],
                       seed: int, sigma: float = 0.02, dtype: torch.dtype = torch.bfloat16) -> Path:
    """Random-weights mode: ``folder/config.json`` (which says so if matrices are in 8 bits) and ``folder/model.safetensors``."""
    folder = Path(folder)
    folder.mkdir(parents=True, exist_ok=True)
    said = dict(config)
    if dtype == block_scaled.DTYPE and any(s.block_scaled for s in specs.values()):
        said["quantization_config"] = block_scaled.CONFIG
    (folder / "config.json").write_text(json.dumps(said, indent=1))
    safetensors_io.write_file(folder / "model.safetensors", random_tensors(specs, seed, sigma, dtype))
    return folder
