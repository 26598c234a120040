"""Matrices stored in 8 bits: e4m3 codes [out, in] and a 32-bit scale for each block of 128 x 128, which a checkpoint keeps
as two tensors, ``name`` and ``name`` + "_scale_inv" ([ceil(out / 128), ceil(in / 128)]; an element is its code times its block's
scale).  No counterpart in the reference, which stores BF16 and F32."""

from __future__ import annotations

from typing import List, Sequence, Tuple

import torch

BLOCK = 128
DTYPE = torch.float8_e4m3fn
SCALE_SUFFIX = "_scale_inv"
# what a folder's config.json says of such tensors ("quantization_config")
CONFIG = {"quant_method": "fp8", "fmt": "e4m3", "activation_scheme": "dynamic", "weight_block_size": [BLOCK, BLOCK]}


def blocks(n: int) -> int:
    return -(-int(n) // BLOCK)


class BlockScaled:
    """One stored matrix, or several stacked ones (``parts``, each with scale blocks of its own).  ``shape`` and ``dtype`` are those of
    the codes, so that a part can ask it what it asks a tensor."""

    dtype = DTYPE

    def __init__(self, parts: Sequence[Tuple[torch.Tensor, torch.Tensor]], in_features: int):
        self.parts: List[Tuple[torch.Tensor, torch.Tensor]] = list(parts)
        self.codes = self.scales = None                       # (all parts in one tensor each: ``on``)
        self.in_features = int(in_features)
        for codes, scales in self.parts:
            if codes.dtype != DTYPE or codes.dim() != 2 or codes.shape[1] not in (self.in_features, blocks(in_features) * BLOCK):
                raise ValueError(f"a matrix in 8 bits is e4m3 codes [out, {in_features}], got {codes.dtype} {tuple(codes.shape)}")
            if scales.dtype != torch.float32 or tuple(scales.shape) != (blocks(codes.shape[0]), blocks(in_features)):
                raise ValueError(f"codes {tuple(codes.shape)} need 32-bit scales {(blocks(codes.shape[0]), blocks(in_features))}, "
                                 f"got {scales.dtype} {tuple(scales.shape)}")

    @property
    def shape(self) -> Tuple[int, int]:
        return sum(c.shape[0] for c, _ in self.parts), self.in_features

    def dim(self) -> int:
        return 2

    def nbytes(self) -> int:
        return sum(c.numel() + 4 * s.numel() for c, s in self.parts)

    def on(self, device) -> "BlockScaled":
        """On a device, as the products take it: the rows of codes padded with zeros to whole blocks, all parts under one another
        in one tensor each (``codes``, ``scales``), of which the parts are views.  Parts of whole blocks become one part."""
        width, padded = blocks(self.in_features) * BLOCK, []
        for codes, _ in self.parts:
            c = codes.to(device).view(torch.uint8)
            padded.append(torch.nn.functional.pad(c, (0, width - c.shape[1])) if c.shape[1] != width else c)
        codes = torch.cat(padded, dim=0).contiguous().view(DTYPE)
        scales = torch.cat([s.to(device) for _, s in self.parts], dim=0).contiguous()
        views, row, block = [], 0, 0
        for c, s in self.parts:
            views.append((codes[row:row + c.shape[0]], scales[block:block + s.shape[0]]))
            row, block = row + c.shape[0], block + s.shape[0]
        if all(c.shape[0] % BLOCK == 0 for c, _ in self.parts[:-1]):
            views = [(codes, scales)]
        out = BlockScaled(views, self.in_features)
        out.codes, out.scales = codes, scales
        return out

    def widened(self) -> torch.Tensor:
        """The 32-bit matrix: code times scale, one rounding an element."""
        out = []
        for codes, scales in self.parts:
            n, k = codes.shape[0], self.in_features
            spread = scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
            out.append(codes[:, :k].float() * spread)
        return torch.cat(out, dim=0)


def stacked(matrices: Sequence) -> "torch.Tensor | BlockScaled":
    """Matrices of one input under one another: tensors of one dtype, or matrices in 8 bits (which stay apart: each begins its own
    scale blocks)."""
    if not any(isinstance(m, BlockScaled) for m in matrices):
        return torch.cat(list(matrices), dim=0)
    return BlockScaled([p for m in matrices for p in m.parts], matrices[0].in_features)


def quantize(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of a matrix: scale = the block's largest magnitude / 448 (of a block of zeros 2^-126), codes rounded to
    nearest even."""
    n, k = w.shape
    nb, kb = blocks(n), blocks(k)
    t = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    scales = t.abs().amax(dim=(1, 3)).clamp_min(448.0 * 2.0 ** -126) / 448.0
    codes = (t / scales[:, None, :, None]).clamp(-448.0, 448.0).view(nb * BLOCK, kb * BLOCK)[:n, :k]
    return codes.to(DTYPE).contiguous(), scales.contiguous()
