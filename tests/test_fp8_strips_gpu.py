"""Strips whose waves have no block of K in their last pass: what they asked for has come before their workgroup's LDS goes to another one."""

import pytest
import torch

from bitwise_amd.csrc import ops
from test_fp8_gpu import matrix, product_bound, rows_of_codes, same_bits

pytestmark = pytest.mark.gpu


def test_waves_without_a_block_beside_other_products(gpu):
    """Products of 1 to 25 blocks of K, few rows (so by way of LDS), one behind the other on two streams at once: the bits of each alone."""
    calls = []
    for blocks in (1, 2, 3, 5, 7, 9, 15, 17, 23, 25):
        for rows, n in ((1, 500), (8, 3000), (16, 6500), (33, 4000), (60, 1990)):
            k = 128 * blocks
            x, xs, x64 = rows_of_codes(rows, k, rows + blocks, gpu)
            w, ws, w64 = matrix(n, k, blocks, gpu)
            alone = torch.empty(rows, n, device=gpu)
            ops.gemm_fp8(x, xs, w, ws, alone, rows)
            some = slice(0, 64)
            off = (alone[:, some].cpu().double() - x64 @ w64[some].t()).abs()
            assert (off <= product_bound(x64, w64[some], k)).all(), (rows, n, k)
            calls.append((x, xs, w, ws, rows, alone, torch.empty(2, rows, n, device=gpu)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            for x, xs, w, ws, rows, _, out in (calls if i == 0 else calls[::-1]):
                ops.gemm_fp8(x, xs, w, ws, out[i], rows)
    torch.cuda.synchronize()
    for x, xs, w, ws, rows, alone, out in calls:
        assert same_bits(out[0], alone) and same_bits(out[1], alone), (rows, *w.shape)


@pytest.mark.parametrize("rows,n,k", [(3, 4200, 8192), (8, 8200, 640), (9, 4200, 8192), (16, 9001, 16384), (12, 4300, 8320), (5, 5000, 12288), (2, 4100, 24576)],
                         ids=lambda v: str(v))
def test_strips_of_many_columns(gpu, rows, n, k):
    """One strip a workgroup and two, rows of the matrix a multiple of 8,192 bytes apart and not."""
    x, xs, x64 = rows_of_codes(rows, k, rows, gpu)
    w, ws, w64 = matrix(n, k, n, gpu)
    out = torch.full((rows + 1, n), 9.0, device=gpu)
    ops.gemm_fp8(x, xs, w, ws, out, rows)
    assert ((out[:rows].cpu().double() - x64 @ w64.t()).abs() <= product_bound(x64, w64, k)).all() and (out[rows] == 9.0).all()
    residual = torch.randn(rows, n, generator=torch.Generator().manual_seed(5)).to(gpu)
    added = residual.clone()
    ops.gemm_fp8(x, xs, w, ws, added, rows, residual=added)
    assert same_bits(added, residual + out[:rows])
    one = torch.empty(1, n, device=gpu)
    ops.gemm_fp8(x[rows - 1:], xs[:, rows - 1:], w, ws, one, 1)
    assert same_bits(one[0], out[rows - 1])
