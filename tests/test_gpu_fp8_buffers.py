"""GPU: 8-bit linear calls whose buffers are columns of one allocation."""
import pytest
import torch

from test_gpu_fp8 import DEV, E4M3, TYPES, _rows, _same_codes, _whole_product
from zoomkv_revision_amd import fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(3, 100, 384), (40, 200, 640), (150, 301, 384), (300, 2048, 4096)])
@pytest.mark.parametrize("dtype", TYPES)
def test_output_beside_its_residual(M, N, K, dtype):
    codes, scales, w = _whole_product(M + N, M, N, K)
    both = torch.randint(-9, 10, (M, 2 * N), generator=torch.Generator().manual_seed(M)).to(dtype).to(DEV)
    r = both[:, N:].clone()
    want = fp8.linear(codes, scales, w, residual=r, out_dtype=dtype)
    got = fp8.linear(codes, scales, w, residual=both[:, N:], out=both[:, :N])
    assert torch.equal(got, want) and torch.equal(both[:, N:], r)


@pytest.mark.parametrize("M,K", [(9, 300), (70, 427), (5, 2600), (1003, 129)])
@pytest.mark.parametrize("dtype", TYPES)
def test_sum_beside_its_inputs_and_scales_beside_their_codes(M, K, dtype):
    three = _rows(K, M, 3 * K, dtype).clamp(-1000, 1000).to(DEV)
    x, r, w = three[:, :K].clone(), three[:, K:2 * K].clone(), three[0, :K].clone()
    want = fp8.rms_norm_quant(x, w, 1e-6, residual=r)
    wide, nb = want[0].shape[1], want[1].shape[1]
    record = torch.full((M, wide + 8 * nb), 7, dtype=torch.uint8, device=DEV)        # codes, then scales, of each row
    scales = record.view(torch.float32)[:, wide // 4:wide // 4 + nb]
    got = fp8.rms_norm_quant(three[:, :K], w, 1e-6, residual=three[:, K:2 * K], sum_out=three[:, 2 * K:],
                             codes=record[:, :wide].view(E4M3), scales=scales)
    assert _same_codes(got[0].contiguous(), want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert torch.equal(three[:, :K], x) and torch.equal(three[:, K:2 * K], r) and (record[:, wide + 4 * nb:] == 7).all()
