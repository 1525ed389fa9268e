"""GPU: a gated product at its limit of 2^37 outputs, whose tiles need more threads
than one launch holds.  Rows and blocks of outputs repeat a small product, of whole
numbers and so exact whichever kernel computes it."""
import pytest
import torch

from test_gpu_fp8 import DEV, E4M3, _whole_product
from zoomkv_revision_amd import fp8

pytestmark = pytest.mark.gpu


def test_two_to_the_37th_gated_outputs():
    M, F, P, Q = 1 << 18, 1 << 19, 1009, 5
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("needs 160 GiB of free device memory")
    codes, scales, w = _whole_product(7, P, Q * 128, 128, parts=2)
    w.scales.mul_(2.0 ** -6)
    small, s = (t.contiguous() for t in fp8.gated_linear(codes, scales, w))
    row, block = torch.arange(M, device=DEV) % P, torch.arange(F // 128, device=DEV) % Q
    big = w.codes.view(torch.uint8).view(2, Q, 128, 128)[:, block].reshape(2 * F, 128).view(E4M3)
    got = fp8.gated_linear(codes.view(torch.uint8)[row].view(E4M3), scales[row],
                           fp8.Fp8Weight(big, w.scales.view(2, Q, 1)[:, block].reshape(-1, 1), parts=2))
    assert got[0].shape == (M, F) and s.isfinite().all()
    for i in range(0, M, 1 << 13):
        at = row[i:i + (1 << 13)]
        blocks = got[0][i:i + (1 << 13)].view(torch.uint8).view(len(at), -1, 128)
        want = small.view(torch.uint8)[at].view(len(at), Q, 128)
        assert all(bool((blocks[:, q::Q] == want[:, q:q + 1]).all()) for q in range(Q))
        assert torch.equal(got[1][i:i + (1 << 13)], s[at][:, block])
    del got, blocks
    torch.cuda.empty_cache()
