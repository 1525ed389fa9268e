"""GPU: 8-bit products at a size for each kernel and number of runs of k: exact for
linear products of whole numbers; for gated ones each code is the one of the 64-bit
value, or the next where that value lies next to the border of two."""
import pytest
import torch

from fp8_cases import ACT_REL, B, E4M3, blocks, padded, scales_of, values, weight_values
from fp8_sizes import CASES
from zoomkv_revision_amd import fp8

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _codes(g, rows, K):
    return padded(torch.randint(-4, 5, (rows, K), generator=g, device=DEV, dtype=torch.int8).float()).to(E4M3)


def _scales(g, *shape):
    return torch.exp2(torch.randint(-2, 3, shape, generator=g, device=DEV).float())


def _operands(parts, M, N, K):
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    codes, scales = _codes(g, M, K), _scales(g, M, blocks(K))
    return g, codes, scales, fp8.Fp8Weight(_codes(g, parts * N, K), _scales(g, parts * blocks(N), blocks(K)), parts)


def _product(codes, scales, w):
    """(the product in 64 bits, the largest sum of magnitudes)."""
    x, v = values(codes, scales), weight_values(w.codes, w.scales, w.parts)
    return x @ v.t(), float((x.abs() @ v.abs().t()).max())


@pytest.mark.parametrize("kernel,runs,M,N,K", [c[1:] for c in CASES if c[0] == 1])
def test_linear(kernel, runs, M, N, K):
    g, codes, scales, w = _operands(1, M, N, K)
    want, mass = _product(codes, scales, w)
    assert mass < 2.0 ** 20                                    # in steps of 2^-4: 24 bits
    assert torch.equal(fp8.linear(codes, scales, w, out_dtype=torch.float32).double(), want)
    r = torch.randint(-9, 10, (M, N), generator=g, device=DEV).float()
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        got = fp8.linear(codes, scales, w, residual=r.to(dtype), out_dtype=dtype)
        assert torch.equal(got, (want + r).float().to(dtype))


@pytest.mark.parametrize("kernel,runs,M,F,K", [c[1:] for c in CASES if c[0] == 2])
def test_gated(kernel, runs, M, F, K):
    """Gates and ups are exact.  A value is off by ACT_REL of itself and its block's scale
    by as much, and their quotient is rounded once (2^-24): its code lies between those
    of the exact quotient made smaller and larger by that."""
    _, codes, scales, w = _operands(2, M, F, K)
    w.scales.mul_(2.0 ** -6)                                      # gates of a few units, exact
    product, mass = _product(codes, scales, w)
    assert mass < 2.0 ** 14
    gate, up = product.chunk(2, 1)
    y = padded(gate / (1 + torch.exp(-gate)) * up)
    got, s = fp8.gated_linear(codes, scales, w)
    want = scales_of(y)
    assert ((s.double() - want).abs() <= ACT_REL * want).all()
    q, rel = y / want.repeat_interleave(B, 1), 2 * ACT_REL + 2.0 ** -23
    low, high = ((q - q.abs() * rel * sign).float().to(E4M3).float() for sign in (1, -1))
    assert ((got.float() >= low) & (got.float() <= high)).all()
    assert int((low != high).sum()) <= 0.01 * low.numel() + 2      # (few values lie so near a border: 2 rel of 2^-4)
    assert (got.float()[:, F:] == 0).all()
