"""CPU: the decode step's 8-bit projections in torch ops, and the step with them."""
import pytest
import torch

from fp8_cases import B, blocks, coded, power_scales, scales_of, values, weight_values, whole_codes
from test_decode_step import TINY, DenseCache
from zoomkv_revision_amd import decode_step as ds
from zoomkv_revision_amd.fp8 import Fp8Weight


@pytest.mark.parametrize("M,K", [(1, 1), (3, 130), (4, 384), (2, 1000)])
def test_rows_and_weights_as_the_kernels_quantise_them(M, K):
    g = torch.Generator().manual_seed(K)
    x = torch.randn(M, K, generator=g)
    codes, scale = ds.quantize_rows_torch(x)
    want, s = coded(x)
    assert torch.equal(codes.float(), want.float()) and torch.equal(scale, s)
    w = torch.randn(2 * 150, K, generator=g).to(torch.bfloat16)
    W = ds.quantize_weight_torch(w, parts=2)
    assert W.codes.shape == (300, blocks(K) * B) and W.scales.shape == (4, blocks(K))
    off = (W.dequantize()[:, :K] - w.float()).abs()
    step = W.scales.view(2, 2, -1).repeat_interleave(B, 1)[:, :150].reshape(300, -1).repeat_interleave(B, 1)[:, :K]
    assert (off <= w.float().abs() * (2.0 ** -4 + 2.0 ** -20) + step * 2.0 ** -10).all()


def test_a_product_of_whole_numbers():
    g = torch.Generator().manual_seed(5)
    codes = whole_codes(g, 40, 300)
    w = Fp8Weight(codes, power_scales(g, (1, 3)))
    x = torch.randint(-4, 5, (7, 300), generator=g).float()
    x[:, 0], x[:, 128], x[:, 256] = 7.0, 7.0, 7.0                 # scales of 1 / 64: codes are whole
    c, s = coded(x)
    assert torch.equal(s, torch.full_like(s, 1 / 64)) and torch.equal(values(c, s)[:, :300], x.double())
    want = values(c, s) @ weight_values(w.codes, w.scales).T
    assert torch.equal(ds.linear_fp8_torch(x, w).double(), want)


def test_the_step_with_8_bit_weights():
    """Same seed, same weights but for their rounding: the 8-bit step is the bf16
    one with every product's operands off by 2^-4 at most, and nothing else."""
    tok = torch.tensor([1, 7])
    logits = {}
    for weights in ("bf16", "fp8"):
        m = ds.RandomQwen3(TINY, "cpu", seed=3, max_position=64, weights=weights)
        cache = DenseCache(TINY.layers, 2, TINY.kv_heads)
        logits[weights] = [m.decode_step(tok, cache) for _ in range(3)]
        assert cache.context == 3
    small = ds.RandomQwen3(TINY, "cpu", seed=3, max_position=64, weights="fp8")
    L = small.layers[0]
    assert isinstance(L["gate_up"], Fp8Weight) and L["gate_up"].parts == 2
    full = ds.RandomQwen3(TINY, "cpu", seed=3, max_position=64)
    for name in ("wqkv", "wo", "gate_up", "down"):
        w, W = full.layers[1][name].float(), small.layers[1][name]
        assert ((W.dequantize()[:, :w.shape[1]] - w).abs() <= w.abs() * 2.0 ** -4 * 1.001 + 0.02 * 5 / 448 * 2.0 ** -9).all()
    assert small.parameter_bytes() < full.parameter_bytes()
    for a, b in zip(logits["bf16"], logits["fp8"]):
        assert torch.isfinite(b).all() and not torch.equal(a, b)


def test_rows_of_a_step_do_not_depend_on_their_neighbours():
    m = ds.RandomQwen3(TINY, "cpu", seed=4, max_position=64, weights="fp8")
    both = m.decode_step(torch.tensor([3, 9]), DenseCache(TINY.layers, 2, TINY.kv_heads))
    for r, t in enumerate((3, 9)):
        alone = m.decode_step(torch.tensor([t]), DenseCache(TINY.layers, 1, TINY.kv_heads))
        assert torch.allclose(alone[0], both[r], atol=8 * 2.0 ** -7 * float(both[r].abs().max()))


def test_other_weights_are_refused():
    with pytest.raises(ValueError, match="bf16 or fp8"):
        ds.RandomQwen3(TINY, "cpu", weights="int8")


def test_scales_of_zeros():
    assert torch.equal(scales_of(torch.zeros(2, 130)), torch.full((2, 2), 2.0 ** -100))
    codes, scale = ds.quantize_rows_torch(torch.zeros(2, 130))
    assert torch.equal(scale, torch.full((2, 2), 2.0 ** -100)) and not codes.float().any()
