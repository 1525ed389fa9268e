"""GPU: rows and weights in 8 bits, their products and the gated product.

Quantising alone rounds like IEEE divisions and conversions, so codes and scales
are compared bit by bit.  Products are compared exactly, on whole numbers and scales
that are powers of two whose sums fit 24 bits: a lost, doubled or misplaced element
shows.  Other results are held against 64 bits with the bounds derived in
fp8_cases."""
import math

import pytest
import torch

from fp8_cases import ACT_REL, B, E4M3, NORM_REL, blocks, check_gated, check_linear, check_norm, code_bound, coded, \
    padded, power_scales, scales_of, values, weight_values, whole_codes
from zoomkv_revision_amd import fp8
from zoomkv_revision_amd._lib import ZkvError

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same(a, b):
    """Equal, NaN where NaN is."""
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _same_codes(a, b):
    """Equal codes (those of -0 and 0 alike: a zero's sign is not kept)."""
    return _same(a.cpu().float(), b.cpu().float())


def _rows(seed, M, K, dtype):
    g = _gen(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(2.0 * torch.randn(M, 1, generator=g))
    x[:, ::37] *= 20.0
    return x.to(dtype)


# ---------------------------------------------------------------------------
# rows and weights
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (2, 128), (9, 130), (17, 2560), (5, 2600), (3, 8200), (2, 70001),
                                 (1000, 68), (77, 200), (41, 427), (33, 512), (9, 513)])
def test_quantised_rows_bit_by_bit(dtype, M, K):
    x = _rows(M + K, M, K, dtype)
    codes, scales = fp8.quantize_rows(x.to(DEV))
    want, s = coded(x.float())                  # (1000 rows of fp16 hold an infinity)
    assert _same(scales.cpu(), s)
    assert _same_codes(codes, want)


def test_quantised_rows_at_the_ends_of_the_range():
    """Zeros, the smallest and the largest magnitudes of fp32, ties between codes."""
    tiny = torch.tensor([1e-45, 1e-38, -1e-30, 2.0 ** -100, 448 * 2.0 ** -100, 0.0])
    big = torch.tensor([3.4028e38, -3.0e38, 1.0, 0.0, -0.0, 1e30])
    ties = torch.cat([torch.tensor([448.0, 432.0, 17.0, 19.0, -21.0, 0.0009765625, 0.0029296875])])
    x = torch.zeros(4, 300)
    x[0, 3:9], x[1, 130:136], x[2, 293:300], x[3, 0] = tiny, big, ties, 2.0 ** -99
    codes, scales = fp8.quantize_rows(x.to(DEV))
    want, s = coded(x)
    assert torch.equal(scales.cpu(), s) and _same_codes(codes, want)
    assert torch.equal(scales.cpu()[0, 1:], torch.full((2,), 2.0 ** -100))


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_block_that_is_not_finite_is_nan_and_no_other(value):
    x = _rows(1, 3, 400, torch.bfloat16)
    x[1, 140] = value
    codes, scales = (t.cpu() for t in fp8.quantize_rows(x.to(DEV)))
    v = values(codes, scales)
    assert v[1, 128:256].isnan().all() and codes[1, 128:256].float().isnan().all()
    assert v[0].isfinite().all() and v[2].isfinite().all() and v[1, :128].isfinite().all() and v[1, 256:].isfinite().all()
    weight = torch.randn(5, 400, generator=_gen(2)).to(DEV)
    y = fp8.linear(codes.to(DEV), scales.to(DEV), fp8.quantize_weight(weight)).cpu()
    assert y[1].isnan().all() and y[0].isfinite().all() and y[2].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,residual", [(1, 1, False), (2, 100, True), (5, 128, False), (3, 2560, True),
                                          (33, 2600, True), (4, 8192, False), (3, 10001, True), (2, 30000, True),
                                          (1, 65536, True), (1000, 68, False), (70, 200, True), (37, 427, True),
                                          (33, 512, True), (9, 513, True), (1, 7405, True)])
def test_normed_rows(dtype, M, K, residual):
    x, w = _rows(M + K, M, K, dtype), (1 + torch.randn(K, generator=_gen(K))).to(dtype)
    r = _rows(M + K + 1, M, K, dtype) if residual else None
    x, w, r = (None if t is None else t.to(DEV) for t in (x, w, r))
    got = fp8.rms_norm_quant(x, w, 1e-5, residual=r)
    check_norm(x, w, 1e-5, r, *got)
    assert ((got[0].float()[:, K:] == 0) | got[1][:, -1:].isnan()).all()     # (a NaN block: all of it)


def test_normed_rows_of_zeros_and_of_one_infinity():
    x = torch.zeros(3, 256, device=DEV)
    x[1, 5] = float("inf")
    x[2] = 1e-30
    codes, scales = fp8.rms_norm_quant(x, torch.ones(256, device=DEV), 1e-6)
    assert (codes[0].float() == 0).all() and torch.equal(scales[0].cpu(), torch.full((2,), 2.0 ** -100))
    assert scales[1, 0].isnan()
    want = 1e-30 * 1e3
    assert ((values(codes, scales)[2] - want).abs() <= want * (2.0 ** -4 + 2 * NORM_REL)).all()


@pytest.mark.parametrize("K", [100, 201, 427, 2600])
@pytest.mark.parametrize("which", ["x", "residual"])
def test_the_sum_in_place(which, K):
    x, r, w = (_rows(i, 7, K, torch.bfloat16).to(DEV) for i in (1, 2, 3))
    w = w[0].contiguous()
    want = fp8.rms_norm_quant(x, w, 1e-6, residual=r)
    a, b = x.clone(), r.clone()
    got = fp8.rms_norm_quant(a, w, 1e-6, residual=b, sum_out=a if which == "x" else b)
    assert got[2].data_ptr() == (a if which == "x" else b).data_ptr()
    assert _same_codes(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert torch.equal(b if which == "x" else a, r if which == "x" else x)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_other_strides_and_offsets(dtype):
    """Views of wider buffers, rows that start on two bytes, scales by rows; what
    lies between the rows stays."""
    M, K = 9, 300
    for offset, ld in ((0, 512), (8, 304), (1, 301), (3, 1000)):
        buf = _rows(offset, M, ld + 8, dtype).to(DEV).view(-1)
        x = buf.as_strided((M, K), (ld, 1), offset)
        place = torch.full((M, 640), 7, dtype=torch.uint8, device=DEV).view(E4M3)
        codes, scales = place[:, 128:512], torch.full((M, 5), -1.0, device=DEV)[:, 1:4]
        fp8.quantize_rows(x, codes, scales)
        want, s = coded(x.float().cpu())
        assert _same_codes(codes.contiguous(), want) and torch.equal(scales.cpu(), s)
        raw = place.view(torch.uint8)
        assert (raw[:, :128] == 7).all() and (raw[:, 512:] == 7).all()
        w = buf.as_strided((K,), (1,), offset)
        total = torch.zeros(M, K + 5, dtype=dtype, device=DEV)
        got = fp8.rms_norm_quant(x, w, 1e-6, residual=x, sum_out=total[:, 2:K + 2])
        ref = fp8.rms_norm_quant(x.contiguous(), w.clone(), 1e-6, residual=x.clone())
        assert _same_codes(got[0], ref[0]) and torch.equal(got[1], ref[1]) and torch.equal(got[2], ref[2])
        assert (total[:, :2] == 0).all() and (total[:, K + 2:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,parts", [(1, 1, 1), (128, 128, 1), (300, 200, 1), (1000, 2600, 2), (2, 130, 2),
                                       (390, 257, 3)])
def test_quantised_weights_bit_by_bit(dtype, N, K, parts):
    w = _rows(N + K, N, K, dtype)
    W = fp8.quantize_weight(w.to(DEV), parts)
    n = N // parts
    for p in range(parts):
        x = padded(w[p * n:(p + 1) * n].float())
        x = torch.nn.functional.pad(x, (0, 0, 0, -n % B)).view(blocks(n), B, blocks(K), B)
        amax = x.abs().amax((1, 3))
        s = torch.maximum(amax / torch.full_like(amax, 448.0), torch.full_like(amax, 2.0 ** -100))
        codes = (x / s[:, None, :, None]).view(-1, blocks(K) * B)[:n].to(E4M3)
        assert torch.equal(W.scales.cpu()[p * blocks(n):(p + 1) * blocks(n)], s)
        assert _same_codes(W.codes[p * n:(p + 1) * n], codes)
    assert torch.equal(W.dequantize(), weight_values(W.codes, W.scales, parts).float())


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _whole_product(seed, M, N, K, parts=1):
    """(codes, scales, weight) of whole numbers and powers of two."""
    g = _gen(seed)
    codes, w = whole_codes(g, M, K), whole_codes(g, parts * N, K)
    scales, ws = power_scales(g, (M, blocks(K))), power_scales(g, (parts * blocks(N), blocks(K)))
    return codes.to(DEV), scales.to(DEV), fp8.Fp8Weight(w.to(DEV), ws.to(DEV), parts)


def _product(codes, scales, weight):
    return values(codes, scales) @ weight_values(weight.codes, weight.scales, weight.parts).t()


SIZES = [(1, 1, 1), (1, 16, 128), (2, 7, 130), (4, 384, 2560), (5, 100, 384), (16, 130, 1000), (17, 24, 256),
         (33, 257, 640), (48, 72, 9728), (64, 200, 2600), (65, 64, 128), (66, 1, 256), (127, 129, 384),
         (128, 256, 1152), (129, 300, 640), (200, 1000, 2600), (257, 513, 16384), (600, 2560, 640), (1100, 80, 256),
         # sizes at which each of the kernels is chosen, with k whole and in runs, as linear and as gated product
         (2376, 2390, 600), (971, 2482, 300), (129, 7420, 700), (66, 5164, 69), (67, 6274, 2960), (39, 7542, 1835),
         (33, 5894, 1093), (65, 4787, 1262), (37, 4675, 336), (38, 5186, 649), (19, 300, 4518), (700, 2235, 600),
         (67, 5539, 4103), (454, 3494, 130), (34, 3588, 9044), (38, 38, 15934), (67, 7803, 357), (18, 1813, 9498),
         (194, 4874, 1095), (78, 5919, 6368), (67, 5553, 67), (34, 65, 16047), (7, 333, 5000), (13, 200, 6000), (30, 40, 16384),
         (3, 100, 16000), (12, 60, 14000), (37, 2704, 12343), (33, 6774, 8170), (915, 1194, 4974), (2730, 69, 2190)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_products_of_whole_numbers_are_exact(M, N, K):
    """|sum| <= 16 * 2^4 * K <= 2^22 in steps of 2^-4 for K of a few blocks, and
    far below that on random signs: every partial sum is exact in fp32."""
    codes, scales, w = _whole_product(M + N + K, M, N, K)
    want = _product(codes, scales, w)
    mass = values(codes, scales).abs() @ weight_values(w.codes, w.scales).abs().t()
    assert float(mass.max()) < 2.0 ** 20                       # in steps of 2^-4: 24 bits
    got = fp8.linear(codes, scales, w, out_dtype=torch.float32)
    assert torch.equal(got.double(), want)
    for dtype in (torch.bfloat16, torch.float16):
        got = fp8.linear(codes, scales, w, out_dtype=dtype)
        assert torch.equal(got, want.float().to(dtype))
    r = torch.randint(-9, 10, (M, N), generator=_gen(M)).float().to(DEV)
    got = fp8.linear(codes, scales, w, residual=r, out=torch.empty_like(r))
    assert torch.equal(got.double(), want + r)


@pytest.mark.parametrize("M,N,K", [(1, 64, 256), (16, 40, 384), (100, 300, 384), (300, 64, 256)])
def test_small_terms_beside_large_ones_that_cancel(M, N, K):
    """448 - 448 + 2^-6 within 8 neighbouring places: the small term is 15 bits
    below the large ones, so the sum is exact in fp32 in any order, and would be 0
    or 2^-5 where terms are cut 14 bits below the largest."""
    g = _gen(M)
    codes, w = torch.zeros(M, padded(torch.zeros(1, K)).shape[1]), torch.zeros(N, padded(torch.zeros(1, K)).shape[1])
    w[:, :K] = 1.0
    want = torch.zeros(M, dtype=torch.float64)
    for m in range(M):
        at = int(torch.randint(0, K // 8, (1,), generator=g)) * 8
        i, j, k = (at + torch.randperm(8, generator=g)[:3]).tolist()
        codes[m, i], codes[m, j], codes[m, k] = 448.0, -448.0, 0.015625
        want[m] = 0.015625
    one = lambda r, c: torch.ones(r, c, device=DEV)
    got = fp8.linear(codes.to(E4M3).to(DEV), one(M, blocks(K)),
                     fp8.Fp8Weight(w.to(E4M3).to(DEV), one(blocks(N), blocks(K))), out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want[:, None].expand(M, N))


@pytest.mark.parametrize("M,N,K", [(1, 640, 2560), (16, 256, 9728), (40, 77, 16384), (333, 1000, 2600),
                                   (512, 256, 9728)])
@pytest.mark.parametrize("dtype", TYPES)
def test_products_of_random_rows(M, N, K, dtype):
    g = _gen(M + N)
    x = torch.randn(M, K, generator=g) * torch.exp(0.5 * torch.randn(M, 1, generator=g))
    codes, scales = (t.to(DEV) for t in coded(x))
    w = fp8.quantize_weight((0.05 * torch.randn(N, K, generator=g)).to(DEV))
    r = torch.randn(M, N, generator=g).to(dtype).to(DEV)
    got = fp8.linear(codes, scales, w, residual=r, out_dtype=dtype)
    check_linear(codes, scales, w, r, got)
    want = _product(codes, scales, w) + r.double()
    # typical sums are far nearer: 2^-24 per rounding, not all of one sign
    if dtype == torch.float32:
        assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -21


def _act(weight, codes, scales):
    """float64 silu(gate) * up, whole blocks."""
    gate, up = _product(codes, scales, weight).chunk(2, 1)
    return padded(gate / (1 + torch.exp(-gate)) * up)


@pytest.mark.parametrize("M,F,K", SIZES)
def test_gated_products_of_whole_numbers(M, F, K):
    codes, scales, w = _whole_product(M + F + K, M, F, K, parts=2)
    w.scales.mul_(2.0 ** -6)                                      # gates of a few units, exact
    y = _act(w, codes, scales)
    got, s = fp8.gated_linear(codes, scales, w)
    want = scales_of(y)
    assert ((s.double() - want).abs() <= ACT_REL * want).all()
    assert ((values(got, s) - y).abs() <= code_bound(y, want, ACT_REL) + 1e-36).all()
    assert (got.float()[:, F:] == 0).all()


def test_gates_far_from_zero():
    """silu of very negative gates is 0 and of large ones the gate; no NaN from
    an exponential that overflows."""
    K, F = 128, 4
    codes = torch.zeros(1, K)
    codes[0, 0] = 1.0
    w = torch.zeros(2 * F, K)
    w[:F, 0] = torch.tensor([-448.0, 448.0, -1.0, 0.0])
    w[F:, 0] = 2.0
    got, s = fp8.gated_linear(codes.to(E4M3).to(DEV), torch.ones(1, 1, device=DEV),
                              fp8.Fp8Weight(w.to(E4M3).to(DEV), torch.ones(2, 1, device=DEV), parts=2))
    v = values(got, s)[0, :F].tolist()
    assert v[0] == 0 and v[1] == 896 and v[3] == 0
    assert abs(v[2] + 2 / (1 + math.e)) <= 2 / (1 + math.e) * 2.0 ** -4 + 2 * 2.0 ** -10


@pytest.mark.parametrize("M,N,K", [(3, 100, 384), (40, 200, 640), (150, 300, 384), (257, 513, 16384), (971, 2482, 300),
                                   (2376, 2390, 600)])
def test_products_of_other_strides(M, N, K):
    """Rows, scales, outputs and residuals as views of wider buffers; what lies
    between them stays."""
    codes, scales, w = _whole_product(M, M, N, K)
    want = fp8.linear(codes, scales, w, out_dtype=torch.float32)
    wide = torch.full((M, codes.shape[1] + 256), 0x7F, dtype=torch.uint8, device=DEV).view(E4M3)
    wide[:, 128:-128].view(torch.uint8).copy_(codes.view(torch.uint8))
    ww = torch.full((N, codes.shape[1] + 16), 0x7F, dtype=torch.uint8, device=DEV).view(E4M3)
    ww[:, :-16].view(torch.uint8).copy_(w.codes.view(torch.uint8))
    by_rows = torch.full((M, scales.shape[1] + 3), float("nan"), device=DEV)
    by_rows[:, 1:-2] = scales
    columns = scales.t().contiguous().t()
    for dtype in TYPES:
        for pad in (1, 3, 4):
            out = torch.full((M, N + 2 * pad), 5.0, dtype=dtype, device=DEV)
            got = fp8.linear(wide[:, 128:-128], by_rows[:, 1:-2], fp8.Fp8Weight(ww[:, :-16], w.scales),
                             out=out[:, pad:-pad])
            assert torch.equal(got, want.to(dtype))
            assert (out[:, :pad] == 5).all() and (out[:, -pad:] == 5).all()
            r = torch.full((M, N + pad), 1.0, dtype=dtype, device=DEV)
            got = fp8.linear(codes, columns, w, out=out[:, pad:-pad], residual=r[:, pad:])
            assert torch.equal(got, (want + 1).to(dtype))
    r = torch.full((M, N), 2.0, device=DEV)
    assert fp8.linear(codes, scales, w, out=r, residual=r) is r and torch.equal(r, want + 2)
    # one scale for all blocks of a row
    one = torch.ones(M, 1, device=DEV).expand(M, scales.shape[1])
    assert torch.equal(fp8.linear(codes, one, w), fp8.linear(codes, one.contiguous(), w))


@pytest.mark.parametrize("M,F,K", [(70, 200, 384), (300, 2048, 4096), (700, 2235, 600)])
def test_gated_products_of_other_strides(M, F, K):
    codes, scales, w = _whole_product(3, M, F, K, parts=2)
    wide = blocks(F) * B
    for m in (5, M):
        want = fp8.gated_linear(codes[:m], scales[:m], w)
        place = torch.full((m, wide + 256), 7, dtype=torch.uint8, device=DEV).view(E4M3)
        s = torch.full((m, blocks(F) + 2), -1.0, device=DEV)
        got = fp8.gated_linear(codes[:m], scales[:m], w, out_codes=place[:, 128:-128], out_scales=s[:, 1:-1])
        assert _same_codes(got[0].contiguous(), want[0]) and torch.equal(got[1], want[1])
        raw = place.view(torch.uint8)
        assert (raw[:, :128] == 7).all() and (raw[:, -128:] == 7).all() and (s[:, 0] == -1).all() and (s[:, -1] == -1).all()


def test_no_rows():
    w = fp8.quantize_weight(torch.randn(40, 200, device=DEV))
    codes, scales = fp8.quantize_rows(torch.empty(0, 200, device=DEV))
    assert codes.shape == (0, 256) and scales.shape == (0, 2)
    got = fp8.rms_norm_quant(torch.empty(0, 200, device=DEV), torch.ones(200, device=DEV), 1e-6,
                             residual=torch.empty(0, 200, device=DEV))
    assert got[2].shape == (0, 200)
    assert fp8.linear(codes, scales, w).shape == (0, 40)
    w.parts, w.scales = 2, w.scales.repeat(2, 1)
    assert fp8.gated_linear(codes, scales, w)[0].shape == (0, 128)


def test_refused_by_the_library():
    """What the C entries refuse before a launch."""
    codes, scales, w = _whole_product(1, 4, 32, 256, parts=2)
    with pytest.raises(ValueError, match="workspace"):
        fp8.gated_linear(codes, scales, w, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    from zoomkv_revision_amd._lib import check, lib, ptr
    L = lib()
    args = lambda K, x: (x, 256, ptr(scales), 2, 1, ptr(w.codes), 256, ptr(w.scales), 4, 16, K, None, 0,
                         ptr(torch.empty(4, 16, device=DEV)), 16, 2, None, 0, 0)
    for K, x in ((200, ptr(codes)), (0, ptr(codes)), (256, None), (256, ptr(codes) + 8), (512, ptr(codes))):
        with pytest.raises(ZkvError):
            check(L.zkv_fp8_linear(*args(K, x)))
    with pytest.raises(ZkvError):
        check(L.zkv_fp8_gated_linear(ptr(codes), 256, ptr(scales), 2, 1, ptr(w.codes), 256, ptr(w.scales), 4, 16, 256,
                                     ptr(codes), 256, ptr(scales), 2, 1, ptr(codes), 8, 0))


# ---------------------------------------------------------------------------
# streams, graphs, large offsets
# ---------------------------------------------------------------------------
def _block(x, r, norm, gate_up, down):
    """A gated feed-forward block on a residual stream."""
    codes, scales, h = fp8.rms_norm_quant(x, norm, 1e-6, residual=r)
    act, act_scales = fp8.gated_linear(codes, scales, gate_up)
    return fp8.linear(act, act_scales, down, residual=h)


def _block_inputs(M, K=384, F=320, seed=1):
    g = _gen(seed)
    x, r = (torch.randn(M, K, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    norm = torch.ones(K, dtype=torch.bfloat16, device=DEV)
    gate_up = fp8.quantize_weight((0.1 * torch.randn(2 * F, K, generator=g)).to(DEV), parts=2)
    down = fp8.quantize_weight((0.1 * torch.randn(K, F, generator=g)).to(DEV))
    return x, r, norm, gate_up, down


@pytest.mark.parametrize("M", [1, 4, 16, 50, 65, 200])
def test_a_feed_forward_block_against_64_bits(M):
    """Each operator on what the one before left (its codes and scales as they
    are), so that every bound is one operator's own."""
    x, r, norm, gate_up, down = _block_inputs(M)
    codes, scales, h = fp8.rms_norm_quant(x, norm, 1e-6, residual=r)
    check_norm(x, norm, 1e-6, r, codes, scales, h)
    act, act_scales = fp8.gated_linear(codes, scales, gate_up)
    check_gated(codes, scales, gate_up, act, act_scales)
    out = fp8.linear(act, act_scales, down, residual=h)
    check_linear(act, act_scales, down, h, out)
    assert torch.equal(out, _block(x, r, norm, gate_up, down))


@pytest.mark.parametrize("M", [4, 50, 200])
def test_on_another_stream_and_in_two_at_once(M):
    inputs = [_block_inputs(M, seed=s) for s in (1, 2)]
    want = [_block(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_block(*inputs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("M", [1, 16, 50, 200])
def test_captured_and_replayed(M):
    """Two graphs of a block, replayed in turn with eager calls between, on new
    inputs: every replay is the eager result."""
    x, r, norm, gate_up, down = _block_inputs(M)
    _block(x, r, norm, gate_up, down)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_block(x, r, norm, gate_up, down))
        graphs.append(g)
    for i in range(6):
        x.copy_(_rows(i, M, x.shape[1], torch.bfloat16).clamp(-100, 100))
        want = _block(x, r, norm, gate_up, down)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want)


@pytest.mark.parametrize("M,F,K", [(257, 513, 16384), (300, 2048, 4096), (700, 2235, 600), (4, 1000, 6000)])
def test_larger_products_at_once_and_replayed(M, F, K):
    """Tiles, and runs of k in a workspace, on two streams and in two graphs at once."""
    codes, scales, w = _whole_product(M, M, F, K, parts=2)
    one = fp8.Fp8Weight(w.codes[:F], w.scales[:blocks(F)])
    both = lambda: (*fp8.gated_linear(codes, scales, w), fp8.linear(codes, scales, one, out_dtype=torch.float32))
    want = [t.clone() for t in both()]
    same = lambda got: _same_codes(got[0], want[0]) and all(torch.equal(g, t) for g, t in zip(got[1:], want[1:]))
    streams, graphs, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both())
        graphs.append(g)
    for _ in range(4):
        got = []
        for o in outs:
            for t in o:
                (t.view(torch.uint8) if t.dtype == E4M3 else t).zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
                got.append(both())
        torch.cuda.synchronize()
        assert all(same(g) for g in got) and all(same(o) for o in outs)


@pytest.mark.parametrize("M", [3, 100])
def test_plans_over_fixed_buffers(M):
    x, r, norm, gate_up, down = _block_inputs(M)
    a = fp8.RmsNormQuantPlan(x, norm, 1e-6, residual=r)
    b = fp8.GatedLinearPlan(a.out[0], a.out[1], gate_up)
    c = fp8.LinearPlan(*b.out, down, residual=a.out[2])
    for i in range(3):
        x.copy_(_rows(i, M, x.shape[1], torch.bfloat16).clamp(-100, 100))
        a.run(), b.run()
        assert torch.equal(c.run(), _block(x, r, norm, gate_up, down))


def test_offsets_beyond_31_bits():
    """Weights, rows and outputs of more than 2^31 elements."""
    N, K = 140000, 16384
    w = torch.zeros(N, K, dtype=torch.uint8, device=DEV).view(E4M3)
    ws = torch.ones(blocks(N), K // B, device=DEV)
    for n in (0, 131072, N - 1):
        w[n].fill_(1.0)
    for M in (2, 70):
        codes, scales = torch.ones(M, K, device=DEV).to(E4M3), torch.ones(M, K // B, device=DEV)
        y = fp8.linear(codes, scales, fp8.Fp8Weight(w, ws), out_dtype=torch.float32)
        assert (y[:, [0, 131072, N - 1]] == K).all() and int((y != 0).sum()) == 3 * M
        # the same memory as rows of x
        x = fp8.linear(w, torch.ones(N, 1, device=DEV).expand(N, K // B),
                       fp8.Fp8Weight(codes, torch.ones(blocks(M), K // B, device=DEV)), out_dtype=torch.float32)
        assert (x[[0, 131072, N - 1]] == K).all() and int((x != 0).sum()) == 3 * M
    del w, y, x
    M, N = 70000, 32000
    codes, scales = torch.ones(M, B, device=DEV).to(E4M3), torch.ones(M, 1, device=DEV)
    scales[:, 0] = torch.arange(M, device=DEV) % 7
    w = torch.ones(N, B, device=DEV).to(E4M3)
    y = fp8.linear(codes, scales, fp8.Fp8Weight(w, torch.ones(blocks(N), 1, device=DEV)))
    want = (128.0 * scales).to(torch.bfloat16)
    assert all(torch.equal(y[i:i + 7000], want[i:i + 7000].expand(-1, N)) for i in range(0, M, 7000))
