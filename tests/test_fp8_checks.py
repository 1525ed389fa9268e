"""What the 8-bit linear calls refuse before any launch (host checks only, on CPU
tensors: the last check is that they are on the GPU)."""
import ctypes

import pytest
import torch

from fp8_cases import E4M3
from zoomkv_revision_amd import fp8
from zoomkv_revision_amd._lib import SIGNATURES, ZkvError, lib, packed_args

BF = torch.bfloat16
M, N, K = 3, 40, 200


def _codes(rows, wide=256):
    return torch.zeros(rows, wide, dtype=torch.uint8).view(E4M3)


def _norm(**changed):
    return {**dict(x=torch.zeros(M, K, dtype=BF), weight=torch.ones(K, dtype=BF), eps=1e-6,
                   residual=torch.zeros(M, K, dtype=BF)), **changed}


def _rows(**changed):
    return {**dict(x=torch.zeros(M, K, dtype=BF)), **changed}


def _weight(**changed):
    return fp8.Fp8Weight(**{**dict(codes=_codes(N), scales=torch.ones(1, 2), parts=1), **changed})


def _linear(**changed):
    return {**dict(codes=_codes(M), scales=torch.ones(M, 2), weight=_weight()), **changed}


def _gated(**changed):
    return {**dict(codes=_codes(M), scales=torch.ones(M, 2),
                   weight=_weight(scales=torch.ones(2, 2), parts=2)), **changed}


CALLS = [(fp8.rms_norm_quant, _norm), (fp8.RmsNormQuantPlan, _norm), (fp8.quantize_rows, _rows),
         (fp8.QuantizeRowsPlan, _rows), (fp8.linear, _linear), (fp8.LinearPlan, _linear), (fp8.gated_linear, _gated),
         (fp8.GatedLinearPlan, _gated), (fp8.quantize_weight, lambda **c: {**dict(w=torch.zeros(N, K)), **c})]


@pytest.mark.parametrize("call,args", CALLS)
def test_matching_buffers_pass_the_host_checks(call, args):
    with pytest.raises(ZkvError, match="device tensors"):
        call(**args())


@pytest.mark.parametrize("changed,text", [
    (dict(x=torch.zeros(M, K, dtype=torch.float64)), "bfloat16, float16 or float32"),
    (dict(x=torch.zeros(K, dtype=BF)), r"\[rows, channels\]"),
    (dict(x=torch.zeros(M, 0, dtype=BF)), r"\[rows, channels\]"),
    (dict(x=torch.zeros(K, M, dtype=BF).t()), "contiguous and apart"),
    (dict(x=torch.zeros(1, K, dtype=BF).expand(M, K)), "contiguous and apart"),
    (dict(weight=None), "needs its weight"),
    (dict(weight=torch.ones(K)), "norm's weight"),
    (dict(weight=torch.ones(K + 1, dtype=BF)), "norm's weight"),
    (dict(residual=torch.zeros(M, K)), "residual must be"),
    (dict(residual=torch.zeros(M, K + 1, dtype=BF)), "residual must be"),
    (dict(residual=None, sum_out=torch.zeros(M, K, dtype=BF)), "goes with a residual"),
    (dict(sum_out=torch.zeros(M, K)), "sum_out must be"),
    (dict(codes=torch.zeros(M, 256, dtype=torch.uint8)), "float8_e4m3fn"),
    (dict(codes=_codes(M, K + 8)), "codes must be"),
    (dict(codes=_codes(M, 260)[:, 1:257]), "start on 8 bytes"),
    (dict(scales=torch.zeros(M, 1)), "scales must be"),
    (dict(scales=torch.zeros(M, 2, dtype=BF)), "scales must be"),
    (dict(scales=torch.zeros(M, 1).expand(M, 2)), "a place for every scale"),
])
def test_norm_refusals(changed, text):
    with pytest.raises((ValueError, TypeError), match=text):
        fp8.rms_norm_quant(**_norm(**changed))


def test_a_sum_that_overlaps_its_inputs_is_refused():
    buf = torch.zeros((M + 1) * K, dtype=BF)
    x, shifted = buf[:M * K].view(M, K), buf[8:8 + M * K].view(M, K)
    with pytest.raises(ValueError, match="x itself or lie apart"):
        fp8.rms_norm_quant(**_norm(x=x, sum_out=shifted))
    with pytest.raises(ValueError, match="residual itself or lie apart"):
        fp8.rms_norm_quant(**_norm(residual=x, sum_out=shifted))
    with pytest.raises(ZkvError, match="device tensors"):
        fp8.rms_norm_quant(**_norm(x=x, sum_out=x))


def test_rows_that_are_too_long():
    long = torch.zeros(1, fp8.MAX_NORM_K + 1, dtype=BF)
    with pytest.raises(ValueError, match="at most 65536"):
        fp8.rms_norm_quant(long, long[0], 1e-6)
    wide = fp8.MAX_K + 128
    with pytest.raises(ValueError, match="at most 16384"):
        fp8.linear(_codes(1, wide), torch.ones(1, wide // 128), fp8.Fp8Weight(_codes(4, wide), torch.ones(1, wide // 128)))


@pytest.mark.parametrize("changed,text", [
    (dict(codes=torch.zeros(M, 256, dtype=torch.uint8)), "float8_e4m3fn"),
    (dict(codes=_codes(M, 384)), "one length"),
    (dict(codes=_codes(M, 200), weight=_weight(codes=_codes(N, 200))), "one length"),
    (dict(codes=_codes(M, 272)[:, 8:264]), "start on 16 bytes"),
    (dict(codes=_codes(1).expand(M, 256)), "contiguous and apart"),
    (dict(scales=torch.ones(M, 3)), "scales must be"),
    (dict(scales=torch.ones(M, 2, dtype=torch.float64)), "scales must be"),
    (dict(weight=_weight(parts=2, scales=torch.ones(2, 2))), r"2 part\(s\), not 1"),
    (dict(weight=_weight(scales=torch.ones(2, 2))), "the weight's scales"),
    (dict(weight=_weight(scales=torch.ones(1, 4)[:, ::2])), "the weight's scales"),
    (dict(weight=_weight(codes=torch.zeros(N, 256))), "float8_e4m3fn"),
    (dict(out_dtype=torch.float64), "out_dtype"),
    (dict(out=torch.zeros(M, N + 1)), "out must be"),
    (dict(out=torch.zeros(N, M).t()), "contiguous and apart"),
    (dict(residual=torch.zeros(M, N)), "residual must be"),
    (dict(residual=torch.zeros(N, dtype=BF)), "residual must be"),
])
def test_linear_refusals(changed, text):
    with pytest.raises((ValueError, TypeError), match=text):
        fp8.linear(**_linear(**changed))


def test_an_output_that_overlaps_the_residual_is_refused():
    buf = torch.zeros((M + 1) * N)
    with pytest.raises(ValueError, match="the residual itself or lie apart"):
        fp8.linear(**_linear(residual=buf[:M * N].view(M, N), out=buf[4:4 + M * N].view(M, N)))


@pytest.mark.parametrize("changed,text", [
    (dict(weight=_weight()), r"1 part\(s\), not 2"),
    (dict(weight=_weight(codes=_codes(N + 1), parts=2, scales=torch.ones(2, 2))), "in 2 part"),
    (dict(weight=_weight(parts=2)), "the weight's scales"),
    (dict(out_codes=_codes(M)), "out_codes must be"),
    (dict(out_scales=torch.ones(M, 2)), "out_scales must be"),
    (dict(out_scales=torch.ones(1, 1).expand(M, 1)), "a place for every scale"),
])
def test_gated_refusals(changed, text):
    with pytest.raises((ValueError, TypeError), match=text):
        fp8.gated_linear(**_gated(**changed))


def test_gated_output_over_its_input_is_refused():
    codes = _codes(M)
    with pytest.raises(ValueError, match="apart from the input"):
        fp8.gated_linear(**_gated(codes=codes, out_codes=codes[:, :128]))


@pytest.mark.parametrize("w,parts,text", [(torch.zeros(N, K, dtype=torch.int32), 1, "bfloat16, float16 or float32"),
                                          (torch.zeros(N), 1, "rows a multiple"), (torch.zeros(N, K), 3, "rows a multiple"),
                                          (torch.zeros(N, K), 0, "rows a multiple"),
                                          (torch.zeros(K, N).t(), 1, "contiguous and apart")])
def test_weight_refusals(w, parts, text):
    with pytest.raises((ValueError, TypeError), match=text):
        fp8.quantize_weight(w, parts)


@pytest.mark.parametrize("entry", ["zkv_fp8_linear", "zkv_fp8_gated_linear"])
@pytest.mark.parametrize("sizes", [(0, 8, 128), (8, 0, 128), (8, 8, 0), (8, 8, 130), (8, 8, 16512), (1 << 20, 8, 128),
                                   (8, 1 << 22, 128), (1 << 19, 1 << 19, 128), (-5, 8, 128)])
def test_the_library_refuses_sizes_its_grids_do_not_hold(entry, sizes):
    """The entry points' own checks, before any launch (the addresses are never read)."""
    at, (m, n, k) = 4096, sizes
    tail = ((0, 0, at, n, 0) if entry == "zkv_fp8_linear" else (at, 1 << 23, at, 1, 1)) + (0, 0, 0)
    assert getattr(lib(), entry)(at, 1 << 20, at, 1, 1, at, 1 << 20, at, m, n, k, *tail) != 0


def _raw(t):
    return t.view(-1).view(torch.uint8)


def test_outputs_over_inputs_are_refused():
    """An output or a workspace that lies in what other workgroups still read."""
    square, ones = _codes(256), torch.ones(256, 2)
    gate = fp8.Fp8Weight(_codes(512), torch.ones(4, 2), parts=2)
    half = fp8.Fp8Weight(_codes(128), torch.ones(1, 2))
    x, single = torch.zeros(256, 256, dtype=BF), torch.zeros(256, 256)
    flat = torch.zeros(256 * 256 * 2, dtype=torch.uint8)
    for call in (
            lambda: fp8.rms_norm_quant(flat.view(BF).view(256, 256), x[0], 1e-6,
                                       codes=flat[:1 << 16].view(E4M3).view(256, 256)),
            lambda: fp8.rms_norm_quant(x.clone(), x[0], 1e-6, residual=x.clone(), sum_out=x),
            lambda: fp8.quantize_rows(single, scales=single[:, :2]),
            lambda: fp8.linear(square, ones, half, out=_raw(square).view(BF).view(256, 128)),
            lambda: fp8.gated_linear(square, ones, gate, out_codes=square),
            lambda: fp8.gated_linear(square, ones, gate, out_scales=ones),
            lambda: fp8.gated_linear(square, ones, gate, out_codes=gate.codes[:256]),
            lambda: fp8.gated_linear(square[:17], ones[:17], gate, workspace=_raw(gate.codes))):
        with pytest.raises(ValueError, match="apart from the input"):
            call()


@pytest.mark.parametrize("entry", ["zkv_fp8_rows", "zkv_fp8_linear", "zkv_fp8_gated_linear"])
def test_packed_arguments_are_the_entrys_own(entry):
    """A null operand with packed arguments is refused as without."""
    values = [0] * (len(SIGNATURES[entry][1]) - 1)
    assert getattr(lib(), entry)(*values, 0) != 0
    text = lib().zkv_last_error()
    packed = packed_args(entry, values)
    assert getattr(lib(), entry + "_call")(ctypes.addressof(packed), 0) != 0
    assert lib().zkv_last_error() == text and b"null pointer" in text
    assert getattr(lib(), entry + "_call")(0, 0) != 0
