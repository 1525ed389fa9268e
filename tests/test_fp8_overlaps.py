"""What the 8-bit linear calls take for buffers that share memory (host checks only)."""
import random

import pytest
import torch

from fp8_cases import E4M3
from test_fp8_checks import BF, K, M, N, _gated, _linear, _norm, _rows
from zoomkv_revision_amd import fp8
from zoomkv_revision_amd._lib import ZkvError


def _bytes(t):
    """The bytes of a 2-D tensor's elements, by enumeration."""
    at, size = t.storage_offset() * t.element_size(), t.element_size()
    starts = [at + (i * t.stride(0) + j * t.stride(1)) * size for i in range(t.shape[0]) for j in range(t.shape[1])]
    return {b for s in starts for b in range(s, s + size)}


def test_overlaps_against_enumeration():
    """Never a shared byte missed; exact for rows of one pitch, and for one row among
    them."""
    r, buf = random.Random(1), torch.zeros(4096, dtype=torch.uint8)
    seen = {False: 0, True: 0}
    for _ in range(6000):
        pitch, pair = 4 * r.randint(2, 12), []
        for _ in range(2):
            b = buf.view(r.choice([torch.uint8, torch.bfloat16, torch.float32]))
            size = b.element_size()
            rows, cols = r.randint(0, 6), r.randint(1, pitch // size)
            pair.append(b.as_strided((rows, cols), (pitch // size, 1), r.randint(0, 200 // size)))
        shared = bool(_bytes(pair[0]) & _bytes(pair[1]))
        assert fp8._overlap(*pair) == shared
        seen[shared] += 1
        other = buf.as_strided((r.randint(0, 6), r.randint(1, 6)), (r.choice([1, 3, 9, 40]), r.choice([1, 2, 7])), r.randint(0, 200))
        for t in pair:
            assert fp8._overlap(t, other) or not _bytes(t) & _bytes(other)
    assert min(seen.values()) > 500


def test_columns_of_one_buffer_are_apart():
    """An output beside its residual, a sum beside its inputs, codes beside their
    scales, in rows of one buffer: no element is shared."""
    both = torch.zeros(M, 2 * N, dtype=BF)
    three = torch.zeros(M, 3 * K, dtype=BF)
    record = torch.zeros(M, 272, dtype=torch.uint8)
    short = torch.zeros(M, 144, dtype=torch.uint8)
    for call in (
            lambda: fp8.linear(**_linear(out=both[:, :N], residual=both[:, N:])),
            lambda: fp8.rms_norm_quant(**_norm(x=three[:, :K], residual=three[:, K:2 * K], sum_out=three[:, 2 * K:])),
            lambda: fp8.quantize_rows(**_rows(codes=record[:, :256].view(E4M3), scales=record.view(torch.float32)[:, 64:66])),
            lambda: fp8.gated_linear(**_gated(out_codes=short[:, :128].view(E4M3),
                                              out_scales=short.view(torch.float32)[:, 32:33]))):
        with pytest.raises(ZkvError, match="device tensors"):
            call()


def test_columns_that_meet_are_refused():
    both = torch.zeros(M, 2 * N, dtype=BF)
    with pytest.raises(ValueError, match="the residual itself or lie apart"):
        fp8.linear(**_linear(out=both[:, :N], residual=both[:, N - 1:2 * N - 1]))
    three = torch.zeros(M, 3 * K, dtype=BF)
    with pytest.raises(ValueError, match="residual itself or lie apart"):
        fp8.rms_norm_quant(**_norm(x=three[:, :K], residual=three[:, K:2 * K], sum_out=three[:, 2 * K - 1:3 * K - 1]))


def test_codes_over_scales_are_refused():
    flat = torch.zeros(M * 256 + 16, dtype=torch.uint8)
    codes = flat[:M * 256].view(E4M3).view(M, 256)
    over = lambda rows, cols: flat[-4 * rows * cols - 16:-16].view(torch.float32).view(rows, cols)
    beside = torch.zeros(M, 272, dtype=torch.uint8)
    for call in (lambda: fp8.quantize_rows(**_rows(codes=codes, scales=over(M, 2))),
                 lambda: fp8.rms_norm_quant(**_norm(codes=codes, scales=over(M, 2))),
                 lambda: fp8.quantize_rows(**_rows(codes=beside[:, :256].view(E4M3),
                                                   scales=beside.view(torch.float32)[:, 63:65])),
                 lambda: fp8.gated_linear(**_gated(out_codes=flat[-16 - M * 128:-16].view(E4M3).view(M, 128),
                                                     out_scales=over(M, 1)))):
        with pytest.raises(ValueError, match="apart from the inputs and the other outputs"):
            call()


def test_scales_that_share_places_are_refused():
    """By enumeration over strides; single rows and blocks have none to share."""
    buf = torch.zeros(4096)
    for rows in (1, 2, 4, 5):
        for nb in (1, 2, 3):
            for s0 in range(7):
                for s1 in range(7):
                    t = buf.as_strided((rows, nb), (s0, s1))
                    places = {i * s0 + j * s1 for i in range(rows) for j in range(nb)}
                    check = lambda: fp8._check_scales("scales", t, rows, 128 * nb, apart=True)
                    if len(places) == rows * nb:
                        check()
                    else:
                        with pytest.raises(ValueError, match="a place for every scale"):
                            check()


def test_calls_refuse_scales_that_share_places():
    wide = torch.zeros(256, 256, dtype=BF)
    over = torch.zeros(512).as_strided((256, 2), (1, 1))
    with pytest.raises(ValueError, match="a place for every scale"):
        fp8.quantize_rows(wide, scales=over)
    gate = fp8.Fp8Weight(torch.zeros(512, 256, dtype=torch.uint8).view(E4M3), torch.ones(4, 2), parts=2)
    codes = torch.zeros(256, 256, dtype=torch.uint8).view(E4M3)
    with pytest.raises(ValueError, match="a place for every scale"):
        fp8.gated_linear(codes, torch.ones(256, 2), gate, out_scales=over)
