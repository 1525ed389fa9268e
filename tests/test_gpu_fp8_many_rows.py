"""GPU: more rows than one launch takes (2^21; a launch holds fewer than 2^32 threads).
Rows repeat a pattern whose length divides no launch, so that a row taken for
another shows; the pattern's own result is what the other tests check."""
import pytest
import torch

from test_gpu_fp8 import DEV, E4M3, TYPES, _rows
from zoomkv_revision_amd import fp8

pytestmark = pytest.mark.gpu


def _repeats(got, pattern, period):
    """Whether row i of got is row i % period of pattern, in runs of rows."""
    if got.dtype == E4M3:
        got, pattern = got.view(torch.uint8), pattern.view(torch.uint8)
    step = 1 << 19
    for i in range(0, got.shape[0], step):
        part = got[i:i + step]
        at = torch.arange(i, i + part.shape[0], device=DEV) % period
        if not torch.equal(part, pattern[at]):
            return False
    return True


def _repeated(pattern, rows):
    out = torch.empty(rows, pattern.shape[1], dtype=pattern.dtype, device=DEV)
    step = 1 << 19
    for i in range(0, rows, step):
        n = min(step, rows - i)
        out[i:i + n] = pattern[torch.arange(i, i + n, device=DEV) % pattern.shape[0]]
    return out


def _finite(codes, scales):
    return bool(scales.isfinite().all()) and bool(codes.float().isfinite().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [((1 << 21) - 3, 20), ((1 << 21) + 1, 24), ((1 << 22) + 77, 130)])
def test_rows_of_several_launches(dtype, M, K):
    P = 1009
    x, r = (_rows(i, P, K, dtype).clamp(-2000, 2000).to(DEV) for i in (1, 2))
    w = _rows(3, 1, K, dtype).clamp(-10, 10).to(DEV)[0]
    many, other = _repeated(x, M), _repeated(r, M)
    codes, scales = fp8.quantize_rows(x)
    got = fp8.quantize_rows(many)
    assert _finite(codes, scales) and _repeats(got[0], codes, P) and _repeats(got[1], scales, P)
    want = fp8.rms_norm_quant(x, w, 1e-6, residual=r)
    got = fp8.rms_norm_quant(many, w, 1e-6, residual=other)
    assert _finite(*want[:2]) and all(_repeats(g, t, P) for g, t in zip(got, want))
    # plans: scales by rows, the sum in place
    by_rows = torch.empty(M, scales.shape[1], device=DEV)
    fp8.RmsNormQuantPlan(many, w, 1e-6, residual=other, sum_out=other, scales=by_rows).run()
    assert _repeats(other, want[2], P) and _repeats(by_rows, want[1].contiguous(), P)


def test_rows_beyond_the_threads_of_a_launch():
    """2^25 rows of two waves each: 2^32 threads."""
    M, K, P = (1 << 25) + 77, 513, 4099
    x = _rows(5, P, K, torch.bfloat16).to(DEV)
    w = torch.ones(K, dtype=torch.bfloat16, device=DEV)
    many = _repeated(x, M)
    for one in (lambda t: fp8.quantize_rows(t), lambda t: fp8.rms_norm_quant(t, w, 1e-6)):
        codes, scales = one(x)
        got = one(many)
        assert _finite(codes, scales) and _repeats(got[0], codes, P) and _repeats(got[1], scales, P)
        del got
    del many
    torch.cuda.empty_cache()
