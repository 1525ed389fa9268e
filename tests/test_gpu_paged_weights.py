"""What the weights of paged attention may lose, with keys that set every
token's weight: vanishing weights on large values, and infinite values.

Bound of an fp32 output element (no rounding but fp32's): with the exact
weights' mass A = sum p |v|, M the largest |v| and T tiles of 32 tokens in a
wave's run,

  * the score is exact here but for one scaling and the exponent's argument x,
    |x| < 2^8: 2^-24 2^8 + 2^-23 < 2^-15 relative, in numerator and denominator;
  * parts: 2^-21 relative, and in fp16 an absolute step of 2^-47 of the largest
    weight: n 2^-47 M;
  * sums of 32 T terms of up to three parts, and the joins of 16 waves and up to
    256 workgroups: (96 T + 300) 2^-24, in numerator and denominator,

so |out - ref| <= A (2^-13 + (96 T + 300) 2^-23) + n 2^-47 M + 2^-24 |ref|."""
import numpy as np
import pytest
import torch

from zoomkv_revision_amd import paged

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16
PAGE = 128


class Steps:
    """One pool for all requests of a batch (they share their pages), the keys 0
    but for channel 0, which times q = 1 and the scale ln 2 is log2 of the
    token's weight."""

    def __init__(self, log2_weights, values, bs, kv, dtype, fp8):
        """log2_weights [n], values [n, d] float64."""
        n, d = values.shape
        cell = torch.float8_e4m3fn if fp8 else dtype
        pages = -(-n // PAGE)
        rows = torch.zeros(2, pages * PAGE, d, dtype=torch.float64)
        rows[0, :n, 0], rows[1, :n] = log2_weights, values
        stored = rows.to(cell)
        assert torch.equal(torch.nan_to_num(stored.double()), torch.nan_to_num(rows))       # nothing is rounded
        self.k, self.v = (stored[i].view(pages, 1, PAGE, d).to(DEV).view(torch.uint8).repeat(1, kv, 1, 1).view(cell)
                          for i in range(2))
        self.table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(bs, pages)
        self.lens = torch.full((bs,), n, dtype=torch.int32, device=DEV)
        self.q = torch.zeros(bs, 2 * kv, d, dtype=dtype, device=DEV)
        self.q[..., 0] = 1.0
        self.p, self.rows, self.n = torch.exp2(log2_weights), values, n
        self.tiles = -(-(bs * kv * (-(-n // 32) + 2)) // 256) // (4 if d == 256 else 8) + 2

    def attend(self):
        out = torch.empty(self.q.shape, dtype=torch.float32, device=DEV)
        return paged.paged_attention(self.q, self.k, self.v, self.table, self.lens, softmax_scale=float(np.log(2.0)),
                                     out=out).double().cpu()

    def check(self, got, channels=slice(None)):
        p = self.p / self.p.sum()
        v = torch.nan_to_num(self.rows, posinf=0.0, neginf=0.0)
        ref, mass = p @ v, p @ v.abs()
        tol = mass * (2.0 ** -13 + (96 * self.tiles + 300) * 2.0 ** -23) + self.n * 2.0 ** -47 * v.abs().max() + \
            2.0 ** -24 * ref.abs()
        err = (got - ref).abs()[..., channels]
        assert bool((err <= tol[channels]).all()), float((err - tol[channels]).max())


@pytest.mark.parametrize("dtype,fp8", [(FP, False), (FP, True), (BF, False), (BF, True)])
@pytest.mark.parametrize("n,bs,kv,d", [(131072, 64, 8, 64), (8192, 64, 8, 128), (20000, 16, 4, 256), (131072, 1, 1, 128),
                                       (700, 1, 2, 64)])
@pytest.mark.parametrize("at", ["first", "last"])
def test_weights_that_vanish_add_nothing(dtype, fp8, n, bs, kv, d, at):
    """One token holds all the weight, with small values; the others have 2^-192
    or 2^-40 of it (on two channels' worth of values that are large and of one
    sign).  Batches whose waves have runs of up to 32768 tokens."""
    for low in (-192.0, -40.0):
        weights = torch.full((n,), low, dtype=torch.float64)
        values = torch.full((n, d), 4.0, dtype=torch.float64)
        values[:, 1::2] = 1.0
        top = 0 if at == "first" else n - 1
        weights[top] = 0.0
        values[top] = 0.0
        values[top, 2:] = 2.0 ** -9
        c = Steps(weights, values, bs, kv, dtype, fp8)
        c.check(c.attend())


@pytest.mark.parametrize("dtype,fp8", [(FP, False), (FP, True), (BF, False), (BF, True)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_weights_of_every_size(dtype, fp8, d):
    """Powers of two from 1 down to 2^-60, each on a channel of its own class:
    what is small against the whole is held to its own size."""
    n = 3000
    step = torch.arange(n) % d
    weights = -4.0 * (torch.arange(n) % 16).double()
    values = torch.zeros(n, d, dtype=torch.float64)
    values[torch.arange(n), step] = 1.0 + (torch.arange(n) % 8).double() / 8
    c = Steps(weights, values, 3, 2, dtype, fp8)
    c.check(c.attend())


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("n,bs,kv,d", [(40, 1, 1, 64), (40, 3, 2, 256), (5000, 2, 2, 128), (9000, 40, 4, 64)])
@pytest.mark.parametrize("low", [0.0, -12.0, -34.0, -100.0])
def test_infinite_values_stay_infinite(dtype, n, bs, kv, d, low):
    """A value of infinity or NaN shows in its channel, whatever its weight is,
    and leaves the other channels as they are."""
    g = torch.Generator().manual_seed(n)
    weights = torch.where(torch.arange(n) % 7 == 3, 0.0, low).double()
    values = torch.randint(-32, 33, (n, d), generator=g).double() / 8
    inf = float("inf")
    places = (0, n // 3, n // 2 + 1, n - 1)
    values[places[0], 5] = inf
    values[places[1], 6] = -inf
    values[places[2], 7], values[places[3], 7] = inf, -inf
    values[places[2], d - 1] = float("nan")
    values[places[3], d - 2] = inf
    values[places[1], 0], values[places[0], 0] = -inf, -inf
    c = Steps(weights, values, bs, kv, dtype, False)
    got = c.attend()
    assert bool((got[..., 5] == inf).all()) and bool((got[..., d - 2] == inf).all())
    assert bool((got[..., 6] == -inf).all()) and bool((got[..., 0] == -inf).all())
    assert bool(got[..., [7, d - 1]].isnan().all())
    finite = [i for i in range(d) if i not in (0, 5, 6, 7, d - 1, d - 2)]
    c.rows[:, [7, d - 1]] = 0.0
    c.check(got, finite)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_infinite_values_of_tokens_that_are_left_out(dtype):
    """Behind the window, past the length and on a page outside the pool."""
    n, d = 300, 128
    values = torch.randint(-32, 33, (n, d), generator=torch.Generator().manual_seed(1)).double() / 8
    c = Steps(torch.zeros(n, dtype=torch.float64), values, 1, 1, dtype, False)
    v = c.v.view(-1, d)
    v[:57], v[290:] = float("inf"), float("nan")
    c.lens.fill_(290)
    out = torch.empty(c.q.shape, dtype=torch.float32, device=DEV)
    paged.paged_attention(c.q, c.k, c.v, c.table, c.lens, softmax_scale=1.0, window=233, out=out)
    c.rows, c.p = values[57:290], torch.ones(233, dtype=torch.float64)
    c.check(out.double().cpu())
