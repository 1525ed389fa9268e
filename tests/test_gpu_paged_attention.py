"""Paged one-token attention on the GPU against float64 softmax attention over
the same rows (oracle/paged.py).

Bound of an output element, from the kernel's arithmetic (u = half a step of
the output's type; A = sum p |v| of the exact weights, n tokens, head dim d):

  * the score is an fp32 sum of d exact products, scaled once:
    |ds| <= (d + 2) 2^-24 scale sum |q k| =: e, and the weights move by at most
    2 e relative (numerator and denominator); exp2 of an fp32 argument x adds
    2^-24 |x| + 2^-23, below 2^-19 for |x| < 2^4.5, beyond which 131072 tokens
    together weigh less than one at x = 0;
  * P enters the product as three 8-bit or two 11-bit parts: 2^-21 relative;
  * sums of n fp32 terms, and the joining of partials: (n + 64) 2^-24, twice;

so |out - ref| <= u |ref| + A (2 e + 2^-17 + (n + 64) 2^-23), as 2^-21 + 2 *
2^-19 < 2^-17.  The log-sum-exp (of the unsplit P) moves by at most e + 2^-16 +
(n + 64) 2^-23, plus its own fp32 rounding 2^-23 |lse|."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from zoomkv_revision_amd import paged
from zoomkv_revision_amd._lib import ZkvError, lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, FP: 2.0 ** -11, torch.float32: 2.0 ** -24}


class Case:
    """A pool, a table and lengths; rows that no request holds are NaN."""

    def __init__(self, lens, hq, kv, d, page, dtype=BF, fp8=False, nhd=False, seed=0, spread=2.0, width=None, extra=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        bs = len(lens)
        used = [-(-n // page) for n in lens]
        pages = sum(used) + extra
        cell = torch.float8_e4m3fn if fp8 else dtype
        pools = []
        for _ in range(2):
            x = torch.randn(pages, kv, page, d, generator=g, device=DEV)
            x = (x * 60).to(cell) if fp8 else x.to(cell)
            pools.append(x)
        perm = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int32)
        width = max(max(used), 1) + 1 if width is None else width
        self.table = torch.full((bs, width), -1, dtype=torch.int32, device=DEV)
        held = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
        at = 0
        for b, (n, u) in enumerate(zip(lens, used)):
            self.table[b, :u] = perm[at:at + u]
            t = torch.arange(n, device=DEV)
            held[self.table[b].long()[t // page], t % page] = True
            at += u
        nan = 0x7F if fp8 else float("nan")
        for i, x in enumerate(pools):
            raw = x.view(torch.uint8) if fp8 else x
            raw.masked_fill_(~held[:, None, :, None], nan)
            if nhd:
                y = raw.transpose(1, 2).contiguous().transpose(1, 2)
                pools[i] = y.view(cell) if fp8 else y
        self.k, self.v = pools
        self.scales = [0.01 + 0.02 * torch.rand(kv, generator=g, device=DEV) for _ in range(2)] if fp8 else [None, None]
        self.q = (spread * torch.randn(bs, 1, hq, d, generator=g, device=DEV)).to(dtype)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.page, self.d, self.hq, self.kv = page, d, hq, kv

    def rows(self, b, h, tokens):
        """K and V of one head's tokens (a list of positions), float64."""
        t = torch.as_tensor(tokens, device=DEV, dtype=torch.long)
        ids, off = self.table[b].long()[t // self.page], t % self.page
        out = []
        for pool, s in zip((self.k, self.v), self.scales):
            x = pool[:, h]
            x = x.view(torch.uint8)[ids, off].view(pool.dtype) if s is not None else x[ids, off]
            out.append((x.double() * (1.0 if s is None else s[h].double())).cpu().numpy())
        return out

    def check(self, out, lse=None, window=0, scale=None, tokens=None, requests=None):
        scale = self.d ** -0.5 if scale is None else scale
        group = self.hq // self.kv
        q = self.q.double().cpu().numpy()
        got = out.double().cpu().numpy().reshape(len(self.lens), self.hq, self.d)
        assert np.isfinite(got).all()
        for b in range(len(self.lens)) if requests is None else requests:
            n = int(self.lens[b])
            seen = list(range(max(0, n - window) if window else 0, n)) if tokens is None else tokens[b]
            for h in range(self.kv):
                k, v = self.rows(b, h, seen)
                heads = slice(h * group, (h + 1) * group)
                ref, ref_lse, mass = op.attention(q[b, 0, heads], k, v, scale)
                e = (self.d + 2) * 2.0 ** -24 * abs(scale) * \
                    (np.abs(q[b, 0, heads]) @ np.abs(k).T).max(initial=0.0)
                sums = (len(seen) + 64) * 2.0 ** -23
                err = np.abs(got[b, heads] - ref)
                tol = U[out.dtype] * np.abs(ref) + mass * (2 * e + 2.0 ** -17 + sums) + 2.0 ** -25
                assert (err <= tol).all(), (b, h, float((err - tol).max()))
                if lse is not None:
                    gl = lse.double().cpu().numpy()[b, heads, 0]
                    if len(seen) == 0:
                        assert np.isneginf(gl).all()
                    else:
                        assert (np.abs(gl - ref_lse) <= e + 2.0 ** -16 + sums + 2.0 ** -23 * np.abs(ref_lse)).all()

    def attend(self, **kw):
        return paged.paged_attention(self.q, self.k, self.v, self.table, self.lens, k_scale=self.scales[0],
                                     v_scale=self.scales[1], **kw)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (FP, False), (BF, True), (FP, True)])
@pytest.mark.parametrize("page,nhd", [(16, False), (24, True), (1, False), (64, True)])
def test_types_dims_and_pages(d, dtype, fp8, page, nhd):
    c = Case([1, 0, 31, 32, 33, 200, 517], 8, 2, d, page, dtype, fp8, nhd, seed=d + page)
    out, lse = c.attend(return_softmax_lse=True)
    assert out.shape == c.q.shape and out.dtype == dtype and lse.shape == (7, 8, 1)
    c.check(out, lse)
    assert not out[1].any()


@pytest.mark.parametrize("hq,kv", [(1, 1), (2, 2), (16, 1), (17, 1), (40, 1), (21, 3), (32, 8), (64, 2)])
def test_head_layouts(hq, kv):
    c = Case([5, 97, 1300, 64], hq, kv, 128, 16, seed=hq)
    out = torch.empty(4, 1, hq, 128, dtype=torch.float32, device=DEV)
    got, lse = c.attend(out=out, return_softmax_lse=True)
    assert got is out
    c.check(out, lse)


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [63], [255], [256], [257], [700], [4097], [20000],
                                  [1] * 300, [3000, 1, 1, 1, 9000], [0, 0, 5, 0], list(range(64)),
                                  [8192, 0, 33, 4000, 1, 77, 16, 2500]])
def test_lengths(lens):
    c = Case(lens, 4, 1, 128, 16, seed=len(lens))
    out, lse = c.attend(return_softmax_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("hq,kv,d,dtype", [(16, 16, 64, FP), (1, 1, 64, BF), (2, 1, 256, BF), (8, 8, 128, FP)])
@pytest.mark.parametrize("n", [1500, 6000])
def test_units_cut_on_both_sides(hq, kv, d, dtype, n):
    """Few query heads, units longer than a workgroup's run: most workgroups
    share a unit with the one before and another with the one after."""
    c = Case([n + 37 * i for i in range(9)] + [40, 3, 0, 700], hq, kv, d, 24, dtype, seed=n)
    for window in (0, n - 100):
        out, lse = c.attend(window=window, return_softmax_lse=True)
        c.check(out, lse, window=window, requests=[0, 4, 8, 9, 10, 11, 12])


@pytest.mark.parametrize("seed", range(24))
def test_random_calls(seed):
    rng = np.random.default_rng(seed)
    kv = int(rng.choice([1, 2, 3, 8]))
    hq = kv * int(rng.choice([1, 2, 4, 5, 16, 24]))
    top = int(rng.choice([20, 300, 5000]))
    lens = [int(x) for x in rng.integers(0, top + 1, int(rng.integers(1, 40)))]
    fp8 = bool(rng.integers(2))
    c = Case(lens, hq, kv, int(rng.choice([64, 128, 256])), int(rng.choice([1, 8, 16, 24, 32, 100])),
             [BF, FP][int(rng.integers(2))], fp8, bool(rng.integers(2)), seed=seed)
    window = int(rng.choice([0, 0, 1, 33, 1000]))
    out, lse = c.attend(window=window, return_softmax_lse=True)
    c.check(out, lse, window=window, requests=sorted({0, len(lens) - 1, len(lens) // 2, int(np.argmax(lens))}))


def test_long_sequence_of_one_head():
    """131072 tokens of one KV head: every workgroup holds a part of the unit."""
    c = Case([131072], 2, 1, 128, 128, seed=3)
    out = torch.empty(1, 1, 2, 128, dtype=torch.float32, device=DEV)
    _, lse = c.attend(out=out, return_softmax_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("lens,hq,kv,d,dtype,fp8", [
    ([4200], 16, 1, 128, BF, False),                 # 17 workgroups and a few more
    ([4400, 0, 3], 16, 1, 128, FP, True),
    ([20000], 24, 1, 128, BF, False),                # 16 heads in two steps, 8 in one or two
    ([66000], 8, 1, 128, BF, False),                 # 256 workgroups
    ([30000, 31000], 40, 1, 64, FP, False),
    ([33333, 1, 700, 20011], 16, 1, 128, BF, False),  # long units that meet inside a workgroup
    ([9000, 9000, 9000], 16, 1, 256, BF, False),
    ([12000, 50], 20, 2, 256, FP, True)])
def test_units_of_many_workgroups(lens, hq, kv, d, dtype, fp8):
    """Partials joined in two steps; the counts are ready for the next call,
    and the bits are the same from call to call."""
    c = Case(lens, hq, kv, d, 16, dtype, fp8, seed=hq + d)
    out, lse = c.attend(return_softmax_lse=True)
    c.check(out, lse)
    workspace = paged.new_workspace(torch.device(DEV), lib().zkv_paged_attention_workspace_size(d))
    for window in (0, 0, lens[0] - 77, 0):
        got, gl = c.attend(return_softmax_lse=True, workspace=workspace, window=window)
        if window:
            c.check(got, gl, window=window)
        else:
            assert torch.equal(got, out) and torch.equal(gl, lse)


@pytest.mark.parametrize("lens,hq,kv,d,dtype,fp8", [
    ([70000], 16, 4, 128, BF, False),                      # sets of four heads
    ([40000, 0, 31, 9000, 1], 64, 8, 128, BF, False),      # of two
    ([5000] * 20 + [3, 0, 700], 10, 2, 64, FP, False),     # of two, five query heads each
    ([3000 + 7 * i for i in range(15)], 8, 8, 128, BF, True),   # of eight
    ([33000, 2000], 8, 4, 256, FP, True),
    ([4100] * 9 + [60, 8000], 6, 6, 64, BF, False),        # of two: three sets
    ([60000, 20000], 48, 2, 64, FP, False)])               # more than 16 query heads a KV head: none
def test_heads_of_a_token_together(lens, hq, kv, d, dtype, fp8):
    """Pools [page, token, head] over enough tokens that neighbouring waves take
    the heads of a set: the same results, with a window, and every time."""
    c = Case(lens, hq, kv, d, 16, dtype, fp8, nhd=True, seed=hq + d)
    some = sorted({0, len(lens) // 2, len(lens) - 2, len(lens) - 1})
    out, lse = c.attend(return_softmax_lse=True)
    c.check(out, lse, requests=some)
    again, lse2 = c.attend(return_softmax_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    window = max(lens) - 500
    c.check(*c.attend(return_softmax_lse=True, window=window), window=window, requests=some)


@pytest.mark.parametrize("hq,kv,d,dtype,fp8", [(64, 8, 64, BF, True), (8, 8, 128, BF, False), (96, 4, 256, FP, False)])
@pytest.mark.parametrize("lens", [[66] * 235, [1 + 37 * i % 160 for i in range(250)],
                                  [0, 1, 2, 33] * 40 + [4000] + [5, 0, 96] * 60])
def test_many_short_units(hq, kv, d, dtype, fp8, lens):
    """Several units a wave, long ones among them."""
    c = Case(lens, hq, kv, d, 16, dtype, fp8, seed=len(lens) + d)
    out, lse = c.attend(return_softmax_lse=True)
    c.check(out, lse, requests=sorted({*range(0, len(lens), 9), *range(150, 170), len(lens) - 1}))


@pytest.mark.parametrize("window", [1, 5, 32, 100, 512, 100000])
@pytest.mark.parametrize("page", [16, 24])
def test_windows(window, page):
    c = Case([1, 4, 33, 100, 101, 512, 513, 2000, 0], 6, 2, 128, page, seed=window)
    out, lse = c.attend(window=window, return_softmax_lse=True)
    c.check(out, lse, window=window)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_other_scales(scale):
    c = Case([40, 300], 4, 2, 64, 8, seed=4)
    out, lse = c.attend(softmax_scale=scale, return_softmax_lse=True)
    c.check(out, lse, scale=scale)


def test_peaked_scores():
    """Scores with a spread of hundreds: most weights vanish, the running
    maximum moves often."""
    c = Case([3000, 64, 1], 8, 2, 128, 16, seed=5, spread=100.0)
    out, lse = c.attend(return_softmax_lse=True)
    c.check(out, lse)


def test_rising_scores():
    """Every tile's maximum is above the last one's."""
    c = Case([2000], 4, 1, 128, 16, FP, seed=6)
    ramp = torch.linspace(-3, 3, 2000, device=DEV)
    c.q.fill_(1.0)
    t = torch.arange(2000, device=DEV)
    c.k[c.table[0].long()[t // 16], 0, t % 16] = (ramp[:, None] + 0 * c.q[0, 0, 0].float()).to(FP)
    out, lse = c.attend(return_softmax_lse=True)
    c.check(out, lse)


def test_pages_outside_the_pool_are_left_out():
    c = Case([100, 64, 40, 16], 4, 2, 128, 16, seed=7)
    table = c.table.clone()
    table[0, 2] = -1                       # tokens 32 .. 47
    table[1, 0] = c.k.shape[0]             # 0 .. 15
    table[1, 3] = 2 ** 31 - 1              # 48 .. 63
    table[2, :] = -5                       # none left
    out, lse = paged.paged_attention(c.q, c.k, c.v, table, c.lens, return_softmax_lse=True)
    c.check(out, lse, tokens=[[*range(32), *range(48, 100)], list(range(16, 48)), [], list(range(16))])
    assert not out[2].any()


def test_lengths_outside_the_table():
    c = Case([48, 20, 48], 4, 2, 128, 16, seed=8, width=3)
    lens = torch.tensor([2 ** 31 - 1, -3, 49], dtype=torch.int32, device=DEV)
    out, lse = paged.paged_attention(c.q, c.k, c.v, c.table, lens, return_softmax_lse=True)
    c.lens = torch.tensor([48, 0, 48], dtype=torch.int32, device=DEV)
    c.check(out, lse)


def test_infinities_and_nan_of_the_cache():
    """A key of -inf scores takes no weight; a NaN or an infinite value that a
    weight meets shows in its own request, head and channel only."""
    c = Case([50, 50, 50, 50, 50], 4, 2, 128, 16, seed=9)
    cell = lambda pool, b, h, t: pool[int(c.table[b, t // 16]), h, t % 16]
    c.q[0] = c.q[0].abs()
    cell(c.k, 0, 0, 17).fill_(float("-inf"))          # score -inf for every query head
    cell(c.v, 1, 0, 3)[5] = float("inf")
    cell(c.k, 2, 1, 40)[7] = float("nan")
    cell(c.v, 3, 1, 49)[0] = float("nan")
    out, lse = c.attend(return_softmax_lse=True)
    seen = [t for t in range(50) if t != 17]
    k, v = c.rows(0, 0, seen)
    q = c.q.double().cpu().numpy()
    ref, ref_lse, mass = op.attention(q[0, 0, :2], k, v, 128 ** -0.5)
    got = out.double().cpu().numpy()
    assert (np.abs(got[0, 0, :2] - ref) <= U[BF] * np.abs(ref) + mass * 2.0 ** -12).all()
    assert np.abs(lse[0, :2, 0].cpu().numpy() - ref_lse).max() < 2.0 ** -12
    assert (got[1, 0, :2, 5] == np.inf).all() and np.isfinite(np.delete(got[1, 0], 5, axis=-1)).all()
    assert np.isfinite(got[1, 0, 2:]).all()
    assert np.isnan(got[2, 0, 2:]).all() and np.isfinite(got[2, 0, :2]).all()
    assert np.isnan(got[3, 0, 2:, 0]).all() and np.isfinite(got[3, 0, 2:, 1:]).all() and np.isfinite(got[3, 0, :2]).all()
    assert np.isfinite(got[4]).all()


def test_keys_of_minus_infinity_everywhere():
    """No score above -inf: zeros, as for no tokens."""
    c = Case([40, 70], 2, 1, 64, 16, seed=10)
    c.q.copy_(c.q.abs() + 0.5)
    t = torch.arange(40, device=DEV)
    c.k[c.table[0].long()[t // 16], 0, t % 16] = float("-inf")
    out, lse = c.attend(return_softmax_lse=True)
    assert not out[0].any() and bool(torch.isneginf(lse[0]).all())
    c.check(out, lse, tokens=[[], list(range(70))])


def test_strided_arguments():
    """q inside a fused projection, table columns inside a wider one, a layer's
    pools inside one tensor of all layers, 3-D q."""
    c = Case([70, 9], 4, 2, 128, 16, seed=11)
    wide_q = torch.randn(2, 12, 128, device=DEV).to(BF)
    wide_q[:, 4:8] = c.q[:, 0]
    wide_t = torch.full((2, 3 * c.table.shape[1]), 1 << 20, dtype=torch.int32, device=DEV)
    wide_t[:, 2:2 + c.table.shape[1]] = c.table
    pools = torch.stack([c.k, c.k * 0, c.v], 1)           # [pages, 3, kv, page, d]
    out = paged.paged_attention(wide_q[:, 4:8], pools[:, 0], pools[:, 2], wide_t[:, 2:2 + c.table.shape[1]], c.lens)
    assert out.shape == (2, 4, 128)
    c.check(out)
    assert torch.equal(out, c.attend()[:, 0])
    odd = torch.randn(2, 4, 129, device=DEV).to(BF)
    odd[..., 1:] = c.q[:, 0]
    assert torch.equal(paged.paged_attention(odd[..., 1:], c.k, c.v, c.table, c.lens), out)


def test_offsets_past_32_bits():
    """Two pools in one tensor of 2^32 + bf16 cells: rows beyond 2^31 elements
    and 2^32 bytes of a pool's base."""
    page, kv, d, stride = 16, 2, 128, 1 << 21
    pages = 1100
    base = torch.empty(pages * stride, dtype=BF, device=DEV)           # 4.6 GB
    pool = lambda off: base.as_strided((pages, kv, page, d), (stride, page * d, d, 1), off)
    k, v = pool(0), pool(1 << 20)
    g = torch.Generator(device=DEV).manual_seed(12)
    ids = torch.tensor([[1099, 0, 1025, 1024, 512, 1098]], dtype=torch.int32, device=DEV)
    slots = (ids[0].long()[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:90].contiguous()
    rows = [torch.randn(90, kv, d, generator=g, device=DEV).to(BF) for _ in range(2)]
    paged.paged_write(*rows, slots, k, v)
    q = torch.randn(1, 4, d, generator=g, device=DEV).to(BF)
    out = paged.paged_attention(q, k, v, ids, torch.tensor([90], dtype=torch.int32, device=DEV))
    for h in range(kv):
        assert torch.equal(k[ids[0].long()[torch.arange(90, device=DEV) // 16], h, torch.arange(90, device=DEV) % 16],
                           rows[0][:, h])
        ref, _, mass = op.attention(*(x.double().cpu().numpy() for x in (q[0, 2 * h:2 * h + 2], rows[0][:, h],
                                                                        rows[1][:, h])), d ** -0.5)
        err = np.abs(out[0, 2 * h:2 * h + 2].double().cpu().numpy() - ref)
        assert (err <= U[BF] * np.abs(ref) + mass * 2.0 ** -12).all()


def test_many_requests():
    c = Case([1 + i % 40 for i in range(paged.MAX_REQUESTS)], 2, 2, 64, 16, seed=13)
    out, lse = c.attend(return_softmax_lse=True)
    c.check(out, lse, requests=[0, 1, 39, 40, 2047, 4094, 4095])


def test_the_same_bits_every_time():
    c = Case([9000, 1, 500, 0, 4444], 16, 2, 128, 16, seed=14)
    first = c.attend(return_softmax_lse=True)
    for _ in range(20):
        again = c.attend(return_softmax_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    plan = paged.PagedAttentionPlan(c.q, c.k, c.v, c.table, c.lens, return_softmax_lse=True)
    for _ in range(3):
        out, lse = plan.run()
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


@pytest.mark.parametrize("lens,hq,kv,dtype,fp8", [([32926] * 4 + [0], 4, 1, BF, True), ([2268] * 79, 4, 1, BF, False),
                                                  ([6017] * 6 + [3], 8, 4, FP, True), ([4613, 800, 77, 3000], 64, 8, BF, False),
                                                  ([20126, 700, 15000], 20, 4, FP, False), ([3578] * 75, 8, 2, BF, False)])
def test_the_same_bits_whoever_ends_last(lens, hq, kv, dtype, fp8):
    """Workgroups that share units on both sides, whose last arrivals change
    from run to run."""
    c = Case(lens, hq, kv, 128, 16, dtype, fp8, seed=16)
    out = torch.empty(len(lens), 1, hq, 128, dtype=torch.float32, device=DEV)
    first = [x.clone() for x in c.attend(out=out, return_softmax_lse=True)]
    for _ in range(60):
        again = c.attend(out=out, return_softmax_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_two_streams_at_once():
    """Two calls that overlap on the device, each on its stream's workspace."""
    cs = [Case([6000, 3000, 40], 8, 2, 128, 16, seed=15 + i) for i in range(2)]
    want = [c.attend() for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.attend())
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_two_captured_graphs_at_once():
    """Graphs captured on one stream have workspaces of their own; replays
    follow new queries, lengths and table entries."""
    cs = [Case([5000, 700, 33], 8, 2, 128, 16, seed=20 + i) for i in range(2)]
    for c in cs:
        c.attend()
    torch.cuda.synchronize()
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(c.attend(return_softmax_lse=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cs]
    for step in range(5):
        for c in cs:
            c.q.copy_(c.q.flip(-1) * (-1) ** step)
            c.lens.copy_((c.lens * 3 + step * 7) % 5001)
            c.lens[1:].clamp_(max=33)
        want = [c.attend(return_softmax_lse=True) for c in cs]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (wo, wl), (o, l) in zip(want, outs):
            assert torch.equal(wo, o) and torch.equal(wl, l), step


@pytest.mark.parametrize("hq,kv,d", [(16, 1, 128), (64, 4, 256), (40, 1, 64)])
def test_captured_with_the_largest_partials(hq, kv, d):
    """16 query heads a unit: the launch asks for the most LDS, also inside a
    capture."""
    c = Case([9000, 40, 3000], hq, kv, d, 16, seed=40)
    plan = paged.PagedAttentionPlan(c.q, c.k, c.v, c.table, c.lens, return_softmax_lse=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.run()
    for n in (9000, 100, 7777):
        c.lens[0] = n
        g.replay()
        out, lse = (x.clone() for x in plan.out)
        c.check(out, lse, requests=[0, 2])
        again, _ = c.attend(return_softmax_lse=True)
        assert torch.equal(again, out)


def test_a_plan_on_another_stream():
    c = Case([2000, 7], 8, 2, 128, 16, seed=41)
    want = c.attend()
    plan = paged.PagedAttentionPlan(c.q, c.k, c.v, c.table, c.lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(4):
            got = plan.run().clone()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_out_in_place_of_q():
    c = Case([2000, 7, 0, 300], 8, 2, 128, 16, seed=42)
    want = c.attend()
    q = c.q.clone()
    assert paged.paged_attention(q, c.k, c.v, c.table, c.lens, out=q) is q and torch.equal(q, want)


def test_a_workspace_too_small_is_refused():
    c = Case([10], 2, 1, 64, 16, seed=30)
    with pytest.raises(ValueError, match="workspace"):
        c.attend(workspace=torch.empty(1024, dtype=torch.uint8, device=DEV))
    with pytest.raises((ValueError, ZkvError)):
        paged.paged_attention(c.q, c.k, c.v, c.table.cpu(), c.lens)
    with pytest.raises((ValueError, ZkvError)):
        paged.paged_attention(c.q.cpu(), c.k, c.v, c.table, c.lens)


# ---------------------------------------------------------------------------
# the operators together: a batch served over a paged cache
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (FP, True)])
def test_a_serving_loop(dtype, fp8):
    """Requests come with prompts, decode, stop and are replaced, over a pool
    that holds them just so: after every step each request's attention equals
    the float64 one over the rows it was given, wherever they lie."""
    page, kv, hq, d, slots_n, width = 8, 2, 6, 128, 5, 12
    rng = np.random.default_rng(31)
    g = torch.Generator(device=DEV).manual_seed(31)
    tables = paged.PageTables.allocate(slots_n, width * page, 40, page, device=DEV)
    cell = torch.float8_e4m3fn if fp8 else dtype
    kp, vp = (torch.zeros(40, kv, page, d, device=DEV).to(cell) for _ in range(2))
    scales = [torch.full((kv,), 0.01, device=DEV) for _ in range(2)] if fp8 else [None, None]
    told = [[] for _ in range(slots_n)]                 # each request's (k, v) rows as stored
    store = lambda x: x if not fp8 else (x.float() / 0.01).clamp(-448, 448).to(cell).to(torch.float64) * \
        float(torch.tensor(0.01))
    positions = torch.empty(64, dtype=torch.int32, device=DEV)
    slots = torch.empty(64, dtype=torch.int64, device=DEV)
    for step in range(25):
        new = []
        for r in range(slots_n):
            if not told[r]:
                new.append(int(rng.integers(0, 13)))
            elif len(told[r]) > 60 or rng.random() < 0.1:
                new.append(-len(told[r]) if rng.random() < 0.7 else -3)
            else:
                new.append(1)
        lens = [len(t) for t in told]
        paged.page_advance(tables, torch.tensor(new, dtype=torch.int32, device=DEV), slots, positions)
        tables.check()
        n = sum(max(x, 0) for x in new)
        k, v = (torch.randn(n, kv, d, generator=g, device=DEV).to(dtype) for _ in range(2))
        paged.paged_write(k, v, slots[:n], kp, vp, *scales)
        at = 0
        for r, x in enumerate(new):
            if x < 0:
                told[r] = told[r][:max(len(told[r]) + x, 0)]
            for i in range(max(x, 0)):
                told[r].append((store(k[at + i]), store(v[at + i])))
            if x > 0:
                assert positions[at:at + x].tolist() == list(range(lens[r], lens[r] + x))
            at += max(x, 0)
        assert tables.seq_lens.tolist() == [len(t) for t in told]
        held = [p for r in range(slots_n) for p in tables.block_table[r, :-(-len(told[r]) // page)].tolist()]
        assert len(set(held)) == len(held) and len(held) + int(tables.state[1]) == 40
        q = torch.randn(slots_n, 1, hq, d, generator=g, device=DEV).to(dtype)
        out = paged.paged_attention(q, kp, vp, tables.block_table, tables.seq_lens, k_scale=scales[0], v_scale=scales[1])
        for r in range(slots_n):
            for h in range(kv):
                rows = [np.stack([x[i][h].double().cpu().numpy() for x in told[r]]) if told[r] else np.zeros((0, d))
                        for i in range(2)]
                ref, _, mass = op.attention(q[r, 0, 3 * h:3 * h + 3].double().cpu().numpy(), *rows, d ** -0.5)
                err = np.abs(out[r, 0, 3 * h:3 * h + 3].double().cpu().numpy() - ref)
                assert (err <= U[dtype] * np.abs(ref) + mass * 2.0 ** -12).all()


def test_plans_and_captures_in_any_order():
    """Captures begun on a side stream right behind the making of the plan, a
    plan made inside a capture, eager runs of either before and after replays."""
    c = Case([9000, 7, 0, 1500], 8, 2, 128, 16, seed=43)
    want, want_lse = c.attend(return_softmax_lse=True)
    nbytes = lib().zkv_paged_attention_workspace_size(128)
    torch.full((nbytes,), 255, dtype=torch.uint8, device=DEV)       # (freed: what torch.empty may find)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs, plans = [torch.cuda.CUDAGraph() for _ in range(2)], []
    plans.append(paged.PagedAttentionPlan(c.q, c.k, c.v, c.table, c.lens, return_softmax_lse=True))
    for i, g in enumerate(graphs):
        with torch.cuda.stream(side):
            g.capture_begin()
            if i == 1:
                plans.append(paged.PagedAttentionPlan(c.q, c.k, c.v, c.table, c.lens, return_softmax_lse=True))
            plans[i].run()
            g.capture_end()

    def same(plan):
        side.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(plan.out[0], want) and torch.equal(plan.out[1], want_lse)
        for x in plan.out:
            x.fill_(9.0)
        torch.cuda.synchronize()

    plans[1].run()                                # eager, before the graph it was made in has run
    same(plans[1])
    for _ in range(3):
        for g, plan in zip(graphs, plans):
            with torch.cuda.stream(side):
                g.replay()
            same(plan)
            plan.run()
            same(plan)
