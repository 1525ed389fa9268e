"""Paged attention on calls whose result shows every tile (tests/paged_cases.py):
long requests divided over waves and workgroups, with joins in one step and in
two, heads in sets, cuts moved out of short units.  tests/test_paged_bounds.py has
what the bounds can see."""
import numpy as np
import pytest
import torch

from tests.paged_cases import CALLS, TILE, name
from zoomkv_revision_amd import paged

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PAGE = 48


def _inputs(c):
    """The requests share their pages, which lie in the pool in another order."""
    dtype = TYPES[c.type]
    n = max(c.lens)
    pages = -(-n // PAGE)
    t = torch.arange(pages * PAGE, device=DEV)
    rows = torch.zeros(2, pages * PAGE, c.kv, c.d, device=DEV)
    rows[0, :, :, 0] = c.log2_weight(t)[:, None].float()
    for h in range(c.kv):
        rows[1, t, h, t // TILE % c.d] = 1.0 + h
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).to(DEV)
    table = order.int().repeat(len(c.lens), 1)
    pools = []
    for x in rows:
        x = x.to(torch.float8_e4m3fn if c.fp8 else dtype).view(pages, PAGE, c.kv, c.d)
        raw = x.view(torch.uint8) if c.fp8 else x
        there = torch.empty_like(raw)
        there[order] = raw                                            # [page, token, head]
        there = there.transpose(1, 2)
        there = there if c.nhd else there.contiguous()
        pools.append(there.view(torch.float8_e4m3fn) if c.fp8 else there)
    q = torch.zeros(len(c.lens), c.hq, c.d, dtype=dtype, device=DEV)
    q[..., 0] = torch.tensor([c.times(h) for h in range(c.hq)], device=DEV).to(dtype)
    return q, *pools, table, torch.tensor(c.lens, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("call", CALLS, ids=name)
@pytest.mark.parametrize("out_f32", [True, False])
def test_every_tile_is_there_once(call, out_f32):
    args = _inputs(call)
    out = torch.empty(args[0].shape, dtype=torch.float32, device=DEV) if out_f32 else None
    out, lse = paged.paged_attention(*args, softmax_scale=float(np.log(2.0)), window=call.window, out=out,
                                     return_softmax_lse=True)
    half_step = 2.0 ** -24 if out_f32 else torch.finfo(TYPES[call.type]).eps / 2
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()[..., 0]
    known = {}
    for b, n in enumerate(call.lens):
        for h in range(call.hq):
            key = n, h // (call.hq // call.kv), call.times(h)
            if key not in known:
                known[key] = call.reference(n, h)
            ref, ref_lse = known[key]
            # (values below fp16's smallest normal number are rounded to a step of 2^-24)
            assert (np.abs(got[b, h] - ref) <= call.out_bound(ref, half_step) + (not out_f32) * 2.0 ** -25).all(), (b, h)
            if n == 0:
                assert np.isneginf(got_lse[b, h])
            else:
                assert abs(got_lse[b, h] - ref_lse) <= call.lse_bound(ref_lse), (b, h)


@pytest.mark.parametrize("call", [c for c in CALLS if c.sets], ids=name)
def test_heads_in_sets_give_the_same_bits_every_time(call):
    q, k, v, table, lens = _inputs(call)
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(q.shape, generator=g, device=DEV).to(q.dtype)
    first = paged.paged_attention(q, k, v, table, lens, window=call.window, return_softmax_lse=True)
    for _ in range(20):
        again = paged.paged_attention(q, k, v, table, lens, window=call.window, return_softmax_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
