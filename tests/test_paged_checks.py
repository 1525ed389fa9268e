"""What the paged-cache calls refuse before any launch (host checks only, on
CPU tensors: the last check is that they are on the GPU)."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from zoomkv_revision_amd import paged
from zoomkv_revision_amd._lib import ZkvError

P, KV, PAGE, D, BS, HQ, W = 6, 2, 16, 128, 3, 8, 4
BF = torch.bfloat16


def _pool(dtype=BF, shape=(P, KV, PAGE, D)):
    return torch.zeros(shape, dtype=dtype)


def _attend(**changed):
    a = dict(q=torch.zeros(BS, 1, HQ, D, dtype=BF), k_pages=_pool(), v_pages=_pool(),
             block_table=torch.zeros(BS, W, dtype=torch.int32), seq_lens=torch.ones(BS, dtype=torch.int32))
    a.update(changed)
    return a


def _write(**changed):
    a = dict(k=torch.zeros(5, KV, D, dtype=BF), v=torch.zeros(5, KV, D, dtype=BF),
             slots=torch.zeros(5, dtype=torch.int64), k_pages=_pool(), v_pages=_pool())
    a.update(changed)
    return a


def _rope(**changed):
    a = dict(qkv=torch.zeros(5, (HQ + 2 * KV) * D, dtype=BF), heads=HQ, kv_heads=KV, q_norm=torch.ones(D, dtype=BF),
             k_norm=torch.ones(D, dtype=BF), eps=1e-6, cos=torch.ones(32, D // 2), sin=torch.zeros(32, D // 2),
             positions=torch.zeros(5, dtype=torch.int32), slots=torch.zeros(5, dtype=torch.int64),
             q_out=torch.zeros(5, HQ, D, dtype=BF), k_pages=_pool(), v_pages=_pool())
    a.update(changed)
    return a


def _tables(**changed):
    t = paged.PageTables.allocate(BS, 64, 40, PAGE, device="cpu")
    for k, v in changed.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("call,args", [(paged.paged_attention, _attend), (paged.paged_write, _write),
                                       (paged.paged_qk_norm_rope, _rope), (paged.PagedAttentionPlan, _attend),
                                       (paged.PagedWritePlan, _write), (paged.PagedRopePlan, _rope)])
def test_matching_buffers_pass_the_host_checks(call, args):
    with pytest.raises(ZkvError, match="device tensors"):
        call(**args())
    with pytest.raises(ZkvError, match="device tensors"):
        call(**args(k_pages=_pool(torch.float8_e4m3fn), v_pages=_pool(torch.float8_e4m3fn),
                    k_scale=torch.ones(KV), v_scale=torch.ones(KV)))
    nhd = torch.zeros(P, PAGE, KV, D, dtype=BF).transpose(1, 2)
    with pytest.raises(ZkvError, match="device tensors"):
        call(**args(k_pages=nhd, v_pages=nhd))


def test_matching_tables_pass_the_host_checks():
    with pytest.raises(ZkvError, match="device tensors"):
        paged.page_advance(_tables(), torch.ones(BS, dtype=torch.int32), torch.zeros(4, dtype=torch.int64),
                           torch.zeros(4, dtype=torch.int32))


POOL_CHANGES = [
    dict(k_pages=_pool(torch.float16)),                                        # K and V of two types
    dict(k_pages=_pool(torch.float32), v_pages=_pool(torch.float32)),
    dict(k_pages=_pool(torch.float16), v_pages=_pool(torch.float16)),          # not the rows' type
    dict(v_pages=_pool(shape=(P, KV, PAGE // 2, D))),
    dict(k_pages=_pool(shape=(P, KV, PAGE, 96)), v_pages=_pool(shape=(P, KV, PAGE, 96))),
    dict(k_pages=_pool()[0], v_pages=_pool()[0]),
    dict(k_pages=_pool(shape=(0, KV, PAGE, D)), v_pages=_pool(shape=(0, KV, PAGE, D))),
    dict(v_pages=_pool(shape=(P, PAGE, KV, D)).transpose(1, 2)),               # other strides than K
    dict(k_pages=_pool(shape=(P, KV, PAGE, 2 * D))[..., ::2], v_pages=_pool(shape=(P, KV, PAGE, 2 * D))[..., ::2]),
    dict(k_pages=_pool(shape=(P, KV, PAGE, D + 4))[..., :D], v_pages=_pool(shape=(P, KV, PAGE, D + 4))[..., :D]),
    dict(k_pages=_pool(shape=(P, KV, PAGE, D + 8))[..., 4:D + 4], v_pages=_pool(shape=(P, KV, PAGE, D + 8))[..., 4:D + 4]),
    dict(k_scale=torch.ones(KV)),                                              # a scale without codes
    dict(k_pages=_pool(torch.float8_e4m3fn), v_pages=_pool(torch.float8_e4m3fn), k_scale=torch.ones(KV + 1)),
    dict(k_pages=_pool(torch.float8_e4m3fn), v_pages=_pool(torch.float8_e4m3fn), v_scale=torch.ones(KV, dtype=BF)),
    dict(k_pages=_pool(torch.float8_e4m3fn), v_pages=_pool(torch.float8_e4m3fn), v_scale=torch.ones(2 * KV)[::2]),
    dict(k_pages=_pool(torch.float8_e5m2), v_pages=_pool(torch.float8_e5m2)),
    dict(k_pages=_pool(shape=(1, KV, 1, D)).expand(1 << 16, KV, 1 << 15, D),
         v_pages=_pool(shape=(1, KV, 1, D)).expand(1 << 16, KV, 1 << 15, D)),  # 2^31 tokens
]


@pytest.mark.parametrize("call,args", [(paged.paged_attention, _attend), (paged.paged_write, _write),
                                       (paged.paged_qk_norm_rope, _rope)])
@pytest.mark.parametrize("i", range(len(POOL_CHANGES)))
def test_pools_the_kernels_cannot_read_are_refused(call, args, i):
    with pytest.raises((ValueError, TypeError)):
        call(**args(**POOL_CHANGES[i]))


@pytest.mark.parametrize("changed", [
    dict(q=torch.zeros(BS, 2, HQ, D, dtype=BF)),                   # two query tokens
    dict(q=torch.zeros(BS, 1, HQ, 64, dtype=BF)),
    dict(q=torch.zeros(BS, 1, 7, D, dtype=BF)),                    # 7 heads over 2
    dict(q=torch.zeros(BS, 1, HQ, D)),
    dict(q=torch.zeros(0, 1, HQ, D, dtype=BF), block_table=torch.zeros(0, W, dtype=torch.int32),
         seq_lens=torch.zeros(0, dtype=torch.int32)),
    dict(q=torch.zeros(4097, 1, HQ, D, dtype=BF), block_table=torch.zeros(4097, W, dtype=torch.int32),
         seq_lens=torch.zeros(4097, dtype=torch.int32)),
    dict(block_table=torch.zeros(BS, W, dtype=torch.int64)),
    dict(block_table=torch.zeros(BS + 1, W, dtype=torch.int32)),
    dict(block_table=torch.zeros(BS, 0, dtype=torch.int32)),
    dict(block_table=torch.zeros(BS, 2 * W, dtype=torch.int32)[:, ::2]),
    dict(block_table=torch.zeros(1, 1, dtype=torch.int32).expand(BS, 1 << 27)),  # 2^31 tokens a request
    dict(seq_lens=torch.ones(BS, dtype=torch.int64)),
    dict(seq_lens=torch.ones(BS + 1, dtype=torch.int32)),
    dict(seq_lens=torch.ones(2 * BS, dtype=torch.int32)[::2]),
    dict(window=-1),
    dict(k_pages=_pool(shape=(1, KV, PAGE, D)).expand(1 << 20, KV, PAGE, D).as_strided(
        (1 << 20, KV, PAGE, D), (0, PAGE * D, D, 1)), v_pages=_pool(), q=torch.zeros(BS, 1, HQ, D, dtype=BF)),
    dict(out=torch.zeros(BS, 1, HQ, D, dtype=torch.float16)),
    dict(out=torch.zeros(BS, 1, HQ, 2 * D, dtype=BF)[..., :D]),
    dict(out=torch.zeros(BS, 1, HQ - 1, D, dtype=BF)),
])
def test_attention_refusals(changed):
    with pytest.raises((ValueError, TypeError)):
        paged.paged_attention(**_attend(**changed))


@pytest.mark.parametrize("changed", [
    dict(k=torch.zeros(5, KV + 1, D, dtype=BF), v=torch.zeros(5, KV + 1, D, dtype=BF)),
    dict(v=torch.zeros(5, KV, D, dtype=torch.float16)),
    dict(v=torch.zeros(4, KV, D, dtype=BF)),
    dict(slots=torch.zeros(4, dtype=torch.int64)),
    dict(slots=torch.zeros(5, dtype=torch.int32)),
    dict(slots=torch.zeros(10, dtype=torch.int64)[::2]),
])
def test_write_refusals(changed):
    with pytest.raises((ValueError, TypeError)):
        paged.paged_write(**_write(**changed))


@pytest.mark.parametrize("changed", [
    dict(heads=HQ + 1), dict(kv_heads=KV + 1), dict(heads=0),
    dict(q_norm=torch.ones(D)), dict(k_norm=torch.ones(D - 8, dtype=BF)), dict(q_norm=torch.ones(2 * D, dtype=BF)[::2]),
    dict(cos=torch.ones(32, D)), dict(sin=torch.ones(31, D // 2)), dict(cos=torch.ones(32, D // 2, dtype=BF)),
    dict(cos=torch.ones(0, D // 2), sin=torch.ones(0, D // 2)),
    dict(positions=torch.zeros(5, dtype=torch.int64)), dict(positions=torch.zeros(4, dtype=torch.int32)),
    dict(slots=torch.zeros(5, dtype=torch.int32)),
    dict(q_out=torch.zeros(5, HQ, D)), dict(q_out=torch.zeros(5, 2 * HQ, D, dtype=BF)[:, ::2]),
    dict(q_out=torch.zeros(4, HQ, D, dtype=BF)),
])
def test_rope_refusals(changed):
    with pytest.raises((ValueError, TypeError)):
        paged.paged_qk_norm_rope(**_rope(**changed))


@pytest.mark.parametrize("plan,args,changed", [
    (paged.PagedAttentionPlan, _attend, dict(q=torch.zeros(BS, 1, HQ, D + 4, dtype=BF)[..., :D])),
    (paged.PagedWritePlan, _write, dict(k=torch.zeros(5, KV, D + 4, dtype=BF)[..., :D])),
    (paged.PagedRopePlan, _rope, dict(qkv=torch.zeros(5, (HQ + 2 * KV) * D + 4, dtype=BF)[:, :(HQ + 2 * KV) * D])),
])
def test_plans_refuse_inputs_that_a_call_would_copy(plan, args, changed):
    with pytest.raises(ValueError, match="in place"):
        plan(**args(**changed))


def test_tables_refusals():
    new = torch.ones(BS, dtype=torch.int32)
    slots, i32 = torch.zeros(4, dtype=torch.int64), dict(dtype=torch.int32)
    for tables in (_tables(block_table=torch.zeros(BS, 4, dtype=torch.int64)),
                   _tables(block_table=torch.zeros(BS + 1, 4, **i32)),
                   _tables(block_table=torch.zeros(BS, 0, **i32)),
                   _tables(block_table=torch.zeros(1, 4, **i32).expand(BS, 4)),     # rows that are one
                   _tables(block_table=torch.zeros(BS, 8, **i32)[:, ::2]),
                   _tables(seq_lens=torch.zeros(BS, dtype=torch.int64)),
                   _tables(free_pages=torch.zeros(0, **i32)),
                   _tables(state=torch.zeros(3, **i32)),
                   _tables(page_size=0), _tables(page_size=1 << 30)):
        with pytest.raises(ValueError):
            paged.page_advance(tables, new, slots)
    for changed in (dict(new_tokens=new.long()), dict(new_tokens=new[:2]), dict(slots=slots.int()),
                    dict(slots=torch.zeros(8, dtype=torch.int64)[::2]), dict(positions=torch.zeros(3, **i32)),
                    dict(starts=torch.zeros(BS, **i32)), dict(lens_out=torch.zeros(BS + 1, **i32)),
                    dict(state_out=torch.zeros(5, **i32)), dict(row=-1), dict(row=1),
                    dict(slots=torch.zeros(BS, dtype=torch.int64), row=1, starts=torch.zeros(BS + 1, **i32))):
        with pytest.raises(ValueError):
            paged.page_advance(**{**dict(tables=_tables(), new_tokens=new, slots=slots), **changed})
    big = paged.MAX_TABLE_REQUESTS + 1
    with pytest.raises(ValueError):
        paged.page_advance(paged.PageTables.allocate(big, 16, 4, 16, device="cpu"), torch.ones(big, **i32), slots)
    for bad in (dict(requests=0), dict(max_tokens=0), dict(num_pages=0), dict(page_size=0)):
        with pytest.raises(ValueError):
            paged.PageTables.allocate(**{**dict(requests=1, max_tokens=1, num_pages=1, page_size=1, device="cpu"), **bad})


def test_status_bits_become_an_error():
    t = _tables()
    t.check()
    t.state[2] = paged.POOL_EMPTY | paged.TABLE_FULL
    with pytest.raises(RuntimeError, match="no free pages.*block table"):
        t.check()


def test_the_c_entries_refuse_too():
    """Sizes the Python layer would have stopped, straight at the C ABI (no
    launch is reached), on a thread of their own: the error text is the
    thread's."""
    with ThreadPoolExecutor(1) as ex:
        ex.submit(_c_refusals).result()


def _c_refusals():
    from zoomkv_revision_amd._lib import lib
    L = lib()
    x = torch.zeros(1 << 16, dtype=torch.uint8).data_ptr() // 16 * 16 + 16
    attend = lambda **c: L.zkv_paged_attention(*{**dict(
        q=x, q_sb=1024, q_sh=128, f16=0, k=x, v=x, fp8=0, ks=None, vs=None, pages=4, page=16, ps=4096, hs=2048, ts=128,
        table=x, tstride=4, width=4, lens=x, bs=1, hq=8, kv=2, d=128, scale=1.0, window=0, out=x, f32=0, lse=None,
        ws=x, wsb=1 << 30, stream=None), **c}.values())
    for c in (dict(q=None), dict(d=96), dict(bs=0), dict(bs=4097), dict(hq=7), dict(kv=0), dict(width=0),
              dict(pages=0), dict(page=0), dict(ts=4), dict(ps=-8), dict(q_sb=4), dict(q=x + 2), dict(window=-1),
              dict(width=1 << 27), dict(pages=1 << 28), dict(pages=1 << 20, ps=1 << 16), dict(bs=4096, width=1 << 20), dict(ws=x + 8)):
        assert attend(**c) == 1, c
    assert attend(wsb=1000) == 3
    assert L.zkv_paged_attention_workspace_size(96) == 0
    write = lambda **c: L.zkv_paged_write(*{**dict(
        k=x, kt=256, kh=128, v=x, vt=256, vh=128, slots=x, n=4, kv=2, d=128, f16=0, kp=x, vp=x, fp8=0, ks=None, vs=None,
        pages=4, page=16, ps=4096, hs=2048, ts=128, stream=None), **c}.values())
    for c in (dict(slots=None), dict(n=-1), dict(kt=4), dict(d=80), dict(kp=x + 2), dict(n=1 << 30), dict(ts=4)):
        assert write(**c) == 1, c
    assert write(n=0) == 0
    advance = lambda **c: L.zkv_page_advance(*{**dict(
        lens=x, new=x, n=4, table=x, tstride=8, width=8, ring=x, pages=4, page=16, state=x, slots=x, pos=None, cap=4,
        row=0, starts=None, lo=x, so=x, stream=None), **c}.values())
    for c in (dict(n=0), dict(n=8193), dict(width=0), dict(tstride=7), dict(page=0), dict(pages=0), dict(cap=-1),
              dict(slots=None), dict(state=None), dict(page=1 << 30), dict(row=-1), dict(row=2),
              dict(row=1, starts=x)):
        assert advance(**c) == 1, c
    rope = lambda **c: L.zkv_paged_qk_norm_rope(*{**dict(
        qkv=x, stride=1536, n=4, hq=8, kv=2, d=128, f16=0, qn=x, kn=x, eps=1e-6, cos=x, sin=x, maxp=4, pos=x, slots=x,
        qo=x, kp=x, vp=x, fp8=0, ks=None, vs=None, pages=4, page=16, ps=4096, hs=2048, ts=128, stream=None), **c}.values())
    for c in (dict(pos=None), dict(n=-1), dict(hq=0), dict(maxp=0), dict(stride=12), dict(cos=x + 4), dict(n=1 << 27),
              dict(d=32)):
        assert rope(**c) == 1, c
    assert rope(n=0) == 0
    assert L.zkv_last_error().startswith(b"zkv_paged_qk_norm_rope: ")
