"""paged_cache on the GPU: its bookkeeping and attention against float64 over
the rows it was given, the decode step of the model over it (fused launches,
torch ops, captured and replayed), and the paged arguments of
flash_attn_with_kvcache_compat."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from zoomkv_revision_amd import decode_step as ds
from zoomkv_revision_amd.attention import flash_attn_with_kvcache_compat
from zoomkv_revision_amd.paged_cache import paged_cache

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
BF = torch.bfloat16


def _cache(batch=3, layers=2, kv=2, hq=4, d=128, max_length=200, page=8, **kw):
    kw = {"dtype": BF, "valid_start": [0] * batch, **kw}
    return paged_cache(layer_num=layers, batch_size=batch, max_length=max_length, num_key_value_heads=kv, num_heads=hq,
                       head_dim=d, layer_mapping={"0": "cuda:0"}, max_new_length=50, page_size=page, **kw)


def _check_attention(c, told, layer, g, half_step=2.0 ** -8):
    q = torch.randn(c.batch_size, 1, c.num_heads, c.head_dim, generator=g, device=DEV).to(c.dtype)
    out = c.compute(q, layer).double().cpu().numpy()
    group = c.num_heads // c.kv_head
    for r, rows in enumerate(told[layer]):
        for h in range(c.kv_head):
            k, v = (np.stack([x[i][h] for x in rows]) if rows else np.zeros((0, c.head_dim)) for i in range(2))
            ref, _, mass = op.attention(q[r, 0, h * group:(h + 1) * group].double().cpu().numpy(), k, v,
                                        c.head_dim ** -0.5)
            err = np.abs(out[r, 0, h * group:(h + 1) * group] - ref)
            assert (err <= half_step * np.abs(ref) + mass * 2.0 ** -12).all(), (layer, r, h)


@pytest.mark.parametrize("dtype,kv_dtype", [(BF, None), (torch.float16, None), (BF, torch.float8_e4m3fn)])
def test_requests_of_their_own_lengths(dtype, kv_dtype):
    """A left-padded batch, decode steps, a request that ends and one that
    takes its row; the pool is shared and holds just what is used."""
    c = _cache(dtype=dtype, kv_dtype=kv_dtype, valid_start=[5, 0, 29], num_pages=22)
    g = torch.Generator(device=DEV).manual_seed(1)
    scales = [0.01, 0.02]
    if kv_dtype is not None:
        for i in range(2):
            c.k_scale[i] = torch.full((2,), scales[0], device=DEV)
            c.v_scale[i] = torch.full((2,), scales[1], device=DEV)
    new = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)

    def stored(x, s):
        if kv_dtype is None:
            return x.double().cpu().numpy()
        one = torch.tensor(s, device=DEV)
        return ((x.float() / one).clamp(-448, 448).to(kv_dtype).double() * one.double()).cpu().numpy()

    def rows(k, v):
        return list(zip(stored(k, scales[0]), stored(v, scales[1])))

    told = [[[] for _ in range(3)] for _ in range(2)]
    seq, step = 33, {BF: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    for layer in range(2):
        k, v = new(3, seq, 2, 128), new(3, seq, 2, 128)
        kk, vv = c.prefill_update_kv_cache(None, k, v, layer, 0)
        assert torch.equal(kk, k) and torch.equal(vv, v)
        for b in (1, 2):
            c.prefill_update_kv_cache(None, k, v, layer, b)          # (rows beyond the first: nothing left to do)
        for r, s in enumerate((5, 0, 29)):
            told[layer][r] = rows(k[r, s:], v[r, s:])
    assert c.tables.seq_lens.tolist() == [28, 33, 4] and c.context == 33

    def decode():
        k, v = [new(3, 1, 2, 128) for _ in range(2)], [new(3, 1, 2, 128) for _ in range(2)]
        for layer in range(2):
            c.decode_update_kv_cache(k[layer], v[layer], layer)
            for r in range(3):
                if told[layer][r]:
                    told[layer][r] += rows(k[layer][r], v[layer][r])
            _check_attention(c, told, layer, g, step)

    for _ in range(6):
        decode()
    assert c.context == 39 and c.lengths == [34, 39, 10]
    c.release(1)
    for layer in range(2):
        told[layer][1] = []
    decode()
    assert c.tables.seq_lens.tolist() == [35, 0, 11] and c.slots[1] == -1 and c.positions.tolist() == [34, -1, 10]
    # a prompt for the free row, and one that replaces a running request
    for r, n in ((1, 20), (0, 50)):
        c.valid_start = [0, 3, 0]
        s = 3 if r == 1 else 0
        for layer in range(2):
            k, v = new(1, n + s, 2, 128), new(1, n + s, 2, 128)
            kk, _ = c.prefill_update_kv_cache(None, k, v, layer, r)
            assert kk.shape[1] == n
            told[layer][r] = rows(k[0, s:], v[0, s:])
    decode()
    c.check()
    assert c.lengths == [51, 21, 12] == c.tables.seq_lens.tolist()
    held = sum(-(-n // 8) for n in c.lengths)
    assert int(c.tables.state[1]) == 22 - held


def test_refusals():
    c = _cache(num_pages=9)
    new = lambda *s: torch.zeros(*s, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="layer 0"):
        c.prefill_update_kv_cache(None, new(1, 8, 2, 128), new(1, 8, 2, 128), 1, 0)
    with pytest.raises(RuntimeError, match="max_length"):
        c.prefill_update_kv_cache(None, new(1, 201, 2, 128), new(1, 201, 2, 128), 0, 0)
    with pytest.raises(RuntimeError, match="pages"):
        c.prefill_update_kv_cache(None, new(1, 80, 2, 128), new(1, 80, 2, 128), 0, 0)
    with pytest.raises(ValueError):
        c.prefill_update_kv_cache(None, new(2, 8, 2, 128), new(2, 8, 2, 128), 0, 0)
    with pytest.raises(ValueError):
        c.prefill_update_kv_cache(None, new(1, 8, 2, 64), new(1, 8, 2, 64), 0, 0)
    with pytest.raises(ValueError):
        c.release(3)
    assert c.lengths == [0, 0, 0] and c.tables.seq_lens.tolist() == [0, 0, 0]
    for layer in range(2):
        c.prefill_update_kv_cache(None, new(1, 72, 2, 128), new(1, 72, 2, 128), layer, 2)
    with pytest.raises(RuntimeError, match="pages"):
        c.decode_begin(0)
    c.check()
    for bad in (dict(dtype=torch.float32), dict(kv_dtype=torch.float16), dict(d=96), dict(hq=3), dict(batch=0)):
        with pytest.raises(ValueError):
            _cache(**bad)


GEO = ds.Qwen3Geometry(layers=3, hidden=512, heads=8, kv_heads=2, ffn=1024, vocab=1000)


def _prompted(lens, seed=7, idle=(), **kw):
    model = ds.RandomQwen3(GEO, DEV, seed=seed, max_position=2048)
    cache = ds.build_paged_cache(GEO, len(lens), 1500, DEV, **kw)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for r, n in enumerate(lens):
        for layer in range(GEO.layers):
            k, v = (torch.randn(1, n, 2, 128, generator=g, device=DEV).to(BF) for _ in range(2))
            if r not in idle:
                cache.prefill_update_kv_cache(None, k, v, layer, r)
    return model, cache


def test_decode_step_equals_the_torch_layer():
    """The fused launches against the torch ops of the same layer, rows at
    positions of their own, one of them idle.  The torch layer rounds the normed
    heads, the rotated ones and every product to bf16; logits of this width stay
    within 8 of their bf16 units of each other, as for polar_cache."""
    lens = [1000, 17, 300, 64, 5]
    model, a = _prompted(lens, idle=(3,))
    _, b = _prompted(lens, idle=(3,))
    tok = torch.tensor([1, 20, 300, 4, 999], device=DEV)
    for step in range(4):
        model.fused = True
        la = model.decode_step(tok, a)
        model.fused = False
        lb = model.decode_step(tok, b)
        unit = lb.abs().amax(-1, keepdim=True) * 2.0 ** -7
        keep = [0, 1, 2, 4]
        assert bool(((la - lb).abs() <= 8 * unit)[keep].all()), step
        assert a.positions.tolist() == [1000 + step, 17 + step, 300 + step, -1, 5 + step] == b.positions.tolist()
        tok = la.argmax(-1)
    assert a.context == 1004 and a.lengths == [1004, 21, 304, 0, 9]


def test_rows_do_not_depend_on_their_neighbours():
    """Each request decodes alone as in the batch (the attention's cuts, and with
    them the last bits, follow the whole batch's lengths)."""
    lens = [700, 33, 120]
    model, cache = _prompted(lens)
    tok = torch.tensor([5, 6, 7], device=DEV)
    logits = [model.decode_step(tok, cache) for _ in range(3)]
    for r in range(3):
        _, alone = _prompted(lens, idle=[i for i in range(3) if i != r])
        for step in range(3):
            got, want = model.decode_step(tok, alone)[r], logits[step][r]
            assert bool(((got - want).abs() <= 8 * 2.0 ** -7 * want.abs().max()).all()), (r, step)


@pytest.mark.parametrize("kv_dtype", [None, torch.float8_e4m3fn])
def test_captured_steps_replay_as_the_next_ones(kv_dtype):
    """A whole decode step in a graph: each replay appends one more token to
    every row, and gives the eager step's logits bit for bit; a release between
    replays is followed."""
    lens = [600, 15, 31]
    model, eager = _prompted(lens, kv_dtype=kv_dtype)
    _, cache = _prompted(lens, kv_dtype=kv_dtype)
    tok = torch.tensor([1, 2, 3], device=DEV)
    for c in (eager, cache):
        model.decode_step(tok, c)                      # warm-up: a step of its own
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode_step(tok, cache)
    cache.lengths = [n - 1 for n in cache.lengths]      # (captured, not run)
    cache.context -= 1
    for step in range(20):
        tok.copy_((tok * 7 + step) % GEO.vocab)
        if step == 12:
            for c in (eager, cache):
                c.release([1])
        want = model.decode_step(tok, eager)
        graph.replay()
        cache.replayed()
        torch.cuda.synchronize()
        rows = [0, 1, 2] if step < 12 else [0, 2]
        assert torch.equal(logits[rows], want[rows]), step
        assert torch.equal(cache.tables.seq_lens, eager.tables.seq_lens) and cache.lengths == eager.lengths
        assert torch.equal(cache.tables.block_table, eager.tables.block_table)
    cache.check()
    assert cache.context == eager.context == 621


def test_flash_attn_compat_takes_a_block_table():
    g = torch.Generator(device=DEV).manual_seed(4)
    new = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)
    k, v, q = new(20, 16, 2, 128), new(20, 16, 2, 128), new(3, 1, 8, 128)
    table = torch.randperm(20, generator=g, device=DEV, dtype=torch.int32)[:18].view(3, 6)
    lens = torch.tensor([90, 1, 40], dtype=torch.int32, device=DEV)
    out, lse = flash_attn_with_kvcache_compat(q, k, v, cache_seqlens=lens, block_table=table, softmax_scale=0.1,
                                              return_softmax_lse=True)
    assert out.shape == (3, 1, 8, 128) and lse.shape == (3, 8, 1)
    for b, n in enumerate(lens.tolist()):
        rows = [x[table[b].long()].reshape(-1, 1, 2, 128)[:n, 0].unsqueeze(0) for x in (k, v)]
        ref, ref_lse = flash_attn_with_kvcache_compat(q[b:b + 1], *rows, softmax_scale=0.1, return_softmax_lse=True,
                                                      out=torch.empty(1, 1, 8, 128, device=DEV))
        assert float((out[b:b + 1].float() - ref).abs().max()) <= 2e-3 + float(ref.abs().max()) * 2.0 ** -8
        assert float((lse[b:b + 1] - ref_lse).abs().max()) <= 1e-4
    with pytest.raises(NotImplementedError):
        flash_attn_with_kvcache_compat(q, k, v, cache_seqlens=lens)
    with pytest.raises(NotImplementedError):
        flash_attn_with_kvcache_compat(q, k, v, cache_seqlens=lens, block_table=table, window_size=(5, 0))
    with pytest.raises(ValueError):
        flash_attn_with_kvcache_compat(q, k, v, block_table=table)
    with pytest.raises(ValueError):
        flash_attn_with_kvcache_compat(q, k, v, cache_seqlens=lens, block_table=table, n_splits=2)


def test_the_capture_counts_as_the_first_replay():
    lens = [40, 15, 31]
    model, cache = _prompted(lens)
    tok = torch.tensor([1, 2, 3], device=DEV)
    model.decode_step(tok, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.decode_step(tok, cache)
    graph.replay()
    assert cache.tables.seq_lens.tolist() == cache.lengths == [n + 2 for n in lens]
    for _ in range(5):
        graph.replay()
    cache.replayed(5)
    cache.check()
    assert cache.tables.seq_lens.tolist() == cache.lengths == [n + 7 for n in lens] and cache.context == 47


@pytest.mark.parametrize("fused", [True, False])
def test_a_step_beyond_the_rope_table_is_refused(fused):
    """The model's RoPE table ends before the cache does: the step that would
    need a row beyond is refused with the cache as it was, and goes on once the
    long request has ended."""
    model = ds.RandomQwen3(GEO, DEV, seed=7, max_position=66, fused=fused)
    cache = ds.build_paged_cache(GEO, 2, 100, DEV)
    zeros = torch.zeros(1, 64, 2, 128, dtype=BF, device=DEV)
    for r, n in enumerate((64, 20)):
        for layer in range(GEO.layers):
            cache.prefill_update_kv_cache(None, zeros[:, :n], zeros[:, :n], layer, r)
    tok = torch.tensor([1, 2], device=DEV)
    for _ in range(2):
        assert bool(torch.isfinite(model.decode_step(tok, cache)).all())
    with pytest.raises(RuntimeError, match="position 66"):
        model.decode_step(tok, cache)
    assert cache.lengths == [66, 22] == cache.tables.seq_lens.tolist() and cache.context == 66
    cache.release(0)
    model.decode_step(tok, cache)
    assert cache.lengths == [0, 23] == cache.tables.seq_lens.tolist()
    cache.check()


def test_a_refused_prompt_leaves_the_running_request():
    """A prompt for a row that holds a request, too long for the pool or for
    max_length: the request goes on, its attention bit for bit."""
    c = _cache(layers=1, num_pages=12, max_length=80)
    g = torch.Generator(device=DEV).manual_seed(3)
    new = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)
    for r, n in ((0, 40), (2, 33)):
        c.prefill_update_kv_cache(None, new(1, n, 2, 128), new(1, n, 2, 128), 0, r)
    q = new(3, 1, 4, 128)
    before = [x.clone() for x in (c.compute(q, 0), c.tables.seq_lens, c.tables.block_table, c.tables.state, c.active)]
    for n, why in ((81, "max_length"), (64, "pages")):
        with pytest.raises(RuntimeError, match=why):
            c.prefill_update_kv_cache(None, new(1, n, 2, 128), new(1, n, 2, 128), 0, 0)
    after = c.compute(q, 0), c.tables.seq_lens, c.tables.block_table, c.tables.state, c.active
    assert all(torch.equal(a, b) for a, b in zip(after, before)) and c.lengths == [40, 0, 33]
    c.prefill_update_kv_cache(None, new(1, 56, 2, 128), new(1, 56, 2, 128), 0, 0)    # all the pages the other leaves
    assert c.lengths == [56, 0, 33] == c.tables.seq_lens.tolist()
    c.check()


def test_a_new_cache_is_ready_for_any_stream():
    """Made behind a queue of work on one stream and used on another at once."""
    g = torch.Generator(device=DEV).manual_seed(5)
    k, v, q = (torch.randn(*s, generator=g, device=DEV).to(BF) for s in ((1, 5000, 2, 128), (1, 5000, 2, 128), (3, 1, 4, 128)))
    outs = []
    side, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), side):
        for _ in range(20):
            busy = busy @ busy * 1e-3
        c = _cache(layers=1, max_length=5100)
        with torch.cuda.stream(stream):
            c.prefill_update_kv_cache(None, k, v, 0, 1)
            outs.append(c.compute(q, 0))
        torch.cuda.synchronize()
        c.check()
    assert torch.equal(*outs) and not outs[0][[0, 2]].any() and bool(outs[0][1].any())


@pytest.mark.parametrize("rows", [16, 17, 70])
def test_wide_batches_decode(rows):
    """The most rows that decode_linear takes and more: the fused step against the
    torch layer, within the bound of test_decode_step_equals_the_torch_layer, and
    replayed from a graph bit for bit."""
    lens = [1 + 37 * r % 300 for r in range(rows)]
    model, fused = _prompted(lens, idle=(3,))
    _, plain = _prompted(lens, idle=(3,))
    _, replayed = _prompted(lens, idle=(3,))
    tok = torch.arange(rows, device=DEV) * 13 % GEO.vocab
    keep = [r for r in range(rows) if r != 3]
    model.decode_step(tok, replayed)                   # warm-up: a step of its own
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode_step(tok, replayed)
    steps = []
    for step in range(5):
        model.fused = True
        steps.append(model.decode_step(tok, fused))
        model.fused = False
        want = model.decode_step(tok, plain)
        unit = want.abs().amax(-1, keepdim=True) * 2.0 ** -7
        assert bool(((steps[-1] - want).abs() <= 8 * unit)[keep].all()), step
        if step:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(logits[keep], steps[-1][keep]), step
    assert fused.lengths == plain.lengths == [0 if r == 3 else n + 5 for r, n in enumerate(lens)]
    assert torch.equal(fused.tables.seq_lens, replayed.tables.seq_lens)
    fused.check()
