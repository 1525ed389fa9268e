"""GPU: the model's decode step with 8-bit projections over the paged cache and
over polar_cache: every call it makes against 64 bits on that call's own inputs,
what goes from one to the next, and whole steps replayed from a graph.

(Against another evaluation of the whole step there is no useful bound: where a
value lies next to the border of two codes, sums that differ in their last bits
take different ones, a step of 2^-3.)"""
import pytest
import torch

from fp8_cases import check_gated, check_linear, check_norm, check_rows, weight_values
from zoomkv_revision_amd import decode_step as ds
from zoomkv_revision_amd import fp8

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
BF = torch.bfloat16
GEO = ds.Qwen3Geometry(layers=3, hidden=512, heads=8, kv_heads=2, ffn=1000, vocab=1000)


def _prompted(lens, seed=7, idle=(), **kw):
    model = ds.RandomQwen3(GEO, DEV, seed=seed, max_position=2048, weights="fp8")
    cache = ds.build_paged_cache(GEO, len(lens), 1500, DEV, **kw)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for r, n in enumerate(lens):
        for layer in range(GEO.layers):
            k, v = (torch.randn(1, n, 2, 128, generator=g, device=DEV).to(BF) for _ in range(2))
            if r not in idle:
                cache.prefill_update_kv_cache(None, k, v, layer, r)
    return model, cache


def test_weights_quantised_on_the_device_as_on_the_host():
    model = ds.RandomQwen3(GEO, DEV, seed=1, max_position=64, weights="fp8")
    g = torch.Generator(device=DEV).manual_seed(1)
    w = (torch.randn(2 * GEO.ffn, GEO.hidden, generator=g, device=DEV) * 0.02).to(BF)
    a, b = fp8.quantize_weight(w, 2), ds.quantize_weight_torch(w.cpu(), 2)
    assert torch.equal(a.codes.cpu().float(), b.codes.float()) and torch.equal(a.scales.cpu(), b.scales)
    L = model.layers[0]
    assert torch.equal(L["down"].dequantize().double(), weight_values(L["down"].codes, L["down"].scales).float().double())


class Recorder:
    """Calls of the fp8 operators and of cache.compute, with their results."""

    def __init__(self, monkeypatch, cache):
        self.calls = []
        for where, name in [(fp8, n) for n in ("rms_norm_quant", "quantize_rows", "linear", "gated_linear")] + \
                [(cache, "compute")]:
            monkeypatch.setattr(where, name, self._wrapped(name, getattr(where, name)))

    def _wrapped(self, name, fn):
        def call(*args, **kw):
            out = fn(*args, **kw)
            self.calls.append((name, args, kw, out))
            return out
        return call


def _check_step(model, calls, hidden):
    """The calls of one decode step whose layers start from `hidden`."""
    per = ["rms_norm_quant", "linear", "compute", "quantize_rows", "linear", "rms_norm_quant", "gated_linear", "linear"]
    assert [c[0] for c in calls] == per * len(model.layers)
    for i, L in enumerate(model.layers):
        norm1, qkv, attn, rows, o, norm2, gated, down = calls[8 * i:8 * i + 8]
        assert norm1[1][0].data_ptr() == hidden.data_ptr() and norm1[1][1] is L["input_ln"] and not norm1[2]
        check_norm(hidden, L["input_ln"], GEO.eps, None, *norm1[3])
        assert qkv[1][0] is norm1[3][0] and qkv[1][1] is norm1[3][1] and qkv[1][2] is L["wqkv"] and not qkv[2]
        check_linear(*qkv[1], None, qkv[3])
        x = rows[1][0]
        assert x.data_ptr() == attn[3].data_ptr() and x.shape == (hidden.shape[0], attn[3][0].numel())
        check_rows(x, *rows[3])
        assert o[1][0] is rows[3][0] and o[1][2] is L["wo"] and not o[2]
        check_linear(*o[1], None, o[3])
        assert norm2[1][0] is o[3] and norm2[1][1] is L["post_ln"] and norm2[2]["residual"].data_ptr() == hidden.data_ptr()
        check_norm(o[3], L["post_ln"], GEO.eps, hidden, *norm2[3])
        assert gated[1][0] is norm2[3][0] and gated[1][1] is norm2[3][1] and gated[1][2] is L["gate_up"]
        check_gated(*gated[1], *gated[3])
        assert down[1][0] is gated[3][0] and down[1][2] is L["down"] and down[2]["residual"] is norm2[3][2]
        check_linear(*down[1], norm2[3][2], down[3])
        hidden = down[3]
    return hidden


@pytest.mark.parametrize("rows", [1, 5, 16, 17, 70])
def test_every_call_of_a_step(rows, monkeypatch):
    model, cache = _prompted([1 + 37 * r % 300 for r in range(rows)])
    tok = torch.arange(rows, device=DEV) * 13 % GEO.vocab
    for _ in range(2):
        with monkeypatch.context() as m:
            rec = Recorder(m, cache)
            logits = model.decode_step(tok, cache)
        # (the embedding's rows, as the first layer was given them)
        hidden = rec.calls[0][1][0]
        assert torch.equal(hidden, model.embed[tok])
        last = _check_step(model, rec.calls, hidden)
        want = ds.rms_norm(last, model.final_norm, GEO.eps).double() @ model.embed.double().t()
        assert ((logits.double() - want).abs() <= 4 * 2.0 ** -8 * want.abs().amax(-1, keepdim=True)).all()
        tok = logits.argmax(-1)
    cache.check()


@pytest.mark.parametrize("rows", [1, 5, 16, 17, 70])
def test_captured_steps_replay_as_the_next_ones(rows):
    lens = [1 + 37 * r % 300 for r in range(rows)]
    idle = (3,) if rows > 3 else ()
    model, eager = _prompted(lens, idle=idle)
    _, replayed = _prompted(lens, idle=idle)
    tok = torch.arange(rows, device=DEV) * 13 % GEO.vocab
    keep = [r for r in range(rows) if r not in idle]
    model.decode_step(tok, replayed)                   # warm-up: a step of its own
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode_step(tok, replayed)
    for step in range(6):
        got = model.decode_step(tok, eager)
        if step:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(logits[keep], got[keep]), step
    eager.check()


def test_rows_do_not_depend_on_their_neighbours():
    """A row of zeros where a request is idle, or one that is not finite, leaves
    the others' bits as they are."""
    model, _ = _prompted([5])
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(6, GEO.hidden, generator=g, device=DEV).to(BF)
    L = model.layers[1]

    def block(x):
        codes, scales = fp8.rms_norm_quant(x, L["post_ln"], GEO.eps)
        return fp8.linear(*fp8.gated_linear(codes, scales, L["gate_up"]), L["down"], residual=x)

    want = block(x)
    for bad in (0.0, float("nan"), float("inf")):
        y = x.clone()
        y[2] = bad
        got = block(y)
        keep = [0, 1, 3, 4, 5]
        assert torch.equal(got[keep], want[keep])
        assert bool(got[2].isnan().all()) == (bad != 0.0)


def test_polar_cache_step(monkeypatch):
    for k, v in ds.PRODUCTION_ENV.items():
        monkeypatch.setenv(k, v)
    monkeypatch.delenv("POLAR_FORCE_CAND_TOKENS", raising=False)
    geo = ds.Qwen3Geometry(layers=2, hidden=256, heads=32, kv_heads=8, head_dim=128, ffn=512, vocab=1000)
    model = ds.RandomQwen3(geo, DEV, seed=42, max_position=8192, weights="fp8")
    cache = ds.build_cache(geo, 2, 4096, 8, 64, 2048, DEV)
    ds.fill_cache(cache, geo, 2, 4096, 43, DEV)
    tok = torch.tensor([5, 77], device=DEV)
    for step in range(3):
        with monkeypatch.context() as m:
            rec = Recorder(m, cache)
            model.decode_step(tok, cache)
        _check_step(model, rec.calls, rec.calls[0][1][0])
        assert cache.context == 4096 + step + 1


def test_the_torch_layer_takes_the_same_weights():
    """layer_decode_torch on the device: its products of the same rows, to the bound
    of an fp32 matrix product and a bf16 rounding."""
    model, _ = _prompted([5])
    x = torch.randn(9, GEO.hidden, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    for name in ("wqkv", "gate_up"):
        codes, scales = ds.quantize_rows_torch(x)
        check_rows(x, codes, scales)
        check_linear(codes, scales, model.layers[0][name], None, ds.linear_fp8_torch(x, model.layers[0][name]))
