"""The 8-bit linear operators, in their plain form and through the library.

Three kinds of call, over the sizes a decode step or a batch of prompts makes
them with:

  rows    a hidden state's rows as e4m3 codes with one scale per 128 channels:
          with the residual's addition and the RMS norm before it ("norm", the
          input of the qkv and gate / up projections, fp8.rms_norm_quant), or as
          they are (the attention's output, fp8.quantize_rows)
  linear  the product of such rows with a weight of e4m3 codes that has one
          scale per block of 128 x 128 (fp8.linear), a residual added on the way
          out where there is one
  gated   both projections of a gated feed-forward block, silu(gate) * up, and
          the result as codes and scales for the down projection
          (fp8.gated_linear)

Rows of codes are as long as whole blocks: ceil(K / 128) * 128, zeros behind K.
A code stands for code * scale.  The scale of a block is its largest magnitude
/ 448, the largest e4m3 value, and not below 2^-100.
"""
from __future__ import annotations

import math

import torch

own = False
_DEV = "cuda:0"
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn
_MAX = 448.0
_LEAST = 2.0 ** -100
_B = 128


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # a small decode batch between two blocks: launch and latency
        {"name": "norm_4", "kind": "rows", "M": 4, "K": 2560, "norm": True, "residual": True, "type": "bf16"},
        # the attention's output of a batch, on its way into the o-projection
        {"name": "rows_64", "kind": "rows", "M": 64, "K": 4096, "norm": False, "residual": False, "type": "bf16"},
        # rows that end inside a block, an odd number of them
        {"name": "norm_ragged", "kind": "rows", "M": 1003, "K": 2600, "norm": True, "residual": False,
         "type": "fp16"},
        # the tokens of a batch of prompts
        {"name": "norm_16384", "kind": "rows", "M": 16384, "K": 4096, "norm": True, "residual": True,
         "type": "bf16"},
        # one token's fused q, k and v
        {"name": "linear_1_qkv", "kind": "linear", "M": 1, "N": 6144, "K": 2560, "residual": False, "type": "bf16"},
        # a decode batch's down projection onto the residual stream
        {"name": "linear_16_down", "kind": "linear", "M": 16, "N": 2560, "K": 9728, "residual": True,
         "type": "bf16"},
        # sizes that end inside every tile, unrounded sums
        {"name": "linear_ragged", "kind": "linear", "M": 333, "N": 1000, "K": 2600, "residual": False,
         "type": "fp32"},
        # a short prompt, or a large decode batch: few tiles, long sums
        {"name": "linear_512_down", "kind": "linear", "M": 512, "N": 2560, "K": 9728, "residual": True,
         "type": "bf16"},
        # a batch of prompts through a wide model
        {"name": "linear_8192", "kind": "linear", "M": 8192, "N": 8192, "K": 8192, "residual": False,
         "type": "bf16"},
        # a small decode batch's gate and up
        {"name": "gated_4", "kind": "gated", "M": 4, "F": 9728, "K": 2560},
        # a block that ends inside every tile
        {"name": "gated_ragged", "kind": "gated", "M": 100, "F": 1000, "K": 2600},
        # a prompt's gate and up
        {"name": "gated_4096", "kind": "gated", "M": 4096, "F": 9728, "K": 2560},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _size(rng, lo: int, hi: int) -> int:
    """As _log, three in four of them whole blocks."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(_B, n // _B * _B)


def draw(rng) -> dict:
    kind = rng.choice(["rows", "linear", "linear", "gated"])
    if kind == "rows":
        K = _size(rng, 64, 16384)
        # at most the elements of the largest listed one, for the widest type
        return {"kind": kind, "M": _log(rng, 1, (1 << 25) // K), "K": K, "norm": rng.random() < 0.7,
                "residual": rng.random() < 0.5, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    K = _size(rng, 128, 16384)
    N = _size(rng, 64, min(151936, (1 << 27) // K))     # at most 128 MB of weights
    # half of them decode batches; at most a quarter of the largest listed one's products
    M = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 65, max(66, min(16384, (1 << 37) // (N * K))))
    if kind == "linear":
        return {"kind": kind, "M": M, "N": N, "K": K, "residual": rng.random() < 0.4,
                "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    return {"kind": kind, "M": M, "F": max(8, N // 2), "K": K}


def _blocks(n: int) -> int:
    return -(-n // _B)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _hidden(g, M: int, K: int) -> torch.Tensor:
    """Rows of a residual stream: channels and tokens of their own sizes, a few
    channels far larger than the others."""
    x = torch.randn(M, K, generator=g, device=_DEV)
    x *= (0.5 * torch.randn(K, generator=g, device=_DEV)).exp()
    x *= (0.3 * torch.randn(M, 1, generator=g, device=_DEV)).exp()
    x[:, torch.randint(0, K, (max(1, K // 512),), generator=g, device=_DEV)] *= 12.0
    return x


def _codes(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return (x / scale).clamp(-_MAX, _MAX).to(_E4M3)


def _coded_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (fp32) as codes [M, whole blocks] and scales [M, blocks]."""
    M, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % _B)).view(M, _blocks(K), _B)
    scale = (x.abs().amax(-1) / _MAX).clamp(min=_LEAST)
    return _codes(x, scale[..., None]).view(M, -1), scale


def _coded_weight(g, rows: int, K: int) -> tuple[torch.Tensor, torch.Tensor]:
    """A weight [rows, K] with a scale per block of 128 x 128."""
    nb, kb = _blocks(rows), _blocks(K)
    w = 0.02 * torch.randn(rows, K, generator=g, device=_DEV)
    w *= (0.4 * torch.randn(rows, 1, generator=g, device=_DEV)).exp()
    w = torch.nn.functional.pad(w, (0, -K % _B, 0, -rows % _B)).view(nb, _B, kb, _B)
    scale = (w.abs().amax((1, 3)) / _MAX).clamp(min=_LEAST)
    return _codes(w, scale[:, None, :, None]).view(nb * _B, kb * _B)[:rows].contiguous(), scale


def _inputs(c: dict, seed: int) -> dict:
    g = torch.Generator(device=_DEV).manual_seed(seed)
    M, K = c["M"], c["K"]
    if c["kind"] == "rows":
        dtype = _TYPES[c["type"]]
        s = {"x": _hidden(g, M, K).to(dtype), "weight": None, "residual": None, "eps": 1.0e-6}
        if c["norm"]:
            s["weight"] = (1.0 + 0.2 * torch.randn(K, generator=g, device=_DEV)).to(dtype)
        if c["norm"] and c["residual"]:
            s["residual"] = (4.0 * _hidden(g, M, K)).to(dtype)
        return s
    codes, scales = _coded_rows(_hidden(g, M, K))
    if c["kind"] == "gated":
        gate, up = _coded_weight(g, c["F"], K), _coded_weight(g, c["F"], K)
        w, ws = (torch.cat(t).contiguous() for t in zip(gate, up))
        return {"codes": codes, "scales": scales, "w": w, "w_scales": ws}
    w, ws = _coded_weight(g, c["N"], K)
    dtype = _TYPES[c["type"]]
    s = {"codes": codes, "scales": scales, "w": w, "w_scales": ws, "dtype": dtype, "residual": None}
    if c["residual"]:
        s["residual"] = (4.0 * _hidden(g, M, c["N"])).to(dtype)
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from zoomkv_revision_amd import fp8
        if case["kind"] == "rows":
            if case["norm"]:
                s["plan"] = fp8.RmsNormQuantPlan(s["x"], s["weight"], s["eps"], residual=s["residual"])
            else:
                s["plan"] = fp8.QuantizeRowsPlan(s["x"])
        elif case["kind"] == "linear":
            s["plan"] = fp8.LinearPlan(s["codes"], s["scales"], fp8.Fp8Weight(s["w"], s["w_scales"]),
                                       out_dtype=s["dtype"], residual=s["residual"])
        else:
            s["plan"] = fp8.GatedLinearPlan(s["codes"], s["scales"], fp8.Fp8Weight(s["w"], s["w_scales"], parts=2))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state: dict):
    if own:
        return state["plan"].run()
    return {"rows": _plain_rows, "linear": _plain_linear, "gated": _plain_gated}[state["case"]["kind"]](state)


def _plain_rows(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    total = x.to(s["x"].dtype) if s["residual"] is not None else None
    if s["weight"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    codes, scales = _coded_rows(x)
    return (codes, scales) if total is None else (codes, scales, total)


def _rows_of(s) -> torch.Tensor:
    M = s["codes"].shape[0]
    return (s["codes"].float().view(M, -1, _B) * s["scales"][..., None]).view(M, -1)


def _matrix(codes, scales) -> torch.Tensor:
    rows = codes.shape[0]
    w = codes.float().view(rows, -1, _B) * scales.repeat_interleave(_B, 0)[:rows, :, None]
    return w.view(rows, -1)


def _plain_linear(s):
    y = torch.mm(_rows_of(s), _matrix(s["w"], s["w_scales"]).t())
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["dtype"])


def _plain_gated(s):
    F, nb, x = s["w"].shape[0] // 2, s["w_scales"].shape[0] // 2, _rows_of(s)
    gate = torch.mm(x, _matrix(s["w"][:F], s["w_scales"][:nb]).t())
    up = torch.mm(x, _matrix(s["w"][F:], s["w_scales"][nb:]).t())
    return _coded_rows(gate / (1.0 + torch.exp(-gate)) * up)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    c = case
    M, K = c["M"], c["K"]
    kb = _blocks(K)
    coded = M * kb * (_B + 4)
    if c["kind"] == "rows":
        item = {"bf16": 2, "fp16": 2, "fp32": 4}[c["type"]]
        passes = 3 if c["norm"] and c["residual"] else 1      # x, residual in, sum out
        return {"bytes": M * K * item * passes + coded + (K * item if c["norm"] else 0), "flops": 0}
    if c["kind"] == "linear":
        N = c["N"]
        item = {"bf16": 2, "fp16": 2, "fp32": 4}[c["type"]]
        return {"bytes": coded + N * kb * _B + _blocks(N) * kb * 4 + M * N * item * (2 if c["residual"] else 1),
                "flops": 2 * M * N * K}
    F = c["F"]
    return {"bytes": coded + 2 * F * kb * _B + 2 * _blocks(F) * kb * 4 + M * _blocks(F) * (_B + 4),
            "flops": 4 * M * F * K}


# ---------------------------------------------------------------------------
# the results in 64 bits
# ---------------------------------------------------------------------------
def _quotients(x):
    """(x / scale, scale) per 128 channels of a row, nothing rounded."""
    M, K = x.shape
    out = torch.zeros(M, _blocks(K) * _B, dtype=torch.float64, device=_DEV)
    scales = torch.empty(M, _blocks(K), dtype=torch.float64, device=_DEV)
    for b in range(_blocks(K)):
        part = x[:, b * _B:(b + 1) * _B]
        scale = torch.maximum(part.max(1)[0], -part.min(1)[0]) / _MAX
        scale[scale < _LEAST] = _LEAST
        scales[:, b] = scale
        out[:, b * _B:b * _B + part.shape[1]] = part / scale.unsqueeze(1)
    return out, scales


def _products(s, rows: slice, blocks: slice):
    """Rows of the product, block of channels by block of channels."""
    w, ws = s["w"][rows], s["w_scales"][blocks].double()
    M, N = s["codes"].shape[0], w.shape[0]
    out = torch.zeros(M, N, dtype=torch.float64, device=_DEV)
    at = torch.arange(N, device=_DEV) // _B
    for b in range(ws.shape[1]):
        cols = slice(b * _B, (b + 1) * _B)
        x = s["codes"][:, cols].double() * s["scales"][:, b].double().unsqueeze(1)
        out.addmm_(x, (w[:, cols].double() * ws[at, b].unsqueeze(1)).t().contiguous())
    return out


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    if case["kind"] == "rows":
        x = s["x"].double()
        total = None
        if s["residual"] is not None:
            x = total = x + s["residual"].double()
        if s["weight"] is not None:
            x = x / (x.square().sum(1, keepdim=True) / case["K"] + s["eps"]).sqrt() * s["weight"].double()
        got = _quotients(x)
        return got if total is None else (*got, total)
    if case["kind"] == "linear":
        y = _products(s, slice(None), slice(None))
        return y if s["residual"] is None else y + s["residual"].double()
    F, nb = case["F"], _blocks(case["F"])
    gate, up = _products(s, slice(0, F), slice(0, nb)), _products(s, slice(F, 2 * F), slice(nb, 2 * nb))
    return _quotients(gate * torch.sigmoid(gate) * up)
