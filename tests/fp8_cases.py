"""Inputs and 64-bit results of the 8-bit linear operators (tests/test_gpu_fp8*.py,
tests/test_fp8_checks.py)."""
from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn
B = 128
LEAST = 2.0 ** -100


def blocks(n: int) -> int:
    return -(-n // B)


def padded(x: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % B))


def scales_of(x: torch.Tensor) -> torch.Tensor:
    """The scale of each row's blocks of 128, in x's type (fp32: the IEEE quotient)."""
    amax = padded(x).view(x.shape[0], -1, B).abs().amax(-1)
    s = torch.maximum(amax / torch.full_like(amax, 448.0), torch.full_like(amax, LEAST))
    return torch.where(amax.isfinite(), s, torch.full_like(s, float("nan")))      # (an infinity: NaN, as its codes)


def coded(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows as codes and scales, each operation rounded as IEEE has it."""
    s = scales_of(x)
    q = padded(x).view(x.shape[0], -1, B) / s[..., None]
    return q.to(E4M3).view(x.shape[0], -1), s


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of rows of codes."""
    return (codes.double().view(codes.shape[0], -1, B) * scales.double()[..., None]).view(codes.shape[0], -1)


def code_bound(y: torch.Tensor, scales: torch.Tensor, rel: float) -> torch.Tensor:
    """How far code * scale may be from y (float64, whole blocks), whose fp32
    computation is off by `rel` relative and whose scale by as much: half a
    step of e4m3 (2^-4 of the value, or 2^-10 where it is subnormal) and `rel` twice."""
    s = scales.double().repeat_interleave(B, 1)
    return y.abs() * (2.0 ** -4 + 2 * rel) + s * 2.0 ** -10 * (1 + 2 * rel)


def whole_codes(g, rows: int, K: int, most: int = 4) -> torch.Tensor:
    """Codes of whole numbers in [-most, most]; zeros behind K."""
    x = torch.randint(-most, most + 1, (rows, K), generator=g).float()
    return padded(x).to(E4M3)


def power_scales(g, shape, low: int = -2, high: int = 2) -> torch.Tensor:
    return torch.exp2(torch.randint(low, high + 1, shape, generator=g).float())


def weight_values(codes, scales, parts: int = 1) -> torch.Tensor:
    """float64 values of a weight [rows, whole blocks]."""
    n = codes.shape[0] // parts
    s = scales.double().view(parts, blocks(n), -1)
    out = []
    for p in range(parts):
        rows = codes[p * n:(p + 1) * n].double().view(n, -1, B)
        out.append((rows * s[p][torch.arange(n, device=codes.device) // B][:, :, None]).view(n, -1))
    return torch.cat(out)


# ---------------------------------------------------------------------------
# a call's result against 64 bits, on the call's own inputs
# ---------------------------------------------------------------------------
# A norm's rows: the sum of squares adds at most 64 terms in a thread, 6 steps over
# lanes and 16 over waves (86 roundings, halved by the square root), then the
# division by K, the root (two units), two products and the sum with the
# residual: fewer than 64 of 2^-24.
NORM_REL = 64 * 2.0 ** -24
# silu(g) u from given g and u: exp (2 units of 2^-23), 1 + (2^-24), the division
# and the product (2^-24 each): fewer than 8 of 2^-24.
ACT_REL = 8 * 2.0 ** -24


def sum_rel(K: int) -> float:
    """Of a product's sum of magnitudes: sums of a block in any order, each
    addition cut rather than rounded, a product of scales and a multiply-add per
    block, sums over runs of k."""
    return (2 * B + 4 + 2 * blocks(K)) * 2.0 ** -24


def check_rows(x, codes, scales):
    want, s = coded(x.float().cpu())
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu().float(), want.float())


def _near(got, want, bound) -> bool:
    """Within the bound, NaN where NaN is."""
    return bool((((got - want).abs() <= bound) | (got.isnan() & want.isnan())).all())


def check_norm(x, weight, eps, residual, codes, scales, total=None):
    h = x.double() + (0 if residual is None else residual.double())
    y = h * (h.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()
    s = scales_of(y)
    assert _near(scales.double(), s, NORM_REL * s)
    y = torch.where(s.isnan().repeat_interleave(B, 1), float("nan"), padded(y))     # (an infinity: its whole block)
    assert _near(values(codes, scales), y, code_bound(y, s, NORM_REL))
    if residual is not None:
        assert torch.equal(total, (x.float() + residual.float()).to(x.dtype))


def check_linear(codes, scales, weight, residual, out):
    w, x = weight_values(weight.codes, weight.scales, weight.parts), values(codes, scales)
    r = 0 if residual is None else residual.double()
    want, mass = x @ w.t() + r, x.abs() @ w.abs().t() + (0 if residual is None else r.abs())
    # (fp16's subnormal step is 2^-24)
    bound = mass * sum_rel(w.shape[1]) + want.abs() * torch.finfo(out.dtype).eps / 2 + 2.0 ** -25
    assert ((out.double() - want).abs() <= bound).all()


def check_gated(codes, scales, weight, act, act_scales):
    """The errors of gate and up, e of their masses, go through silu, whose slope is
    below 1.1 and whose size is at most |gate|; a block's scale may be off by its
    largest such error / 448."""
    w, x = weight_values(weight.codes, weight.scales, 2), values(codes, scales)
    (gate, up), (ga, ua) = (x @ w.t()).chunk(2, 1), (x.abs() @ w.abs().t()).chunk(2, 1)
    e = sum_rel(w.shape[1])
    y = padded(gate * torch.sigmoid(gate) * up)
    off = padded(1.1 * e * ga * (up.abs() + e * ua) + gate.abs() * e * ua)
    top = off.view(off.shape[0], -1, B).amax(-1)
    s = scales_of(y)
    assert ((act_scales.double() - s).abs() <= ACT_REL * s + top / 448).all()
    slack = off + top.repeat_interleave(B, 1) * 2.0 ** -8
    assert ((values(act, act_scales) - y).abs() <= code_bound(y, s, ACT_REL) + slack).all()
