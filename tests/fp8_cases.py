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
    return torch.maximum(amax / torch.full_like(amax, 448.0), torch.full_like(amax, LEAST))


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
