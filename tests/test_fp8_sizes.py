"""CPU: which kernel an 8-bit product takes, and that none is left without a size that is
computed on the GPU."""
import math
import random

import pytest

from fp8_cases import B, blocks
from fp8_sizes import CASES
from zoomkv_revision_amd._lib import lib


@pytest.mark.parametrize("parts,kernel,runs,M,N,K", CASES)
def test_the_size_takes_its_kernel(parts, kernel, runs, M, N, K):
    assert divmod(lib().zkv_fp8_plan(M, N, blocks(K) * B, parts), 16) == (kernel, runs)


def test_no_size_takes_another():
    """Over the whole range of sizes, spread over their logarithms."""
    r, known, seen = random.Random(0), {c[:3] for c in CASES}, set()
    spread = lambda top: round(math.exp(r.uniform(0, math.log(top))))
    while len(seen) < 20000:
        M, N, nkb, parts = spread((1 << 20) - 1), spread((1 << 22) - 1), spread(128), r.choice((1, 2))
        if M * N <= 1 << 37 and (M, N, nkb, parts) not in seen:
            seen.add((M, N, nkb, parts))
            assert (parts, *divmod(lib().zkv_fp8_plan(M, N, nkb * B, parts), 16)) in known, (M, N, nkb, parts)


# weight rows and rows of x of a unit or tile, and its threads
SHAPE = {3: (32, 32, 256), 4: (256, 128, 512), 5: (128, 128, 512), 6: (128, 64, 512), 7: (64, 64, 256)}


def test_products_fit_a_launch():
    """Fewer than 2^32 threads; only the gated product's own tile, launched in halves then,
    may pass that."""
    r, edge = random.Random(1), [((1 << i) - 1 + d) for i in range(1, 23) for d in (0, 1)]
    for _ in range(20000):
        N = min(r.choice(edge), (1 << 22) - 1)
        M = min((1 << 20) - 1, (1 << 37) // N if r.random() < 0.5 else r.choice(edge))
        if M * N > 1 << 37:
            continue
        parts = r.choice((1, 2))
        kernel, runs = divmod(lib().zkv_fp8_plan(M, N, r.choice((1, 2, 5, 20, 128)) * B, parts), 16)
        if kernel < 3:
            threads = -(-N // 4) * 512                              # (units of 4 weight rows at least, of 8 waves at most)
        elif kernel < 8:
            n, m, t = SHAPE[kernel]
            threads = -(-N // n) * (1 if kernel == 3 else -(-M // m) * parts * runs) * t
        else:
            continue
        assert threads < 1 << 32, (M, N, parts, kernel, runs)


@pytest.mark.parametrize("sizes", [(0, 1, 128, 1), (1, 1, 100, 1), (1, 1, 16512, 1), (1 << 20, 1, 128, 1),
                                   (1, 1 << 22, 128, 2), (1 << 19, 1 << 19, 128, 1), (1, 1, 128, 3), (1, 1, 128, 0)])
def test_refused_sizes_have_no_plan(sizes):
    assert lib().zkv_fp8_plan(*sizes) == -1


@pytest.mark.parametrize("entry", ["zkv_fp8_linear_workspace_size", "zkv_fp8_gated_workspace_size"])
def test_workspaces_of_sizes_at_and_beyond_the_limits(entry):
    """K is rounded up to whole blocks; sizes that the calls refuse need none (they passed 32
    bits in the choice)."""
    size, top = getattr(lib(), entry), (1 << 31) - 1
    assert size(64, 64, 16300) == size(64, 64, 16384) > 0 and size(64, 256, 9728 - 50) == size(64, 256, 9728) > 0
    for sizes in ((top, 64, top), (top, top, 16384), (64, 1 << 22, 16384), (64, 64, top), (64, 64, 16385), (64, 64, 0),
                  (64, 64, -1), (0, 64, 16384), (1 << 20, 64, 16384)):
        assert size(*sizes) == 0
