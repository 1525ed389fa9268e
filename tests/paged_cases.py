"""Calls of paged attention whose result shows every tile of 32 tokens: tile i
has value 1 (times its KV head's number) on channel i % d and 0 elsewhere, and
its tokens have weights 1, 2^-x, 2^-2x in turn, x from 1 to 5 by the query head,
all of it exact in every type.  With the bound of a result and how the kernel
divides a call.

Bound, for T tiles in a wave's run: the exponents' arguments are below 2^5, so a
weight is right to 2^-20 + 2^-23, parts of it to 2^-21; a wave sums at most three
parts of its 32 T terms, and then at most 16 waves and 256 workgroups are joined.
In numerator and denominator: |out - ref| <= ref (2^-17 + (96 T + 300) 2^-23) +
half a step of the output's type; all terms are positive, so ref is the mass.  The
weights' sum has 4 T terms a lane: |lse - ref| <= 2^-18 + (4 T + 300) 2^-24 + 2^-23
|ref|.

How a call is divided (paged_attention.hip): a place on the line for each tile of
each unit and 2 for the unit, workgroups that take equal runs of it, at least a
place a wave, and waves that take equal parts of those."""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

TILE, UNIT_COST, GROUPS, BATCH, STEP_ROUNDS = 32, 2, 256, 8, 2


@dataclass(frozen=True)
class Call:
    lens: tuple
    hq: int
    kv: int
    d: int
    type: str = "bf16"          # or "fp16"
    fp8: bool = False
    nhd: bool = False
    window: int = 0
    two_steps: bool = False     # whether a unit's partials are joined in two steps
    sets: bool = False          # whether neighbouring waves take the KV heads of a set

    def first(self, n: int) -> int:
        return max(0, n - self.window) if self.window else 0

    @property
    def waves(self) -> int:
        return 4 if self.d == 256 else 8

    def line(self):
        """(KV heads of a set, places per workgroup, [(places of a unit, how many of them)])."""
        gqa = self.hq // self.kv
        groups = -(-gqa // 16)
        size = [-(-n // TILE) - self.first(n) // TILE + UNIT_COST for n in self.lens if n]
        set_ = 1
        if self.nhd and self.d < 256 and self.kv > 1 and self.kv * self.d * (1 if self.fp8 else 2) % 512 == 0:
            while 2 * set_ <= self.waves and 2 * set_ * gqa <= 16 and self.kv % (2 * set_) == 0:
                set_ *= 2
        if set_ > 1 and sum(size) * self.kv * groups < 12 * self.waves * GROUPS:
            set_ = 1
        units = self.kv * groups // set_
        runs = self.waves // set_
        return set_, max(runs, -(-sum(size) * units // GROUPS)), [(s, units) for s in size]

    @property
    def run_tiles(self) -> int:
        """Most tiles in a wave's run (a run may grow by a short unit moved into it)."""
        set_, chunk, _ = self.line()
        runs = self.waves // set_
        return -(-(chunk + (30 if set_ == 1 else 0)) // runs)

    def joins_in_two_steps(self) -> bool:
        set_, chunk, units = self.line()
        most = max(s for s, _ in units) - UNIT_COST
        n, fan = -(-most // chunk), 2 * self.waves
        heads = min(16, set_ * self.hq // self.kv)

        def rounds(count):
            at_once = BATCH * max(1, min(64 * self.waves // 2 // (heads * self.d // 4), count))
            return -(-count // at_once)

        return n > fan and rounds(n) > rounds(fan) + rounds(-(-n // fan)) + STEP_ROUNDS

    # --- inputs --------------------------------------------------------------
    def log2_weight(self, t):
        return -(t % 3)

    def times(self, head: int) -> int:
        """What a query head multiplies the tokens' log2 weights by."""
        return 1 + head % 5

    # --- result --------------------------------------------------------------
    def reference(self, n: int, head: int, left_out=()):
        """(out [d], lse) of a query head over n tokens, without those of `left_out`."""
        t = np.arange(self.first(n), n)
        t = t[~np.isin(t, np.asarray(left_out, dtype=np.int64))]
        if len(t) == 0:
            return np.zeros(self.d), -np.inf
        p = np.exp2(self.log2_weight(t) * float(self.times(head)))
        out = np.bincount(t // TILE % self.d, weights=p, minlength=self.d) / p.sum()
        return out * (1 + head // (self.hq // self.kv)), float(np.log(p.sum()))

    def out_bound(self, ref, half_step: float):
        return ref * (2.0 ** -17 + (96 * self.run_tiles + 300) * 2.0 ** -23 + half_step)

    def lse_bound(self, ref: float) -> float:
        return 2.0 ** -18 + (4 * self.run_tiles + 300) * 2.0 ** -24 + 2.0 ** -23 * abs(ref)


def _long(*a, **k):
    return Call(*a, two_steps=True, **k)


CALLS = [
    Call((1,), 1, 1, 64), Call((33, 1, 0, 700), 8, 2, 128, "fp16"), Call((4097,), 32, 8, 128),
    _long((131072,), 2, 1, 128), Call((131072,), 2, 1, 64, "fp16", fp8=True), _long((66000,), 8, 1, 128),
    _long((66000,), 8, 1, 128, fp8=True), _long((11000,), 16, 1, 128), _long((12001, 0, 3), 16, 1, 128, "fp16", fp8=True),
    _long((20000,), 24, 1, 128), _long((33333, 1, 700, 20011), 16, 1, 128), _long((30000, 9000), 16, 1, 256),
    _long((66000,), 8, 1, 256, "fp16"), _long((70000, 50), 20, 1, 64, "fp16"), _long((66000,), 8, 1, 128, window=60001),
    Call((4200,), 16, 1, 128), Call((131072,), 32, 8, 128),
    Call(tuple(1500 + 37 * i for i in range(9)) + (40, 3, 0, 700), 16, 16, 64, "fp16"),
    Call(tuple(6000 + 37 * i for i in range(9)) + (40, 3, 0, 700), 2, 1, 256), Call((66,) * 235, 8, 8, 64),
    Call((8192, 0, 33, 4000, 1, 77, 16, 2500), 32, 8, 128), Call((8000,) * 12, 16, 2, 128, fp8=True, window=4096),
    # pools [page, token, head]
    Call((70000,), 16, 4, 128, nhd=True),                                     # (too few tiles for sets)
    _long((131072,), 32, 8, 128, nhd=True, sets=True),                        # sets of four heads
    _long((131072,), 32, 8, 128, "fp16", nhd=True, window=120001, sets=True),
    _long((90000, 0, 31, 9000, 1), 64, 8, 128, nhd=True, sets=True),          # of two
    Call((65000, 70000), 12, 6, 128, "fp16", nhd=True, sets=True),           # three of two
    Call((5000,) * 80 + (3, 0, 700), 10, 2, 128, nhd=True, sets=True),        # one of two, five query heads each
    Call(tuple(7000 + 7 * i for i in range(15)), 8, 8, 128, fp8=True, nhd=True, sets=True),    # of eight
    Call((5000,) * 40 + (3, 0, 700), 16, 4, 64, "fp16", nhd=True, sets=True),
    Call((7000,) * 15, 40, 8, 64, "fp16", fp8=True, nhd=True, sets=True),
    Call((66000,), 16, 8, 256, nhd=True), Call((30000,) * 4, 10, 2, 64, "fp16", nhd=True),
]


def name(c: Call) -> str:
    lens = f"{len(c.lens)}x{max(c.lens)}"
    return "-".join([lens, f"{c.hq}.{c.kv}.{c.d}", c.type] + ["fp8"] * c.fp8 + ["nhd"] * c.nhd + ["window"] * bool(c.window))
