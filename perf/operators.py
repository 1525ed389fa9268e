"""The paged-cache operators, in their plain form and through the library.

Four kinds of call, over the sizes a serving loop makes them with:

  tables   one step of the page tables of a batch: pages handed out and taken
           back, the block table, the slot and position of every new token
           (paged.page_advance)
  write    key / value rows of new tokens into their slots of a paged cache,
           in the cache's type or as e4m3 with a scale per head
           (paged.paged_write)
  rope     q / k norm, rotary embedding at each row's own position, and the
           K / V rows of a decode batch into their slots
           (paged.paged_qk_norm_rope)
  attend   attention of one new token per request over its pages
           (paged.paged_attention)

A paged cache is one pool of pages [pages, kv heads, page size, head dim] for K
and one for V; "nhd" cases keep the pool as [pages, page size, kv heads, head
dim] and pass the transposed view.  A slot is page * page_size + offset, -1 for
a row that has none.
"""
from __future__ import annotations

import math
import random

import torch

own = False
_DEV = "cuda:0"
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3_MAX = 448.0


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # the step of a decode batch: every request gets one token, one in
        # sixteen a new page
        {"name": "tables_decode_64", "kind": "tables", "requests": 64, "len": 4096, "prompt": 1, "mix": "decode",
         "page": 16, "cap": 64, "tight": False, "lens": 1},
        # a busy server's step: prompts admitted, others decoding, idle,
        # rolled back or finished
        {"name": "tables_mixed_1024", "kind": "tables", "requests": 1024, "len": 8192, "prompt": 2048,
         "mix": "mixed", "page": 16, "cap": 65536, "tight": False, "lens": 2},
        # one prompt of one layer, as the 32 / 8-head model with head dim 128 has it
        {"name": "write_prompt_4097", "kind": "write", "tokens": 4097, "kv": 8, "d": 128, "type": "bf16",
         "fp8": False, "page": 16, "nhd": False, "padded": 0, "pool": 320},
        # a batch of prompts into an 8-bit cache, with padding behind the last
        {"name": "write_fp8_32768", "kind": "write", "tokens": 32768, "kv": 8, "d": 128, "type": "bf16",
         "fp8": True, "page": 32, "nhd": False, "padded": 500, "pool": 1100},
        # a small decode batch's rows, between the QKV projection and the attention
        {"name": "rope_8", "kind": "rope", "tokens": 8, "hq": 32, "kv": 8, "d": 128, "type": "bf16", "page": 16,
         "nhd": False, "positions": 65536, "pool": 64, "padded": 0},
        # a large one, a few of its rows padding
        {"name": "rope_512", "kind": "rope", "tokens": 512, "hq": 32, "kv": 8, "d": 128, "type": "bf16", "page": 16,
         "nhd": False, "positions": 65536, "pool": 560, "padded": 9},
        # one short chat: latency
        {"name": "attend_1x700", "kind": "attend", "bs": 1, "hq": 32, "kv": 8, "d": 128, "type": "bf16",
         "fp8": False, "page": 16, "nhd": False, "len": 700, "shape": "equal", "window": 0, "empty": 0,
         "lse": False, "f32": False, "lens": 1},
        # an ordinary decode batch: lengths from one token to 8192
        {"name": "attend_64_ragged", "kind": "attend", "bs": 64, "hq": 32, "kv": 8, "d": 128, "type": "bf16",
         "fp8": False, "page": 16, "nhd": False, "len": 8192, "shape": "ragged", "window": 0, "empty": 3,
         "lse": False, "f32": False, "lens": 2},
        # the headline decode shape: 16 sequences of 32K tokens, 32 / 8 heads
        {"name": "attend_16x32k", "kind": "attend", "bs": 16, "hq": 32, "kv": 8, "d": 128, "type": "bf16",
         "fp8": False, "page": 16, "nhd": False, "len": 32768, "shape": "equal", "window": 0, "empty": 0,
         "lse": True, "f32": False, "lens": 3},
        # one long document, pages of 64 as [page, token, head]
        {"name": "attend_1x131k", "kind": "attend", "bs": 1, "hq": 32, "kv": 8, "d": 128, "type": "bf16",
         "fp8": False, "page": 64, "nhd": True, "len": 131072, "shape": "equal", "window": 0, "empty": 0,
         "lse": True, "f32": True, "lens": 4},
        # the 8-bit cache under a batch of long requests
        {"name": "attend_fp8_32", "kind": "attend", "bs": 32, "hq": 32, "kv": 8, "d": 128, "type": "bf16",
         "fp8": True, "page": 32, "nhd": False, "len": 32768, "shape": "ragged", "window": 0, "empty": 0,
         "lse": False, "f32": False, "lens": 5},
        # a head per query head, narrow heads, a sliding window, pages that
        # are no power of two
        {"name": "attend_mha_d64", "kind": "attend", "bs": 12, "hq": 16, "kv": 16, "d": 64, "type": "fp16",
         "fp8": False, "page": 24, "nhd": False, "len": 20000, "shape": "ragged", "window": 4096, "empty": 0,
         "lse": False, "f32": False, "lens": 6},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    kind = rng.choice(["tables", "write", "rope", "attend", "attend", "attend"])
    kv = rng.choice([1, 2, 4, 8, 8])
    gqa = rng.choice([1, 2, 4, 4, 5, 7, 8, 16, 24])
    d = rng.choice([64, 128, 128, 128, 256])
    page = rng.choice([1, 8, 16, 16, 16, 24, 32, 64, 128])
    base = {"kind": kind, "page": page}
    if kind == "tables":
        requests = _log(rng, 1, 1024)
        mix = rng.choice(["decode", "mixed", "mixed"])
        prompt = 1 if mix == "decode" else _log(rng, 2, 2048)
        page = max(page, 8)
        cap = requests if mix == "decode" else min(65536, max(16, requests * prompt // rng.choice([1, 4, 16])))
        return {**base, "page": page, "requests": requests, "len": _log(rng, 1, 8192), "prompt": prompt, "mix": mix,
                "cap": cap, "tight": rng.random() < 0.3, "lens": rng.randrange(1 << 30)}
    if kind == "write":
        # at most the bytes of the largest listed write
        tokens = _log(rng, 1, max(1, 32768 * 8 * 128 // (kv * d * 2)))
        return {**base, "tokens": tokens, "kv": kv, "d": d, "type": rng.choice(["bf16", "bf16", "fp16"]),
                "fp8": rng.random() < 0.4, "nhd": rng.random() < 0.4,
                "padded": min(rng.choice([0, 0, 1, 17]), tokens // 2),
                "pool": -(-(tokens * 5 // 4 + 40) // page)}
    if kind == "rope":
        gqa = min(gqa, 8)
        tokens = _log(rng, 1, min(1024, max(1, 512 * 44 * 128 // (kv * (gqa + 2) * d))))
        return {**base, "tokens": tokens, "hq": kv * gqa, "kv": kv, "d": d,
                "type": rng.choice(["bf16", "bf16", "fp16"]), "nhd": rng.random() < 0.4, "positions": rng.choice([4096, 65536, 131072]),
                "pool": -(-(tokens * 5 // 4 + 40) // page), "padded": min(rng.choice([0, 0, 1, 5]), tokens // 2)}
    bs = _log(rng, 1, 256)
    fp8 = rng.random() < 0.3
    # at most a quarter of the cells of the largest listed call and half its
    # products, at most 131072 tokens a request
    length = _log(rng, 1, min(131072, max(1, (1 << 30) // (bs * kv * d * max(8, gqa)))))
    shape = rng.choice(["equal", "ragged", "ragged"])
    empty = rng.choice([0, 0, 1, bs // 4])
    return {**base, "bs": bs, "hq": kv * gqa, "kv": kv, "d": d, "type": rng.choice(["bf16", "bf16", "fp16"]),
            "fp8": fp8, "nhd": rng.random() < 0.4, "len": length, "shape": shape,
            "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)]), "empty": min(empty, bs - 1),
            "lse": empty == 0 and rng.random() < 0.5, "f32": rng.random() < 0.3, "lens": rng.randrange(1 << 30)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=_DEV).manual_seed(seed)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=_DEV).to(dtype)


def _attend_lens(c) -> list[int]:
    """The lengths of an attend case: all the same, or spread over the
    logarithm from 1 to the longest (which one request has); the last
    ``empty`` requests have none (the padding of a fixed batch)."""
    r = random.Random(c["lens"])
    n = [c["len"] if c["shape"] == "equal" else _log(r, 1, c["len"]) for _ in range(c["bs"])]
    n[0] = c["len"]
    for i in range(c["empty"]):
        n[c["bs"] - 1 - i] = 0
    return n


def _table_lens(c) -> tuple[list[int], list[int]]:
    """Lengths before the step and new tokens of a tables case."""
    r = random.Random(c["lens"])
    have, new = [], []
    for _ in range(c["requests"]):
        n = _log(r, 1, c["len"])
        if c["mix"] == "decode":
            what = "decode"
        else:
            what = r.choice(["decode", "decode", "decode", "prompt", "idle", "rollback", "done"])
        if what == "prompt":
            have.append(r.choice([0, 0, n]))
            new.append(_log(r, 1, c["prompt"]))
        else:
            have.append(n)
            new.append({"decode": 1, "idle": 0, "rollback": -min(n, 3), "done": -n}[what])
    return have, new


def _pages_of(n: int, page: int) -> int:
    return -(-n // page)


def _pool(g, c, pages: int):
    """One pool of K or V pages [pages, kv, page, d], values as a cache holds
    them (e4m3: scaled so that the largest of a head come near its range)."""
    shape = (pages, c["page"], c["kv"], c["d"]) if c["nhd"] else (pages, c["kv"], c["page"], c["d"])
    dtype = torch.float8_e4m3fn if c.get("fp8") else _TYPES[c["type"]]
    t = torch.empty(shape, dtype=dtype, device=_DEV)
    step = max(1, (1 << 26) // (c["page"] * c["kv"] * c["d"]))
    for i in range(0, pages, step):
        x = torch.randn(t[i:i + step].shape, generator=g, device=_DEV)
        t[i:i + step] = (x * 80.0).clamp(-_E4M3_MAX, _E4M3_MAX).to(dtype) if c.get("fp8") else x.to(dtype)
    return t.transpose(1, 2) if c["nhd"] else t


def _scales(g, c):
    """A positive scale per head, about what maps N(0, 1) rows to e4m3."""
    return 0.0125 * (0.75 + 0.5 * torch.rand(c["kv"], generator=g, device=_DEV)) if c.get("fp8") else None


def _slots(g, c) -> torch.Tensor:
    """Distinct slots of a scattered set of pages for every token but the last
    ``padded``, which have none."""
    perm = torch.randperm(c["pool"], generator=g, device=_DEV)
    t = torch.arange(c["tokens"], device=_DEV) + 3 % c["page"]      # starts inside a page
    s = perm[t // c["page"]] * c["page"] + t % c["page"]
    if c["padded"]:
        s[max(0, c["tokens"] - c["padded"]):] = -1
    return s


def _inputs(c, seed: int) -> dict:
    g = _gen(seed)
    kind, page = c["kind"], c["page"]
    if kind == "tables":
        have, new = _table_lens(c)
        width = _pages_of(max(h + max(n, 0) for h, n in zip(have, new)), page)
        used = [_pages_of(h, page) for h in have]
        grow = sum(_pages_of(h + max(n, 0), page) - u for h, n, u in zip(have, new, used))
        free = grow // 2 if c["tight"] else grow + grow // 4 + 8    # tight: the pool runs dry
        pages = sum(used) + free
        perm = torch.randperm(pages, generator=g, device=_DEV, dtype=torch.int32)
        table = torch.full((c["requests"], width), -1, dtype=torch.int32, device=_DEV)
        owner = torch.arange(width, device=_DEV)[None] < torch.tensor(used, device=_DEV)[:, None]
        table[owner] = perm[:sum(used)]
        ring = torch.full((pages,), -1, dtype=torch.int32, device=_DEV)
        head = int(torch.randint(0, pages, (1,), generator=g, device=_DEV))
        at = (head + torch.arange(free, device=_DEV)) % pages
        ring[at] = perm[sum(used):]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=_DEV)
        return {"seq_lens": i32(have), "new": i32(new), "table": table, "free": ring,
                "state": i32([head, free, 0, 0])}
    if kind == "write":
        dtype = _TYPES[c["type"]]
        shape = (c["tokens"], c["kv"], c["d"])
        return {"k": _randn(g, dtype, *shape), "v": _randn(g, dtype, *shape),
                "slots": _slots(g, c), "k_pages": _pool(g, c, c["pool"]), "v_pages": _pool(g, c, c["pool"]),
                "k_scale": _scales(g, c), "v_scale": _scales(g, c)}
    if kind == "rope":
        dtype = _TYPES[c["type"]]
        d, n = c["d"], c["tokens"]
        inv = 1.0 / (1.0e6 ** (torch.arange(0, d, 2, dtype=torch.float64, device=_DEV) / d))
        ang = torch.arange(c["positions"], dtype=torch.float64, device=_DEV)[:, None] * inv
        pos = torch.randint(0, c["positions"], (n,), generator=g, device=_DEV, dtype=torch.int32)
        slots = _slots(g, c)
        pos[slots < 0] = -1
        return {"qkv": _randn(g, dtype, n, (c["hq"] + 2 * c["kv"]) * d), "positions": pos, "slots": slots,
                "q_norm": (1.0 + 0.1 * torch.randn(d, generator=g, device=_DEV)).to(dtype),
                "k_norm": (1.0 + 0.1 * torch.randn(d, generator=g, device=_DEV)).to(dtype),
                "cos": ang.cos().float(), "sin": ang.sin().float(), "eps": 1.0e-6,
                "q_out": torch.zeros(n, c["hq"], d, dtype=dtype, device=_DEV),
                "k_pages": _pool(g, c, c["pool"]), "v_pages": _pool(g, c, c["pool"])}
    lens = _attend_lens(c)
    used = [_pages_of(n, page) for n in lens]
    pages = sum(used) + 8
    perm = torch.randperm(pages, generator=g, device=_DEV, dtype=torch.int32)
    table = torch.full((c["bs"], max(used) + 2), -1, dtype=torch.int32, device=_DEV)
    owner = torch.arange(max(used) + 2, device=_DEV)[None] < torch.tensor(used, device=_DEV)[:, None]
    table[owner] = perm[:sum(used)]
    return {"q": (2.0 * torch.randn(c["bs"], 1, c["hq"], c["d"], generator=g, device=_DEV)).to(_TYPES[c["type"]]),
            "k_pages": _pool(g, c, pages), "v_pages": _pool(g, c, pages), "table": table,
            "seq_lens": torch.tensor(lens, dtype=torch.int32, device=_DEV), "lens": lens,
            "k_scale": _scales(g, c), "v_scale": _scales(g, c)}


def prepare(case: dict, seed: int) -> dict:
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if c["kind"] == "tables":
        n = c["cap"]
        s["slots"] = torch.empty(n, dtype=torch.int64, device=_DEV)
        s["positions"] = torch.empty(n, dtype=torch.int32, device=_DEV)
        s["starts"] = torch.empty(c["requests"] + 1, dtype=torch.int32, device=_DEV)
        s["lens_out"] = torch.empty_like(s["seq_lens"])
        s["state_out"] = torch.zeros_like(s["state"])
    if own:
        from zoomkv_revision_amd import paged
        if c["kind"] == "tables":
            tables = paged.PageTables(s["table"], s["seq_lens"], s["free"], s["state"], c["page"])
            s["plan"] = paged.PageAdvancePlan(tables, s["new"], s["slots"], s["positions"], s["starts"],
                                              lens_out=s["lens_out"], state_out=s["state_out"])
        elif c["kind"] == "write":
            s["plan"] = paged.PagedWritePlan(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"],
                                             s["k_scale"], s["v_scale"])
        elif c["kind"] == "rope":
            s["plan"] = paged.PagedRopePlan(s["qkv"], c["hq"], c["kv"], s["q_norm"], s["k_norm"], s["eps"], s["cos"],
                                            s["sin"], s["positions"], s["slots"], s["q_out"], s["k_pages"],
                                            s["v_pages"])
        else:
            out = torch.empty(s["q"].shape, dtype=torch.float32, device=_DEV) if c["f32"] else None
            s["plan"] = paged.PagedAttentionPlan(s["q"], s["k_pages"], s["v_pages"], s["table"], s["seq_lens"],
                                                 window=c["window"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                                 return_softmax_lse=c["lse"], out=out)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state: dict):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        got = s["plan"].run()
        if kind == "tables":
            return s["slots"], s["positions"], s["starts"], s["lens_out"], s["state_out"], s["table"], s["free"]
        if kind == "write":
            return s["k_pages"], s["v_pages"]
        if kind == "rope":
            return s["q_out"], s["k_pages"], s["v_pages"]
        return got
    return {"tables": _plain_tables, "write": _plain_write, "rope": _plain_rope, "attend": _plain_attend}[kind](s, c)


def _plain_tables(s, c):
    """Request i goes from seq_lens[i] to seq_lens[i] + new[i] tokens (never
    below 0).  Pages come off the ring of free pages from its head in request
    order, and go back behind its last; a request grows whole or not at all:
    its tokens have to fit the table's width and the slot map, and its pages
    those that are free (counted with every earlier request's)."""
    page, (R, width) = c["page"], s["table"].shape
    table, ring = s["table"], s["free"]
    cap, pages = s["slots"].numel(), ring.numel()
    have, new = s["seq_lens"].long(), s["new"].long()
    head, count = s["state"][0].long(), s["state"][1].long()
    ceil = lambda n: (n + page - 1) // page
    ok = (have >= 0) & (have <= width * page)
    grow = new.clamp(min=0)
    ends = torch.cumsum(grow, 0).clamp(max=cap + 1)
    starts = torch.cat((ends.new_zeros(1), ends))
    wide = have + grow <= width * page
    fits = ok & wide & (ends <= cap) & (new > 0)
    need = torch.where(fits, ceil(have + grow) - ceil(have), 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= count))
    kept = torch.where(ok & (new < 0), (have + new).clamp(min=0), have)
    give = ceil(kept.clamp(min=0)) - ceil(have.clamp(min=0))
    give = torch.where(ok & (new < 0), -give, 0)
    back = torch.cumsum(give, 0)
    # the slot and position of every token
    t = torch.arange(cap, device=table.device)
    r = torch.searchsorted(ends, t, right=True).clamp(max=R - 1)
    live = (t < ends[-1]) & granted[r]
    pos = have[r] + t - starts[r]
    at = torch.where(live, pos // page, 0)
    fresh = live & (at >= ceil(have)[r])
    order = head + (upto - need)[r] + at - ceil(have)[r]
    new_page = ring[torch.where(fresh, order, 0) % pages]
    old_page = table[r, torch.where(fresh, 0, at)]
    got = torch.where(fresh, new_page, old_page).long()
    s["slots"].copy_(torch.where(live, got * page + pos % page, -1))
    s["positions"].copy_(torch.where(live, pos, -1))
    s["starts"].copy_(starts)
    # pages taken back: the j-th of the step to the ring's place head + count + j
    j = torch.arange(pages, device=table.device)
    fr = torch.searchsorted(back, j, right=True).clamp(max=R - 1)
    fj = ceil(kept)[fr] + j - (back - give)[fr]
    freed = (j < back[-1]) & (count + j < pages)
    old = table[fr, torch.where(freed, fj, 0)]
    where = torch.where(freed, (head + count + j) % pages, pages)
    grown = torch.cat((ring, ring.new_zeros(1)))
    grown[where] = old
    # the table's new entries
    rows = torch.where(fresh, r, R)
    wider = torch.cat((table, table.new_zeros(1, width)))
    wider[rows, at] = got.int()
    table.copy_(wider[:R])
    ring.copy_(grown[:pages])
    taken = torch.where(granted & (need > 0), upto, 0).max()
    s["lens_out"].copy_(torch.where(granted, have + grow, kept))
    dry = (fits & ~granted).any()
    status = s["state"][2].long() | dry.long() | ((ok & (new > 0) & ~wide).any().long() << 1) | \
        ((ok & wide & (new > 0) & (ends > cap)).any().long() << 2) | ((~ok).any().long() << 3) | \
        ((count + back[-1] - taken > pages).long() << 4)
    left = torch.minimum(count + back[-1], count * 0 + pages) - taken
    s["state_out"].copy_(torch.stack(((head + taken) % pages, left, status, status * 0)))
    return s["slots"], s["positions"], s["starts"], s["lens_out"], s["state_out"], table, ring


def _store(pages, rows, slots, scale):
    """rows [n, kv, d] (fp32) into the slots that a row has."""
    page = pages.shape[2]
    live = slots >= 0
    at, x = slots[live], rows[live]
    if pages.dtype == torch.float8_e4m3fn:
        x = (x / scale[None, :, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        raw = x.to(torch.float8_e4m3fn).view(torch.uint8)
        pages.view(torch.uint8)[at // page, :, at % page] = raw
    else:
        pages[at // page, :, at % page] = x.to(pages.dtype)


def _plain_write(s, c):
    _store(s["k_pages"], s["k"].float(), s["slots"], s["k_scale"])
    _store(s["v_pages"], s["v"].float(), s["slots"], s["v_scale"])
    return s["k_pages"], s["v_pages"]


def _plain_rope(s, c):
    """x * rsqrt(mean(x^2) + eps) * w for the heads of q and k, then (x1, x2)
    -> (x1 cos - x2 sin, x2 cos + x1 sin) of a head's two halves."""
    n, hq, kv, d = c["tokens"], c["hq"], c["kv"], c["d"]
    x = s["qkv"].float().view(n, hq + 2 * kv, d)
    live = s["positions"] >= 0
    pos = s["positions"].clamp(min=0).long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w.float()
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q, k = turned(x[:, :hq], s["q_norm"]), turned(x[:, hq:hq + kv], s["k_norm"])
    s["q_out"].copy_(torch.where(live[:, None, None], q.to(s["q_out"].dtype), s["q_out"]))
    _store(s["k_pages"], k, s["slots"], None)
    _store(s["v_pages"], x[:, hq + kv:], s["slots"], None)
    return s["q_out"], s["k_pages"], s["v_pages"]


def _rows(pages, table_row, first: int, n: int, scale, dtype):
    """Tokens [first, n) of one request from its pages: [kv, n - first, d]."""
    page = pages.shape[2]
    p0 = first // page
    ids = table_row[p0:_pages_of(n, page)].long()
    x = pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn) if pages.dtype == torch.float8_e4m3fn else pages[ids]
    x = x.to(dtype).transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, first - p0 * page:n - p0 * page]
    return x if scale is None else x * scale.to(dtype)[:, None, None]


def _plain_attend(s, c):
    bs, hq, kv, d = c["bs"], c["hq"], c["kv"], c["d"]
    out = torch.zeros(bs, 1, hq, d, device=_DEV)
    lse = torch.full((bs, hq, 1), float("-inf"), device=_DEV)
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        first = max(0, n - c["window"]) if c["window"] else 0
        k = _rows(s["k_pages"], s["table"][b], first, n, s["k_scale"], torch.float32)
        v = _rows(s["v_pages"], s["table"][b], first, n, s["v_scale"], torch.float32)
        q = s["q"][b, 0].float().view(kv, hq // kv, d)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
        m = x.max(-1, keepdim=True)[0]
        p = (x - m).exp()
        z = p.sum(-1, keepdim=True)
        out[b, 0] = (torch.matmul(p, v) / z).view(hq, d)
        lse[b] = (m + z.log()).view(hq, 1)
    out = out if c["f32"] else out.to(s["q"].dtype)
    return (out, lse) if c["lse"] else out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    c = case
    kind = c["kind"]
    if kind == "tables":
        have, new = _table_lens(c)
        moved = sum(abs(_pages_of(max(h + n, 0), c["page"]) - _pages_of(h, c["page"])) for h, n in zip(have, new))
        # lengths, new tokens, new lengths and starts; slot and position of
        # every token; a page id read and written for every page that moves
        return {"bytes": c["requests"] * 16 + c["cap"] * 12 + moved * 8, "flops": 0}
    item = {"bf16": 2, "fp16": 2, "fp32": 4}[c["type"]]
    cell = 1 if c.get("fp8") else item
    if kind == "write":
        n = c["tokens"] - min(c["padded"], c["tokens"])
        return {"bytes": 2 * n * c["kv"] * c["d"] * (item + cell) + c["tokens"] * 8, "flops": 0}
    if kind == "rope":
        n = c["tokens"] - min(c["padded"], c["tokens"])
        heads = c["hq"] + 2 * c["kv"]
        return {"bytes": 2 * n * heads * c["d"] * item + n * c["d"] * 4 + c["tokens"] * 12,
                "flops": n * (c["hq"] + c["kv"]) * c["d"] * 7}
    seen = sum(min(n, c["window"]) if c["window"] else n for n in _attend_lens(c))
    out = c["bs"] * c["hq"] * c["d"]
    return {"bytes": 2 * seen * c["kv"] * c["d"] * cell + out * (item + (4 if c["f32"] else item)) +
            _pages_of(seen, c["page"]) * 4 + (c["bs"] * c["hq"] * 4 if c["lse"] else 0),
            "flops": 4 * seen * c["hq"] * c["d"]}


# ---------------------------------------------------------------------------
# the results in 64 bits
# ---------------------------------------------------------------------------
def exact(case: dict, seed: int):
    c = case
    s = _inputs(c, seed)
    if c["kind"] == "tables":
        return None      # whole numbers only
    if c["kind"] == "attend":
        return _exact_attend(s, c)
    new_k, new_v = s.get("k"), s.get("v")
    q = None
    if c["kind"] == "rope":
        n, hq, kv, d = c["tokens"], c["hq"], c["kv"], c["d"]
        x = s["qkv"].double().reshape(n, -1, d)
        at = s["positions"].long().clamp(min=0)
        # the pair (x_i, x_{i + d/2}) as one complex number, turned by the row's angle
        turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]

        def rotated(heads, weight):
            y = heads * weight.double() / (heads.square().sum(-1, keepdim=True) / d + s["eps"]).sqrt()
            z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        q = rotated(x[:, :hq], s["q_norm"])
        q[s["positions"] < 0] = 0.0
        new_k, new_v = rotated(x[:, hq:hq + kv], s["k_norm"]), x[:, hq + kv:]
    pages = []
    for name, rows in (("k", new_k), ("v", new_v)):
        pool = s[name + "_pages"].to(torch.float64)
        scale = s.get(name + "_scale")
        rows = rows.double() if scale is None else rows.double() / scale.double()[:, None]
        if scale is not None:
            rows = rows.clamp(-_E4M3_MAX, _E4M3_MAX)
        for h in range(c["kv"]):
            flat = torch.empty(pool.shape[0] * c["page"], c["d"], dtype=torch.float64, device=_DEV)
            flat.copy_(pool[:, h].reshape(flat.shape))
            keep = s["slots"] >= 0
            flat.index_copy_(0, s["slots"][keep], rows[keep, h])
            pool[:, h] = flat.view(pool.shape[0], c["page"], c["d"])
        pages.append(pool)
    return tuple(pages) if q is None else (q, *pages)


def _exact_attend(s, c):
    bs, hq, kv, d = c["bs"], c["hq"], c["kv"], c["d"]
    out = torch.zeros(bs, 1, hq, d, dtype=torch.float64, device=_DEV)
    lse = torch.full((bs, hq, 1), float("-inf"), dtype=torch.float64, device=_DEV)
    page = c["page"]
    for b, n in enumerate(_attend_lens(c)):
        if n == 0:
            continue
        t = torch.arange(max(0, n - c["window"]) if c["window"] else 0, n, device=_DEV)
        where = s["table"][b].long()[t // page]
        for h in range(kv):
            heads = slice(h * (hq // kv), (h + 1) * (hq // kv))
            kk, vv = (_cells(s[x + "_pages"][:, h], where, t % page, s[x + "_scale"], h) for x in "kv")
            x = torch.mm(s["q"][b, 0, heads].double(), kk.t()) * d ** -0.5
            z = torch.logsumexp(x, -1, keepdim=True)
            out[b, 0, heads] = torch.mm((x - z).exp(), vv)
            lse[b, heads] = z
    return (out, lse) if c["lse"] else out


def _cells(pool, where, off, scale, h):
    """Rows (where, off) of one head's pages in 64 bits."""
    if pool.dtype == torch.float8_e4m3fn:
        return pool.view(torch.uint8)[where, off].view(torch.float8_e4m3fn).double() * scale[h].double()
    return pool[where, off].double()
