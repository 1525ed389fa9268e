"""The paged K / V cache: page tables, writes and one-token attention (gfx950).

One pool of pages per layer for K and one for V, ``[num_pages, kv, page_size,
d]`` (or any view of that shape whose rows are contiguous and start on 16
bytes, such as the transpose of ``[num_pages, page_size, kv, d]``), shared by
all requests of a batch through a block table:

  * ``PageTables`` / ``page_advance``: one step of a batch's tables on the
    device.  Pages are handed out from a ring of free ids and taken back, the
    block table grows, and every new token gets its slot and position; nothing
    is read by the host, so the step can be captured with the layers after it.
  * ``paged_write``: K / V rows of new tokens into their slots.
  * ``paged_qk_norm_rope``: the same for a decode batch straight from the fused
    QKV projection, with the per-head norms and RoPE at each row's own position
    (``decode_step.qk_norm_rope`` has one position for the whole batch).
  * ``paged_attention``: softmax(q K^T) V of one new token per request over the
    pages of its row of the block table (``attention.gather_attention`` and
    ``flash_attn_with_kvcache_compat`` read one run of rows per sequence).

Cells are bf16 or fp16, or e4m3 (``torch.float8_e4m3fn``) with an fp32 scale
per KV head: a code stands for code * scale.  Each function checks its
arguments on every call; the ``*Plan`` classes check once for fixed buffers and
then make one C-ABI call per ``run()``.

The reference has no paged cache: its layers hold one run of tokens per
sequence, all of the same length (S:519-611).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ._lib import check, device_stream, lib, ptr, require_gpu

HEAD_DIMS = (64, 128, 256)
MAX_REQUESTS = 4096          # of one attention call
MAX_TABLE_REQUESTS = 8192    # of one page_advance call

# status bits of PageTables (ZKV_PAGES_*)
POOL_EMPTY, TABLE_FULL, SLOTS_FULL, BAD_LENGTH, RING_FULL = 1, 2, 4, 8, 16
_STATUS_TEXT = {POOL_EMPTY: "no free pages for a request", TABLE_FULL: "a request exceeds the block table's width",
                SLOTS_FULL: "new tokens exceed the slot map", BAD_LENGTH: "a length is negative or beyond the table",
                RING_FULL: "more pages were given back than the ring holds"}

_WS: dict = {}
_ARRIVAL_BYTES = 1024        # of an attention workspace (ZKV_PAGED_ARRIVAL_BYTES)


def _capturing(device: torch.device) -> bool:
    """Whether the current stream of `device`, which need not be the current
    device, is being captured."""
    if torch.cuda.current_device() == device.index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Arrival counts and partials per (device, stream); under graph capture a
    buffer of the graph's own, so that two graphs never share one (its counts
    are then cleared in the graph, a launch more: a plan, or a workspace that
    is passed in, saves it)."""
    if _capturing(device):
        return new_workspace(device, nbytes)
    key = (device, device_stream(device))
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = _WS[key] = new_workspace(device, nbytes)
    return ws


def new_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """A workspace for paged_attention (zkv_paged_attention_workspace_size(d)
    bytes).  The arrival counts, at the front, are 0 between calls; the partials
    behind them need no clearing.  It is cleared on the current stream: order
    the calls of another stream behind it."""
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    ws[:_ARRIVAL_BYTES].zero_()
    return ws


def _launch(fn, device: torch.device, args) -> None:
    """One C-ABI call on the current stream of `device`, which need not be the
    current device."""
    if torch.cuda.current_device() == device.index:
        check(fn(*args, device_stream(device)))
    else:
        with torch.cuda.device(device):
            check(fn(*args, device_stream(device)))


class _Plan:
    """A checked call over fixed buffers: ``run()`` is one C-ABI call on the
    current stream of their device.  The tensors must stay alive and keep their
    shapes and strides."""

    def __init__(self, fn, device, args, result, keep):
        self._fn, self._device, self._args, self.out, self._keep = fn, device, args, result, keep

    def run(self):
        _launch(self._fn, self._device, self._args)
        return self.out


def _same_device(first: torch.Tensor, **others) -> None:
    device = first.device
    for name, t in others.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _strides(t: torch.Tensor) -> tuple[int, ...]:
    """Strides in elements; those of single-entry dims (any number in torch)
    as 0."""
    strides, shape = t.stride(), t.shape
    return tuple([0 if n == 1 else s for n, s in zip(shape, strides)]) if 1 in shape else strides


def _check_rows(t: torch.Tensor, strides: tuple[int, ...]) -> bool:
    """Whether t's rows are contiguous and start on 16 bytes (strides: t's)."""
    cells = 16 // t.element_size()
    if strides[-1] != 1 or t.data_ptr() % 16:
        return False
    for s in strides[:-1]:
        if s % cells:
            return False
    return True


def _check_pools(k_pages: torch.Tensor, v_pages: torch.Tensor, dtype: torch.dtype, k_scale, v_scale):
    """(is_fp8, num_pages, kv, page_size, d, page / head / token strides)."""
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"rows must be bfloat16 or float16; got {dtype}")
    if k_pages.dtype != v_pages.dtype or k_pages.dtype not in (dtype, torch.float8_e4m3fn):
        raise TypeError(f"pages must be {dtype} or float8_e4m3fn, K and V alike; got {k_pages.dtype}, {v_pages.dtype}")
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError(f"pages must be [num_pages, kv, page_size, d], K and V alike; got {tuple(k_pages.shape)}, "
                         f"{tuple(v_pages.shape)}")
    pages, kv, page, d = k_pages.shape
    if d not in HEAD_DIMS:
        raise ValueError(f"the head dim must be one of {HEAD_DIMS}; got {d}")
    if min(pages, kv, page) < 1 or pages * page >= 1 << 31:
        raise ValueError(f"a pool of {pages} pages of {page} tokens, {kv} heads")
    strides = _strides(k_pages)
    if strides != _strides(v_pages):
        raise ValueError(f"K and V pages must have the same strides; got {k_pages.stride()}, {v_pages.stride()}")
    if not (_check_rows(k_pages, strides) and _check_rows(v_pages, strides)):
        raise ValueError("the rows of a pool must be contiguous and start on 16 bytes")
    fp8 = k_pages.dtype == torch.float8_e4m3fn
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s is None:
            continue
        if not fp8:
            raise ValueError(f"{name} goes with float8_e4m3fn pages")
        if s.dtype != torch.float32 or tuple(s.shape) != (kv,) or (kv > 1 and s.stride(0) != 1):
            raise ValueError(f"{name} must be contiguous float32 [{kv}]")
    _same_device(k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale)
    return int(fp8), pages, kv, page, d, strides[:3]


def _check_ints(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} {list(shape)}; got {t.dtype} {list(t.shape)}")


# ---------------------------------------------------------------------------
# page tables
# ---------------------------------------------------------------------------
@dataclass
class PageTables:
    """The page tables of a batch of requests, on the device.

    block_table int32 [requests, width]: page ids of each request's tokens;
    entries past a request's length are not read.  seq_lens int32 [requests].
    free_pages int32 [num_pages] and state int32 [4]: a ring of the ids that no
    request holds, from place state[0], state[1] of them; state[2] collects
    status bits, state[3] is 0 between calls."""

    block_table: torch.Tensor
    seq_lens: torch.Tensor
    free_pages: torch.Tensor
    state: torch.Tensor
    page_size: int

    @classmethod
    def allocate(cls, requests: int, max_tokens: int, num_pages: int, page_size: int = 16, device="cuda"):
        """Empty tables of `requests` requests of up to max_tokens tokens over
        a pool of num_pages pages, all of them free."""
        if min(requests, max_tokens, num_pages, page_size) < 1:
            raise ValueError("requests, max_tokens, num_pages and page_size must be positive")
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.full((requests, -(-max_tokens // page_size)), -1, **i32), torch.zeros(requests, **i32),
                   torch.arange(num_pages, **i32), torch.tensor([0, num_pages, 0, 0], **i32), int(page_size))

    def check(self) -> None:
        """Raise RuntimeError if any step so far left a request as it was
        (reads the device: call it where the caller synchronises anyway)."""
        bits = int(self.state[2])
        if bits:
            raise RuntimeError("page tables: " + "; ".join(t for b, t in _STATUS_TEXT.items() if bits & b))


def _advance_args(tables, new_tokens, slots, positions, starts, lens_out, state_out, row):
    t = tables
    requests = t.seq_lens.numel()
    if t.block_table.dtype != torch.int32 or t.block_table.dim() != 2 or t.block_table.shape[0] != requests or \
            t.block_table.shape[1] < 1 or (t.block_table.shape[1] > 1 and t.block_table.stride(1) != 1) or \
            (requests > 1 and t.block_table.stride(0) < t.block_table.shape[1]):
        raise ValueError(f"block_table must be int32 [{requests}, width] with contiguous rows")
    if not 1 <= requests <= MAX_TABLE_REQUESTS:
        raise ValueError(f"{requests} requests outside [1, {MAX_TABLE_REQUESTS}]")
    _check_ints("seq_lens", t.seq_lens, torch.int32, (requests,))
    _check_ints("new_tokens", new_tokens, torch.int32, (requests,))
    _check_ints("free_pages", t.free_pages, torch.int32, (t.free_pages.numel(),))
    _check_ints("state", t.state, torch.int32, (4,))
    pages, width, cap = t.free_pages.numel(), t.block_table.shape[1], 0 if slots is None else slots.numel()
    if t.page_size < 1 or pages < 1 or pages > 1 << 30 or pages * t.page_size >= 1 << 31 or \
            width * t.page_size >= 1 << 31:
        raise ValueError(f"{pages} pages of {t.page_size} tokens, {width} a request")
    row = int(row)
    if cap > 1 << 30 or row < 0 or (row and (row * requests != cap or starts is not None)):
        raise ValueError(f"a slot map of {cap} for {requests} requests" + (f" in rows of {row}" if row else ""))
    if slots is not None:
        _check_ints("slots", slots, torch.int64, (cap,))
    if positions is not None:
        _check_ints("positions", positions, torch.int32, (cap,))
    if starts is not None:
        _check_ints("starts", starts, torch.int32, (requests + 1,))
    lens_out = t.seq_lens if lens_out is None else lens_out
    state_out = t.state if state_out is None else state_out
    _check_ints("lens_out", lens_out, torch.int32, (requests,))
    _check_ints("state_out", state_out, torch.int32, (4,))
    _same_device(t.seq_lens, block_table=t.block_table, free_pages=t.free_pages, state=t.state,
                 new_tokens=new_tokens, slots=slots, positions=positions, starts=starts, lens_out=lens_out,
                 state_out=state_out)
    require_gpu(t.seq_lens)
    args = (ptr(t.seq_lens), ptr(new_tokens), requests, ptr(t.block_table),
            t.block_table.stride(0) if requests > 1 else width, width, ptr(t.free_pages), pages, t.page_size,
            ptr(t.state), ptr(slots) if cap else None, ptr(positions) if cap else None, cap, row, ptr(starts),
            ptr(lens_out), ptr(state_out))
    return args, (slots, positions), (t, new_tokens, slots, positions, starts, lens_out, state_out)


class PageAdvancePlan(_Plan):
    """``page_advance`` with its checks done once for fixed buffers."""

    def __init__(self, tables: PageTables, new_tokens, slots=None, positions=None, starts=None, lens_out=None,
                 state_out=None, row=0):
        args, out, keep = _advance_args(tables, new_tokens, slots, positions, starts, lens_out, state_out, row)
        super().__init__(lib().zkv_page_advance, new_tokens.device, args, out, keep)


def page_advance(tables: PageTables, new_tokens: torch.Tensor, slots: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, starts: torch.Tensor | None = None,
                 lens_out: torch.Tensor | None = None, state_out: torch.Tensor | None = None, row: int = 0):
    """One step of the page tables, one launch: request i goes from
    seq_lens[i] to seq_lens[i] + new_tokens[i] tokens (int32; 0: stays; negative:
    drops that many, at most all, which ends the request).

    Pages a request lacks come from the ring's head in request order and are
    written into block_table; pages it no longer needs go behind the ring's
    last, for later steps.  A request grows whole or not at all: one whose
    pages are not free, or whose tokens exceed the block table's width or
    the slot map, keeps its length and sets a status bit (``tables.check()``),
    and from the first that the ring cannot serve on, only requests that need
    no page grow.  slots int64 [capacity] and positions int32 [capacity] get the
    slot and position of each new token, packed in request order, or with
    row > 0 each request's at the end of its row of that many (capacity =
    requests * row: a left-padded batch; 1: a decode batch with idle rows), -1
    for those of a request that was not served and where there is no token;
    starts int32 [requests + 1] (packed only) the running sum of the new tokens,
    at most capacity + 1.
    seq_lens and state are updated in place unless lens_out / state_out are
    given.  Returns (slots, positions)."""
    return PageAdvancePlan(tables, new_tokens, slots, positions, starts, lens_out, state_out, row).run()


# ---------------------------------------------------------------------------
# writes
# ---------------------------------------------------------------------------
def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t if _check_rows(t, _strides(t)) else t.contiguous()


def _write_args(k, v, slots, k_pages, v_pages, k_scale, v_scale, copies: bool):
    fp8, pages, kv, page, d, strides = _check_pools(k_pages, v_pages, k.dtype, k_scale, v_scale)
    if v.dtype != k.dtype:
        raise TypeError(f"k and v must have one type; got {k.dtype}, {v.dtype}")
    if k.dim() != 3 or k.shape != v.shape or tuple(k.shape[1:]) != (kv, d):
        raise ValueError(f"k / v must be [tokens, {kv}, {d}]; got {tuple(k.shape)}, {tuple(v.shape)}")
    n = k.shape[0]
    _check_ints("slots", slots, torch.int64, (n,))
    _same_device(k_pages, k=k, v=v, slots=slots)
    if n * kv * (d // 8) >= (1 << 31) - 1024:
        raise ValueError(f"{n} tokens of {kv} heads in one call")
    if n and not (_check_rows(k, _strides(k)) and _check_rows(v, _strides(v))):
        if not copies:
            raise ValueError("a write plan reads k and v in place: their rows must be contiguous and start on 16 bytes")
        k, v = _aligned(k), _aligned(v)
    require_gpu(k_pages)
    ks, vs = _strides(k), _strides(v)
    args = (ptr(k), ks[0], ks[1], ptr(v), vs[0], vs[1], ptr(slots), n, kv, d, int(k.dtype == torch.float16),
            ptr(k_pages), ptr(v_pages), fp8, ptr(k_scale), ptr(v_scale), pages, page, *strides)
    return args, (k, v, slots, k_pages, v_pages, k_scale, v_scale)


class PagedWritePlan(_Plan):
    """``paged_write`` with its checks done once for fixed buffers."""

    def __init__(self, k, v, slots, k_pages, v_pages, k_scale=None, v_scale=None):
        args, keep = _write_args(k, v, slots, k_pages, v_pages, k_scale, v_scale, copies=False)
        super().__init__(lib().zkv_paged_write if k.shape[0] else _nothing, k_pages.device, args, None, keep)


def _nothing(*_args) -> int:
    return 0


def paged_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """K / V rows [tokens, kv, d] (any token and head strides) into slots int64
    [tokens] of the pools; a slot outside the pool (-1) drops its row.  Slots of
    one call must be distinct.  e4m3 pools take row / scale[head] (scale None:
    1), rounded to nearest even, magnitudes above 448 as 448, NaN kept."""
    args, keep = _write_args(k, v, slots, k_pages, v_pages, k_scale, v_scale, copies=True)
    if keep[0].shape[0]:
        _launch(lib().zkv_paged_write, k_pages.device, args)


def _rope_args(qkv, heads, kv_heads, q_norm, k_norm, eps, cos, sin, positions, slots, q_out, k_pages, v_pages,
               k_scale, v_scale, copies: bool):
    fp8, pages, kv, page, d, strides = _check_pools(k_pages, v_pages, qkv.dtype, k_scale, v_scale)
    heads, kv_heads = int(heads), int(kv_heads)
    if kv_heads != kv or heads < 1:
        raise ValueError(f"{heads} / {kv_heads} heads over pools of {kv}")
    if qkv.dim() != 2 or qkv.shape[1] != (heads + 2 * kv) * d:
        raise ValueError(f"qkv must be [rows, ({heads} + 2 * {kv}) * {d}]; got {tuple(qkv.shape)}")
    n = qkv.shape[0]
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w.dtype != qkv.dtype or tuple(w.shape) != (d,) or w.stride(0) != 1 or w.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous {qkv.dtype} [{d}] on 16 bytes")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != d // 2 or t.shape != cos.shape or \
                not t.is_contiguous() or t.data_ptr() % 16 or t.shape[0] < 1:
            raise ValueError(f"{name} must be contiguous float32 [positions, {d // 2}]")
    _check_ints("positions", positions, torch.int32, (n,))
    _check_ints("slots", slots, torch.int64, (n,))
    if q_out.dtype != qkv.dtype or not q_out.is_contiguous() or q_out.numel() != n * heads * d or \
            q_out.data_ptr() % 16:
        raise ValueError(f"q_out must be contiguous {qkv.dtype} [{n}, {heads}, {d}]")
    if n * (heads + 2 * kv) * (d // 8) >= (1 << 31) - 256:
        raise ValueError(f"{n} rows of {heads + 2 * kv} heads in one call")
    _same_device(k_pages, qkv=qkv, q_norm=q_norm, k_norm=k_norm, cos=cos, sin=sin, positions=positions, slots=slots,
                 q_out=q_out)
    if n and not _check_rows(qkv, _strides(qkv)):
        if not copies:
            raise ValueError("a rope plan reads qkv in place: its rows must be contiguous and start on 16 bytes")
        qkv = qkv.contiguous()
    require_gpu(k_pages)
    args = (ptr(qkv), _strides(qkv)[0], n, heads, kv, d, int(qkv.dtype == torch.float16), ptr(q_norm), ptr(k_norm),
            float(eps), ptr(cos), ptr(sin), cos.shape[0], ptr(positions), ptr(slots), ptr(q_out), ptr(k_pages),
            ptr(v_pages), fp8, ptr(k_scale), ptr(v_scale), pages, page, *strides)
    return args, (qkv, q_norm, k_norm, cos, sin, positions, slots, q_out, k_pages, v_pages, k_scale, v_scale)


class PagedRopePlan(_Plan):
    """``paged_qk_norm_rope`` with its checks done once for fixed buffers."""

    def __init__(self, qkv, heads, kv_heads, q_norm, k_norm, eps, cos, sin, positions, slots, q_out, k_pages, v_pages,
                 k_scale=None, v_scale=None):
        args, keep = _rope_args(qkv, heads, kv_heads, q_norm, k_norm, eps, cos, sin, positions, slots, q_out, k_pages,
                                v_pages, k_scale, v_scale, copies=False)
        super().__init__(lib().zkv_paged_qk_norm_rope if qkv.shape[0] else _nothing, k_pages.device, args, q_out, keep)


def paged_qk_norm_rope(qkv: torch.Tensor, heads: int, kv_heads: int, q_norm: torch.Tensor, k_norm: torch.Tensor,
                       eps: float, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                       q_out: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                       k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Per-head RMSNorm of q and k, rotate-half RoPE at each row's position and
    the K / V rows into their slots: qkv [rows, (heads + 2 kv_heads) * d] ->
    q_out [rows, heads, d]; cos / sin float32 [max_positions, d / 2], positions
    int32 [rows], slots int64 [rows].  fp32 throughout, rounded once to the
    result's type (``decode_step.qk_norm_rope`` rounds the normed heads to bf16
    first, as the torch layer does).  A row whose position is outside [0,
    max_positions) writes nothing; one whose slot is outside the pool writes
    only q.  Returns q_out."""
    args, keep = _rope_args(qkv, heads, kv_heads, q_norm, k_norm, eps, cos, sin, positions, slots, q_out, k_pages,
                            v_pages, k_scale, v_scale, copies=True)
    if keep[0].shape[0]:
        _launch(lib().zkv_paged_qk_norm_rope, k_pages.device, args)
    return q_out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention_args(q, k_pages, v_pages, block_table, seq_lens, softmax_scale, window, k_scale, v_scale,
                    return_softmax_lse, out, workspace, copies: bool):
    fp8, pages, kv, page, d, strides = _check_pools(k_pages, v_pages, q.dtype, k_scale, v_scale)
    if q.dim() not in (3, 4) or (q.dim() == 4 and q.shape[1] != 1) or q.shape[-1] != d:
        raise ValueError(f"q must be [bs, 1, hq, {d}] or [bs, hq, {d}]; got {tuple(q.shape)}")
    q3 = q[:, 0] if q.dim() == 4 else q
    bs, hq, _ = q3.shape
    if not 1 <= bs <= MAX_REQUESTS:
        raise ValueError(f"{bs} requests outside [1, {MAX_REQUESTS}]")
    if hq < 1 or hq % kv:
        raise ValueError(f"{hq} query heads over {kv} KV heads")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != bs or \
            block_table.shape[1] < 1 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 [{bs}, width] with contiguous rows; got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    _check_ints("seq_lens", seq_lens, torch.int32, (bs,))
    width, window = block_table.shape[1], int(window)
    if window < 0:
        raise ValueError(f"window must not be negative (0: the whole sequence); got {window}")
    window = min(window, (1 << 31) - 1)
    if ((pages - 1) * strides[0] + (page - 1) * strides[2]) * k_pages.element_size() >= 1 << 36:
        raise ValueError("the rows of a pool must start within 64 GiB")
    groups = -(-(hq // kv) // 16)
    if width * page >= (1 << 31) - 32 or bs * kv * groups * (-(-width * page // 32) + 2) >= (1 << 31) - (1 << 20):
        raise ValueError(f"{bs} requests of up to {width * page} tokens in one call")
    out_shape = tuple(q.shape)
    if out is None:
        out = torch.empty(out_shape, dtype=q.dtype, device=q.device)
    elif out.dtype not in (q.dtype, torch.float32) or not out.is_contiguous() or out.numel() != bs * hq * d or \
            out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous {list(out_shape)} tensor of q's dtype or float32 on 16 bytes")
    _same_device(q, k_pages=k_pages, block_table=block_table, seq_lens=seq_lens, out=out, workspace=workspace)
    if not _check_rows(q3, _strides(q3)):
        if not copies:
            raise ValueError("an attention plan reads q in place: its rows must be contiguous and start on 16 bytes")
        q3 = q3.contiguous()
    require_gpu(q)
    lse = torch.empty(bs, hq, 1, dtype=torch.float32, device=q.device) if return_softmax_lse else None
    scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    L = lib()
    need = L.zkv_paged_attention_workspace_size(d)
    ws = _workspace(q.device, need) if workspace is None else workspace
    if ws.dtype != torch.uint8 or ws.numel() < need or not ws.is_contiguous() or ws.data_ptr() % 16:
        raise ValueError(f"workspace must be contiguous uint8 of at least {need} bytes on 16 bytes")
    qs = _strides(q3)
    args = (ptr(q3), qs[0], qs[1], int(q.dtype == torch.float16), ptr(k_pages), ptr(v_pages), fp8, ptr(k_scale),
            ptr(v_scale), pages, page, *strides, ptr(block_table), block_table.stride(0) if bs > 1 else 0, width,
            ptr(seq_lens), bs, hq, kv, d, scale, window, ptr(out), int(out.dtype == torch.float32), ptr(lse), ptr(ws),
            ws.numel())
    keep = (q3, k_pages, v_pages, k_scale, v_scale, block_table, seq_lens, out, lse, ws)
    return args, (out, lse) if return_softmax_lse else out, keep


class PagedAttentionPlan(_Plan):
    """``paged_attention`` with its checks done once for fixed buffers (a
    decode loop: new query, lengths, table entries and pages in the same
    tensors).  A plan has a workspace of its own unless one is given, ready for
    any stream and any capture once the plan is made (which waits for its
    clearing); runs of one plan must not overlap on the device."""

    def __init__(self, q, k_pages, v_pages, block_table, seq_lens, softmax_scale=None, window=0, k_scale=None,
                 v_scale=None, return_softmax_lse=False, out=None, workspace=None):
        self._counts = None       # arrival counts that no run has cleared yet
        if workspace is None and q.is_cuda and q.shape[-1] in HEAD_DIMS:
            nbytes = lib().zkv_paged_attention_workspace_size(q.shape[-1])
            if _capturing(q.device):
                # nothing runs here: each captured run clears the counts in its
                # graph, and so does the first eager one, whichever comes first
                workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
                self._counts = workspace[:_ARRIVAL_BYTES]
            else:
                workspace = new_workspace(q.device, nbytes)
                torch.cuda.current_stream(q.device).synchronize()
        args, result, keep = _attention_args(q, k_pages, v_pages, block_table, seq_lens, softmax_scale, window, k_scale,
                                             v_scale, return_softmax_lse, out, workspace, copies=False)
        super().__init__(lib().zkv_paged_attention, q.device, args, result, keep)

    def run(self):
        if self._counts is not None:
            self._counts.zero_()
            if not _capturing(self._device):
                self._counts = None
        return super().run()


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, softmax_scale: float | None = None, window: int = 0,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    return_softmax_lse: bool = False, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None):
    """softmax(q K^T * scale) V of one query token per request over its pages,
    one launch: q [bs, 1, hq, d] or [bs, hq, d] (bf16 or fp16; hq a multiple of
    the pools' KV heads), block_table int32 [bs, width], seq_lens int32 [bs]
    with the new token counted in (its K / V already written).  window > 0
    attends the last `window` tokens only.

    Returns out in q's shape and dtype (a float32 ``out`` buffer receives the
    unrounded result) and with ``return_softmax_lse`` also the fp32 LSE [bs,
    hq, 1].  Lengths are read on the device (limited to [0, width *
    page_size]); a request without tokens gives zeros and -inf, and tokens on
    a page id outside the pool are left out.  The result does not depend on
    what other rows of the pages hold, NaN included, and is the same from run
    to run."""
    args, result, _keep = _attention_args(q, k_pages, v_pages, block_table, seq_lens, softmax_scale, window, k_scale,
                                          v_scale, return_softmax_lse, out, workspace, copies=True)
    _launch(lib().zkv_paged_attention, q.device, args)
    return result
