"""``paged_cache``: full attention over a paged K / V cache, for a batch whose
requests have lengths of their own.

The counterpart of ``cache.polar_cache`` for requests that attend every token
(below the sparse path's threshold, or a model that is not to select): the same
methods the runtime calls (``prefill_update_kv_cache``, ``sync``,
``decode_update_kv_cache``, ``compute``, the ``context`` counter), selected by
module name like it (``POLAR_CACHE_MODULE=zoomkv_revision_amd.paged_cache``), on
the operators of ``paged``.  Where ``polar_cache`` keeps one run of tokens per
sequence and every sequence at the same position (the reference's layout,
S:519-611), here

  * all requests share one pool of pages per layer, K and V bf16, fp16 or e4m3
    with a scale per head, through one block table for all layers;
  * prompts of a batch may differ in length (``valid_start`` per row), a request
    may end (``release``) and another take its row (a prefill of that row), and
    rows without a request stay idle;
  * a decode step's tables, positions and slots are made on the device
    (``paged.page_advance``), so a captured step replays as the next one.
"""
from __future__ import annotations

import torch

from . import paged
from ._lib import lib


class paged_cache:
    """Paged full-attention decode cache on gfx950 (see module docstring).

    ``page_size`` tokens a page, ``num_pages`` pages a layer (default: enough
    for every row at ``max_length``), ``kv_dtype`` the cells' type (default
    ``dtype``; torch.float8_e4m3fn stores 8 bits, with ``k_scale[layer]`` /
    ``v_scale[layer]`` float32 [kv] once they are set, else 1).

    Its calls share one set of tables, slots and positions and one workspace:
    calls on several streams, and replays beside eager calls, are to be ordered
    one behind the other by the caller.  A cache is ready for any stream once it
    is made."""

    def __init__(self, valid_start, layer_num: int, batch_size: int, max_length: int, num_key_value_heads: int,
                 num_heads: int, head_dim: int, dtype: torch.dtype, layer_mapping: dict, max_new_length: int,
                 num_gpus: int = 1, model_size: int = 0, page_size: int = 16, num_pages: int | None = None,
                 kv_dtype: torch.dtype | None = None) -> None:
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"the model dtype must be bfloat16 or float16 (got {dtype})")
        kv_dtype = dtype if kv_dtype is None else kv_dtype
        if kv_dtype not in (dtype, torch.float8_e4m3fn):
            raise ValueError(f"kv_dtype must be {dtype} or torch.float8_e4m3fn (got {kv_dtype})")
        if head_dim not in paged.HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {paged.HEAD_DIMS} (got {head_dim})")
        if num_heads % num_key_value_heads:
            raise ValueError(f"{num_heads} query heads over {num_key_value_heads} KV heads")
        if not 1 <= batch_size <= paged.MAX_REQUESTS:
            raise ValueError(f"batch_size {batch_size} outside [1, {paged.MAX_REQUESTS}]")
        self.layer_num, self.batch_size, self.max_length = layer_num, batch_size, max_length
        self.kv_head, self.num_heads, self.head_dim = num_key_value_heads, num_heads, head_dim
        self.dtype, self.kv_dtype, self.layer_mapping = dtype, kv_dtype, layer_mapping
        self.num_gpus, self.model_size = num_gpus, model_size
        self.max_new_length, self.input_length = max_new_length, max_length - max_new_length
        self.valid_start = valid_start
        self.page_size = int(page_size)
        self.device = torch.device(list(layer_mapping.values())[0] if layer_mapping else "cuda:0")
        if self.device.type != "cuda":
            raise RuntimeError("paged_cache needs a GPU device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if num_pages is None:
            num_pages = batch_size * -(-max_length // self.page_size)
        self.num_pages = int(num_pages)
        self.tables = paged.PageTables.allocate(batch_size, max_length, self.num_pages, self.page_size, self.device)
        shape = (self.num_pages, num_key_value_heads, self.page_size, head_dim)
        new = lambda: torch.zeros(shape, dtype=kv_dtype, device=self.device)
        self.k_pages = [new() for _ in range(layer_num)]
        self.v_pages = [new() for _ in range(layer_num)]
        self.k_scale: list = [None] * layer_num
        self.v_scale: list = [None] * layer_num
        self.context = 0
        self.lengths = [0] * batch_size          # tokens of each row, as the host has ordered them
        self._max_positions: int | None = None   # rows of the RoPE table that the last decode step was given
        # one decode step: which rows get a token, and where it goes
        self.active = torch.zeros(batch_size, dtype=torch.int32, device=self.device)
        self.slots = torch.full((batch_size,), -1, dtype=torch.int64, device=self.device)
        self.positions = torch.full((batch_size,), -1, dtype=torch.int32, device=self.device)
        self._step = paged.PageAdvancePlan(self.tables, self.active, self.slots, self.positions, row=1)
        self._prompt_slots: dict = {}
        self._workspace = paged.new_workspace(self.device, lib().zkv_paged_attention_workspace_size(head_dim))
        torch.cuda.current_stream(self.device).synchronize()    # the buffers are filled, whatever stream comes first

    # ------------------------------------------------------------------
    # bookkeeping
    # ------------------------------------------------------------------
    def _pages(self, n: int) -> int:
        return -(-n // self.page_size)

    def _fitted(self, lengths: list[int], new: list[int]) -> list[int]:
        """Rows of these lengths after a step; refuses one that does not fit."""
        after = [n + max(x, -n) for n, x in zip(lengths, new)]
        # pages that this step gives back serve later steps
        held = sum(self._pages(max(a, b)) for a, b in zip(after, lengths))
        if max(after) > self.max_length:
            raise RuntimeError(f"a request of {max(after)} tokens exceeds max_length {self.max_length}")
        if held > self.num_pages:
            raise RuntimeError(f"{held} pages needed, the pool has {self.num_pages}")
        return after

    def _grow(self, new: list[int]) -> None:
        """The host's count of the rows after a step; refuses one that does
        not fit before anything is launched (tables.check() has the device's
        word, for steps that were replayed)."""
        self.lengths = self._fitted(self.lengths, new)

    def _refuse_positions(self, max_positions: int | None, length: int) -> None:
        """A step whose longest row ends at `length` tokens rotates it at
        position length - 1: that is to be a row of the RoPE table."""
        if max_positions is not None and length > max_positions:
            raise RuntimeError(f"position {length - 1} is beyond the RoPE table's {max_positions} rows")

    def _rows_tensor(self, values: list[int]) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.device)

    def check(self) -> None:
        """Raise RuntimeError if a step, replayed ones included, could not
        serve a request (reads the device: call it where the caller
        synchronises anyway)."""
        self.tables.check()

    def replayed(self, steps: int = 1) -> None:
        """Count `steps` replays of a captured decode step beyond the first
        (which the capture counted), each one more token of every active row;
        refuses what the host can count, the pool and the captured step's RoPE
        table among it: call it before the replays where they may run out."""
        for _ in range(steps):
            self._refuse_positions(self._max_positions, max(n + 1 if n else 0 for n in self.lengths))
            self._grow([1 if n else 0 for n in self.lengths])
            self.context += 1

    def release(self, rows) -> None:
        """End the requests of these rows: their pages serve later steps, the
        rows are idle until a prefill gives them a request (one that has not
        reached its last layer ends with them)."""
        rows = [int(r) for r in ([rows] if isinstance(rows, int) else rows)]
        if any(not 0 <= r < self.batch_size for r in rows):
            raise ValueError(f"rows {rows} outside [0, {self.batch_size})")
        new = [0] * self.batch_size
        for r in rows:
            new[r] = -self.lengths[r]
        self._grow(new)
        # the slots of a prompt on its way may be another request's from now on
        self._prompt_slots = {(bsz, r): slots for (bsz, r), slots in self._prompt_slots.items()
                              if not any(r <= x < r + bsz for x in rows)}
        paged.page_advance(self.tables, self._rows_tensor(new))
        self.active.copy_(self._rows_tensor([int(n > 0) for n in self.lengths]))

    # ------------------------------------------------------------------
    # prefill
    # ------------------------------------------------------------------
    def prefill_update_kv_cache(self, query_states, key_states, value_states, layer_idx, batch_idx):
        """key_states / value_states [bsz, seq_len, kv, d], left-padded by
        valid_start; bsz == 1 writes row batch_idx, bsz == batch_size writes
        all rows (on batch_idx 0), each with its own valid_start.  Layer 0 comes
        first and makes the pages (a row that holds a request is released; a
        prompt that is refused leaves it running).  Returns the inputs without
        the padding that all rows share."""
        del query_states
        bsz, seq = key_states.shape[:2]
        if key_states.shape != value_states.shape or tuple(key_states.shape[2:]) != (self.kv_head, self.head_dim):
            raise ValueError(f"keys / values must be [bsz, seq, {self.kv_head}, {self.head_dim}]; got "
                             f"{tuple(key_states.shape)}, {tuple(value_states.shape)}")
        if key_states.device != self.device or value_states.device != self.device:
            raise ValueError(f"keys / values are on {key_states.device}, {value_states.device}, not on {self.device}")
        if bsz != 1 and bsz != self.batch_size:
            raise ValueError(f"bsz ({bsz}) must be 1 or the cache batch_size ({self.batch_size})")
        start = lambda r: int(self.valid_start[r]) if hasattr(self.valid_start, "__len__") else int(self.valid_start)
        rows = [range(self.batch_size)[batch_idx]] if bsz == 1 else list(range(bsz))
        starts = [start(r) for r in rows]
        if any(not 0 <= s <= seq for s in starts):
            raise ValueError(f"valid_start {starts} outside [0, {seq}]")
        shared = min(starts)
        if bsz > 1 and batch_idx != 0:
            return key_states[:, shared:], value_states[:, shared:]
        key = (bsz, rows[0])
        if layer_idx == 0:
            new, others = [0] * self.batch_size, self.lengths[:]
            for r, s in zip(rows, starts):
                new[r], others[r] = seq - s, 0
            self._fitted(others, new)
            slots = torch.empty(self.batch_size * seq if bsz > 1 else seq, dtype=torch.int64, device=self.device)
            if any(self.lengths[r] for r in rows):
                self.release([r for r in rows if self.lengths[r]])
            self._grow(new)
            paged.page_advance(self.tables, self._rows_tensor(new), slots, row=seq if bsz > 1 else 0)
            if bsz == 1:          # (packed: the row's tokens from place 0 on; its padding has no slot)
                slots = torch.cat((slots.new_full((starts[0],), -1), slots[:seq - starts[0]]))
            self._prompt_slots[key] = slots
            self.active.copy_(self._rows_tensor([int(n > 0) for n in self.lengths]))
            self.context = max(self.lengths)
        slots = self._prompt_slots.get(key)
        if slots is None or slots.numel() != bsz * seq:
            raise RuntimeError(f"prefill of layer {layer_idx} without layer 0 of the same rows before it")
        flat = lambda t: t.reshape(bsz * seq, self.kv_head, self.head_dim).to(self.dtype)
        paged.paged_write(flat(key_states), flat(value_states), slots, self.k_pages[layer_idx],
                          self.v_pages[layer_idx], self.k_scale[layer_idx], self.v_scale[layer_idx])
        if layer_idx == self.layer_num - 1:
            del self._prompt_slots[key]
        return key_states[:, shared:], value_states[:, shared:]

    def sync(self, layer_idx, batch_idx):
        """Nothing to wait for: every write is on the caller's stream."""
        del layer_idx, batch_idx

    # ------------------------------------------------------------------
    # decode
    # ------------------------------------------------------------------
    def decode_begin(self, layer_idx, max_positions: int | None = None) -> None:
        """The bookkeeping of a decode step, without the write: at layer 0 every
        active row gets its next place (``positions`` int32 [bs], ``slots``
        int64 [bs], -1 for idle rows), which serve all layers.  max_positions:
        the rows of the RoPE table that the step goes on with; a step (or a
        replay of it) that needs a row beyond is refused before anything is
        launched."""
        if layer_idx == 0:
            self._refuse_positions(max_positions, max(n + 1 if n else 0 for n in self.lengths))
            self._grow([1 if n else 0 for n in self.lengths])
            self._max_positions = max_positions
            self._step.run()
        if layer_idx == self.layer_num - 1:
            self.context += 1

    def decode_write(self, key_states, value_states, layer_idx) -> None:
        """K / V [bs, 1, kv, d] of the step's token into its slots."""
        paged.paged_write(key_states[:, 0].to(self.dtype), value_states[:, 0].to(self.dtype), self.slots,
                          self.k_pages[layer_idx], self.v_pages[layer_idx], self.k_scale[layer_idx],
                          self.v_scale[layer_idx])

    def decode_update_kv_cache(self, key_states, value_states, layer_idx):
        """Append one token ([bs, 1, kv, d]) of one layer to every active row.
        Returns (None, None)."""
        self.decode_begin(layer_idx)
        self.decode_write(key_states, value_states, layer_idx)
        return None, None

    def decode_norm_rope(self, qkv, q_norm, k_norm, eps, cos, sin, layer_idx) -> torch.Tensor:
        """decode_write from the fused projection qkv [bs, (heads + 2 kv) d],
        with the q / k norms and RoPE at each row's position; the query heads
        [bs, 1, heads, d] (idle rows 0).  Refuses tables cos / sin that a row's
        position lies beyond (its token would not be written)."""
        if cos.shape[0] != self._max_positions:      # (else decode_begin or the layer before has looked)
            self._refuse_positions(cos.shape[0], max(self.lengths))
            self._max_positions = cos.shape[0]
        q = torch.zeros(self.batch_size, 1, self.num_heads, self.head_dim, dtype=self.dtype, device=self.device)
        return paged.paged_qk_norm_rope(qkv, self.num_heads, self.kv_head, q_norm, k_norm, eps, cos, sin,
                                        self.positions, self.slots, q, self.k_pages[layer_idx],
                                        self.v_pages[layer_idx], self.k_scale[layer_idx], self.v_scale[layer_idx])

    def compute(self, queries, layer_idx):
        """queries [bs, 1, num_heads, d] -> attention over each row's tokens, of
        the same shape (zeros for idle rows)."""
        return paged.paged_attention(queries, self.k_pages[layer_idx], self.v_pages[layer_idx],
                                     self.tables.block_table, self.tables.seq_lens, k_scale=self.k_scale[layer_idx],
                                     v_scale=self.v_scale[layer_idx], workspace=self._workspace)


polar_cache = paged_cache   # the class name the runtime imports (Z/model_hub/qwen.py:336-350)
