"""What paged_cache counts and refuses on the host, on CPU tensors: its tables
advance by oracle/paged.py's plain form, and every launch is written down."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from zoomkv_revision_amd import paged
from zoomkv_revision_amd.paged_cache import paged_cache

BF = torch.bfloat16


@pytest.fixture
def make(monkeypatch):
    """A cache of `batch` rows over `pages` pages of 4 tokens, one KV head of 64,
    two layers; cache.launched lists what reached the device."""

    def build(batch=3, pages=12, max_length=40):
        c = object.__new__(paged_cache)
        c.layer_num, c.batch_size, c.max_length, c.page_size, c.num_pages = 2, batch, max_length, 4, pages
        c.kv_head, c.num_heads, c.head_dim, c.dtype, c.kv_dtype = 1, 1, 64, BF, BF
        c.valid_start, c.device = [0] * batch, torch.device("cpu")
        c.tables = paged.PageTables.allocate(batch, max_length, pages, 4, device="cpu")
        c.k_pages, c.v_pages = ([torch.zeros(pages, 1, 4, 64, dtype=BF) for _ in range(2)] for _ in range(2))
        c.k_scale, c.v_scale = [None, None], [None, None]
        c.context, c.lengths, c._prompt_slots, c._max_positions = 0, [0] * batch, {}, None
        c.active = torch.zeros(batch, dtype=torch.int32)
        c.slots = torch.full((batch,), -1, dtype=torch.int64)
        c.positions = torch.full((batch,), -1, dtype=torch.int32)
        c.launched = []

        def advance(tables, new, slots=None, positions=None, row=0, **_):
            c.launched.append("page_advance")
            n = [t.numpy() for t in (tables.seq_lens, new, tables.block_table, tables.free_pages, tables.state)]
            out = op.advance(*n, tables.page_size, 0 if slots is None else slots.numel(), row)
            for t, x in zip((tables.seq_lens, tables.block_table, tables.free_pages, tables.state, slots, positions), out):
                if t is not None:
                    t.copy_(torch.from_numpy(x))

        class Step:
            def run(self):
                advance(c.tables, c.active, c.slots, c.positions, row=1)

        c._step = Step()
        monkeypatch.setattr(paged, "page_advance", advance)
        monkeypatch.setattr(paged, "paged_write", lambda *a: c.launched.append("paged_write"))
        monkeypatch.setattr(paged, "paged_qk_norm_rope", lambda *a: c.launched.append("paged_qk_norm_rope"))
        return c

    return build


def _prefill(c, row, n):
    for layer in range(c.layer_num):
        c.prefill_update_kv_cache(None, *(torch.zeros(1, n, 1, 64, dtype=BF) for _ in range(2)), layer, row)


def _state(c):
    t = c.tables
    return [c.lengths[:], c.context, *(x.tolist() for x in (t.seq_lens, t.block_table, t.free_pages, t.state, c.active))]


def test_the_host_and_the_tables_count_alike(make):
    c = make()
    for row, n in ((0, 7), (2, 12)):
        _prefill(c, row, n)
    for _ in range(3):
        for layer in range(2):
            c.decode_begin(layer)
    assert c.lengths == [10, 0, 15] == c.tables.seq_lens.tolist() and c.positions.tolist() == [9, -1, 14]
    c.release([0])
    _prefill(c, 2, 3)
    assert c.lengths == [0, 0, 3] == c.tables.seq_lens.tolist() and int(c.tables.state[1]) == 11


# ---------------------------------------------------------------------------
# positions beyond the RoPE table
# ---------------------------------------------------------------------------
def _table(rows):
    return torch.ones(rows, 32)


def test_a_step_beyond_the_rope_table_is_refused_before_it_is_launched(make):
    c = make()
    _prefill(c, 0, 7)
    _prefill(c, 1, 3)
    c.decode_begin(0, 8)              # position 7, the table's last row
    c.decode_begin(1, 8)
    c.launched.clear()
    before = _state(c)
    with pytest.raises(RuntimeError, match="position 8 .* 8 rows"):
        c.decode_begin(0, 8)
    assert _state(c) == before and not c.launched
    c.decode_begin(0, 9)              # a longer table goes on
    c.release(0)
    c.decode_begin(0, 8)              # and so do the others, once the long request has ended
    assert c.lengths == [0, 6, 0]


def test_rope_tables_shorter_than_a_row_are_refused(make):
    """For a step whose decode_begin was not told the table."""
    c = make()
    _prefill(c, 1, 8)
    c.decode_begin(0)
    c.launched.clear()
    w = torch.ones(64, dtype=BF)
    with pytest.raises(RuntimeError, match="position 8 .* 8 rows"):
        c.decode_norm_rope(torch.zeros(3, 192, dtype=BF), w, w, 1e-6, _table(8), _table(8), 0)
    assert not c.launched
    c.decode_norm_rope(torch.zeros(3, 192, dtype=BF), w, w, 1e-6, _table(9), _table(9), 0)
    assert c.launched == ["paged_qk_norm_rope"]


def test_replays_beyond_the_rope_table_are_refused(make):
    c = make()
    _prefill(c, 1, 3)
    for layer in range(2):
        c.decode_begin(layer, 6)      # (the captured step: position 3)
    c.replayed(2)                     # positions 4 and 5
    with pytest.raises(RuntimeError, match="position 6 .* 6 rows"):
        c.replayed()
    assert c.lengths == [0, 6, 0]
    other = make()
    _prefill(other, 1, 3)
    other.decode_begin(0)             # rotated by the caller: no table to run out of
    other.replayed(20)
    assert other.lengths == [0, 24, 0]


# ---------------------------------------------------------------------------
# prompts that are refused
# ---------------------------------------------------------------------------
def test_a_refused_prompt_leaves_the_running_request(make):
    c = make(pages=12, max_length=40)
    _prefill(c, 0, 20)                # 5 pages
    _prefill(c, 1, 17)                # 5 pages
    before = _state(c)
    c.launched.clear()
    rows = lambda n, b=1: [torch.zeros(b, n, 1, 64, dtype=BF) for _ in range(2)]
    with pytest.raises(RuntimeError, match="max_length"):
        c.prefill_update_kv_cache(None, *rows(41), 0, 0)
    with pytest.raises(RuntimeError, match="pages"):
        c.prefill_update_kv_cache(None, *rows(29), 0, 0)          # 8 pages with 5 held by the other row
    with pytest.raises(RuntimeError, match="pages"):
        c.prefill_update_kv_cache(None, *rows(20, 3), 0, 0)
    with pytest.raises(ValueError, match="not on cpu"):
        c.prefill_update_kv_cache(None, *(x.to("meta") for x in rows(4)), 0, 0)
    with pytest.raises(IndexError):
        c.prefill_update_kv_cache(None, *rows(4), 0, 3)
    assert _state(c) == before and not c.launched
    _prefill(c, 0, 28)                # 7 pages: the row's own 5 and the 2 that were free
    assert c.lengths == [28, 17, 0] == c.tables.seq_lens.tolist() and int(c.tables.state[1]) == 0
    assert int(c.tables.state[2]) == 0
    c.release([0, 1])
    for layer in range(2):
        c.prefill_update_kv_cache(None, *rows(16, 3), layer, 0)
    assert c.lengths == [16, 16, 16] == c.tables.seq_lens.tolist()


# ---------------------------------------------------------------------------
# prompts on their way
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("batch", [False, True])
def test_a_prompt_whose_row_is_released_writes_no_more(make, batch):
    """Its pages may be another request's by the time of its next layer."""
    c = make(pages=12)
    rows = lambda n: [torch.zeros(3 if batch else 1, n, 1, 64, dtype=BF) for _ in range(2)]
    at = 0 if batch else 1
    c.prefill_update_kv_cache(None, *rows(8), 0, at)
    c.release(1)
    _prefill(c, 1 if batch else 2, 16)  # a request that takes the row, or another that takes the pages
    c.launched.clear()
    with pytest.raises(RuntimeError, match="without layer 0"):
        c.prefill_update_kv_cache(None, *rows(8), 1, at)
    assert not c.launched


def test_a_prompt_on_its_way_does_not_mind_another_row(make):
    c = make(pages=12)
    rows = lambda n: [torch.zeros(1, n, 1, 64, dtype=BF) for _ in range(2)]
    _prefill(c, 0, 5)
    c.prefill_update_kv_cache(None, *rows(8), 0, 1)
    c.release(0)
    _prefill(c, 2, 16)
    c.prefill_update_kv_cache(None, *rows(8), 1, 1)
    assert c.lengths == [0, 8, 16] and not c._prompt_slots
