"""oracle/paged.py against closed forms."""
import numpy as np

from oracle import paged as op


def _i32(*x):
    return np.array(x, np.int32)


def test_decode_steps_fill_pages_in_ring_order():
    """Two requests growing token by token from nothing take the ring's pages
    alternately; slots and positions count up inside them."""
    lens, table = _i32(0, 0), np.full((2, 3), -1, np.int32)
    ring, state = _i32(5, 3, 1, 0, 2, 4), _i32(0, 6, 0, 0)
    for t in range(6):
        lens, table, ring, state, slots, pos, starts = op.advance(lens, _i32(1, 1), table, ring, state, 2, 2)
        assert pos.tolist() == [t, t] and starts.tolist() == [0, 1, 2]
        assert slots.tolist() == [table[0, t // 2] * 2 + t % 2, table[1, t // 2] * 2 + t % 2]
    assert table.tolist() == [[5, 1, 2], [3, 0, 4]] and state.tolist() == [0, 0, 0, 0]
    assert lens.tolist() == [6, 6]
    # full tables and an empty ring: nothing moves
    again = op.advance(lens, _i32(1, 0), table, ring, state, 2, 2)
    assert again[0].tolist() == [6, 6] and again[3].tolist() == [0, 0, op.TABLE_FULL, 0]
    assert again[4].tolist() == [-1, -1]


def test_pages_given_back_are_handed_out_later():
    lens, table = _i32(5, 0), _i32(7, 8, 9, -1).reshape(1, 4).repeat(2, 0)
    ring, state = np.zeros(10, np.int32), _i32(9, 1, 0, 0)
    ring[9] = 6
    out = op.advance(lens, _i32(-5, 3), table, ring, state, 2, 3)
    # one page free, two needed: not served; three given back behind it
    assert out[0].tolist() == [0, 0] and out[3].tolist() == [9, 4, op.POOL_EMPTY, 0]
    assert [int(out[2][(9 + i) % 10]) for i in range(4)] == [6, 7, 8, 9]
    out = op.advance(out[0], _i32(0, 3), out[1], out[2], out[3], 2, 3)
    assert out[0].tolist() == [0, 3] and out[1][1, :2].tolist() == [6, 7] and out[3].tolist() == [1, 2, op.POOL_EMPTY, 0]


def test_rows_end_with_their_tokens():
    out = op.advance(_i32(0, 3, 0), _i32(2, 0, 4), np.full((3, 2), -1, np.int32), np.arange(4, dtype=np.int32),
                     _i32(0, 4, 0, 0), 2, 9, row=3)
    assert out[4].tolist() == [-1, 0, 1, -1, -1, -1, -1, -1, -1] and out[5].tolist() == [-1, 0, 1] + [-1] * 6
    assert out[0].tolist() == [2, 3, 0] and out[3][2] == op.SLOTS_FULL


def test_every_status_bit():
    t = np.zeros((1, 2), np.int32)
    one = lambda have, n, count=4, cap=8: op.advance(_i32(have), _i32(n), t, np.arange(4, dtype=np.int32),
                                                    _i32(0, count, 0, 0), 2, cap)[3][2]
    assert one(0, 4) == 0
    assert one(0, 4, count=1) == op.POOL_EMPTY
    assert one(0, 5) == op.TABLE_FULL
    assert one(0, 3, cap=2) == op.SLOTS_FULL
    assert one(-1, 1) == one(5, 0) == op.BAD_LENGTH
    assert one(4, -4, count=3) == op.RING_FULL


def test_attention_of_equal_keys_is_the_mean():
    v = np.arange(12.0).reshape(4, 3)
    out, lse, mass = op.attention(np.ones((2, 3)), np.zeros((4, 3)), v, 1.0)
    assert np.allclose(out, v.mean(0)) and np.allclose(lse, np.log(4)) and np.allclose(mass, np.abs(v).mean(0))
    out, lse, _ = op.attention(np.ones((2, 3)), np.zeros((0, 3)), np.zeros((0, 3)), 1.0)
    assert not out.any() and np.isneginf(lse).all()


def test_norm_rope_turns_pairs():
    x = np.array([3.0, 4.0, 0.0, 0.0])
    turned = op.norm_rope(x, np.ones(4), 0.0, np.zeros(2), np.ones(2))     # by 90 degrees
    assert np.allclose(turned, [0, 0, 3 / 2.5, 4 / 2.5])
    assert np.allclose(op.norm_rope(x, 2 * np.ones(4), 0.0, np.ones(2), np.zeros(2)), x / 1.25)
