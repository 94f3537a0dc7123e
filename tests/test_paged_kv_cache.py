"""PagedKVCache's bookkeeping on the CPU, where a stand-in for the operator keeps the slots that it is given."""
import pytest
import torch

from pytorch_amd.contrib.module import PagedKVCache

BATCH, HEADS, DIM, PAGE = 2, 3, 8, 4


class Bookkeeping(PagedKVCache):
    def __init__(self, max_tokens=8, **more):
        super().__init__(BATCH, max_tokens, HEADS, DIM, block_size=PAGE, **more)

    def replayed(self, name, *args):
        """The call as a replay of a captured one makes it: past the host's count."""
        held, self._held = self._held, [0] * BATCH
        getattr(self, name)(*args)
        self._held = held


@pytest.fixture(autouse=True)
def operator(monkeypatch):
    """npu_paged_cache_write's checks of shape and type, and a list of the slots."""
    def write(key, value, key_cache, value_cache, slots, *, key_scale=None, value_scale=None):
        if key.shape != (slots.shape[0], HEADS, DIM) or value.shape != key.shape or key.dtype != key_cache.dtype:
            raise RuntimeError("key must have shape")
        write.slots.append(slots.tolist())

    write.slots = []
    monkeypatch.setattr(torch.ops.npu, "npu_paged_cache_write", write)
    return write


def rows(n):
    return (torch.zeros(n, HEADS, DIM, dtype=torch.bfloat16),) * 2


def test_places_and_positions(operator):
    c = Bookkeeping(budget=6)
    c.prefill(0, *rows(5))
    c.append(*rows(BATCH))
    assert operator.slots == [[0, 1, 2, 3, 4], [5, 8]]
    assert c.context_lens.tolist() == c.next_position.tolist() == [6, 1]
    assert c.positions[0].tolist() == [[0, 1, 2, 3, 4, 5, -1, -1]] * HEADS and c.positions[1].tolist() == [[0] + [-1] * 7] * HEADS


def test_replays_that_overfill_append_nothing(operator):
    c = Bookkeeping(budget=6)
    c.prefill(0, *rows(7))
    for _ in range(4):
        c.replayed("append", *rows(BATCH))
    assert operator.slots[1:] == [[7, 8], [-1, 9], [-1, 10], [-1, 11]]
    assert c.context_lens.tolist() == [8, 4]
    assert c.positions[0].tolist() == [list(range(8))] * HEADS          # of the tokens that are held
    assert c.positions[1].tolist() == [[0, 1, 2, 3, -1, -1, -1, -1]] * HEADS
    assert c.next_position.tolist() == [8, 4]                           # the next one that is held follows them


def test_replays_that_overfill_prefill_what_fits(operator):
    c = Bookkeeping(budget=6)
    c.prefill(1, *rows(6))
    for _ in range(2):
        c.replayed("prefill", 1, *rows(5))
    assert operator.slots[1:] == [[14, 15, -1, -1, -1], [-1] * 5]
    assert c.context_lens.tolist() == [0, 8] and c.next_position.tolist() == [0, 8]
    assert c.positions[1].tolist() == [list(range(8))] * HEADS


def test_refused_calls_do_not_count(operator):
    """What the operator does not take leaves the host's count, and everything else, as it was."""
    c = Bookkeeping()
    c.prefill(0, *rows(5))
    wrong = torch.zeros(3, HEADS, DIM, dtype=torch.float16)
    for call in (lambda: c.prefill(0, wrong, wrong), lambda: c.append(wrong, wrong), lambda: c.append(*rows(BATCH + 1))):
        for _ in range(3):
            with pytest.raises(RuntimeError, match="key must have shape"):
                call()
    with pytest.raises(RuntimeError, match="sequence 0 holds up to 5 tokens, 4 more do not fit into 8"):
        c.prefill(0, *rows(4))
    c.prefill(0, *rows(3))
    assert c.context_lens.tolist() == [8, 0]
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(*rows(BATCH))


def test_blocks_that_the_table_does_not_name_take_nothing(operator):
    """Whatever stands in the table: no slot of the cache comes of a number that names no block."""
    c = Bookkeeping()
    for entry in (-1, -2 ** 31, 2 ** 31 - 1, 2 ** 30, 2 ** 30 + 1, BATCH * 2):
        c.block_table[0, 0] = entry
        c.append(*rows(BATCH))
        c.context_lens.zero_()
        c._held = [0] * BATCH
        assert not 0 <= operator.slots[-1][0] < BATCH * 8 and operator.slots[-1][1] == 8


def test_read_of_blocks_that_the_table_does_not_name(operator, monkeypatch):
    c = Bookkeeping()
    c.block_table[1] = torch.tensor([2 ** 30, 3])
    monkeypatch.setattr(torch.ops.npu, "npu_paged_cache_read", lambda key_cache, value_cache, slots, **more: slots.tolist())
    assert c.read(1, 2, 7) == [2 ** 32 + 2, 2 ** 32 + 3, 12, 13, 14]
    assert c.read(0, 3, 3) == []
