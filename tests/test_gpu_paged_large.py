"""The paged operators where a call has more rows than one launch takes: the threads of a grid are numbered in 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


@pytest.mark.parametrize("kind", [torch.float16, "int8"])
def test_write_and_read_more_rows_than_a_grid_takes(pa, kind):
    """2^26 rows and a few, of one element, a wavefront each; in an int8 cache an element is 127 times its scale, or 0."""
    tokens, heads, page = 2 ** 21 + 5, 32, 1 << 14
    blocks = -(-tokens // page)
    cache = [torch.zeros(blocks, page, heads, 1, dtype=torch.int8 if kind == "int8" else kind, device="cuda") for _ in range(2)]
    scale = [torch.zeros(blocks, page, heads, device="cuda") if kind == "int8" else None for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(1)
    new = [torch.randint(-9, 10, (tokens, heads, 1), generator=g, device="cuda").half() * 127 for _ in range(2)]
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:tokens]
    more = {"key_scale": scale[0], "value_scale": scale[1]}
    pa.npu_paged_cache_write(*new, *cache, slots, **more)
    for c, s, x in zip(cache, scale, new):
        stored = c.flatten(0, 1)[slots]
        assert torch.equal(stored if s is None else (stored.float() * s.flatten(0, 1)[slots][..., None]).half(), x)
    for got, x in zip(pa.npu_paged_cache_read(*cache, slots, **more, dtype=torch.float16), new):
        assert torch.equal(got, x)


def test_evict_in_more_heads_than_a_grid_takes(pa):
    """2^22 heads and a few, a workgroup of 1024 threads each; every other sequence has one token too many."""
    batch, heads, d = 2 ** 19 + 3, 8, 8
    cache = [torch.arange(batch * 2 * heads, device="cuda").mul(k).remainder(251).half().reshape(-1, 1, heads, 1).expand(-1, 1, heads, d).contiguous() for k in (3, 7)]
    was = [c.reshape(batch, 2, heads, d).clone() for c in cache]
    table = torch.arange(batch * 2, dtype=torch.int32, device="cuda").reshape(batch, 2)
    lens = torch.arange(batch, dtype=torch.int32, device="cuda") % 2 + 1
    g = torch.Generator(device="cuda").manual_seed(2)
    sums = torch.rand(batch, heads, 2, generator=g, device="cuda")
    positions = torch.tensor([4, 9], dtype=torch.int32, device="cuda").expand(batch, heads, 2).contiguous()
    got = pa.npu_paged_cache_evict(*cache, table, lens, sums, positions, 1, 0)
    second = (sums[..., 1] > sums[..., 0]) & (lens == 2)[:, None]                       # its token stays, and moves
    assert bool((got[0] == 1).all())
    assert torch.equal(got[1][..., 0], torch.where(second, sums[..., 1], sums[..., 0])) and bool((got[1][..., 1] == 0).all())
    assert torch.equal(got[2][..., 0], torch.where(second, 9, 4).int()) and bool((got[2][..., 1] == -1).all())
    for c, w in zip(cache, was):
        now = c.reshape(batch, 2, heads, d)
        assert torch.equal(now[:, 1], w[:, 1]) and torch.equal(now[:, 0], torch.where(second[..., None], w[:, 1], w[:, 0]))


def test_evict_in_more_heads_than_the_moves_of_a_launch(pa):
    """2^16 heads and a few, whose rows are moved by a second launch: the second half of every other sequence takes the first one's place."""
    batch, heads, d, keep = 8193, 8, 256, 33
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = [torch.randint(-99, 100, (batch, 2 * keep, heads, d), generator=g, dtype=torch.int8, device="cuda").half() for _ in range(2)]
    was = [c.clone() for c in cache]
    table = torch.arange(batch, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lens = torch.full((batch,), 2 * keep, dtype=torch.int32, device="cuda")
    late = (torch.arange(batch, device="cuda") % 2 == 1)[:, None, None]
    sums = torch.rand(batch, heads, 2 * keep, generator=g, device="cuda")
    sums = sums + ((torch.arange(2 * keep, device="cuda") >= keep) == late)
    positions = torch.arange(2 * keep, dtype=torch.int32, device="cuda").expand(batch, heads, 2 * keep).contiguous()
    got = pa.npu_paged_cache_evict(*cache, table, lens, sums, positions, keep, 0)
    assert bool((got[0] == keep).all())
    for new, old, rest in ((got[1], sums, 0), (got[2], positions, -1)):
        assert torch.equal(new[..., :keep], torch.where(late, old[..., keep:], old[..., :keep])) and bool((new[..., keep:] == rest).all())
    for c, w in zip(cache, was):
        assert torch.equal(c[:, keep:], w[:, keep:]) and torch.equal(c[:, :keep], torch.where(late[..., None], w[:, keep:], w[:, :keep]))
