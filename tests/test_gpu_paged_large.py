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
