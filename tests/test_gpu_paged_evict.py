"""Eviction over the lengths that real caches have, for every number of held rounds and every width of the moves, by the choosing
kernel and by a second one, against a selection in 64 bits on the CPU.  Everything is exact."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


def chosen(sums, positions, n, keep, recent):
    """Where the tokens of the first min(n, keep) places come from, for one head."""
    places = np.arange(min(n, keep))
    if n <= keep:
        return places
    w, p = sums[:n].astype(np.float64), positions[:n].astype(np.int64)
    order = np.lexsort((np.arange(n), -np.nan_to_num(w, nan=0.0, posinf=np.inf, neginf=-np.inf), np.isnan(w), p <= p.max() - recent))
    kept = np.zeros(n, bool)
    kept[order[:keep]] = True
    places[~kept[:keep]] = np.nonzero(kept[keep:])[0] + keep
    return places


def run(pa, kind, d, pad, page, n, keep, recent, lens, seed):
    g = torch.Generator().manual_seed(seed)
    hkv, batch = 2, len(lens)
    width = -(-n // page)
    cap, blocks = width * page, batch * width + 1
    quant = kind == "int8"
    rows = torch.randint(-128, 128, (2, blocks, hkv, page, d + pad), generator=g)
    key, value = ((r.to(torch.int8) if quant else r.to(kind))[..., :d].transpose(1, 2) for r in rows)
    scales = [torch.rand(blocks, page, hkv, generator=g) if quant else None for _ in range(2)]
    table = torch.randperm(blocks, generator=g)[: batch * width].reshape(batch, width).to(torch.int32)
    sums = torch.exp(2 * torch.randn(batch, hkv, cap, generator=g))
    sums[:, 1] = (sums[:, 1] * 2).round()                           # one head of each sequence with many equal sums
    sums[-1, 1] = 0.0                                               # and one with nothing else, as after a prefill
    for at, x in ((5, np.nan), (n // 3, -np.inf), (n // 2, np.inf), (n - 1, -0.0)):
        sums[0, 0, at] = x
    positions = torch.argsort(torch.rand(batch, hkv, cap, generator=g), -1).to(torch.int32)
    whole = [torch.empty_strided(c.shape, c.stride(), dtype=c.dtype, device="cuda").copy_(c) for c in (key, value)]
    dev = whole + [None if s is None else s.cuda() for s in scales]
    got = pa.npu_paged_cache_evict(dev[0], dev[1], table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), sums.cuda(), positions.cuda(), keep, recent,
                                   key_scale=dev[2], value_scale=dev[3])
    want_sums, want_positions = torch.zeros_like(sums), torch.full_like(positions, -1)
    caches = [t.clone() for t in (key, value, *scales) if t is not None]
    for b, length in enumerate(lens):
        for h in range(hkv):
            src = torch.from_numpy(chosen(sums[b, h].numpy(), positions[b, h].numpy(), length, keep, recent))
            to = torch.arange(len(src))
            want_sums[b, h, : len(src)], want_positions[b, h, : len(src)] = sums[b, h][src], positions[b, h][src]
            for c in caches:
                c[table[b].long()[to // page], to % page, h] = c[table[b].long()[src // page], src % page, h]
    assert got[0].tolist() == [min(length, keep) for length in lens]
    assert torch.equal(got[1].cpu().nan_to_num(nan=-7.0), want_sums.nan_to_num(nan=-7.0)) and torch.equal(got[2].cpu(), want_positions)
    for mine, want in zip([t for t in dev if t is not None], caches):
        assert torch.equal(mine.cpu(), want)


@pytest.mark.parametrize("kind,d,pad,page", [(torch.bfloat16, 128, 0, 16), ("int8", 128, 0, 64), (torch.float16, 33, 3, 24), ("int8", 40, 1, 7)])
@pytest.mark.parametrize("n", [1500, 2100, 2900, 4097, 4500, 8193, 9000, 16385, 17000])
def test_half(pa, kind, d, pad, page, n):
    """Prompts of several lengths brought down to half: many moves, by a second kernel."""
    keep = n // 2
    run(pa, kind, d, pad, page, n, keep, keep // 4, [n, keep + 1, keep, n - n // 5], n + d)


@pytest.mark.parametrize("kind,d,pad,page", [(torch.bfloat16, 128, 0, 16), ("int8", 128, 0, 64), (torch.float16, 33, 3, 24), ("int8", 40, 1, 7)])
@pytest.mark.parametrize("over", [1, 5])
@pytest.mark.parametrize("n", [2060, 4097, 8193, 16385, 33001])
def test_a_few_over(pa, kind, d, pad, page, over, n):
    """A cache that is kept at a budget: few moves, by the choosing kernel."""
    run(pa, kind, d, pad, page, n, n - over, 64, [n, n - over, n - 1], n + d + over)


@pytest.mark.parametrize("kind,d,pad,page", [(torch.bfloat16, 64, 0, 16), ("int8", 16, 1, 16)])
def test_more_places_than_are_held(pa, kind, d, pad, page):
    run(pa, kind, d, pad, page, 40000, 15000, 3000, [40000, 15001], 9)
