"""4-bit attention, one way of cutting the work up after the other: whole sequences (in one round of workgroups and in several), single steps,
equal pieces of several steps, and ranges that end one sequence and begin the next.

`plan` is the rule of csrc/paged_decode_attention.hip (Ranges) on the host; every test says which way it means to take.  Inputs and tolerances are
those of test_gpu_paged_int4_precision.py, whose weight lies on few positions, the first and last ones of 16 and 32 among them, where pieces
begin and end; calls are made twice and give the same bits.
"""
import math

import pytest
import torch

from test_gpu_paged import gpu, tables
from test_gpu_paged_int4 import Cache, attend, check_attention, pa  # noqa: F401
from test_gpu_paged_int4_precision import check_outputs, exact_scores, unlike

pytestmark = pytest.mark.gpu

STEP, START, CUT = 8, 24, 16                                # kStep, kStart, kCut


def plan(lens, page, width, heads, kv, dim):
    """"whole 1" (of so many rounds), "steps", "cut 2" (of so many steps) or "dense 24" (of so many halves of a tile)"""
    pairs = kv * -(-heads // kv // 16)
    per_block = -(-page // 16)
    shares = 256 * (3 if dim <= 128 else 2)
    ranges = max(min(shares // pairs, len(lens) * -(-width * per_block // STEP)), 1)
    halves = [n // page * per_block + -(-(n % page) // 16) for n in (min(max(n, 0), page * width) for n in lens)]
    units = [-(-h // STEP) for h in halves]
    sequences, steps, tallest = sum(h > 0 for h in halves), sum(units), max(units)
    if sequences <= ranges and tallest <= 2:
        return "whole 1"
    if steps <= ranges:
        return "steps"
    average = max(-(-(sum(halves) + sequences * START) // ranges), STEP)
    u, cut = -(-average // STEP) if average <= 2 * STEP else average // STEP, False
    if len(lens) <= 64:
        while u > 1 and sum(-(-n // u) for n in units) <= ranges:
            u, cut = u - 1, True
        u += cut
    elif sequences < ranges:
        cut = steps <= u * (ranges - sequences)
    rounds = -(-sequences // ranges)
    if rounds * (START + tallest * STEP) < START + CUT + (u * STEP if cut else average):
        return f"whole {rounds}"
    return f"cut {u}" if cut else f"dense {average}"


def alternating(n, *lens):
    return [lens[i % len(lens)] for i in range(n)]


# lengths, blocks, heads, key/value heads, head_dim, plan
CASES = {
    "dense": ([3000, 40, 0, 900, 2100], 16, 32, 32, 128, "dense 20"),
    "dense, few ranges": (alternating(20, 700, 30, 0, 350, 17), 16, 64, 64, 128, "dense 56"),
    "dense, heads of 64": ([2500, 0, 0, 17, 1300, 16, 800, 40, 2900], 48, 96, 48, 64, "dense 41"),
    "dense, heads of 256": ([900, 1, 1500, 0, 333, 17, 600], 16, 64, 32, 256, "dense 23"),
    "dense, groups of 20": ([3000, 40, 0, 900, 2100], 32, 320, 16, 80, "dense 20"),
    "dense, more than 64 sequences": (alternating(90, 700, 0, 3, 260, 16, 17, 500), 16, 12, 12, 64, "dense 49"),
    "dense, blocks of 24": ([2600, 24, 0, 25, 1700, 23], 24, 32, 32, 128, "dense 21"),
    "dense, blocks of 40": ([2900, 300, 1, 0, 1290, 1500], 40, 40, 40, 96, "dense 31"),
    "cut": ([1000, 900, 0, 700], 16, 48, 48, 128, "cut 2"),
    "cut in threes": ([2900, 3000, 0, 2960], 64, 32, 32, 128, "cut 3"),
    "cut, heads of 256": ([1000, 980, 0, 1024], 16, 32, 32, 256, "cut 2"),
    "cut, more than 64 sequences": (alternating(70, 520, 500, 0, 510), 32, 4, 4, 64, "cut 2"),
    "cut, blocks of 24": ([0, 0, 3200, 0, 200], 24, 32, 32, 128, "cut 2"),
    "whole, two rounds": ([300] * 64, 16, 16, 16, 128, "whole 2"),
    "whole, three rounds": (alternating(195, 300, 0, 280), 16, 16, 16, 64, "whole 3"),
    "whole, long": ([600] * 30 + [0, 590], 16, 24, 24, 128, "whole 1"),
    "steps": ([2000, 0, 130, 129, 128], 16, 8, 4, 128, "steps"),
    "whole": ([256, 0, 1, 255, 17], 32, 8, 4, 128, "whole 1"),
}


def inputs(name, dt, order, seed=0, exact=True):
    lens, page, heads, kv, dim, way = CASES[name]
    g = torch.Generator().manual_seed(seed + len(name))
    batch, width = len(lens), -(-max(lens) // page)
    assert plan(lens, page, width, heads, kv, dim) == way, plan(lens, page, width, heads, kv, dim)
    cache = Cache(g, batch * width + 1, page, kv, dim, order=order)
    table = tables(g, batch, width, batch * width + 1, page)
    lens = torch.tensor(lens, dtype=torch.int32)
    q = exact_scores(g, cache, table, lens, heads, dt) if exact else torch.randn(batch, heads, dim, generator=g).to(dt)
    return cache, q, table, lens


def same_again(pa, first, cache, q, table, lens, **more):  # noqa: F811
    again = attend(pa, cache, q, table, lens, **more)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dt,order", [(torch.bfloat16, "token"), (torch.bfloat16, "head"), (torch.float16, "head")])
@pytest.mark.parametrize("name", list(CASES))
def test_every_way(pa, name, dt, order):  # noqa: F811
    cache, q, table, lens = inputs(name, dt, order)
    got = attend(pa, cache, q, table, lens)
    check_outputs(got, cache, q, table, lens)
    same_again(pa, got, cache, q, table, lens)


@pytest.mark.parametrize("name", ["dense", "dense, groups of 20", "dense, more than 64 sequences", "cut", "whole, two rounds"])
def test_random_keys(pa, name):  # noqa: F811
    cache, q, table, lens = inputs(name, torch.float16, "head", exact=False)
    check_attention(attend(pa, cache, q, table, lens), cache, q, table, lens)


@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("name", ["dense", "dense, heads of 64", "dense, heads of 256", "dense, groups of 20", "dense, more than 64 sequences",
                                  "dense, blocks of 24", "cut", "cut, more than 64 sequences", "cut, blocks of 24", "whole, two rounds", "steps"])
def test_masks_and_sums(pa, name, masked):  # noqa: F811
    """Masks that hide whole stretches and single positions; the sums of a sequence in several pieces."""
    dt = torch.bfloat16 if len(name) % 2 else torch.float16
    cache, q, table, lens = inputs(name, dt, "head" if masked else "token")
    kv, places = cache.key.shape[2], table.shape[1] * cache.key.shape[1]
    g = torch.Generator().manual_seed(9)
    mask = None
    if masked:
        mask = torch.rand(len(lens), places, generator=g) < 0.2
        mask |= (torch.rand(len(lens), -(-places // 100), generator=g) < 0.2).repeat_interleave(100, 1)[:, :places]
        mask[int(lens.argmax()) - 1] = True
    before = torch.rand(len(lens), kv, places, generator=g)
    sums = before.cuda()
    got = attend(pa, cache, q, table, lens, atten_mask=None if mask is None else mask.cuda(), attn_sums=sums)
    check_outputs(got, cache, q, table, lens, mask=mask, sums=(before, sums))
    same_again(pa, got, cache, q, table, lens, atten_mask=None if mask is None else mask.cuda())


@pytest.mark.parametrize("name", ["dense", "dense, more than 64 sequences", "cut"])
def test_blocks_of_nobody(pa, name):  # noqa: F811
    """Entries of the table that name no block, at the ends of pieces too."""
    cache, q, table, lens = inputs(name, torch.float16, "head")
    g = torch.Generator().manual_seed(5)
    table[torch.rand(table.shape, generator=g) < 0.2] = -1
    table[:, 1::7] = cache.key.shape[0]
    check_outputs(attend(pa, cache, q, table, lens), cache, q, table, lens)


def test_replays_that_change_the_plan(pa):  # noqa: F811
    """One captured call; its lengths make it dense, cut, whole and empty in turn, with eager calls of another batch between them."""
    page, heads, kv, dim, width = 16, 32, 32, 128, 200
    g = torch.Generator().manual_seed(3)
    turns = [([3000, 40, 0, 900, 2100], "dense"), ([100, 16, 256, 0, 1], "whole"), ([1500, 1490, 1510, 1530, 1500], "cut"), ([0] * 5, "whole"),
             ([1, 2, 3, 4, 1000], "steps"), ([2100, 900, 3000, 0, 40], "dense"), ([3200, 3200, 3200, 3200, 3200], "dense"), ([0, 0, 3200, 0, 0], "cut")]
    cache = Cache(g, 5 * width, page, kv, dim, order="head")
    table = tables(g, 5, width, 5 * width, page)
    most = torch.full((5,), page * width, dtype=torch.int32)
    q = exact_scores(g, cache, table, most, heads, torch.bfloat16)
    args = cache.on_gpu() | {"block_table": table.cuda()}
    lens = most.cuda()
    call = lambda n: pa.npu_paged_decode_attention(gpu(q), **args, context_lens=n, softmax_lse=True)  # noqa: E731
    query = gpu(q)
    call(lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pa.npu_paged_decode_attention(query, **args, context_lens=lens, softmax_lse=True)
    for now, way in turns:
        assert plan(now, page, width, heads, kv, dim).split()[0] == way, plan(now, page, width, heads, kv, dim)
        now = torch.tensor(now, dtype=torch.int32)
        lens.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        check_outputs(out, cache, q, table, now)
        want = call(now.cuda())
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        call(most.cuda())


# ------------------------------------------------------------------------------------------------ the general kernel and its launches

@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,page", [(64, 16), (80, 24), (128, 16), (128, 12), (192, 32), (256, 8)])
def test_values_that_lie_otherwise(pa, dim, page, dt, masked):  # noqa: F811
    """Keys and values that do not lie alike, in blocks of 8 tokens and more, with and without a mask and sums; short and long sequences."""
    g = torch.Generator().manual_seed(dim + page)
    lens = [5, 3000, 0, 700, 129]
    width = -(-3000 // page)
    cache = Cache(g, 5 * width, page, 4, dim, order="head")
    table = tables(g, 5, width, 5 * width, page)
    lens = torch.tensor(lens, dtype=torch.int32)
    q = exact_scores(g, cache, table, lens, 12, dt)
    unlike(cache)
    mask = None
    if masked:
        mask = torch.rand(5, width * page, generator=g) < 0.3
        mask[0] = True
    check_outputs(attend(pa, cache, q, table, lens, atten_mask=None if mask is None else mask.cuda()), cache, q, table, lens, mask=mask)
    before = torch.rand(5, 4, width * page, generator=g)
    sums = before.cuda()
    got = attend(pa, cache, q, table, lens, atten_mask=None if mask is None else mask.cuda(), attn_sums=sums)
    check_outputs(got, cache, q, table, lens, mask=mask, sums=(before, sums))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [9, 10, 31])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_sums_in_blocks_of_no_multiple_of_four(pa, dim, page, dt):  # noqa: F811
    g = torch.Generator().manual_seed(dim + page)
    lens = torch.tensor([700, 0, 33, page, page + 1], dtype=torch.int32)
    width = -(-700 // page)
    cache = Cache(g, 5 * width, page, 2, dim)
    table = tables(g, 5, width, 5 * width, page)
    q = exact_scores(g, cache, table, lens, 8, dt)
    mask = torch.rand(5, width * page, generator=g) < 0.3
    for m in (None, mask):
        before = torch.rand(5, 2, width * page, generator=g)
        sums = before.cuda()
        got = attend(pa, cache, q, table, lens, atten_mask=None if m is None else m.cuda(), attn_sums=sums)
        check_outputs(got, cache, q, table, lens, mask=m, sums=(before, sums))


@pytest.mark.parametrize("dim", [80, 128])
@pytest.mark.parametrize("order,params", [("token", "head"), ("head", "head"), ("head", "token")])
def test_eviction_of_many_rows(pa, dim, order, params):  # noqa: F811
    """More rows than the workgroup that chooses them moves by itself: codes, scales and offsets by a launch of their own."""
    g = torch.Generator().manual_seed(dim)
    batch, heads, page, n, keep = 2, 2, 16, 2400, 1100
    width = n // page
    cache = Cache(g, batch * width, page, heads, dim, order=order, params=params)
    table = tables(g, batch, width, batch * width, page)
    lens = torch.tensor([2400, 1900], dtype=torch.int32)
    sums = torch.rand(batch, heads, n, generator=g)
    positions = torch.arange(n, dtype=torch.int32).expand(batch, heads, -1).contiguous()
    args = cache.on_gpu()
    new_lens, new_sums, new_pos = pa.npu_paged_cache_evict(**args, block_table=table.cuda(), context_lens=lens.cuda(), attn_sums=sums.cuda(),
                                                           positions=positions.cuda(), keep=keep, recent=100)
    assert new_lens.tolist() == [keep, keep]
    moved = 0
    for b in range(batch):
        ids, at = table[b].long()[torch.arange(n) // page], torch.arange(n) % page
        for h in range(heads):
            came = new_pos[b, h, :keep].cpu().long()       # positions were the places
            worth = sums[b, h, : int(lens[b])].clone()
            worth[int(lens[b]) - 100:] = math.inf
            assert sorted(came.tolist()) == sorted(worth.argsort(descending=True, stable=True)[:keep].tolist())
            assert torch.equal(new_sums[b, h, :keep].cpu(), sums[b, h, came])
            moved = max(moved, int((came != torch.arange(keep)).sum()))
            for name, old in (("key_cache", cache.key), ("value_cache", cache.value), ("key_scale", cache.ks), ("value_scale", cache.vs),
                              ("key_offset", cache.ko), ("value_offset", cache.vo)):
                assert torch.equal(args[name].cpu()[ids[:keep], at[:keep], h], old[ids[came], at[came], h]), name
    assert moved * dim // 2 > 16384
