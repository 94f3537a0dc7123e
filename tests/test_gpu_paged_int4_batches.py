"""4-bit attention over whole batches: ranges that end one sequence and begin the next, maxima that rise, what is not a number, far blocks,
streams and graphs.  Tolerances are those of test_gpu_paged_int4.py; where other ones are taken they are derived there."""
import importlib.util
import math
import os

import pytest
import torch

from test_gpu_paged import gpu, tables
from test_gpu_paged_int4 import Cache, attend, check_attention, pa, pack  # noqa: F401

pytestmark = pytest.mark.gpu


def batch_of(g, lens, page, heads, kv, dim, dt, order):
    batch, width = len(lens), max(-(-int(max(lens)) // page), 1)
    cache = Cache(g, batch * width + 1, page, kv, dim, order=order)
    table = tables(g, batch, width, batch * width + 1, page)
    return cache, torch.randn(batch, heads, dim, generator=g).to(dt), table, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.parametrize("order", ["token", "head"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,longest,page,heads,kv,dim", [
    (2, 2500, 16, 8, 8, 128), (5, 1900, 48, 16, 4, 64), (70, 900, 32, 8, 2, 128), (131, 300, 16, 4, 4, 64), (200, 90, 64, 2, 1, 128), (9, 1200, 16, 6, 2, 256),
    (3, 1500, 16, 5, 1, 80), (20, 400, 80, 20, 1, 96), (33, 33, 16, 3, 3, 16), (1, 6000, 128, 40, 2, 128)])
def test_ragged_batches(pa, batch, longest, page, heads, kv, dim, dt, order):  # noqa: F811
    """Lengths from 0 to `longest`, several empty and several equal ones side by side; the same twice over."""
    g = torch.Generator().manual_seed(batch + dim)
    lens = torch.randint(0, longest + 1, (batch,), generator=g)
    lens[::7], lens[-1] = 0, longest
    lens[1:batch // 3] = min(16, longest)
    cache, q, table, lens = batch_of(g, lens.tolist(), page, heads, kv, dim, dt, order)
    got = attend(pa, cache, q, table, lens)
    check_attention(got, cache, q, table, lens)
    assert bool((got[0][lens.cuda() == 0] == 0).all())
    again = attend(pa, cache, q, table, lens)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("page", [8, 9, 10, 16, 24, 31, 40, 100])
@pytest.mark.parametrize("params", ["head", "token", "spread"])
@pytest.mark.parametrize("masked", [False, True])
def test_blocks_and_masks(pa, page, params, masked):  # noqa: F811
    """Blocks that end inside a tile, with and without a mask; scales and offsets of what is not seen are NaN, unnamed blocks among the others."""
    g = torch.Generator().manual_seed(page)
    dt, order = (torch.bfloat16, "token") if page % 2 else (torch.float16, "head")
    lens = [700, 0, 33, page, page + 1, 250, 1]
    batch, width = len(lens), -(-700 // page)
    cache = Cache(g, batch * width + 1, page, 2, 80, order=order, params=params)
    table = tables(g, batch, width, batch * width + 1, page)
    q, lens = torch.randn(batch, 8, 80, generator=g).to(dt), torch.tensor(lens, dtype=torch.int32)
    mask = torch.rand(batch, width * page, generator=g) < 0.4 if masked else None
    if masked:
        mask[3] = True
    table[0, 2], table[5, 1] = -1, batch * width + 1
    at = torch.arange(width * page)
    unseen = torch.ones(batch * width + 1, page, dtype=torch.bool)
    for b in range(batch):
        see = (at < lens[b]) & ((table[b].long() >= 0) & (table[b] < len(unseen)))[at // page]
        see = see & ~mask[b] if masked else see
        unseen[table[b].long()[at[see] // page], at[see] % page] = False
    for t in (cache.ks, cache.vs, cache.ko, cache.vo):
        t[unseen] = math.nan
    got = attend(pa, cache, q, table, lens, atten_mask=None if mask is None else mask.cuda())
    assert bool(got[0].isfinite().all())
    check_attention(got, cache, q, table, lens, mask=mask)


@pytest.mark.parametrize("page", [8, 12, 24, 64])
def test_sums_over_blocks(pa, page):  # noqa: F811
    """Weights added to the sums of the positions that they belong to, where blocks end inside a tile and sequences are cut."""
    g = torch.Generator().manual_seed(page)
    cache, q, table, lens = batch_of(g, [2100, 30, 0, 333], page, 8, 2, 128, torch.bfloat16, "head")
    width = table.shape[1]
    mask = torch.rand(4, width * page, generator=g) < 0.3
    for m in (None, mask):
        before = torch.rand(4, 2, width * page, generator=g)
        sums = before.cuda()
        got = attend(pa, cache, q, table, lens, atten_mask=None if m is None else m.cuda(), attn_sums=sums)
        check_attention(got, cache, q, table, lens, mask=m, sums=(before, sums))


def test_batches_of_nothing(pa):  # noqa: F811
    g = torch.Generator().manual_seed(0)
    for lens in ([0], [0] * 70, [0, 0, 1, 0], [-3, 5, 0]):
        cache, q, table, n = batch_of(g, [max(x, 1) for x in lens], 16, 4, 2, 64, torch.bfloat16, "head")
        n = torch.tensor(lens, dtype=torch.int32)
        got = attend(pa, cache, q, table, n)
        check_attention(got, cache, q, table, n.clamp(min=0))


def test_lengths_beyond_the_table(pa):  # noqa: F811
    """A length is at most what the table has room for."""
    g = torch.Generator().manual_seed(1)
    cache, q, table, lens = batch_of(g, [64, 64, 64], 16, 8, 2, 128, torch.float16, "head")
    got = attend(pa, cache, q, table, torch.tensor([65, 1 << 30, 2147483647], dtype=torch.int32))
    want = attend(pa, cache, q, table, lens)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_attention(got, cache, q, table, lens)


def test_more_heads_than_workgroups(pa):  # noqa: F811
    g = torch.Generator().manual_seed(2)
    for order in ("token", "head"):
        cache, q, table, lens = batch_of(g, [40, 0, 17], 16, 1600, 800, 16, torch.bfloat16, order)
        check_attention(attend(pa, cache, q, table, lens), cache, q, table, lens)


@pytest.mark.parametrize("climb", ["slow", "steps", "falling", "one high", "far below"])
@pytest.mark.parametrize("order", ["token", "head"])
def test_maxima_that_rise(pa, climb, order):  # noqa: F811
    """Scores that grow slower and faster than the maximum is followed, and that lie far from 0.

    Queries of 1, keys of 128 equal codes 4 with a power of two or a multiple of 2^-6 as scale, offset 0: the products and their sums are whole
    numbers below 2^24, so a score is off by the two roundings of its factor and of the exponent's sum alone, 3 * 2^-24 of the largest |z|,
    and the exponential 2^-20: in all `err`.  Values have scale 1 and offset 0, so each image's sums carry up to 31 + 24."""
    n, dim, kv = 700, 128, 2
    g = torch.Generator().manual_seed(3)
    cache = Cache(g, 44, 16, kv, dim, order=order)
    j = torch.arange(44 * 16.0)
    rise = {"slow": j / 64, "steps": (j // 100) * 2, "falling": 10 - j / 128, "one high": torch.where(j == 333, 12.0, 0.0), "far below": j / 256 - 30}[climb]
    rise = (rise * 64).floor() / 64
    table = torch.arange(44, dtype=torch.int32)[None]
    cache.key = pack(torch.full((44, 16, kv, dim), 4)) if order == "token" else pack(torch.full((44, kv, 16, dim), 4)).transpose(1, 2)
    for t, x in ((cache.ks, rise), (cache.ko, 0 * j), (cache.vs, 1 + 0 * j), (cache.vo, 0 * j)):
        t.copy_(x.view(44, 16, 1).expand(44, 16, kv))
    q = torch.ones(1, 4, dim, dtype=torch.float16)
    lens = torch.tensor([n], dtype=torch.int32)
    out, lse = attend(pa, cache, q, table, lens)
    z = 4.0 * dim * rise[:n].double() / math.sqrt(dim)
    p = torch.softmax(z, 0)
    _, v = cache.values()
    want = (p[:, None, None] * v.flatten(0, 1)[:n]).sum(0).repeat_interleave(2, 0)            # [4, dim]
    err = 3 * 2.0 ** -24 * z.abs().max() * math.log2(math.e) + 2.0 ** -20
    assert bool(((out[0].cpu().double() - want).abs() <= 2.0 ** -11 * want.abs() + 55 * (2 * err + 2.0 ** -16 + 2.0 ** -18)).all())
    assert bool(((lse[0].cpu().double() - torch.logsumexp(z, 0)).abs() <= 2 * err + 2.0 ** -22 * z.abs().max()).all())


@pytest.mark.parametrize("name", ["ks", "ko", "vs", "vo"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_is_no_number(pa, name, value):  # noqa: F811
    """One position of one head with a scale or an offset that is none: outputs of that sequence's heads of it are no numbers, all others as before.
    An infinite scale or offset of a key makes a score of either sign (the sum over the head's codes comes before it is multiplied): a query
    for which it is -infinity does not see the position."""
    g = torch.Generator().manual_seed(4)
    cache, q, table, lens = batch_of(g, [500, 70, 129], 16, 8, 2, 64, torch.bfloat16, "head")
    good = attend(pa, cache, q, table, lens)
    getattr(cache, name)[table[0, 3], 5, 1] = value
    bad = attend(pa, cache, q, table, lens)
    sees = bad[0][0, 4:].isnan().all(-1) | (bad[0][0, 4:].isinf().any(-1))
    if name[0] == "k" and value == math.inf:
        getattr(cache, name)[table[0, 3], 5, 1] = 0.0
        mask = torch.zeros(3, 512, dtype=torch.bool)
        mask[0, 3 * 16 + 5] = True
        without = attend(pa, cache, q, table, lens, atten_mask=mask.cuda())[0][0, 4:]
        # each of the two outputs is off by its rounding, 2^-8, one bf16 term, 2^-5 of the scales, and float32 sums of up to 55 times them
        room = 2 * (2.0 ** -8 * without.abs() + (2.0 ** -5 + 55 * 2.0 ** -12) * cache.vs.abs().max().cuda())
        assert bool((sees | ((bad[0][0, 4:] - without).abs() <= room).all(-1)).all())
    else:
        assert bool(sees.all())
    assert torch.equal(bad[0][0, :4], good[0][0, :4]) and torch.equal(bad[0][1:], good[0][1:]) and torch.equal(bad[1][1:], good[1][1:])
    if name[0] == "v":
        assert torch.equal(bad[1], good[1])


def test_codes_behind_32_bits(pa):  # noqa: F811
    """Codes whose blocks start behind 2^32 bytes, scales and offsets close together."""
    g = torch.Generator().manual_seed(5)
    cache, q, table, lens = batch_of(g, [180, 100], 16, 8, 2, 128, torch.bfloat16, "head")
    block = 1 << 26                                        # words
    blocks, page, heads, words = cache.key.shape
    args = cache.on_gpu()
    for name, t in (("key_cache", cache.key), ("value_cache", cache.value)):
        big = torch.empty(blocks * block, dtype=torch.int32, device="cuda")
        args[name] = torch.as_strided(big, t.shape, (block, words, page * words, 1)).copy_(t)
    got = pa.npu_paged_decode_attention(gpu(q), **args, block_table=table.cuda(), context_lens=lens.cuda(), softmax_lse=True)
    near = attend(pa, cache, q, table, lens)
    assert torch.equal(got[0], near[0]) and torch.equal(got[1], near[1])
    check_attention(got, cache, q, table, lens)


def test_streams(pa):  # noqa: F811
    """Calls on two streams at a time, each with tensors of its own stream."""
    g = torch.Generator().manual_seed(6)
    sets = [batch_of(g, lens, 16, 8, 2, 128, torch.bfloat16, order) for lens, order in (([3000, 40, 900], "head"), ([10, 2000, 0, 1500], "token"))]
    want = [attend(pa, *s) for s in sets]
    inputs = [(s[0].on_gpu(), gpu(s[1]), s[2].cuda(), s[3].cuda()) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                args, q, table, lens = inputs[i]
                got[i].append(pa.npu_paged_decode_attention(q, **args, block_table=table, context_lens=lens, softmax_lse=True))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_two_graphs(pa):  # noqa: F811
    """Two captured calls of different batches, replayed in turn with eager calls and new lengths between them."""
    g = torch.Generator().manual_seed(7)
    sets = [batch_of(g, lens, 16, 8, 2, 128, torch.float16, "head") for lens in ([3000, 40, 900], [900, 2000, 16, 1500, 64])]
    inputs = [(s[0].on_gpu(), gpu(s[1]), s[2].cuda(), s[3].cuda()) for s in sets]
    call = lambda i: pa.npu_paged_decode_attention(inputs[i][1], **inputs[i][0], block_table=inputs[i][2], context_lens=inputs[i][3], softmax_lse=True)  # noqa: E731
    for i in range(2):
        call(i)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    for turn in range(6):
        for i in range(2):
            inputs[i][3].copy_((sets[i][3] * (turn + 1) // 6).int())
            graphs[i].replay()
            want = call(i)
            assert torch.equal(outs[i][0], want[0]) and torch.equal(outs[i][1], want[1])
        torch.cuda.synchronize()


@pytest.mark.parametrize("more", [["--int4-cache"], ["--int4-cache", "--layer"], ["--layer"], ["--int4-cache", "--layer", "--graph"], ["--int8-cache", "--layer", "--graph"]])
def test_example_runs(more):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_paged_cache.py")
    spec = importlib.util.spec_from_file_location("decode_paged_cache", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    y, cache = example.main(["--batch", "3", "--hidden", "512", "--heads", "8", "--kv-heads", "2", "--budget", "64", "--prompt", "60", "--steps", "8"] + more)
    assert y.shape == (3, 512) and bool(torch.isfinite(y).all())
    assert cache.context_lens.tolist() == [64, 64, 64] and cache.bits == (4 if "--int4-cache" in more else 8 if "--int8-cache" in more else 16)
