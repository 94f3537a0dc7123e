"""How exactly 4-bit attention weighs its values, on inputs whose scores leave nothing in doubt.

Scores.  Key codes are all 4, key offsets 0, the elements of a head's query all the same power of two, so the sums of products are whole
multiples of it below 2^24, exact in float32; a position's key scale makes its score.  What is left are the roundings of scale_value, of its
product with log2(e), of that with the key scale, of the score, of the running maximum and of the differences from it: 8 * 2^-24 of the
largest exponent of two, and 2^-20 for the exponential: `err`.

Outputs.  U half a step of the 16-bit type relative to the value (2^-8 bfloat16, 2^-11 float16); p_j the weight, c_j, o_j, s_j code, offset and
scale of a value.  The weight p_j s_j of a code goes into the matrix instructions in two bf16 terms, each off by 2^-8 of what is left: 2^-16 of
the weight, which counts for the image c_j + 24 <= 31: 31 * 2^-16 sum p_j |s_j|.  Sums are of images and of o_j - 24, in float32: with
S = sum p_j |s_j| (31 + |o_j - 24|), a position's part is rounded on its way at most 32 times within a matrix instruction, three times for each
tile of 128 positions of its wavefront (two terms, one new maximum), and 88 times in the sums of wavefronts and pieces: (3 n / 128 + 120) 2^-24 S.
The sum of probabilities has n / 16 + 60 roundings, 2^-24 of the output each.
"""
import math

import pytest
import torch

from test_gpu_paged import U, attend_ref, gpu, tables
from test_gpu_paged_int4 import Cache, attend, pa, pack, unpack  # noqa: F401

pytestmark = pytest.mark.gpu


def check_outputs(got, cache, q, table, lens, mask=None, sums=None):
    """`got` against 64 bits; `cache` and `q` as in the first paragraph above."""
    dt, dim = q.dtype, q.shape[-1]
    k, v = cache.values()
    out, lse, weights, _, _ = attend_ref(q, k, v, table, lens, mask=mask)
    heads, kv, page = q.shape[1], k.shape[2], k.shape[1]
    n = weights.shape[-1]
    zmax = float(cache.ks.abs().max()) * 4 * float(q.double().abs().sum(-1).max()) / math.sqrt(dim)
    err = 8 * 2.0 ** -24 * zmax * math.log2(math.e) + 2.0 ** -20
    at = torch.arange(n)
    ids = table.long()[:, at // page]                                                    # [B, n]
    there = ((ids >= 0) & (ids < k.shape[0]))[..., None]
    ids = ids.clamp(0, k.shape[0] - 1)
    vs, vo = (torch.where(there, t[ids, at % page].double(), 0.0) for t in (cache.vs, cache.vo))       # [B, n, kv]
    total = lambda t: torch.matmul(weights.view(-1, kv, heads // kv, n), t.permute(0, 2, 1)[..., None]).view(-1, heads)  # noqa: E731
    terms = 31 * 2.0 ** -16 * total(vs.abs())
    S = total(vs.abs() * (31 + (vo - 24).abs()))
    longest = int(lens.clamp(0, n).max())
    unit = 2.0 ** -24
    room = (terms + (2 * err + (3 * longest / 128 + 120) * unit) * S)[..., None] + (longest / 16 + 60) * unit * out.abs()
    bound = U[dt] * out.abs() + (1 + U[dt]) * room + unit
    diff = (got[0].cpu().double() - out).abs()
    assert got[0].dtype == dt and bool((diff <= bound).all()), f"output off by {(diff / bound).max():.3g} bounds"
    empty = lse == -math.inf
    have = got[1].cpu().double()
    assert torch.equal(have == -math.inf, empty)
    assert bool(((have - lse).abs()[~empty] <= 2 * err + (longest / 16 + 60) * unit + 2.0 ** -22 * (1 + lse[~empty].abs())).all())
    if sums is not None:
        before, after = sums
        grown = weights.view(-1, kv, heads // kv, n).sum(2)
        far = (after.cpu().double() - before.double() - grown).abs()
        assert bool((far <= (2 * err + 2.0 ** -21 + (longest / 16 + 60) * unit) * grown + 2.0 ** -23 * (before.double().abs() + grown)).all())


def exact_scores(g, cache, table, lens, heads, dt):
    """Keys and scales of `cache` (in place) and a query: most weight on few positions, first and last ones of 16, 32 and of a block among them."""
    blocks, page, kv, _ = cache.key.shape
    dim = cache.key.shape[-1] * 8
    cache.key.copy_(pack(torch.full((blocks, page, kv, dim), 4)))
    cache.ko.zero_()
    n = table.shape[1] * page
    at = torch.arange(n)
    edge = (at % 16 == 0) | (at % 16 == 15) | (at % page == 0) | (at % page == page - 1)
    for b in range(table.shape[0]):
        last = (at >= int(lens[b]) - 2) & (at < int(lens[b]))
        score = torch.rand(n, kv, generator=g) * 2
        high = edge & (torch.rand(n, generator=g) < 0.15) | last
        score[high] += 3 + 4 * torch.rand(int(high.sum()), kv, generator=g)
        ids = table[b].long()[at // page]
        there = (ids >= 0) & (ids < blocks)
        cache.ks[ids[there], at[there] % page] = (score / (4 * dim) * math.sqrt(dim))[there]
    q = torch.ones(table.shape[0], heads, dim) * 2.0 ** -(torch.arange(heads) % 3)[:, None]
    return q.to(dt)


def unlike(cache):
    """Values, and their offsets, that do not lie as the keys."""
    cache.value, cache.vo = cache.value.contiguous(), cache.vo.contiguous()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order,page,alike", [("head", 16, True), ("token", 16, True), ("head", 24, True), ("head", 16, False), ("head", 5, True)])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_one_token(pa, dt, order, page, alike, dim):  # noqa: F811
    """With one token seen the output is its value, also where that is 0 because code and offset cancel: rows whose least or largest value is 0."""
    g = torch.Generator().manual_seed(dim + page)
    batch, kv = 24, 2
    x = torch.rand(batch, kv, dim, generator=g) * torch.rand(batch, 1, 1, generator=g) * 8
    x[..., ::5] = 0.0
    x[batch // 2:] *= -1
    x[-2:] = torch.randn(2, kv, dim, generator=g) + 20.0
    x = x.to(dt)
    cache = Cache(g, batch, page, kv, dim, order=order)
    if not alike:
        unlike(cache)
    args = cache.on_gpu()
    table = tables(g, batch, 1, batch, page)
    lens = torch.ones(batch, dtype=torch.int32)
    slots = table[:, 0].long() * page
    pa.npu_paged_cache_write(x.cuda(), x.cuda(), slots=slots.cuda(), **args)
    for name, t in (("key_cache", "key"), ("value_cache", "value"), ("key_scale", "ks"), ("value_scale", "vs"), ("key_offset", "ko"), ("value_offset", "vo")):
        getattr(cache, t).copy_(args[name].cpu())
    assert bool((unpack(cache.value)[table[:, 0].long(), 0].double() + cache.vo[table[:, 0].long(), 0].double()[..., None] == 0).any())
    q = torch.zeros(batch, 4, dim, dtype=dt)                # every score is 0
    cache.ks[:] = 0.0
    check_outputs(attend(pa, cache, q, table, lens), cache, q, table, lens)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order,page,alike", [("head", 16, True), ("token", 32, True), ("head", 24, True), ("token", 16, False), ("token", 6, True)])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_few_weights(pa, dt, order, page, alike, dim):  # noqa: F811
    """Most of the weight on few positions, of short and of longer sequences."""
    g = torch.Generator().manual_seed(dim + page)
    lens = torch.tensor([1, 37, 130, 0, 517], dtype=torch.int32)
    width = -(-517 // page)
    cache = Cache(g, 5 * width, page, 2, dim, order=order)
    table = tables(g, 5, width, 5 * width, page)
    q = exact_scores(g, cache, table, lens, 8, dt)
    if not alike:
        unlike(cache)
    check_outputs(attend(pa, cache, q, table, lens), cache, q, table, lens)
