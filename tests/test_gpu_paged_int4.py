"""The 4-bit paged cache on the GPU: codes against the write's float32 rule, attention against 64 bits on the CPU.

Tolerances of attention.  u is half a step of the output's type (2^-8 bfloat16, 2^-11 float16).  A kernel's image of a code is c + 24, at
most 31, and the offset o less 24 comes in afterwards, so sums in float32 carry terms of up to (31 + |o - 24|) |q| |scale| where the value
itself may be small:
  exponent   (D + 12) 2^-24 times scale_value * max_j |ks_j| (31 + |ko_j - 24|) * sum_d |q_d|, and 2^-20 for the exponential and the sums
             of probabilities
  output     u |o| for its one rounding; with S = sum_j p_j |vs_j| (31 + |vo_j - 24|): twice the exponent's error, 2^-16 for the two bf16
             terms that a probability times a scale is rounded to, and 2^-18 for float32 sums (of at most 300 terms a lane here), of S.
             bfloat16 outputs may come from one bf16 term r_j = p_j vs_j (1 + e_j), |e_j| <= 2^-8: with the sum of these very r_j the images'
             24 is taken off again, so sum_j r_j (c_j + 24) - 24 sum_j r_j + sum_j p_j vs_j o_j is off by sum_j p_j vs_j e_j c_j, and
             |c_j| <= 8: by 2^-5 of sum_j p_j |vs_j|
  lse        the exponent's error alone;  attn_sums: twice it, and one float32 addition
Codes, scales, offsets, values read back and moved rows are exact.
"""
import math

import pytest
import torch

from test_gpu_paged import U, attend_ref, gpu, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


def pack(codes):
    """int32 words of codes in [-8, 7], [..., D] -> [..., D / 8]"""
    u = (codes.long() & 15).unflatten(-1, (-1, 8)) << torch.arange(0, 32, 4)
    u = u.sum(-1)
    return torch.where(u >= 1 << 31, u - (1 << 32), u).to(torch.int32)


def unpack(words):
    return ((words.long()[..., None] >> torch.arange(0, 32, 4)) & 15 ^ 8).sub(8).flatten(-2)


class Cache:
    """CPU tensors of a 4-bit cache with random codes; `order`: what lies together; `params`: how scales and offsets lie."""

    def __init__(self, g, blocks, page, heads, dim, order="token", pad=0, params="head"):
        def words():
            shape = (blocks, page, heads) if order == "token" else (blocks, heads, page)
            w = pack((torch.randn(*shape, dim, generator=g) * 3).round().clamp(-8, 7))
            w = torch.cat((w, torch.full((*shape, pad), 0x77777777, dtype=torch.int32)), -1)[..., : dim // 8]
            return w if order == "token" else w.transpose(1, 2)

        def param(base, spread):
            t = base + spread * torch.randn(blocks, heads, page, generator=g)
            if params == "head":
                return t.transpose(1, 2)
            t = t.transpose(1, 2).contiguous()
            return t if params == "token" else torch.stack((t, t), -1)[..., 0]

        self.key, self.value = words(), words()
        self.ks, self.vs, self.ko, self.vo = param(0.3, 0.05), param(0.3, 0.05), param(0.5, 0.7), param(0.5, 0.7)

    def values(self):
        """64-bit keys and values"""
        return tuple((unpack(w).double() + o.double()[..., None]) * s.double()[..., None] for w, s, o in ((self.key, self.ks, self.ko), (self.value, self.vs, self.vo)))

    def on_gpu(self):
        return {"key_cache": gpu(self.key), "value_cache": gpu(self.value), "key_scale": gpu(self.ks), "value_scale": gpu(self.vs), "key_offset": gpu(self.ko),
                "value_offset": gpu(self.vo)}


def check_attention(got, cache, q, table, lens, scale=None, mask=None, sums=None):
    dt, dim = q.dtype, q.shape[-1]
    k, v = cache.values()
    out, lse, weights, _, _ = attend_ref(q, k, v, table, lens, scale=scale, mask=mask)
    heads, kv = q.shape[1], k.shape[2]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    bad = cache.ks.isnan() | cache.ko.isnan() | cache.vs.isnan() | cache.vo.isnan()
    span = lambda s, o: torch.where(bad, 0.0, s.double().abs() * (31 + (o.double() - 24).abs()))  # noqa: E731
    err = (dim + 12) * 2.0 ** -24 * abs(scale) * span(cache.ks, cache.ko).max() * q.double().abs().sum(-1) + 2.0 ** -20            # [B, H]
    page = k.shape[1]
    S, one_term = torch.zeros_like(lse), torch.zeros_like(lse)
    for b in range(q.shape[0]):
        n = weights.shape[-1]
        ids, at = table[b].long()[torch.arange(n) // page], torch.arange(n) % page
        there = (ids >= 0) & (ids < k.shape[0])
        wide = torch.where(there[:, None], span(cache.vs, cache.vo)[ids.clamp(0, k.shape[0] - 1), at], 0.0)                         # [n, kv]
        S[b] = (weights[b] * wide.t().repeat_interleave(heads // kv, 0)).sum(-1)
        if dt == torch.bfloat16:
            scales = torch.where(there[:, None], cache.vs.double().abs().nan_to_num(0.0)[ids.clamp(0, k.shape[0] - 1), at], 0.0)
            one_term[b] = 2.0 ** -5 * (weights[b] * scales.t().repeat_interleave(heads // kv, 0)).sum(-1)
    bound = U[dt] * out.abs() + (((2 * err + 2.0 ** -16 + 2.0 ** -18) * S + one_term) * (1 + U[dt]))[..., None] + 2.0 ** -24
    diff = (got[0].cpu().double() - out).abs()
    assert got[0].dtype == dt and bool((diff <= bound).all()), f"output off by {(diff / bound).max():.3g} bounds"
    empty = lse == -math.inf
    have = got[1].cpu().double()
    assert torch.equal(have == -math.inf, empty)
    assert bool(((have - lse).abs()[~empty] <= (2 * err + 2.0 ** -22 * (1 + lse.abs()))[~empty]).all())
    if sums is not None:
        before, after = sums
        grown = weights.view(q.shape[0], kv, heads // kv, -1).sum(2)
        room = (weights * 2 * err[..., None]).view(q.shape[0], kv, heads // kv, -1).sum(2)
        want = before.double() + grown
        assert bool(((after.cpu().double() - want).abs() <= room + 2.0 ** -21 * grown + 2.0 ** -23 * want.abs()).all())


def attend(pa, cache, q, table, lens, **more):
    return pa.npu_paged_decode_attention(gpu(q), **cache.on_gpu(), block_table=table.cuda(), context_lens=lens.cuda(), softmax_lse=True, **more)


# ------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 128])
@pytest.mark.parametrize("params", ["head", "token"])
def test_attention_lengths_and_pages(pa, dt, page, params):
    g = torch.Generator().manual_seed(page)
    lens = torch.tensor([0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 300], dtype=torch.int32)
    B, width = len(lens), -(-300 // page)
    cache = Cache(g, B * width + 2, page, 2, 128, params=params)
    table = tables(g, B, width, B * width + 2, page)
    q = torch.randn(B, 8, 128, generator=g).to(dt)
    got = attend(pa, cache, q, table, lens)
    check_attention(got, cache, q, table, lens)
    assert bool((got[0][0] == 0).all()) and bool((got[1][0] == -math.inf).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 80, 96, 104, 112, 128, 136, 192, 248, 256])
@pytest.mark.parametrize("order", ["token", "head"])
def test_attention_head_widths(pa, dt, dim, order):
    g = torch.Generator().manual_seed(dim)
    lens = torch.tensor([70, 5, 200], dtype=torch.int32)
    cache = Cache(g, 45, 16, 2, dim, order=order)
    table = tables(g, 3, 13, 45, 16)
    q = torch.randn(3, 6, dim, generator=g).to(dt)
    check_attention(attend(pa, cache, q, table, lens), cache, q, table, lens)


@pytest.mark.parametrize("heads,kv", [(1, 1), (7, 7), (8, 1), (16, 1), (17, 1), (40, 2), (64, 2), (28, 4)])
def test_attention_groups(pa, heads, kv):
    g = torch.Generator().manual_seed(heads)
    lens = torch.tensor([90, 33], dtype=torch.int32)
    for dim in (64, 128):
        cache = Cache(g, 20, 16, kv, dim)
        table = tables(g, 2, 6, 20, 16)
        q = torch.randn(2, heads, dim, generator=g).to(torch.bfloat16)
        check_attention(attend(pa, cache, q, table, lens), cache, q, table, lens)


@pytest.mark.parametrize("page", [16, 12, 6])
def test_attention_masks_and_sums(pa, page):
    """Masks that hide everything, all but one position, every other one; the weights are added to the sums where they are seen."""
    g = torch.Generator().manual_seed(page)
    lens = torch.tensor([100, 77, 64, 3, 90], dtype=torch.int32)
    width = -(-100 // page)
    cache = Cache(g, 5 * width, page, 2, 128)
    table = tables(g, 5, width, 5 * width, page)
    mask = torch.rand(5, width * page, generator=g) < 0.3
    mask[0] = True
    mask[1] = torch.arange(width * page) != 40
    mask[2] = torch.arange(width * page) % 2 == 0
    q = torch.randn(5, 8, 128, generator=g).to(torch.bfloat16)
    for m in (mask, None):
        before = torch.rand(5, 2, width * page, generator=g)
        sums = before.cuda()
        got = attend(pa, cache, q, table, lens, atten_mask=None if m is None else m.cuda(), attn_sums=sums)
        check_attention(got, cache, q, table, lens, mask=m, sums=(before, sums))


@pytest.mark.parametrize("page,masked", [(16, False), (16, True), (5, False), (5, True)])
def test_what_is_not_seen_may_be_anything(pa, page, masked):
    """NaN scales and offsets behind the lengths, under the mask, and in blocks of nobody; entries of the table that name no block."""
    g = torch.Generator().manual_seed(2)
    width = -(-80 // page)
    lens = torch.tensor([50, 33, 80], dtype=torch.int32)
    cache = Cache(g, 3 * width + 3, page, 2, 64)
    table = tables(g, 3, width, 3 * width + 3, page)
    mask = torch.rand(3, width * page, generator=g) < 0.4 if masked else None
    table[0, 1], table[1, 0] = -1, 3 * width + 3
    nan = torch.ones(3 * width + 3, page, dtype=torch.bool)
    for b in range(3):
        for j in range(int(lens[b])):
            if 0 <= table[b, j // page] < len(nan) and not (masked and mask[b, j]):
                nan[table[b, j // page], j % page] = False
    for t in (cache.ks, cache.vs, cache.ko, cache.vo):
        t[nan] = float("nan")
    q = torch.randn(3, 8, 64, generator=g).to(torch.float16)
    k, v = cache.values()
    got = attend(pa, cache, q, table, lens, atten_mask=None if mask is None else mask.cuda())
    assert bool(got[0].isfinite().all())
    check_attention(got, cache, q, table, lens, mask=mask)


@pytest.mark.parametrize("order,pad,params", [("token", 0, "spread"), ("token", 1, "head"), ("token", 3, "token"), ("head", 0, "head"), ("head", 2, "head"), ("head", 5, "spread")])
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_attention_layouts(pa, order, pad, params, dim):
    g = torch.Generator().manual_seed(pad + dim)
    lens = torch.tensor([130, 65], dtype=torch.int32)
    cache = Cache(g, 24, 16, 3, dim, order=order, pad=pad, params=params)
    if params == "head" and pad:                           # keys and values, and scales and offsets, that do not lie alike
        cache.value = cache.value.contiguous()
        cache.vo = cache.vo.contiguous()
    table = tables(g, 2, 9, 24, 16)
    q = torch.randn(2, 12, dim, generator=g).to(torch.bfloat16)
    check_attention(attend(pa, cache, q, table, lens), cache, q, table, lens)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 64), (128, 3), (64, 7)])
def test_every_position_by_itself(pa, dim, page):
    """With one position seen the output is its value: every place of every word is where it belongs."""
    g = torch.Generator().manual_seed(dim)
    n = 70
    width = -(-n // page)
    cache = Cache(g, width + 1, page, 1, dim)
    table = tables(g, 1, width, width + 1, page).expand(n, -1)
    mask = torch.ones(n, width * page, dtype=torch.bool)
    mask[torch.arange(n), torch.arange(n)] = False
    q = torch.randn(n, 3, dim, generator=g).to(torch.float16)
    got = attend(pa, cache, q, table, torch.full((n,), n, dtype=torch.int32), atten_mask=mask.cuda())
    _, v = cache.values()
    want = v[table[0].long()[torch.arange(n) // page], torch.arange(n) % page]         # [n, 1, dim]
    # one probability of 1: two bf16 terms of the scale, 2^-16 of 31 times it, and the output's rounding
    assert bool(((got[0].cpu().double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -16 * 55 * cache.vs.abs().max()).all())
    check_attention(got, cache, q, table, torch.full((n,), n, dtype=torch.int32), mask=mask)


@pytest.mark.parametrize("case", [dict(B=1, n=9000, heads=8, kv=1, dim=128), dict(B=3, n=5000, heads=8, kv=2, dim=64), dict(B=2, n=4100, heads=4, kv=1, dim=256)])
def test_sequences_that_are_cut(pa, case):
    """Long sequences are cut into pieces whose sums are added; the result does not change from call to call."""
    g = torch.Generator().manual_seed(case["n"])
    page = 32
    width = -(-case["n"] // page)
    cache = Cache(g, case["B"] * width, page, case["kv"], case["dim"], order="head")
    table = tables(g, case["B"], width, case["B"] * width, page)
    lens = torch.tensor([case["n"] - 77 * b for b in range(case["B"])], dtype=torch.int32)
    q = torch.randn(case["B"], case["heads"], case["dim"], generator=g).to(torch.bfloat16)
    args = cache.on_gpu()
    first = pa.npu_paged_decode_attention(gpu(q), **args, block_table=table.cuda(), context_lens=lens.cuda(), softmax_lse=True)
    check_attention(first, cache, q, table, lens)
    for _ in range(3):
        again = pa.npu_paged_decode_attention(gpu(q), **args, block_table=table.cuda(), context_lens=lens.cuda(), softmax_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_beyond_32_bits(pa):
    """Blocks that start behind 2^32 bytes."""
    g = torch.Generator().manual_seed(4)
    page, heads, dim = 16, 2, 128
    cache = Cache(g, 40, page, heads, dim)
    block = 1 << 26                                        # words
    def far(t):
        big = torch.empty(40 * block, dtype=t.dtype, device="cuda")
        return torch.as_strided(big, t.shape, (block, *t.contiguous().stride()[1:])).copy_(t)
    args = {name: far(t) for name, t in (("key_cache", cache.key), ("value_cache", cache.value), ("key_scale", cache.ks), ("value_scale", cache.vs),
                                         ("key_offset", cache.ko), ("value_offset", cache.vo))}
    table = tables(g, 2, 12, 40, page)
    lens = torch.tensor([180, 100], dtype=torch.int32)
    q = torch.randn(2, 8, dim, generator=g).to(torch.bfloat16)
    got = pa.npu_paged_decode_attention(gpu(q), **args, block_table=table.cuda(), context_lens=lens.cuda(), softmax_lse=True)
    check_attention(got, cache, q, table, lens)
    slots = torch.tensor([39 * page + 3, 5])
    k, v = pa.npu_paged_cache_read(args["key_cache"], args["value_cache"], slots.cuda(), **{n: args[n] for n in args if not n.endswith("cache")})
    want_k, _ = read_ref(cache, slots, torch.bfloat16)
    assert torch.equal(k.cpu(), want_k)


# ------------------------------------------------------------------------------------------------ write, read, evict

def quantise(x):
    """The write's rule in float32: codes, scale, offset."""
    x = x.float()
    lo, hi = x.amin(-1), x.amax(-1)
    span = hi - lo
    flat = span <= 2.0 ** -120
    fifteen = torch.full_like(span, 15.0)
    scale = torch.where(flat, torch.ones_like(span), span / fifteen)
    offset = torch.where(flat, lo, lo / scale + 8.0)
    code = torch.round((x - lo[..., None]) * 15.0 / span[..., None]) - 8.0
    return torch.where(flat[..., None], 0.0, code).long(), scale, offset


def read_ref(cache, slots, dt):
    page = cache.key.shape[1]
    outs = []
    for w, s, o in ((cache.key, cache.ks, cache.ko), (cache.value, cache.vs, cache.vo)):
        at = (slots // page, slots % page)
        outs.append(((unpack(w[at]).float() + o[at][..., None]) * s[at][..., None]).to(dt))
    return outs


def empty(blocks, page, heads, dim, order="token", device="cuda"):
    shape = (blocks, page, heads) if order == "token" else (blocks, heads, page)
    turn = (lambda t: t) if order == "token" else (lambda t: t.transpose(1, 2))
    c = {name: turn(torch.full((*shape, dim // 8), 0x01234567, dtype=torch.int32, device=device)) for name in ("key_cache", "value_cache")}
    return c | {name: turn(torch.full(shape, 7.0, device=device)) for name in ("key_scale", "value_scale", "key_offset", "value_offset")}


def check_written(c, key, value, slots, blocks, page):
    """What lies in the cache after a write of CPU tensors into `empty`."""
    written = torch.zeros(blocks, page, dtype=torch.bool)
    for name, x in (("key", key), ("value", value)):
        codes, scale, offset = quantise(x)
        words, s, o = (c[f"{name}_{part}"].cpu() for part in ("cache", "scale", "offset"))
        for i, slot in enumerate(slots.tolist()):
            if not 0 <= slot < blocks * page:
                continue
            at = (slot // page, slot % page)
            written[at] = True
            assert torch.equal(unpack(words[at]), codes[i]), (name, i)
            assert torch.equal(s[at], scale[i]) and torch.equal(o[at], offset[i]), (name, i)
        assert bool((words[~written] == 0x01234567).all()) and bool((s[~written] == 7.0).all()) and bool((o[~written] == 7.0).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 128, 136, 256, 264, 1032])
@pytest.mark.parametrize("order", ["token", "head"])
def test_write_and_read(pa, dt, dim, order):
    g = torch.Generator().manual_seed(dim)
    blocks, page, heads, tokens = 6, 8, 3, 17
    slots = torch.randperm(blocks * page, generator=g)[:tokens]
    slots[3], slots[9] = -1, blocks * page                 # skipped
    key, value = (torch.randn(tokens, heads, dim, generator=g).to(dt) for _ in range(2))
    c = empty(blocks, page, heads, dim, order)
    pa.npu_paged_cache_write(key.cuda(), value.cuda(), slots=slots.cuda(), **c)
    check_written(c, key, value, slots, blocks, page)
    k, v = pa.npu_paged_cache_read(slots=slots.int().cuda(), dtype=dt, **c)
    for got, x in ((k, key), (v, value)):
        codes, scale, offset = quantise(x)
        want = ((codes.float() + offset[..., None]) * scale[..., None]).to(dt)
        want[3] = want[9] = 0
        assert torch.equal(got.cpu(), want)
        # half a step of the codes, the float32 roundings of offset and value, and the rounding to 16 bits: at most U of what is read, which
        # is at most |x| and that half step.  (U of |x| alone, however often, is too little where x is nearer to 0 than the step.)
        step = scale[..., None].double()
        room = step * (0.5 + 2.0 ** -18) + 2.0 ** -22 * x.double().abs().amax(-1, keepdim=True) + U[dt] * (x.double().abs() + step)
        far = (got.cpu().double() - x.double()).abs()
        far[3] = far[9] = 0
        assert bool((far <= room + 2.0 ** -20).all())


@pytest.mark.parametrize("view", ["odd start", "odd pitch", "projection", "columns"])
@pytest.mark.parametrize("dim", [64, 128])
def test_write_from_views(pa, view, dim):
    g = torch.Generator().manual_seed(3)
    blocks, page, heads, tokens = 5, 16, 4, 40
    slots = torch.randperm(blocks * page, generator=g)[:tokens]
    key, value = (torch.randn(tokens, heads, dim, generator=g).to(torch.bfloat16) for _ in range(2))
    k, v = key.cuda(), value.cuda()
    if view == "odd start":
        k = torch.cat((k, k[..., :8]), -1)[..., 1:dim + 1]
        key = torch.cat((key, key[..., :8]), -1)[..., 1:dim + 1]
    elif view == "odd pitch":
        v = torch.cat((v, v[..., :3]), -1)[..., :dim]
    elif view == "projection":
        both = torch.cat((k, v), 1)
        k, v = both[:, :heads], both[:, heads:]
    else:
        k = k.transpose(1, 2).contiguous().transpose(1, 2)
    c = empty(blocks, page, heads, dim)
    pa.npu_paged_cache_write(k, v, slots=slots.cuda(), **c)
    check_written(c, key, value, slots, blocks, page)


@pytest.mark.parametrize("tokens,heads", [(3000, 8), (1501, 7), (4096, 2)])
@pytest.mark.parametrize("order", ["token", "head"])
def test_write_of_many_tokens(pa, tokens, heads, order):
    """Enough rows for several heads a thread group."""
    g = torch.Generator().manual_seed(tokens)
    page, dim = 16, 128
    blocks = -(-tokens // page) + 1
    slots = torch.randperm(blocks * page, generator=g)[:tokens]
    key, value = (torch.randn(tokens, heads, dim, generator=g).to(torch.float16) for _ in range(2))
    c = empty(blocks, page, heads, dim, order)
    pa.npu_paged_cache_write(key.cuda(), value.cuda(), slots=slots.cuda(), **c)
    codes, scale, offset = quantise(key)
    at = (slots // page, slots % page)
    assert torch.equal(unpack(c["key_cache"].cpu()[at]), codes) and torch.equal(c["key_scale"].cpu()[at], scale)
    assert torch.equal(c["key_offset"].cpu()[at], offset)
    k, v = pa.npu_paged_cache_read(slots=slots.cuda(), dtype=torch.float16, **c)
    codes, scale, offset = quantise(value)
    assert torch.equal(v.cpu(), ((codes.float() + offset[..., None]) * scale[..., None]).half())


@pytest.mark.parametrize("magnitude", [1e-38, 2.0 ** -121, 2.0 ** -70, 1e-8, 1.0, 1e8, 2.0 ** 80, 1e36])
@pytest.mark.parametrize("shift", [0.0, 3.0, -100.0])
def test_magnitudes(pa, magnitude, shift):
    """Ranges inside and outside the one in which codes go by a reciprocal, about 0 and far from it."""
    g = torch.Generator().manual_seed(1)
    x = ((torch.randn(9, 2, 128, generator=g) + shift) * magnitude).to(torch.bfloat16)
    slots = torch.arange(9)
    c = empty(2, 8, 2, 128)
    pa.npu_paged_cache_write(x.cuda(), (-x).cuda(), slots=slots.cuda(), **c)
    check_written(c, x, -x, slots, 2, 8)


def test_ties(pa):
    """Values exactly between two codes take the even one (0, 2, 4 ... above the least)."""
    x = torch.arange(32.0).repeat(4)[None, None] / 2                       # 0 to 15.5: steps of 15.5 / 15
    x = torch.cat((x, (torch.arange(128.0) % 31)[None, None] / 2), 1)     # 0 to 15: every other value is a tie
    for dt in U:
        c = empty(1, 8, 2, 128)
        key = x.to(dt)
        pa.npu_paged_cache_write(key.cuda(), (-key).cuda(), slots=torch.tensor([5]).cuda(), **c)
        check_written(c, key, -key, torch.tensor([5]), 1, 8)
        got = unpack(c["key_cache"].cpu()[0, 5, 1]) + 8
        assert got[:31].tolist() == [0, 0, 1, 2, 2, 2, 3, 4, 4, 4, 5, 6, 6, 6, 7, 8, 8, 8, 9, 10, 10, 10, 11, 12, 12, 12, 13, 14, 14, 14, 15]


def test_rows_of_one_value_and_rows_that_are_not_finite(pa):
    x = torch.randn(8, 1, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    x[0], x[1], x[2] = 0.0, -3.25, 1e-30
    x[3, 0, :32], x[3, 0, 32:] = 0.0, -0.0
    x[4, 0, 5], x[5, 0, 6], x[6, 0, 7] = float("nan"), float("inf"), float("-inf")
    x[7, 0, 0], x[7, 0, 1] = 3e38, -3e38
    for key in (x, torch.cat((x, x[..., :8]), -1)[..., :64]):              # wide loads, and any
        c = empty(1, 8, 1, 64)
        pa.npu_paged_cache_write(key.cuda(), key.cuda(), slots=torch.arange(8).cuda(), **c)
        k, v = pa.npu_paged_cache_read(slots=torch.arange(8).cuda(), **c)
        assert torch.equal(k[:4].cpu(), x[:4]) and torch.equal(v[:4].cpu(), x[:4])
        assert bool(k[4:].isnan().all()) and bool(v[4:].isnan().all())


@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("order,keep", [("token", 40), ("head", 40), ("head", 190)])
def test_evict_moves_codes_scales_and_offsets(pa, dim, order, keep):
    """The rows that stay are those of the 16-bit rule; each arrives whole."""
    g = torch.Generator().manual_seed(dim)
    batch, heads, page, n = 3, 2, 16, 200
    width = -(-n // page)
    cache = Cache(g, batch * width, page, heads, dim, order=order)
    table = tables(g, batch, width, batch * width, page)
    lens = torch.tensor([200, 30, 151], dtype=torch.int32)
    sums = torch.rand(batch, heads, width * page, generator=g)
    positions = torch.arange(width * page, dtype=torch.int32).expand(batch, heads, -1).contiguous()
    args = cache.on_gpu()
    new_lens, new_sums, new_pos = pa.npu_paged_cache_evict(**args, block_table=table.cuda(), context_lens=lens.cuda(), attn_sums=sums.cuda(),
                                                           positions=positions.cuda(), keep=keep, recent=8)
    assert new_lens.tolist() == [min(int(x), keep) for x in lens]
    for b in range(batch):
        ids = table[b].long()[torch.arange(width * page) // page]
        at = torch.arange(width * page) % page
        m = int(new_lens[b])
        for h in range(heads):
            came = new_pos[b, h, :m].cpu().long()          # positions were the places
            worth = sums[b, h, : int(lens[b])].clone()
            worth[int(lens[b]) - 8:] = math.inf
            assert sorted(came.tolist()) == sorted(worth.argsort(descending=True, stable=True)[:m].tolist())
            assert torch.equal(new_sums[b, h, :m].cpu(), sums[b, h, came])
            for name, old in (("key_cache", cache.key), ("value_cache", cache.value), ("key_scale", cache.ks), ("value_scale", cache.vs),
                              ("key_offset", cache.ko), ("value_offset", cache.vo)):
                assert torch.equal(args[name].cpu()[ids[:m], at[:m], h], old[ids[came], at[came], h]), name


# ------------------------------------------------------------------------------------------------ together

@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("budget", [None, 40])
def test_module(pa, dt, budget):
    """PagedKVCache with 4 bits: prompts, steps turned to their positions, eviction; against 64-bit attention over what it reads back."""
    from pytorch_amd.contrib.module import PagedKVCache
    g = torch.Generator().manual_seed(6)
    batch, heads, kv, dim = 3, 8, 2, 64
    cache = PagedKVCache(batch, 80, kv, dim, block_size=16, quantized=True, bits=4, budget=budget, recent=None if budget is None else 8, device="cuda", dtype=dt)
    angle = torch.arange(200.0)[:, None] * 10000.0 ** (-torch.arange(dim // 2) * 2 / dim)
    table = torch.cat((angle.cos(), angle.sin()), 1).cuda()
    new = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()  # noqa: E731
    for b, n in enumerate((50, 20, 33)):
        cache.prefill(b, new(n, kv, dim), new(n, kv, dim))
    delta = torch.tensor([0, -5, 3], device="cuda")
    for step in range(6):
        q, k, v = new(batch, heads, dim), new(batch, kv, dim), new(batch, kv, dim)
        at = torch.tensor([50, 20, 33], device="cuda") + step
        turned = cache.rotate(q, k, table, mrope_section=[8, 12, 12], offset=delta)
        want = pa.npu_mrope((at + delta).expand(3, -1), q, k, table, dim, mrope_section=[8, 12, 12])
        assert all(torch.equal(x, y) for x, y in zip(turned, want))
        assert torch.equal(cache.rotate(q, k, table)[0], pa.npu_mrope(at, q, k, table, dim)[0])
        cache.append(turned[1], v)
        out = cache.attend(turned[0]).cpu().double()
        for b, n in enumerate(cache.context_lens.tolist()):
            kk, vv = (x.cpu().double() for x in cache.read(b, 0, n))
            kk, vv = kk.repeat_interleave(heads // kv, 1), vv.repeat_interleave(heads // kv, 1)
            p = torch.softmax(torch.einsum("hd,thd->ht", turned[0][b].cpu().double(), kk) / math.sqrt(dim), 1)
            ref, size = torch.einsum("ht,thd->hd", p, vv), torch.einsum("ht,thd->hd", p, vv.abs())
            # what is read back is rounded to 16 bits: u of each value, and of each key, whose scores are off by u sum |q||k| / sqrt(D)
            shift = U[dt] * (torch.einsum("hd,thd->ht", turned[0][b].cpu().double().abs(), kk.abs()) / math.sqrt(dim)).amax(1, keepdim=True)
            assert bool(((out[b] - ref).abs() <= (2 * U[dt] + 2 * shift + 2.0 ** -10) * size + 2.0 ** -12).all())
        if budget is not None:
            cache.evict()
    assert cache.context_lens.tolist() == ([56, 26, 39] if budget is None else [40, 26, 39])


def test_a_step_as_a_graph(pa):
    """norm, projection, rotary positions, write, attention and eviction captured; every replay as the eager step."""
    from pytorch_amd.contrib.module import PagedKVCache
    g = torch.Generator().manual_seed(8)
    batch, heads, kv, dim, hidden = 4, 8, 2, 64, 512
    weight = torch.randint(-127, 128, ((heads + 2 * kv) * dim, hidden), generator=g, dtype=torch.int8).cuda()
    scale = torch.full((weight.shape[0],), 1.0 / (74 * hidden ** 0.5), device="cuda")
    gamma = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    angle = torch.arange(300.0)[:, None] * 10000.0 ** (-torch.arange(dim // 2) * 2 / dim)
    table = torch.cat((angle.cos(), angle.sin()), 1).cuda()
    caches = [PagedKVCache(batch, 80, kv, dim, block_size=16, quantized=True, bits=4, budget=48, recent=8, device="cuda") for _ in range(2)]
    for b in range(batch):
        k, v = (torch.randn(40 + b, kv, dim, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        for c in caches:
            c.prefill(b, k, v)

    def step(c):
        codes, row, x = pa.npu_add_rms_norm_dynamic_quant(branch, residual, gamma)
        qkv = pa.npu_quant_matmul(codes, weight.t(), scale, pertoken_scale=row, output_dtype=torch.bfloat16).view(batch, heads + 2 * kv, dim)
        q, k, v = qkv.split((heads, kv, kv), 1)
        q, k = c.rotate(q, k, table, mrope_section=[8, 12, 12])
        c.append(k, v)
        out = c.attend(q)
        c.evict()
        return out, x

    branch, residual = (torch.randn(batch, hidden, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    first = [step(c) for c in caches]
    assert torch.equal(first[0][0], first[1][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, x = step(caches[0])
    for _ in range(10):
        branch.copy_(torch.randn(batch, hidden, generator=g).to(torch.bfloat16))
        residual.copy_(torch.randn(batch, hidden, generator=g).to(torch.bfloat16))
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(x, want[1])
        for name in ("context_lens", "positions", "attn_sums", "next_position", "key_cache", "value_cache", "key_scale", "value_scale", "key_offset", "value_offset"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
