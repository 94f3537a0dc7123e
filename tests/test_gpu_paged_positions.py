"""Decode attention position by position: every cached position counts once, and its value goes with its key, in sequences that
are cut into many pieces and at every edge of a block, a tile, a unit and a piece.

Two probes, both with answers that are exact in 16 bits:
  counts   queries of zeros weigh every position 1/n.  Values are zero but for a window of head_dim positions, where position
           i of the window has a one in element i: out must be 1/n there, 0 for a position that was lost and 2/n for one that was
           taken twice.  The window goes over all positions.  lse must be log n, to a quarter of what one position makes.
  pairs    keys are zero but for such a window; a query along element i attends to one position alone, whose value is the position's
           number in ones and minus ones.
"""
import math

import pytest
import torch

from test_gpu_paged import U, attend_ref, check_attention, gpu, make_cache, run_attention, tables


def check_counts(out, lse, lens, hidden=None):
    """out [windows, B, H, D], lse [windows, B, H]: a window's positions are its elements.  hidden: bool [B, positions]."""
    windows, batch, heads, d = out.shape
    place = torch.arange(windows * d, device=out.device)
    seen = place < torch.tensor(lens, device=out.device)[:, None]
    if hidden is not None:
        seen[:, : hidden.shape[1]] &= ~hidden[:, : windows * d]
    n = seen.sum(1).reshape(1, batch, 1, 1)
    want = torch.where(seen.reshape(batch, windows, 1, d).transpose(0, 1), 1.0 / n.clamp(min=1), 0.0)
    assert bool(((out - want).abs() <= 2 * U[out.dtype] * want).all())       # the division's and the output's rounding
    n = n[..., 0].double()
    assert bool(((lse.double() - n.log()).abs()[(n > 0).expand_as(lse)] < (0.25 / n).expand_as(lse)[(n > 0).expand_as(lse)]).all())
    assert bool((lse[(n == 0).expand_as(lse)] == -math.inf).all())


def check_pairs(out, place, lens, codes):
    """out [probes, B, H, D] of heads that look for position place [probes, H]; codes [positions, H, D]."""
    heads = torch.arange(out.shape[2], device=out.device)
    want = codes[place, heads][:, None]
    seen = place[:, None] < torch.tensor(lens, device=out.device)[:, None]                     # [probes, B, H]
    assert bool((out == want).all(-1)[seen].all())


def number(positions, hkv, d):
    """[positions, hkv, d]: the bits of position and head as ones and minus ones."""
    word = torch.arange(positions)[:, None] * hkv + torch.arange(hkv)
    return ((word[..., None] >> torch.arange(d).clamp(max=24)) & 1).float() * 2 - 1


class Probed:
    def __init__(self, kind, hkv, group, d, page, order, lens, out_type, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.heads, self.d, self.n = lens, hkv, hkv * group, d, max(lens)
        width = -(-self.n // page)
        dtype = torch.int8 if kind == "int8" else kind
        shape = (width + 1, page, hkv, d) if order == "token" else (width + 1, hkv, page, d)
        self.key, self.value = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2))
        if order == "head":
            self.key, self.value = self.key.transpose(1, 2), self.value.transpose(1, 2)
        self.scale = torch.ones(width + 1, hkv, page, device="cuda").transpose(1, 2) if kind == "int8" else None
        table = torch.randperm(width + 1, generator=g)[:width]
        place = torch.arange(self.n)
        self.block, self.spot = table[place // page].cuda(), (place % page).cuda()
        self.table = table.to(torch.int32).expand(len(lens), width).contiguous().cuda()        # all attend to the same blocks
        self.lens_gpu = torch.tensor(lens, dtype=torch.int32).cuda()
        self.out_type = out_type
        self.windows = -(-self.n // d)

    def window(self, cache, k, x):
        places = torch.arange(k * self.d, min((k + 1) * self.d, self.n), device="cuda")
        cache[self.block[places], self.spot[places], :, places - k * self.d] = x

    def attend(self, pa, query, mask=None):
        return pa.npu_paged_decode_attention(query, self.key, self.value, self.table, self.lens_gpu, key_scale=self.scale, value_scale=self.scale,
                                             scale_value=1.0, atten_mask=mask, softmax_lse=True)


SHAPES = [(torch.float16, 1, 16, 128, 64, "token"), (torch.bfloat16, 1, 3, 256, 64, "token"), ("int8", 1, 16, 128, 64, "head"), ("int8", 1, 3, 256, 16, "token"),
          (torch.bfloat16, 2, 20, 64, 24, "head"), (torch.float16, 3, 2, 80, 16, "token"), (torch.bfloat16, 2, 4, 128, 5, "token"), ("int8", 2, 5, 64, 9, "token")]
LENGTHS = [(23001, 40, 0, 9000), (1025, 1024, 129, 17, 16, 1)]


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("kind,hkv,group,d,page,order", SHAPES)
def test_every_position_counts_once(pa, kind, hkv, group, d, page, order, lens, masked):
    """Every one that is seen: with a mask about 0.7 of them."""
    p = Probed(kind, hkv, group, d, page, order, lens, torch.float16 if kind == "int8" else kind)
    query = torch.zeros(len(lens), p.heads, d, dtype=p.out_type, device="cuda")
    mask = torch.rand(len(lens), p.table.shape[1] * page, generator=torch.Generator().manual_seed(2)).cuda() < 0.3 if masked else None
    outs, lses = [], []
    for k in range(p.windows):
        p.window(p.value, k, 1)
        out, lse = p.attend(pa, query, mask)
        p.window(p.value, k, 0)
        outs.append(out), lses.append(lse)
    check_counts(torch.stack(outs), torch.stack(lses), lens, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("kind,hkv,group,d,page,order", SHAPES)
def test_every_value_goes_with_its_key(pa, kind, hkv, group, d, page, order, lens):
    p = Probed(kind, hkv, group, d, page, order, lens, torch.float16 if kind == "int8" else kind)
    codes = number(p.windows * d, hkv, d).cuda()
    p.value[p.block, p.spot] = codes[:p.n].to(p.value.dtype)
    heads = torch.arange(p.heads, device="cuda")
    outs, places = [], []
    for k in range(p.windows):
        p.window(p.key, k, 8)
        for first in range(0, d, p.heads):
            element = (first + heads) % d
            query = torch.zeros(len(lens), p.heads, d, dtype=p.out_type, device="cuda")
            query[:, heads, element] = 8
            outs.append(p.attend(pa, query)[0])
            places.append(k * d + element)
        p.window(p.key, k, 0)
    check_pairs(torch.stack(outs), torch.stack(places), lens, codes.repeat_interleave(group, 1))


def test_the_probes_see_one_position():
    """Planted in answers as they should be: a position that is lost, taken twice, or whose value is another's."""
    n, d, lens = 23001, 128, (23001, 40)
    windows = -(-n // d)
    place = torch.arange(windows * d).reshape(windows, 1, 1, d)
    out = torch.where(place < torch.tensor(lens).reshape(1, 2, 1, 1), 1 / torch.tensor(lens).reshape(1, 2, 1, 1), 0.0).half()
    lse = torch.tensor(lens).float().log().expand(windows, 2)[..., None].contiguous()
    check_counts(out, lse, lens)
    for change in (0.0, 2.0):
        wrong = out.clone()
        wrong[100, 0, 0, 77] *= change
        with pytest.raises(AssertionError):
            check_counts(wrong, lse, lens)
    for by in (-1, 1):
        wrong = lse.clone()
        wrong[100, 0, 0] = math.log(n + by)
        with pytest.raises(AssertionError):
            check_counts(out, wrong, lens)
    codes = number(windows * d, 1, d)
    places = torch.arange(windows * d)[:, None]
    out = codes[:, None].expand(-1, 2, -1, -1).half().contiguous()
    check_pairs(out, places, lens, codes)
    out[12345, 0, 0] = codes[12346, 0].half()
    with pytest.raises(AssertionError):
        check_pairs(out, places, lens, codes)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, "int8"])
@pytest.mark.parametrize("page", [8, 9, 10, 12, 13, 15, 18])
def test_summed_weights_in_blocks_of_any_size(pa, kind, page):
    """Blocks of 8 to 15 tokens, and ones that are no multiple of 4, whose scores are stored one by one."""
    g = torch.Generator().manual_seed(page)
    batch, hkv, group, width = 4, 2, 3, 13
    cap = width * page
    lens = torch.tensor([cap, 0, 37, cap - 1], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, batch * width, page, hkv, 64, kind)
    table = tables(g, batch, width, batch * width, page)
    table[3, 2] = -1
    dt = torch.float16 if kind == "int8" else kind
    q = torch.randn(batch, hkv * group, 64, generator=g).to(dt)
    before = torch.rand(batch, hkv, cap, generator=g)
    sums = gpu(before)
    got = run_attention(pa, q, kc, vc, table, lens, ks, vs, attn_sums=sums)
    want = attend_ref(q, kc, vc, table, lens, ks, vs)
    check_attention(got, want, dt, kind == "int8")
    added = want[2].reshape(batch, hkv, group, cap).sum(2)
    rel = 4 * want[3].reshape(batch, hkv, group).amax(-1)[..., None] + (group + 4) * 2.0 ** -24
    bound = rel * added + 2.0 ** -23 * (before.double() + added)
    assert bool(((sums.cpu().double() - before.double() - added).abs() <= bound).all())
