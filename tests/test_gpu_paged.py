"""The paged key-value cache's operators on the GPU against plain 64-bit implementations on the CPU.

Tolerances.  With u the unit roundoff of a 16-bit type (2^-8 bfloat16, 2^-11 float16):
  output     u |o| for its one rounding, u' sum p|v| for rounding the probabilities (u' = u; 2^-16 on int8 caches, which keep
             two terms), and the relative error of a probability, which is the absolute error of its exponent: float32 sums
             over head_dim terms of size |q||k| give at most (head_dim + 8) 2^-24 times scale * sum |q||k|, another 2^-20 covers
             the exponential and the sums of probabilities
  lse        the exponent's error alone
  attn_sums  the relative error of a probability, and one float32 addition
Codes, scales, copies, chosen tokens and lengths are exact.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


def make_cache(g, blocks, page, hkv, d, kind, order="token", pad=0, scale_order="head"):
    """CPU tensors [blocks, page, hkv, d] (key, value) and their scales or None; `pad`: elements between rows."""
    def one():
        shape = (blocks, page, hkv, d) if order == "token" else (blocks, hkv, page, d)
        x = torch.randn(*shape[:-1], d + pad, generator=g)
        x = (x * 32).round().clamp(-127, 127).to(torch.int8) if kind == "int8" else x.to(kind)
        x = x[..., :d]
        return x if order == "token" else x.transpose(1, 2)

    def scales():
        if kind != "int8":
            return None
        s = torch.rand(blocks, hkv, page, generator=g) * 0.03 + 0.005
        return s.transpose(1, 2) if scale_order == "head" else s.transpose(1, 2).contiguous()

    return one(), one(), scales(), scales()


def gpu(t):
    """The tensor on the GPU with its strides."""
    if t is None:
        return None
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
    out.copy_(t)
    return out


def values(cache, scale):
    return cache.double() if scale is None else cache.double() * scale.double()[..., None]


def attend_ref(q, kc, vc, table, lens, ks=None, vs=None, scale=None, mask=None):
    """64-bit (out, lse, weights [B, H, capacity], bound of the exponent's error [B, H], sum p|v| [B, H, D])."""
    B, H, D = q.shape
    nb, page, hkv, _ = kc.shape
    cap = table.shape[1] * page
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    k, v = values(kc, ks), values(vc, vs)
    out, spread = torch.zeros(B, H, D, dtype=torch.double), torch.zeros(B, H, D, dtype=torch.double)
    lse, err = torch.full((B, H), -math.inf, dtype=torch.double), torch.zeros(B, H, dtype=torch.double)
    weights = torch.zeros(B, H, cap, dtype=torch.double)
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        at = torch.arange(n)
        ids = table[b].long()[at // page]
        seen = (ids >= 0) & (ids < nb)
        if mask is not None:
            seen &= ~mask[b, :n]
        at, ids = at[seen], ids[seen]
        if len(at) == 0:
            continue
        for h in range(H):
            kk, vv = k[ids, at % page, h // (H // hkv)], v[ids, at % page, h // (H // hkv)]
            qq = q[b, h].double()
            s = scale * (kk @ qq)
            lse[b, h] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[b, h])
            out[b, h] = p @ vv
            spread[b, h] = p @ vv.abs()
            weights[b, h, at] = p
            err[b, h] = (D + 8) * 2.0 ** -24 * abs(scale) * (kk.abs() @ qq.abs()).max() + 2.0 ** -20
    return out, lse, weights, err, spread


def check_attention(got, want, dtype, quant):
    out, lse = got
    ref, ref_lse, _, err, spread = want
    u = U[dtype]
    up = 2.0 ** -16 if quant else u
    bound = u * ref.abs() + (up + 2 * err[..., None]) * spread * (1 + u) + 2.0 ** -24
    diff = (out.cpu().double() - ref).abs()
    assert bool((diff <= bound).all()), f"output off by {(diff / bound).max():.3g} bounds"
    lse = lse.cpu().double()
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    rounding = 2.0 ** -22 * (1 + ref_lse[~empty].abs())
    assert bool(((lse - ref_lse).abs()[~empty] <= 2 * err[~empty] + rounding).all())


def tables(g, B, width, blocks, page):
    assert B * width <= blocks
    return torch.randperm(blocks, generator=g)[: B * width].reshape(B, width).to(torch.int32)


def run_attention(pa, q, kc, vc, table, lens, ks=None, vs=None, **more):
    return pa.npu_paged_decode_attention(gpu(q), gpu(kc), gpu(vc), table.cuda(), lens.cuda(), key_scale=gpu(ks), value_scale=gpu(vs),
                                         softmax_lse=True, **more)


# ------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, "int8"])
@pytest.mark.parametrize("page", [1, 3, 16, 24, 128])
def test_attention_lengths_and_pages(pa, kind, page):
    g = torch.Generator().manual_seed(page)
    lens = torch.tensor([0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 300], dtype=torch.int32)
    B, width = len(lens), -(-300 // page)
    kc, vc, ks, vs = make_cache(g, B * width + 2, page, 2, 128, kind)
    table = tables(g, B, width, B * width + 2, page)
    for dt in ([kind] if kind != "int8" else [torch.bfloat16, torch.float16]):
        q = (torch.randn(B, 8, 128, generator=g) * 2).to(dt)
        got = run_attention(pa, q, kc, vc, table, lens, ks, vs)
        check_attention(got, attend_ref(q, kc, vc, table, lens, ks, vs), dt, kind == "int8")
        assert bool((got[0][0] == 0).all()) and bool((got[1][0] == -math.inf).all())


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, "int8"])
@pytest.mark.parametrize("d", [1, 8, 40, 64, 80, 96, 100, 112, 128, 129, 192, 256])
def test_attention_head_widths(pa, kind, d):
    g = torch.Generator().manual_seed(d)
    lens = torch.tensor([70, 5, 200], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 45, 16, 2, d, kind)
    table = tables(g, 3, 13, 45, 16)
    dt = torch.float16 if kind == "int8" else kind
    q = torch.randn(3, 6, d, generator=g).to(dt)
    check_attention(run_attention(pa, q, kc, vc, table, lens, ks, vs), attend_ref(q, kc, vc, table, lens, ks, vs), dt, kind == "int8")


@pytest.mark.parametrize("kind", [torch.bfloat16, "int8"])
@pytest.mark.parametrize("hkv,group", [(1, 1), (1, 15), (1, 16), (2, 17), (1, 40), (3, 5), (8, 4), (32, 1)])
def test_attention_head_layouts(pa, kind, hkv, group):
    g = torch.Generator().manual_seed(hkv * 100 + group)
    lens = torch.tensor([130, 1, 257], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 30, 32, hkv, 64, kind, order="head", scale_order="token")
    table = tables(g, 3, 9, 30, 32)
    q = torch.randn(3, hkv * group, 64, generator=g).to(torch.bfloat16)
    check_attention(run_attention(pa, q, kc, vc, table, lens, ks, vs), attend_ref(q, kc, vc, table, lens, ks, vs), torch.bfloat16, kind == "int8")


@pytest.mark.parametrize("kind", [torch.float16, "int8"])
@pytest.mark.parametrize("order,pad", [("token", 8), ("head", 16), ("token", 3), ("head", 1)])
def test_attention_strides_and_alignment(pa, kind, order, pad):
    g = torch.Generator().manual_seed(pad)
    lens = torch.tensor([50, 99], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 16, 16, 3, 64, kind, order, pad)
    table = torch.stack([tables(g, 2, 7, 16, 16), torch.zeros(2, 7, dtype=torch.int32)], -1)[..., 0]       # inner stride 2
    qkv = torch.randn(2, 6 + 3, 64 + pad, generator=g).to(torch.float16)
    q = qkv[:, :6, pad:]                                                                                    # starts anywhere
    out = pa.npu_paged_decode_attention(gpu(qkv)[:, :6, pad:], gpu(kc), gpu(vc), table.cuda().long(), lens.cuda().long(), key_scale=gpu(ks),
                                        value_scale=gpu(vs), scale_value=0.3, softmax_lse=True)
    check_attention(out, attend_ref(q, kc, vc, table, lens, ks, vs, scale=0.3), torch.float16, kind == "int8")


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, "int8"])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_unseen_places_have_no_influence(pa, kind, page):
    """NaN and infinities behind the length, under the mask and in unnamed blocks; rows whose mask leaves nothing."""
    g = torch.Generator().manual_seed(7)
    B, width = 5, 10
    cap = width * page
    lens = torch.tensor([cap + 100, 77, 40, 1, -3], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, B * width, page, 2, 128, kind)
    table = tables(g, B, width, B * width, page)
    mask = torch.rand(B, cap, generator=g) < 0.3
    mask[2] = True
    mask[0, 64:96] = True                                       # a whole tile
    table[0, 3], table[1, 0] = -1, B * width                    # blocks that do not exist
    dt = torch.bfloat16 if kind == "int8" else kind
    q = torch.randn(B, 8, 128, generator=g).to(dt)
    want = attend_ref(q, kc, vc, table, lens, ks, vs, mask=mask)
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        for j in range(cap):
            blk = int(table[b, j // page])
            if (j >= n or mask[b, j]) and 0 <= blk < B * width:
                bad = [math.nan, math.inf, -math.inf][j % 3]
                if kind == "int8":
                    ks[blk, j % page], vs[blk, j % page] = bad, bad
                else:
                    kc[blk, j % page], vc[blk, j % page] = bad, bad
    got = run_attention(pa, q, kc, vc, table, lens, ks, vs, atten_mask=mask.cuda())
    check_attention(got, want, dt, kind == "int8")
    assert bool((got[0][2] == 0).all()) and bool((got[0][4] == 0).all())
    wide = torch.zeros(B, cap + 9, dtype=torch.bool)
    wide[:, 5:5 + cap] = mask                                   # rows apart, starting anywhere
    again = run_attention(pa, q, kc, vc, table, lens, ks, vs, atten_mask=wide.cuda()[:, 5:5 + cap])
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


def test_attention_nan_that_is_seen_comes_out(pa):
    g = torch.Generator().manual_seed(8)
    kc, vc, _, _ = make_cache(g, 8, 16, 1, 64, torch.bfloat16)
    table, lens = torch.arange(8, dtype=torch.int32).reshape(2, 4), torch.tensor([40, 40], dtype=torch.int32)
    q = torch.randn(2, 2, 64, generator=g).to(torch.bfloat16)
    kc[4:, :] = math.nan                                        # every key of the second sequence
    got = run_attention(pa, q, kc, vc, table, lens)
    assert bool(got[0][1].isnan().all()) and bool(got[1][1].isnan().all()) and not bool(got[0][0].isnan().any())


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_attention_extreme_scores(pa, kind):
    """One key far above the others, all keys alike, and scores of some hundred: the running maximum carries them."""
    g = torch.Generator().manual_seed(9)
    kc, vc, _, _ = make_cache(g, 40, 16, 1, 64, kind)
    table, lens = tables(g, 3, 13, 40, 16), torch.tensor([200, 200, 200], dtype=torch.int32)
    kc[table[1].long()] = 1.0
    kc[table[0, 7].long(), 5] *= 30
    q = (torch.randn(3, 4, 64, generator=g) * 20).to(kind)
    q[1] = 3.0
    want = attend_ref(q, kc, vc, table, lens)
    check_attention(run_attention(pa, q, kc, vc, table, lens), want, kind, False)


@pytest.mark.parametrize("batch", [1, 3, 300, 1030])
def test_attention_work_is_dealt_out_whatever_the_batch(pa, batch):
    """Long and empty sequences side by side: stretches cut between workgroups, workgroups with several sequences."""
    g = torch.Generator().manual_seed(batch)
    hkv, d, page, blocks = 2, 64, 16, 4000
    longest = {1: 30001, 3: 9000}.get(batch, 1500)
    width = -(-longest // page)
    kc, vc, _, _ = make_cache(g, blocks, page, hkv, d, torch.float16)
    table = torch.randint(0, blocks, (batch, width), generator=g, dtype=torch.int32)      # sequences may share blocks
    lens = torch.randint(0, 40, (batch,), generator=g, dtype=torch.int32)
    lens[torch.randperm(batch, generator=g)[: max(1, batch // 50)]] = longest
    lens[-1] = max(int(lens[-1]), 1)
    q = torch.randn(batch, 4, d, generator=g).to(torch.float16)
    got = run_attention(pa, q, kc, vc, table, lens)
    check_attention(got, attend_ref(q, kc, vc, table, lens), torch.float16, False)
    again = run_attention(pa, q, kc, vc, table, lens)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])                 # no order of arrival in the sums


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, "int8"])
@pytest.mark.parametrize("page,group", [(16, 4), (24, 1), (5, 19)])
def test_attention_sums(pa, kind, page, group):
    g = torch.Generator().manual_seed(11)
    B, hkv, width = 4, 2, 20
    cap = width * page
    lens = torch.tensor([cap, 0, 37, cap - 1], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, B * width, page, hkv, 64, kind)
    table = tables(g, B, width, B * width, page)
    mask = torch.rand(B, cap, generator=g) < 0.2
    mask[2] = True
    dt = torch.float16 if kind == "int8" else kind
    q = torch.randn(B, hkv * group, 64, generator=g).to(dt)
    wide = torch.rand(B, hkv + 1, cap + 3, generator=g)
    sums = gpu(wide)[:, :hkv, 1:1 + cap]
    before = wide[:, :hkv, 1:1 + cap].double()
    got = run_attention(pa, q, kc, vc, table, lens, ks, vs, atten_mask=mask.cuda(), attn_sums=sums)
    want = attend_ref(q, kc, vc, table, lens, ks, vs, mask=mask)
    check_attention(got, want, dt, kind == "int8")
    added = want[2].reshape(B, hkv, group, cap).sum(2)
    rel = 4 * want[3].reshape(B, hkv, group).amax(-1)[..., None] + (group + 4) * 2.0 ** -24
    bound = rel * added + 2.0 ** -23 * (before + added)
    assert bool(((sums.cpu().double() - before - added).abs() <= bound).all())
    plain = run_attention(pa, q, kc, vc, table, lens, ks, vs, atten_mask=mask.cuda())
    assert torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[1])


def test_attention_offsets_beyond_32_bits(pa):
    """A cache of over 4 GiB whose last blocks are in use."""
    d, page, hkv = 128, 64, 8
    blocks = 2 ** 32 // (page * hkv * d * 2) + 40
    kc = torch.zeros(blocks, page, hkv, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    g = torch.Generator().manual_seed(12)
    small_k, small_v, _, _ = make_cache(g, 6, page, hkv, d, torch.bfloat16)
    kc[-6:], vc[-6:] = small_k.cuda(), small_v.cuda()
    lens = torch.tensor([190, 129], dtype=torch.int32)
    local = tables(g, 2, 3, 6, page)
    q = torch.randn(2, 32, d, generator=g).to(torch.bfloat16)
    got = pa.npu_paged_decode_attention(q.cuda(), kc, vc, (local + blocks - 6).cuda(), lens.cuda(), softmax_lse=True)
    check_attention(got, attend_ref(q, small_k, small_v, local, lens), torch.bfloat16, False)
    slots = torch.arange(5, dtype=torch.int64) + (blocks - 6) * page
    k, v = pa.npu_paged_cache_read(kc, vc, slots.cuda())
    assert torch.equal(k.cpu(), small_k[0, :5]) and torch.equal(v.cpu(), small_v[0, :5])
    pa.npu_paged_cache_write(k, v, kc, vc, (slots + 7).cuda())
    assert torch.equal(kc[blocks - 6, 7:12].cpu(), small_k[0, :5]) and torch.equal(vc[blocks - 6, 7:12].cpu(), small_v[0, :5])


def test_attention_on_another_stream_and_in_a_graph(pa):
    g = torch.Generator().manual_seed(13)
    kc, vc, _, _ = make_cache(g, 64, 16, 2, 128, torch.bfloat16)
    table, lens = tables(g, 4, 16, 64, 16), torch.tensor([256, 100, 0, 31], dtype=torch.int32)
    q = torch.randn(4, 8, 128, generator=g).to(torch.bfloat16)
    args = [gpu(q), gpu(kc), gpu(vc), table.cuda(), lens.cuda()]
    sums = torch.zeros(4, 2, 256, device="cuda")
    want = pa.npu_paged_decode_attention(*args, softmax_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pa.npu_paged_decode_attention(*args, softmax_lse=True)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = pa.npu_paged_decode_attention(*args, softmax_lse=True, attn_sums=sums)
    one = None
    for i in range(4):
        args[0].copy_(gpu(q) * (i + 1))
        before = sums.clone()
        graph.replay()
        torch.cuda.synchronize()
        eager_sums = before.clone()
        eager = pa.npu_paged_decode_attention(*args, softmax_lse=True, attn_sums=eager_sums)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1]) and torch.equal(sums, eager_sums)
        one = out.clone() if one is None else one
    assert not torch.equal(one, out)


@pytest.mark.parametrize("offset,pitch", [(0, 0), (1, 3), (2, 8), (4, 2)])
def test_attention_mask_that_is_a_view(pa, offset, pitch):
    """Rows of the mask at any address and distance."""
    g = torch.Generator().manual_seed(offset + pitch)
    B, H, hkv, d, page = 4, 4, 2, 64, 16
    kc, vc, _, _ = make_cache(g, 24, page, hkv, d, torch.bfloat16)
    table, lens = tables(g, B, 6, 24, page), torch.tensor([96, 5, 50, 81], dtype=torch.int32)
    whole = torch.rand(B, offset + 96 + pitch, generator=g) < 0.4
    mask = whole[:, offset:offset + 96]
    q = torch.randn(B, H, d, generator=g).to(torch.bfloat16)
    got = run_attention(pa, q, kc, vc, table, lens, atten_mask=whole.cuda()[:, offset:offset + 96])
    check_attention(got, attend_ref(q, kc, vc, table, lens, mask=mask), torch.bfloat16, False)


def test_attention_and_eviction_take_64_bit_tables_and_lengths(pa):
    """What does not fit into 32 bits names no block, and is longer or shorter than anything."""
    g = torch.Generator().manual_seed(8)
    B, H, hkv, d, page = 4, 4, 2, 64, 16
    kc, vc, _, _ = make_cache(g, 24, page, hkv, d, torch.bfloat16)
    table, lens = tables(g, B, 6, 24, page).long(), torch.tensor([96, 2 ** 32 + 5, -2 ** 33 + 7, 40])
    table[0, 2] = 2 ** 32 + 3
    table[3, 0] = -2 ** 32 + 1
    table[1, 1] = 2 ** 40
    q = torch.randn(B, H, d, generator=g).to(torch.bfloat16)
    assert attend_ref(q, kc, vc, table, lens)[1][2].eq(-math.inf).all()
    check_attention(run_attention(pa, q, kc, vc, table, lens), attend_ref(q, kc, vc, table, lens), torch.bfloat16, False)
    sums, positions = torch.rand(B, hkv, 96, generator=g).cuda(), torch.arange(96, dtype=torch.int32).expand(B, hkv, 96).contiguous().cuda()
    kept, _, _ = pa.npu_paged_cache_evict(gpu(kc), gpu(vc), table.cuda(), lens.cuda(), sums, positions, 30, 4)
    assert kept.tolist() == [30, 30, 0, 30]


@pytest.mark.parametrize("kind", [torch.bfloat16, "int8"])
@pytest.mark.parametrize("page,d", [(16, 128), (24, 64), (64, 256)])
def test_attention_keys_and_values_laid_out_differently(pa, kind, page, d):
    """Keys token by token and values head by head, the scales the other way round."""
    g = torch.Generator().manual_seed(page + d)
    B, H, hkv = 5, 6, 3
    kc, _, ks, _ = make_cache(g, 40, page, hkv, d, kind, "token", 16, "head")
    _, vc, _, vs = make_cache(g, 40, page, hkv, d, kind, "head", 0, "token")
    table, lens = tables(g, B, 7, 40, page), torch.tensor([0, 1, page, 5 * page + 3, 7 * page], dtype=torch.int32)
    q = torch.randn(B, H, d, generator=g).to(torch.bfloat16)
    check_attention(run_attention(pa, q, kc, vc, table, lens, ks, vs), attend_ref(q, kc, vc, table, lens, ks, vs), torch.bfloat16, kind == "int8")


@pytest.mark.parametrize("kind", [torch.float16, "int8"])
@pytest.mark.parametrize("hkv,group,d", [(1, 16, 128), (1, 3, 256), (2, 20, 64)])
def test_attention_long_sequences_in_many_pieces(pa, kind, hkv, group, d):
    """More pieces of a pair than are added at once, beside short sequences."""
    g = torch.Generator().manual_seed(hkv * group)
    lens = torch.tensor([23001, 40, 0, 9000], dtype=torch.int32)
    width = 23040 // 64
    kc, vc, ks, vs = make_cache(g, 4 * width, 64, hkv, d, kind)
    table = tables(g, 4, width, 4 * width, 64)
    q = torch.randn(4, hkv * group, d, generator=g).to(torch.float16)
    check_attention(run_attention(pa, q, kc, vc, table, lens, ks, vs), attend_ref(q, kc, vc, table, lens, ks, vs), torch.float16, kind == "int8")


@pytest.mark.parametrize("kind,d", [(torch.bfloat16, 80), (torch.float16, 40), ("int8", 64)])
def test_attention_rows_of_several_heads_in_a_line(pa, kind, d):
    g = torch.Generator().manual_seed(d)
    B, hkv, page = 21, 7, 16
    lens = torch.randint(0, 500, (B,), generator=g).to(torch.int32)
    kc, vc, ks, vs = make_cache(g, B * 32, page, hkv, d, kind)
    table = tables(g, B, 32, B * 32, page)
    dt = torch.bfloat16 if kind == "int8" else kind
    q = torch.randn(B, 2 * hkv, d, generator=g).to(dt)
    check_attention(run_attention(pa, q, kc, vc, table, lens, ks, vs), attend_ref(q, kc, vc, table, lens, ks, vs), dt, kind == "int8")


def test_attention_calls_leave_nothing_behind(pa):
    """Calls of different shapes in turn, whose arrival counters lie at the same addresses: each gives the same bits every time."""
    g = torch.Generator().manual_seed(77)
    calls, first = [], []
    for B, H, hkv, d, n in ((2, 16, 1, 128, 9000), (7, 8, 8, 64, 700), (1, 32, 2, 256, 20000), (130, 4, 2, 128, 300)):
        width = -(-n // 64)
        kc, vc, _, _ = make_cache(g, B * width, 64, hkv, d, torch.bfloat16)
        lens = torch.randint(n // 2, n + 1, (B,), generator=g).to(torch.int32)
        calls.append((torch.randn(B, H, d, generator=g).to(torch.bfloat16).cuda(), gpu(kc), gpu(vc), tables(g, B, width, B * width, 64).cuda(), lens.cuda()))
        first.append(pa.npu_paged_decode_attention(*calls[-1], softmax_lse=True))
    for _ in range(5):
        for args, want in zip(calls, first):
            got = pa.npu_paged_decode_attention(*args, softmax_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------------------------ write and read

def codes_ref(x):
    """npu_dynamic_quant's rule in float32."""
    f = x.float()
    s = f.abs().amax(-1) / torch.tensor(127.0)
    c = torch.where(s[..., None] > 0, torch.round(f / s[..., None]), torch.zeros(()))
    return c.to(torch.int8), s


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, "int8"])
@pytest.mark.parametrize("order,pad", [("token", 0), ("head", 0), ("head", 16), ("token", 5)])
@pytest.mark.parametrize("d", [1, 40, 64, 80, 100, 128, 250, 256, 300])
def test_write_and_read(pa, kind, order, pad, d):
    g = torch.Generator().manual_seed(d)
    hkv, page, blocks, T = 3, 24, 9, 77
    kc, vc, ks, vs = make_cache(g, blocks, page, hkv, d, kind, order, pad)
    dt = torch.bfloat16 if kind == "int8" else kind
    qkv = torch.randn(T, 2 * hkv, d + pad, generator=g).to(dt)
    qkv[3], qkv[4] = 0, 1e-30 if dt == torch.bfloat16 else 6e-8
    key, value = qkv[:, :hkv, :d], qkv[:, hkv:, :d]
    slots = torch.randperm(blocks * page, generator=g)[:T]
    slots[10], slots[20] = -1, blocks * page                    # not written
    dev = [gpu(t) for t in (kc, vc, ks, vs)]
    wide = gpu(qkv)
    for slot_type in (torch.int64, torch.int32):
        pa.npu_paged_cache_write(wide[:, :hkv, :d], wide[:, hkv:, :d], dev[0], dev[1], slots.to(slot_type).cuda(), key_scale=dev[2], value_scale=dev[3])
        there = [t for t in range(T) if t not in (10, 20)]
        b, o = slots[there] // page, slots[there] % page
        if kind == "int8":
            for cache, scale, new in ((kc, ks, key), (vc, vs, value)):
                cache[b, o], scale[b, o] = codes_ref(new[there])
        else:
            kc[b, o], vc[b, o] = key[there], value[there]
        for mine, want in zip(dev, (kc, vc, ks, vs)):
            assert want is None or torch.equal(mine.cpu(), want)
        for out_type in ([torch.bfloat16, torch.float16] if kind == "int8" else [dt]):
            k, v = pa.npu_paged_cache_read(dev[0], dev[1], slots.to(slot_type).cuda(), key_scale=dev[2], value_scale=dev[3], dtype=out_type)
            for got, cache, scale in ((k, kc, ks), (v, vc, vs)):
                want = torch.zeros(T, hkv, d, dtype=out_type)
                want[there] = cache[b, o].to(out_type) if scale is None else (cache[b, o].float() * scale[b, o][..., None]).to(out_type)
                assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_write_int8_is_dynamic_quant(pa, dt):
    """The codes and scales of npu_dynamic_quant, rows with infinities and NaN and subnormal rows among them."""
    g = torch.Generator().manual_seed(3)
    T, hkv, d = 64, 4, 128
    x = torch.randn(T, hkv, d, generator=g) * torch.exp(4 * torch.randn(T, hkv, 1, generator=g))
    x[0, 0, 5], x[1, 1, 7], x[2] = math.inf, math.nan, 1e-7
    x = x.to(dt).cuda()
    kc = torch.zeros(T, 1, hkv, d, dtype=torch.int8, device="cuda")
    vc, ks, vs = torch.zeros_like(kc), torch.zeros(T, 1, hkv, device="cuda"), torch.zeros(T, 1, hkv, device="cuda")
    pa.npu_paged_cache_write(x, x, kc, vc, torch.arange(T, device="cuda"), key_scale=ks, value_scale=vs)
    codes, scales = pa.npu_dynamic_quant(x)
    assert torch.equal(kc[:, 0], codes) and torch.equal(vc[:, 0], codes)
    assert torch.equal(ks[:, 0].nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))
    assert torch.equal(vs[:, 0].nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))


def test_write_and_read_nothing(pa):
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    pa.npu_paged_cache_write(kc[0, :0], kc[0, :0], kc, kc.clone(), empty)
    k, v = pa.npu_paged_cache_read(kc, kc, empty)
    assert k.shape == v.shape == (0, 2, 64)
    out, lse = pa.npu_paged_decode_attention(kc[0, :0], kc, kc, torch.empty(0, 3, dtype=torch.int32, device="cuda"),
                                             torch.empty(0, dtype=torch.int32, device="cuda"), softmax_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    out, lse = pa.npu_paged_decode_attention(kc[0, :3] + 1, kc, kc, torch.empty(3, 0, dtype=torch.int32, device="cuda"),
                                             torch.ones(3, dtype=torch.int32, device="cuda"), softmax_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


# ------------------------------------------------------------------------------------------------ eviction

def evict_ref(kc, vc, ks, vs, table, lens, sums, positions, keep, recent):
    nb, page, hkv, _ = kc.shape
    B, cap = table.shape[0], table.shape[1] * page
    kc, vc = kc.clone(), vc.clone()
    ks, vs = None if ks is None else ks.clone(), None if vs is None else vs.clone()
    new_lens, new_sums, new_pos = torch.zeros(B, dtype=torch.int32), torch.zeros(B, hkv, cap), torch.full((B, hkv, cap), -1, dtype=torch.int32)
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        new_lens[b] = min(n, keep)
        for h in range(hkv):
            w, p = sums[b, h, :n], positions[b, h, :n].long()
            src = list(range(min(n, keep)))
            if n > keep > 0:
                newest = int(p.max())
                worth = [math.inf if int(p[i]) > newest - recent else -math.inf if w[i].isnan() else float(w[i]) for i in range(n)]
                below = [bool(w[i].isnan()) and worth[i] != math.inf for i in range(n)]             # NaN below -infinity
                first = [int(p[i]) > newest - recent for i in range(n)]
                order = sorted(range(n), key=lambda i: (not first[i], below[i], -worth[i], i))[:keep]
                kept = set(order)
                holes, fills = [i for i in range(keep) if i not in kept], sorted(i for i in kept if i >= keep)
                for dst, s in zip(holes, fills):
                    src[dst] = s
                    bd, bs = int(table[b, dst // page]), int(table[b, s // page])
                    if not (0 <= bd < nb and 0 <= bs < nb):
                        continue
                    for x in (kc, vc, ks, vs):
                        if x is not None:
                            x[bd, dst % page, h] = x[bs, s % page, h]
            for i, s in enumerate(src):
                new_sums[b, h, i], new_pos[b, h, i] = w[s], p[s]
    return kc, vc, ks, vs, new_lens, new_sums, new_pos


def same(a, b):
    return torch.equal(a.cpu().float().nan_to_num(nan=-12345.0), b.float().nan_to_num(nan=-12345.0))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, "int8"])
@pytest.mark.parametrize("page,d,order,pad", [(16, 128, "token", 0), (24, 80, "head", 0), (1, 64, "token", 0), (7, 33, "head", 3)])
@pytest.mark.parametrize("keep,recent", [(100, 20), (1, 1), (63, 63), (333, 0), (0, 0), (5000, 7)])
def test_evict(pa, kind, page, d, order, pad, keep, recent):
    g = torch.Generator().manual_seed(page * 1000 + keep)
    lens = torch.tensor([0, 1, 100, 101, 334, 400, 999, -2], dtype=torch.int32)
    B, hkv, width = len(lens), 2, -(-400 // page)
    cap = width * page
    kc, vc, ks, vs = make_cache(g, B * width, page, hkv, d, kind, order, pad)
    table = tables(g, B, width, B * width, page)
    table[5, -1] = -1
    sums = torch.exp(2 * torch.randn(B, hkv, cap, generator=g))
    sums[4] = (sums[4] * 3).round()                             # many equal ones
    sums[5, 0, 3:40:5], sums[5, 0, 4:60:7], sums[5, 1, 8:20] = math.nan, -math.inf, math.inf
    sums[5, 1, 30:90], sums[5, 1, 90:120] = 0.0, -0.0
    positions = torch.argsort(torch.rand(B, hkv, cap, generator=g), -1).to(torch.int32) * 3
    want = evict_ref(kc, vc, ks, vs, table, lens, sums, positions, keep, recent)
    dev = [gpu(t) for t in (kc, vc, ks, vs)]
    got = pa.npu_paged_cache_evict(dev[0], dev[1], table.cuda(), lens.cuda(), sums.cuda(), positions.cuda(), keep, recent, key_scale=dev[2],
                                   value_scale=dev[3])
    assert torch.equal(got[0].cpu(), want[4]) and same(got[1], want[5]) and torch.equal(got[2].cpu(), want[6])
    for mine, ref in zip(dev, want[:4]):
        assert ref is None or torch.equal(mine.cpu(), ref)


@pytest.mark.parametrize("n,keep", [(20000, 12345), (70000, 69999), (70001, 300)])
def test_evict_long(pa, n, keep):
    """More places than the keys of one workgroup fit on the chip, and sums that differ in their last bits only."""
    g = torch.Generator().manual_seed(n)
    page, hkv, d = 16, 1, 16
    width = -(-n // page)
    kc, vc, _, _ = make_cache(g, width, page, hkv, d, torch.bfloat16)
    table, lens = tables(g, 1, width, width, page), torch.tensor([n], dtype=torch.int32)
    sums = 1.0 + torch.randint(0, 5000, (1, 1, width * page), generator=g) * 2.0 ** -23
    positions = torch.arange(width * page, dtype=torch.int32).reshape(1, 1, -1)
    dev = gpu(kc), gpu(vc)
    got = pa.npu_paged_cache_evict(*dev, table.cuda(), lens.cuda(), sums.cuda(), positions.cuda(), keep, 100)
    worth = sums[0, 0, :n].clone()
    worth[n - 100:] = math.inf
    kept = torch.argsort(-worth.double(), stable=True)[:keep].sort().values
    fills, is_kept = kept[kept >= keep], torch.zeros(n, dtype=torch.bool)
    is_kept[kept] = True
    src = torch.arange(keep)
    src[(~is_kept[:keep]).nonzero()[:, 0]] = fills
    flat = table[0].long()
    want_k = kc[flat[src // page], src % page, 0]
    assert torch.equal(got[2][0, 0, :keep].cpu().long(), src) and torch.equal(got[1][0, 0, :keep].cpu(), sums[0, 0][src])
    at = torch.arange(keep)
    assert torch.equal(dev[0].cpu()[flat[at // page], at % page, 0], want_k)


def test_budgeted_cache_over_many_steps(pa):
    """Write, attend with sums, evict, step after step, against the same steps in 64 bits on the CPU."""
    g = torch.Generator().manual_seed(21)
    B, hkv, group, d, page, keep, recent = 2, 2, 2, 64, 16, 32, 8
    width = keep // page + 1
    cap = width * page
    kc, vc, _, _ = make_cache(g, B * width, page, hkv, d, torch.float16)
    dev = [gpu(kc), gpu(vc)]
    table = tables(g, B, width, B * width, page)
    lens = torch.zeros(B, dtype=torch.int32)
    sums, positions = torch.zeros(B, hkv, cap, device="cuda"), torch.full((B, hkv, cap), -1, dtype=torch.int32, device="cuda")
    for step in range(60):
        key, value, q = (torch.randn(B, h, d, generator=g).to(torch.float16) for h in (hkv, hkv, hkv * group))
        slots = table[torch.arange(B), lens.long() // page].long() * page + lens.long() % page
        pa.npu_paged_cache_write(key.cuda(), value.cuda(), *dev, slots.cuda())
        kc[slots // page, slots % page], vc[slots // page, slots % page] = key, value
        positions[torch.arange(B), :, lens.long()] = step
        lens = lens + 1
        before = sums.clone()
        got = pa.npu_paged_decode_attention(q.cuda(), *dev, table.cuda(), lens.cuda(), attn_sums=sums, softmax_lse=True)
        want = attend_ref(q, kc, vc, table, lens)
        check_attention(got, want, torch.float16, False)
        added = want[2].reshape(B, hkv, group, cap).sum(2)
        assert bool(((sums - before).cpu().double() - added).abs().max() < 1e-4)
        ref = evict_ref(kc, vc, None, None, table, lens, sums.cpu(), positions.cpu(), keep, recent)
        new_lens, sums, positions = pa.npu_paged_cache_evict(*dev, table.cuda(), lens.cuda(), sums, positions, keep, recent)
        kc, vc, lens = ref[0], ref[1], ref[4]
        assert torch.equal(new_lens.cpu(), lens) and same(sums, ref[5]) and torch.equal(positions.cpu(), ref[6])
        assert torch.equal(dev[0].cpu(), kc) and torch.equal(dev[1].cpu(), vc)
    assert int(lens.max()) == keep
