"""PagedKVCache: the paged operators together, as a decode step uses them."""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def module():
    from pytorch_amd.contrib import module
    return module


def rows(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g).to(dtype)


def attend(q, k, v):
    """64-bit attention of one token: q [heads, dim], k and v [tokens, kv_heads, dim]; also sum p|v|, the scale of an error."""
    group = q.shape[0] // k.shape[1]
    k, v = (x.double().repeat_interleave(group, 1) for x in (k, v))
    p = torch.softmax(torch.einsum("hd,thd->ht", q.double(), k) / math.sqrt(q.shape[1]), 1)
    return torch.einsum("ht,thd->hd", p, v), torch.einsum("ht,thd->hd", p, v.abs()), p


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steps_without_a_budget(module, quantized, dtype):
    """Prompts of different lengths, one in two pieces, then steps; against attention over the same rows.  The bound: roundings
    of output and probabilities (u each) over sum p|v|, a thousandth for float32 sums, and on an int8 cache the codes themselves,
    which the reference reads back."""
    g = torch.Generator().manual_seed(1)
    batch, heads, kv, d = 3, 8, 2, 80
    cache = module.PagedKVCache(batch, 100, kv, d, block_size=16, quantized=quantized, device="cuda", dtype=dtype)
    kept = [[], [], []]

    def fill(b, n):
        k, v = rows(g, n, kv, d, dtype=dtype), rows(g, n, kv, d, dtype=dtype)
        cache.prefill(b, k.cuda(), v.cuda())
        kept[b].append((k, v))

    fill(0, 40), fill(2, 17), fill(2, 30)
    for _ in range(5):
        k, v, q = (rows(g, batch, n, d, dtype=dtype) for n in (kv, kv, heads))
        cache.append(k.cuda(), v.cuda())
        for b in range(batch):
            kept[b].append((k[b:b + 1], v[b:b + 1]))
        out = cache.attend(q.cuda()).cpu().double()
        for b in range(batch):
            k, v = (torch.cat(x) for x in zip(*kept[b]))
            got_k, got_v = (x.cpu() for x in cache.read(b, 0, len(k)))
            if quantized:
                for got, want in ((got_k, k), (got_v, v)):
                    step = want.double().abs().amax(-1, keepdim=True) / 127
                    assert bool(((got.double() - want.double()).abs() <= step * 0.501 + want.double().abs() * 2 * U[dtype]).all())
                # (what the kernel reads: codes times scales, not rounded to dtype)
                place = torch.arange(len(k))
                slots = (cache.block_table[b].cpu().long()[place // 16], place % 16)
                k, v = (c.cpu()[slots].double() * s.cpu()[slots].double()[..., None]
                        for c, s in ((cache.key_cache, cache.key_scale), (cache.value_cache, cache.value_scale)))
            else:
                assert torch.equal(got_k, k) and torch.equal(got_v, v)
            want, spread, _ = attend(q[b], k, v)
            assert bool(((out[b] - want).abs() <= U[dtype] * (want.abs() + 1.01 * spread) + 1e-3 * spread).all())
    assert cache.context_lens.tolist() == [45, 5, 52]
    cache.clear(1)
    with pytest.raises(RuntimeError, match="do not fit into 112"):
        cache.prefill(2, *(torch.zeros(61, kv, d, dtype=dtype, device="cuda"),) * 2)
    cache.prefill(1, *(torch.zeros(112, kv, d, dtype=dtype, device="cuda"),) * 2)
    with pytest.raises(RuntimeError, match="sequence 1 holds up to 112"):
        cache.append(*(torch.zeros(batch, kv, d, dtype=dtype, device="cuda"),) * 2)
    with pytest.raises(RuntimeError, match="budget"):
        cache.evict()
    with pytest.raises(IndexError):
        cache.read(0, 0, 113)


@pytest.mark.parametrize("quantized", [False, True])
def test_budget_keeps_the_newest_and_the_most_attended(module, quantized):
    """Every head of every sequence, over 30 steps: what it holds is what a plain simulation of its own choices holds, as long
    as those are not closer than the sums' error; rows travel with their positions."""
    g = torch.Generator().manual_seed(2)
    batch, heads, kv, d, budget, recent = 2, 4, 2, 64, 24, 6
    cache = module.PagedKVCache(batch, budget + 4, kv, d, block_size=8, budget=budget, recent=recent, quantized=quantized, device="cuda")
    written = {}
    position = [0] * batch
    held = [[{} for _ in range(kv)] for _ in range(batch)]          # position -> sum

    def note(b, k, v):
        for t in range(len(k)):
            written[b, position[b]] = (k[t], v[t])
            for h in range(kv):
                held[b][h][position[b]] = 0.0
            position[b] += 1

    for b, n in enumerate((20, 9)):
        k, v = rows(g, n, kv, d), rows(g, n, kv, d)
        cache.prefill(b, k.cuda(), v.cuda())
        note(b, k, v)
    for _ in range(30):
        k, v, q = rows(g, batch, kv, d), rows(g, batch, kv, d), rows(g, batch, heads, d) * 2
        cache.append(k.cuda(), v.cuda())
        cache.attend(q.cuda())
        cache.evict()
        places = cache.positions.cpu()
        for b in range(batch):
            note(b, k[b:b + 1], v[b:b + 1])
            n = min(position[b], budget)
            assert int(cache.context_lens[b]) == n
            got_k, got_v = (x.cpu() for x in cache.read(b, 0, n))
            for h in range(kv):
                mine = held[b][h]
                order = list(mine)
                stored = [written[b, j] for j in order]
                ks, vs = (torch.stack([r[i][h] for r in stored])[:, None] for i in (0, 1))
                if quantized:                                       # the scale of a row: its largest value / 127
                    step = ks.float().abs().amax(-1, keepdim=True) / 127
                    ks = (ks.float() / step).round() * step
                for qh in range(heads // kv):
                    p = attend(q[b, h * (heads // kv) + qh][None], ks, vs)[2][0]
                    for j, w in zip(order, p.tolist()):
                        mine[j] += w
                if len(mine) > budget:
                    old = sorted((j for j in mine if j <= position[b] - 1 - recent), key=lambda j: mine[j])
                    gap = mine[old[1]] - mine[old[0]]
                    gone = (set(mine) - set(places[b, h, :n].tolist())).pop()
                    assert gone == old[0] or gap < 1e-4
                    del mine[gone]
                assert sorted(places[b, h, :n].tolist()) == sorted(mine)
                assert places[b, h, n:].eq(-1).all()
                sums = cache.attn_sums[b, h, :n].cpu().tolist()
                for at, j in enumerate(places[b, h, :n].tolist()):
                    assert abs(sums[at] - mine[j]) < 1e-4
                    for got, want in ((got_k[at, h], written[b, j][0][h]), (got_v[at, h], written[b, j][1][h])):
                        bound = want.double().abs().max() / 127 * 0.501 + want.double().abs() * 2.0 ** -7 if quantized else 0
                        assert bool(((got.double() - want.double()).abs() <= bound).all())


def test_captured_step_replays(module):
    """A captured step against eager steps on a second cache, with eager work between the replays."""
    g = torch.Generator().manual_seed(3)
    batch, heads, kv, d = 4, 8, 2, 128
    caches = [module.PagedKVCache(batch, 70, kv, d, budget=48, device="cuda") for _ in range(2)]
    for b in range(batch):
        k, v = rows(g, 40 + b, kv, d).cuda(), rows(g, 40 + b, kv, d).cuda()
        for c in caches:
            c.prefill(b, k, v)
    q, k, v = (torch.zeros(batch, n, d, dtype=torch.bfloat16, device="cuda") for n in (heads, kv, kv))

    def step(c):
        c.append(k, v)
        out = c.attend(q)
        c.evict()
        return out

    step(caches[0]), step(caches[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for _ in range(12):
        for t, n in ((q, heads), (k, kv), (v, kv)):
            t.copy_(rows(g, batch, n, d))
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for name in ("context_lens", "positions", "attn_sums", "next_position", "key_cache", "value_cache"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    assert caches[0].context_lens.tolist() == [48] * batch


@pytest.mark.parametrize("more", [[], ["--int8-cache"], ["--graph"]])
def test_example_runs(more):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_paged_cache.py")
    spec = importlib.util.spec_from_file_location("decode_paged_cache", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    y, cache = example.main(["--batch", "3", "--hidden", "512", "--heads", "8", "--kv-heads", "2", "--budget", "64", "--prompt", "60", "--steps", "8"] + more)
    assert y.shape == (3, 512) and bool(torch.isfinite(y).all())
    assert cache.context_lens.tolist() == [64, 64, 64]
