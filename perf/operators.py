"""The paged key-value cache's operators, as a serving program calls them, beside their plain forms.

A case is one pass through one of four operators, named by ``op``:

* ``write``   the keys and values of new tokens go into their slots of the cache, as they are or quantised to int8 with one
              scale per token and head;
* ``read``    tokens come back out of the cache in the order of a list of slots, in 16 bits: what the next chunk of a long
              prompt attends to;
* ``attend``  one new token of every sequence attends to that sequence's pages; optionally every key/value head adds the
              weight that each cached position got to a running sum;
* ``evict``   a cache that outgrew its budget keeps the newest tokens and those with the largest running sums.

Cache: ``[blocks, page, key/value heads, head width]``, in memory either in that order ("token") or with the heads outside
the page's tokens ("head"); int8 caches have float32 scales ``[blocks, page, heads]``, a head's scales of a page side by side.
With ``own`` false ``run`` is the plain form: elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
# no drawn case has more cached values than the largest listed ones, 2 * 131071 * 8 * 128 of 16 bits each
_MAX_CACHE_BYTES = 5.0e8
_MAX_POSITIONS = 2 ** 19                       # sequences x longest length: what the plain forms pad to


def listed():
    return [
        # a decode step's new tokens, one of each sequence, bf16 cache
        {"name": "write_decode_64", "op": "write", "T": 64, "Hkv": 8, "D": 128, "page": 16, "dtype": "bf16", "int8": False, "order": "token"},
        # a chunk of a prompt into an int8 cache; the codes come back as the values they stand for
        {"name": "write_prefill_int8", "op": "write", "T": 8192, "Hkv": 8, "D": 128, "page": 16, "dtype": "bf16", "int8": True, "order": "head"},
        # a prefix of odd length that the next chunk attends to
        {"name": "read_prefix_2047", "op": "read", "T": 2047, "Hkv": 8, "D": 128, "page": 16, "dtype": "bf16", "int8": False, "order": "token"},
        # a long prefix out of an int8 cache
        {"name": "read_prefix_int8", "op": "read", "T": 32768, "Hkv": 8, "D": 128, "page": 64, "dtype": "fp16", "int8": True, "order": "head"},
        # the first answers to a short prompt, one sequence: the smallest call of a decode step
        {"name": "attend_one_short", "op": "attend", "B": 1, "H": 32, "Hkv": 8, "D": 128, "len": 37, "page": 16, "dtype": "bf16", "int8": False,
         "order": "token", "ragged": False, "mask": False, "sums": False},
        # a decode batch of requests of all ages, grouped heads
        {"name": "attend_batch_32", "op": "attend", "B": 32, "H": 32, "Hkv": 8, "D": 128, "len": 4095, "page": 16, "dtype": "bf16", "int8": False,
         "order": "token", "ragged": True, "mask": False, "sums": False},
        # a large batch on an int8 cache
        {"name": "attend_batch_64_int8", "op": "attend", "B": 64, "H": 32, "Hkv": 8, "D": 128, "len": 8192, "page": 64, "dtype": "bf16", "int8": True,
         "order": "head", "ragged": True, "mask": False, "sums": False},
        # one very long document
        {"name": "attend_one_long", "op": "attend", "B": 1, "H": 32, "Hkv": 8, "D": 128, "len": 131071, "page": 128, "dtype": "fp16", "int8": False,
         "order": "token", "ragged": False, "mask": False, "sums": False},
        # every query head with a key/value head of its own, narrow heads, pages that no tile divides, left-padded prompts
        {"name": "attend_mha_masked", "op": "attend", "B": 16, "H": 32, "Hkv": 32, "D": 80, "len": 1001, "page": 24, "dtype": "fp16", "int8": False,
         "order": "token", "ragged": True, "mask": True, "sums": False},
        # a batch whose attention weights are summed for eviction
        {"name": "attend_sums_16", "op": "attend", "B": 16, "H": 32, "Hkv": 8, "D": 128, "len": 4097, "page": 16, "dtype": "bf16", "int8": False,
         "order": "token", "ragged": False, "mask": False, "sums": True},
        # the steady state of a budgeted cache: one token too many in every sequence
        {"name": "evict_one_over", "op": "evict", "B": 16, "Hkv": 8, "D": 128, "len": 4097, "keep": 4096, "recent": 512, "page": 16, "dtype": "bf16",
         "order": "token", "ragged": False},
        # prompts of several lengths brought down to the budget after their prefill
        {"name": "evict_half", "op": "evict", "B": 8, "Hkv": 8, "D": 128, "len": 8192, "keep": 4096, "recent": 256, "page": 64, "dtype": "fp16",
         "order": "head", "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd_or_tiles(rng, lo, hi):
    """A length: mostly any odd number, now and then a multiple of 256."""
    n = _log_int(rng, lo, hi)
    return max(256, n // 256 * 256) if rng.random() < 0.25 and n >= 256 and n // 256 % 3 else n | 1


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "evict"])
    c = {"op": op, "Hkv": rng.choice([1, 2, 4, 8, 8, 32]), "D": rng.choice([64, 80, 96, 128, 128, 128, 256]), "page": rng.choice([16, 16, 24, 32, 64, 128]),
         "dtype": rng.choice(["bf16", "fp16"]), "order": rng.choice(["token", "head"])}
    row = c["Hkv"] * c["D"] * 4                                  # bytes of one cached token at 16 bits
    if op in ("write", "read"):
        return {**c, "T": min(_odd_or_tiles(rng, 1, 32768), int(_MAX_CACHE_BYTES / 4 / row)), "int8": rng.random() < 0.5}
    if op == "evict":
        n = _odd_or_tiles(rng, 256, 16384)
        n = min(n, int(_MAX_CACHE_BYTES / 2 / row))
        keep = max(64, n - 1 if rng.random() < 0.4 else int(n * rng.uniform(0.3, 0.95)))
        b = max(1, min(_log_int(rng, 1, 32), int(_MAX_CACHE_BYTES / 2 / (n * row)), 128 // c["Hkv"]))
        return {**c, "B": b, "len": n, "keep": keep, "recent": rng.randrange(0, keep // 2), "ragged": rng.random() < 0.5}
    c["H"] = c["Hkv"] * (rng.choice([1, 1, 2]) if c["Hkv"] == 32 else rng.choice([1, 2, 4, 4, 5, 7, 8, 16]))
    c["int8"] = rng.random() < 0.4
    sums = rng.random() < 0.25
    n = min(_odd_or_tiles(rng, 1, 32768 if sums else 131071), int(_MAX_CACHE_BYTES / row))
    b = max(1, min(_log_int(rng, 1, 128), _MAX_POSITIONS // n, int(_MAX_CACHE_BYTES / (n * row))))
    return {**c, "B": b, "len": n, "ragged": rng.random() < 0.6, "mask": rng.random() < 0.2, "sums": sums}


def _lengths(case):
    """The sequences' lengths, sorted: what the pass works on is the same for every seed."""
    b, n = case["B"], case["len"]
    if not case["ragged"]:
        return [n] * b
    lo = 1 if case["op"] == "attend" else case["keep"] // 2
    return [lo + (n - lo) * (i + 1) // b for i in range(b)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op, hkv, d, page, dt = case["op"], case["Hkv"], case["D"], case["page"], _DT[case["dtype"]]
    int8 = case.get("int8", False)
    batch = case.get("B", 1)
    n = case["T"] + 3 * page if "T" in case else case["len"]
    width = -(-n // page)                                       # pages of a sequence
    blocks = batch * width + 5

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def cache(value):
        shape = (blocks, page, hkv, d) if case["order"] == "token" else (blocks, hkv, page, d)
        if op == "write":
            t = torch.zeros(*shape, device=dev, dtype=torch.int8 if int8 else dt)
        elif int8:
            t = torch.empty(*shape, device=dev, dtype=torch.float16).normal_(0.0, 32.0, generator=g).round_().clamp_(-127, 127).to(torch.int8)
        else:
            t = torch.empty(*shape, device=dev, dtype=dt).normal_(0.0, 1.0, generator=g)
            if not value:
                t *= torch.exp(0.5 * normal(d)).to(dt)          # keys have channels that are larger than others
        t = t if case["order"] == "token" else t.transpose(1, 2)
        if not int8:
            return t, None
        s = torch.rand(blocks, hkv, page, generator=g, device=dev) * 0.03 + 0.01 if op != "write" else torch.zeros(blocks, hkv, page, device=dev)
        return t, s.transpose(1, 2)

    state = {"op": op, "dtype": dt}
    state["key_cache"], state["key_scale"] = cache(False)
    state["value_cache"], state["value_scale"] = cache(True)
    pages = torch.randperm(blocks, generator=g, device=dev)[: batch * width].to(torch.int32).reshape(batch, width)
    if op in ("write", "read"):
        at = torch.arange(case["T"], device=dev) + page // 2    # a chunk starts anywhere in its first page
        state["slots"] = pages[0][at // page].long() * page + at % page
        if op == "write":
            qkv = normal(case["T"], 4 * hkv + 2 * hkv, d).to(dt)          # what the fused projection leaves behind
            state["key"], state["value"] = qkv[:, 4 * hkv:5 * hkv], qkv[:, 5 * hkv:]
        return state
    order = torch.randperm(batch, generator=g, device=dev)
    state["block_table"], state["lens"] = pages, torch.tensor(_lengths(case), dtype=torch.int32, device=dev)[order]
    if op == "attend":
        state["query"] = (normal(batch, case["H"], d) * 2.0).to(dt)
        state["mask"] = None
        if case["mask"]:                                        # left-padded prompts, and a few tokens taken back
            spot = torch.arange(width * page, device=dev)
            pad = torch.rand(batch, 1, generator=g, device=dev) * 0.3 * state["lens"][:, None]
            state["mask"] = (spot < pad) | (torch.rand(batch, width * page, generator=g, device=dev) < 0.02)
        state["sums"] = torch.rand(batch, hkv, width * page, generator=g, device=dev) if case["sums"] else None
        return state
    cap = width * page
    spot = torch.arange(cap, device=dev)
    live = spot < state["lens"][:, None, None]
    state["sums"] = torch.where(live, torch.exp(1.5 * normal(batch, hkv, cap)), torch.zeros((), device=dev))
    # earlier evictions have left the tokens in no order
    step = torch.randint(1, 3, (batch, hkv, cap), generator=g, device=dev).cumsum(-1)
    mix = torch.where(live, torch.rand(batch, hkv, cap, generator=g, device=dev), 2.0).argsort(-1)
    state["positions"] = torch.where(live, step.gather(-1, mix), -1).to(torch.int32)
    state["keep"], state["recent"] = case["keep"], case["recent"]
    return state


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


def _own(s):
    import pytorch_amd as pa
    scales = {"key_scale": s["key_scale"], "value_scale": s["value_scale"]}
    if s["op"] == "write":
        pa.npu_paged_cache_write(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"], **scales)
        if s["key_scale"] is not None:
            return pa.npu_paged_cache_read(s["key_cache"], s["value_cache"], s["slots"], **scales, dtype=s["dtype"])
        return s["key_cache"], s["value_cache"]
    if s["op"] == "read":
        return pa.npu_paged_cache_read(s["key_cache"], s["value_cache"], s["slots"], **scales, dtype=s["dtype"])
    if s["op"] == "attend":
        out, lse = pa.npu_paged_decode_attention(s["query"], s["key_cache"], s["value_cache"], s["block_table"], s["lens"], **scales,
                                                 atten_mask=s["mask"], attn_sums=s["sums"], softmax_lse=True)
        return (out, lse) if s["sums"] is None else (out, lse, s["sums"])
    lens, sums, positions = pa.npu_paged_cache_evict(s["key_cache"], s["value_cache"], s["block_table"], s["lens"], s["sums"], s["positions"],
                                                     s["keep"], s["recent"])
    return s["key_cache"], s["value_cache"], lens, sums, positions


def _plain_write(s):
    page = s["key_cache"].shape[1]
    block, spot = s["slots"] // page, s["slots"] % page
    if s["key_scale"] is None:
        s["key_cache"][block, spot] = s["key"]
        s["value_cache"][block, spot] = s["value"]
        return s["key_cache"], s["value_cache"]
    k, v = s["key"].float(), s["value"].float()
    ks, vs = k.abs().amax(-1) / 127.0, v.abs().amax(-1) / 127.0
    s["key_cache"][block, spot] = torch.where(ks[..., None] > 0, torch.round(k / ks[..., None]), 0.0).to(torch.int8)
    s["value_cache"][block, spot] = torch.where(vs[..., None] > 0, torch.round(v / vs[..., None]), 0.0).to(torch.int8)
    s["key_scale"][block, spot] = ks
    s["value_scale"][block, spot] = vs
    return _plain_read(s)


def _plain_read(s):
    page = s["key_cache"].shape[1]
    block, spot = s["slots"] // page, s["slots"] % page
    k, v = s["key_cache"][block, spot], s["value_cache"][block, spot]
    if s["key_scale"] is None:
        return k, v
    return (k.float() * s["key_scale"][block, spot][..., None]).to(s["dtype"]), (v.float() * s["value_scale"][block, spot][..., None]).to(s["dtype"])


def _plain_attend(s):
    q, lens, pages = s["query"], s["lens"], s["block_table"].long()
    batch, heads, d = q.shape
    hkv = s["key_cache"].shape[2]
    k, v = s["key_cache"][pages].flatten(1, 2).float(), s["value_cache"][pages].flatten(1, 2).float()       # [B, S, Hkv, D]
    if s["key_scale"] is not None:
        k = k * s["key_scale"][pages].flatten(1, 2)[..., None]
        v = v * s["value_scale"][pages].flatten(1, 2)[..., None]
    score = torch.matmul(q.float().reshape(batch, hkv, heads // hkv, d), k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    seen = torch.arange(k.shape[1], device=q.device) < lens[:, None]
    if s["mask"] is not None:
        seen = seen & ~s["mask"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = torch.matmul(p, v.transpose(1, 2)).reshape(batch, heads, d).to(q.dtype)
    lse = (top + torch.log(total)).reshape(batch, heads)
    if s["sums"] is None:
        return out, lse
    s["sums"] += p.sum(2)
    return out, lse, s["sums"]


def _plain_evict(s):
    kc, vc, pages, lens, keep, recent = s["key_cache"], s["value_cache"], s["block_table"].long(), s["lens"], s["keep"], s["recent"]
    page, hkv, cap = kc.shape[1], kc.shape[2], s["sums"].shape[-1]
    keep = min(keep, cap)
    spot = torch.arange(cap, device=kc.device)
    live = spot < lens[:, None, None]
    newest = torch.where(live, s["positions"], -1).amax(-1, keepdim=True)
    worth = torch.where(s["positions"] > newest - recent, math.inf, s["sums"])
    order = torch.where(live, worth, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, spot.expand_as(order))
    kept = live & (rank < keep)
    hole, late = live & ~kept & (spot < keep), kept & (spot >= keep)
    sources = torch.where(late, spot, cap).sort(-1).values
    source = torch.where(hole, sources.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), spot)        # where a slot's token comes from
    to = spot[:keep]
    come = source[..., :keep].transpose(1, 2)                                                       # [B, keep, Hkv]
    seq = torch.arange(pages.shape[0], device=kc.device)[:, None, None]
    head = torch.arange(hkv, device=kc.device)
    block, offset = pages[seq, come // page], come % page
    to_block, to_offset = pages[:, to // page][..., None], (to % page)[:, None]
    kc[to_block, to_offset, head] = kc[block, offset, head]
    vc[to_block, to_offset, head] = vc[block, offset, head]
    lens = lens.clamp(max=keep)
    live = spot < lens[:, None, None]
    source = source.clamp(max=cap - 1)
    return kc, vc, lens, torch.where(live, s["sums"].gather(-1, source), 0.0), torch.where(live, s["positions"].gather(-1, source), -1)


_PLAIN = {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "evict": _plain_evict}


def work(case):
    hkv, d = case["Hkv"], case["D"]
    size = 1 if case.get("int8") else 2
    scale = 4 if case.get("int8") else 0
    row = 2 * hkv * (d * size + scale)                          # one token's keys and values in the cache
    if case["op"] in ("write", "read"):
        t = case["T"]
        wide = 2 * hkv * d * 2                                  # the same outside the cache
        again = row + wide if case["op"] == "write" and case["int8"] else 0
        return {"bytes": t * (row + wide + 8 + again), "flops": t * hkv * d * 2 * (3 if scale else 0)}
    tokens = sum(_lengths(case))
    if case["op"] == "attend":
        h = case["H"]
        return {"bytes": tokens * (row + 4 / case["page"] + (8 * hkv if case["sums"] else 0) + (1 if case["mask"] else 0)) + case["B"] * h * (4 * d + 4),
                "flops": tokens * h * d * 4}
    # a token that has to move is read and written; by chance the evicted ones among the first `keep` slots
    moved = sum(max(0, n - case["keep"]) * min(n, case["keep"]) / max(1, n) for n in _lengths(case))
    cap = -(-case["len"] // case["page"]) * case["page"]
    return {"bytes": moved * row * 2 + hkv * (tokens * 8 + case["B"] * cap * 8), "flops": hkv * tokens * 4}


def exact(case, seed):
    s = prepare(case, seed)
    kc, vc = s["key_cache"], s["value_cache"]
    blocks, page, hkv, d = kc.shape

    def rows(cache, scale, slots):                              # [n, heads, d] in 64 bits
        flat = cache[slots.div(page, rounding_mode="floor"), slots.remainder(page)].double()
        return flat if scale is None else flat * scale[slots.div(page, rounding_mode="floor"), slots.remainder(page)].double().unsqueeze(-1)

    if case["op"] == "read":
        return rows(kc, s["key_scale"], s["slots"]), rows(vc, s["value_scale"], s["slots"])
    if case["op"] == "write":
        if case["int8"]:                                        # what the codes stand for
            got = []
            for new in (s["key"], s["value"]):
                step = new.double().abs().max(-1, keepdim=True).values / 127.0
                got.append(torch.round(new.double() / step.clamp(min=1e-300)) * step)
            return tuple(got)
        for cache, new in ((kc, s["key"]), (vc, s["value"])):
            for i, slot in enumerate(s["slots"].tolist() if case["T"] <= 256 else []):
                cache[slot // page, slot % page] = new[i]
            if case["T"] > 256:
                cache.index_put_((s["slots"].div(page, rounding_mode="floor"), s["slots"].remainder(page)), new)
        return kc.double(), vc.double()
    lens = s["lens"].tolist()
    table = s["block_table"].tolist()
    if case["op"] == "attend":
        group = case["H"] // hkv
        outs, lses, sums = [], [], None if s["sums"] is None else s["sums"].double()
        for b, n in enumerate(lens):
            at = torch.arange(n, device=kc.device)
            ids = torch.tensor(table[b], device=kc.device)[at.div(page, rounding_mode="floor")] * page + at.remainder(page)
            if s["mask"] is not None:
                at = at[~s["mask"][b, :n]]
                ids = ids[~s["mask"][b, :n]]
            k, v = rows(kc, s["key_scale"], ids).transpose(0, 1), rows(vc, s["value_scale"], ids).transpose(0, 1)      # [Hkv, n, D]
            q = s["query"][b].double().view(hkv, group, d)
            z = torch.bmm(k.contiguous(), q.transpose(1, 2).contiguous()) / math.sqrt(d)                                # [Hkv, n, group]
            lse = torch.logsumexp(z, 1)
            w = torch.exp(z - lse[:, None])
            outs.append(torch.bmm(w.transpose(1, 2).contiguous(), v.contiguous()).view(-1, d))
            lses.append(lse.reshape(-1))
            if sums is not None:
                sums[b].index_add_(1, at, w.sum(-1))
        got = (torch.stack(outs), torch.stack(lses))
        return got if sums is None else (*got, sums)
    keep, recent = case["keep"], case["recent"]
    new_lens, new_sums, new_pos = [], torch.zeros_like(s["sums"], dtype=torch.float64), torch.full_like(s["positions"], -1)
    for b, n in enumerate(lens):
        new_lens.append(min(n, keep))
        ids = torch.tensor([p * page + t for p in table[b] for t in range(page)], device=kc.device)
        for h in range(hkv):
            w, p = s["sums"][b, h, :n].double().cpu(), s["positions"][b, h, :n].cpu()
            slots = torch.arange(n)
            if n > keep:
                w_sort = torch.where(p > p.max() - recent, torch.tensor(math.inf, dtype=torch.float64), w)
                stay = torch.argsort(-w_sort, stable=True)[:keep]                      # largest first, the lower slot first among equals
                is_kept = torch.zeros(n, dtype=torch.bool)
                is_kept[stay] = True
                holes, movers = slots[:keep][~is_kept[:keep]], slots[keep:][is_kept[keep:]]
                src, dst = ids[movers.to(ids.device)], ids[holes.to(ids.device)]
                for cache in (kc, vc):
                    cache[dst // page, dst % page, h] = cache[src // page, src % page, h]
                slots = slots[:keep].clone()
                slots[holes] = movers
            new_sums[b, h, : len(slots)] = w[slots].to(kc.device)
            new_pos[b, h, : len(slots)] = p[slots].to(kc.device)
    return kc.double(), vc.double(), torch.tensor(new_lens), new_sums, new_pos
