"""What a decoder layer needs between its quantised projections, as a serving program calls it, beside plain forms.

A case is one pass through one operator, named by ``op``:

* ``norm``    the residual stream and a block's output are added and normalised by their root mean square, into 16 bits or,
              with ``int8``, into codes with one scale per token for the next W8A8 projection;
* ``rotate``  queries and keys of a fused projection are turned to their positions, on one axis or on three (time, height and
              width of images and video), from a table of cosines and sines;
* ``store``   tokens go into a paged cache of 4-bit codes, with a scale and an offset per token and head, and come back as the
              values that the codes stand for;
* ``attend``  one new token of every sequence attends to that sequence's pages of such a cache.

A 4-bit cache is int32 words of eight codes in two's complement, the first in the lowest bits, ``[blocks, page, key/value
heads, head width / 8]``, in memory in that order ("token") or with the heads outside the page's tokens ("head"); scales and
offsets are float32 ``[blocks, page, heads]``, a head's of a page side by side; a value is ``(code + offset) * scale``.
With ``own`` false ``run`` is the plain form: elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_MAX_NORM = 8191 * 8192                        # elements of the largest listed norm
_MAX_ROTATE = 32767 * 40 * 128                 # and of queries and keys together
_MAX_STORE = 8192 * 8 * 128                    # and of the keys that are stored
_MAX_ATTEND = 64 * 8192 // 2 * 8 * 144         # and bytes of the cache that is attended to
_MAX_POSITIONS = 2 ** 19                       # sequences x longest length: what the plain form pads to


def listed():
    return [
        # the one token of a chat that is being decoded, on its way into a W8A8 projection
        {"name": "norm_int8_one_token", "op": "norm", "T": 1, "N": 4096, "dtype": "bf16", "int8": True, "residual": True},
        # a long prompt's chunk on the same way
        {"name": "norm_int8_prefill", "op": "norm", "T": 8191, "N": 8192, "dtype": "bf16", "int8": True, "residual": True},
        # a decode batch in front of a weight-only projection, which takes 16 bits
        {"name": "norm_decode_64", "op": "norm", "T": 64, "N": 8192, "dtype": "fp16", "int8": False, "residual": True},
        # a prompt in front of one; its width is no multiple of the usual ones
        {"name": "norm_prefill", "op": "norm", "T": 2047, "N": 5128, "dtype": "bf16", "int8": False, "residual": True},
        # a decode step of a model that sees images: all axes of a token at the same position
        {"name": "rotate_decode_64", "op": "rotate", "T": 64, "H": 32, "Hkv": 8, "D": 128, "R": 128, "t": 16, "h": 24, "w": 24, "mode": "half",
         "dtype": "bf16", "table": "bf16"},
        # a prompt of text and images
        {"name": "rotate_prefill_images", "op": "rotate", "T": 32767, "H": 32, "Hkv": 8, "D": 128, "R": 128, "t": 16, "h": 24, "w": 24, "mode": "half",
         "dtype": "bf16", "table": "fp32"},
        # a decode step's new tokens, one of each sequence
        {"name": "store_decode_64", "op": "store", "T": 64, "Hkv": 8, "D": 128, "page": 16, "dtype": "bf16", "order": "token"},
        # a chunk of a prompt
        {"name": "store_prefill", "op": "store", "T": 8192, "Hkv": 8, "D": 128, "page": 64, "dtype": "bf16", "order": "head"},
        # the start of one chat, where latency counts
        {"name": "attend_one_short", "op": "attend", "B": 1, "H": 32, "Hkv": 8, "D": 128, "len": 37, "page": 16, "dtype": "bf16", "order": "token",
         "ragged": False, "mask": False, "sums": False},
        # a serving batch in the middle of its answers
        {"name": "attend_batch_32", "op": "attend", "B": 32, "H": 32, "Hkv": 8, "D": 128, "len": 4095, "page": 16, "dtype": "bf16", "order": "token",
         "ragged": True, "mask": False, "sums": False},
        # a large batch with long contexts, what 4 bits make room for
        {"name": "attend_batch_64", "op": "attend", "B": 64, "H": 32, "Hkv": 8, "D": 128, "len": 8192, "page": 64, "dtype": "bf16", "order": "head",
         "ragged": True, "mask": False, "sums": False},
        # one very long document
        {"name": "attend_one_long", "op": "attend", "B": 1, "H": 32, "Hkv": 8, "D": 128, "len": 131071, "page": 128, "dtype": "fp16", "order": "head",
         "ragged": False, "mask": False, "sums": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd_or_tiles(rng, lo, hi):
    """A length: mostly any odd number, now and then a multiple of 256."""
    n = _log_int(rng, lo, hi)
    return max(256, n // 256 * 256) if rng.random() < 0.25 and n >= 256 and n // 256 % 3 else n | 1


def draw(rng):
    op = rng.choice(["norm", "norm", "rotate", "store", "attend", "attend"])
    c = {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
    if op == "norm":
        n = _log_int(rng, 64, 16384)
        n = n // 8 * 8 if rng.random() < 0.8 else n              # widths are multiples of 8 as a rule
        return {**c, "T": max(1, min(_odd_or_tiles(rng, 1, 32768), _MAX_NORM // n)), "N": n, "int8": rng.random() < 0.6, "residual": rng.random() < 0.85}
    c |= {"Hkv": rng.choice([1, 2, 4, 8, 8, 32]), "D": rng.choice([64, 80, 96, 128, 128, 128, 256])}
    c["H"] = c["Hkv"] * (rng.choice([1, 1, 2]) if c["Hkv"] == 32 else rng.choice([1, 2, 4, 4, 5, 7, 8, 16]))
    if op == "rotate":
        r = rng.choice([c["D"], c["D"], c["D"], c["D"] // 2])
        t, h, w = r // 2, 0, 0
        if rng.random() < 0.7:                                   # three axes, their sections multiples of 8 or any
            t, h = r // 8, (r // 2 - r // 8) // 2
            t, h = (t, h) if rng.random() < 0.7 else (rng.randrange(1, r // 4), rng.randrange(1, r // 4))
            w = r // 2 - t - h
        heads = (c["H"] + c["Hkv"]) * c["D"]
        return {**c, "T": max(1, min(_odd_or_tiles(rng, 1, 32768), _MAX_ROTATE // heads)), "R": r, "t": t, "h": h, "w": w,
                "mode": rng.choice(["half", "half", "interleave"]), "table": rng.choice(["fp32", c["dtype"]])}
    c |= {"page": rng.choice([16, 16, 24, 32, 64, 128]), "order": rng.choice(["token", "head"])}
    if op == "store":
        del c["H"]
        return {**c, "T": max(1, min(_odd_or_tiles(rng, 1, 32768), _MAX_STORE // (c["Hkv"] * c["D"])))}
    sums = rng.random() < 0.25
    row = c["Hkv"] * (c["D"] + 16 + (8 if sums else 0)) + 2
    n = min(_odd_or_tiles(rng, 1, 32768 if sums else 131071), _MAX_ATTEND // row)
    b = max(1, min(_log_int(rng, 1, 128), _MAX_POSITIONS // n, _MAX_ATTEND // (n * row)))
    return {**c, "B": b, "len": n, "ragged": rng.random() < 0.6, "mask": rng.random() < 0.2, "sums": sums}


def _lengths(case):
    """The sequences' lengths, sorted: what the pass works on is the same for every seed."""
    b, n = case["B"], case["len"]
    return [1 + (n - 1) * (i + 1) // b for i in range(b)] if case["ragged"] else [n] * b


def _sections(case):
    return [case["t"], case["h"], case["w"]] if case["h"] else None


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op, dt = case["op"], _DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    state = {"op": op, "dtype": dt}
    if op == "norm":
        t, n = case["T"], case["N"]
        # a residual stream: a few channels are far larger than the others
        loud = torch.where(torch.rand(n, generator=g, device=dev) < 0.004, 20.0, 1.0)
        state["x1"] = (normal(t, n) * 0.5).to(dt)
        state["x2"] = (normal(t, n) * loud).to(dt) if case["residual"] else None
        state["gamma"] = (1.0 + 0.3 * normal(n)).to(dt)
        state["int8"] = case["int8"]
        return state
    if op == "rotate":
        t, h, hkv, d, r = case["T"], case["H"], case["Hkv"], case["D"], case["R"]
        qkv = normal(t, h + 2 * hkv, d).to(dt)                  # what the fused projection leaves behind
        state["query"], state["key"] = qkv[:, :h], qkv[:, h:h + hkv]
        most = 32768
        angle = torch.arange(most, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(r // 2, device=dev, dtype=torch.float64) * 2 / r)
        state["table"] = torch.cat((angle.cos(), angle.sin()), 1).to(_DT[case["table"]])
        state["sections"], state["mode"], state["head"] = _sections(case), case["mode"], d
        if t <= 256:                                            # decode: a token of each sequence, anywhere
            at = torch.randint(0, most, (t,), generator=g, device=dev)
            state["positions"] = at if state["sections"] is None else at.expand(3, t).contiguous()
            return state
        at = torch.arange(t, device=dev) + int(torch.randint(0, most - t + 1, (), generator=g, device=dev))
        if state["sections"] is not None:                       # every other stretch of 1024 tokens is an image of 32 x 32 patches
            inside = torch.arange(t, device=dev) % 1024
            image = torch.arange(t, device=dev) // 1024 % 2 == 1
            first = at - inside
            at = torch.stack((torch.where(image, first, at), torch.where(image, first + inside // 32, at), torch.where(image, first + inside % 32, at)))
        state["positions"] = at
        return state
    hkv, d, page = case["Hkv"], case["D"], case["page"]
    batch = case.get("B", 1)
    n = case["T"] + 3 * page if op == "store" else case["len"]
    width = -(-n // page)                                       # pages of a sequence
    blocks = batch * width + 5

    def cache():
        shape = (blocks, page, hkv) if case["order"] == "token" else (blocks, hkv, page)
        words = torch.zeros(*shape, d // 8, device=dev, dtype=torch.int32)
        if op == "attend":
            for i in range(8):                                  # codes of normally distributed rows
                code = torch.empty(words.shape, device=dev, dtype=torch.float16).normal_(0.0, 2.8, generator=g).round_().clamp_(-8, 7)
                words |= (code.to(torch.int32) & 15) << (4 * i)
        words = words if case["order"] == "token" else words.transpose(1, 2)
        scale = torch.rand(blocks, hkv, page, generator=g, device=dev) * 0.3 + 0.2
        offset = 0.5 + 0.5 * normal(blocks, hkv, page)
        if op == "store":
            scale.zero_(), offset.zero_()
        return words, scale.transpose(1, 2), offset.transpose(1, 2)

    state["key_cache"], state["key_scale"], state["key_offset"] = cache()
    state["value_cache"], state["value_scale"], state["value_offset"] = cache()
    pages = torch.randperm(blocks, generator=g, device=dev)[: batch * width].to(torch.int32).reshape(batch, width)
    if op == "store":
        at = torch.arange(case["T"], device=dev) + page // 2    # a chunk starts anywhere in its first page
        state["slots"] = pages[0][at // page].long() * page + at % page
        kv = normal(case["T"], 2 * hkv, d)
        kv[:, :hkv] *= torch.exp(0.5 * normal(d))               # keys have channels that are larger than others
        kv = kv.to(dt)
        state["key"], state["value"] = kv[:, :hkv], kv[:, hkv:]
        return state
    order = torch.randperm(batch, generator=g, device=dev)
    state["block_table"], state["lens"] = pages, torch.tensor(_lengths(case), dtype=torch.int32, device=dev)[order]
    state["query"] = normal(batch, case["H"], d).to(dt)
    state["mask"] = None
    if case["mask"]:                                            # left-padded prompts, and a few tokens taken back
        spot = torch.arange(width * page, device=dev)
        pad = torch.rand(batch, 1, generator=g, device=dev) * 0.3 * state["lens"][:, None]
        state["mask"] = (spot < pad) | (torch.rand(batch, width * page, generator=g, device=dev) < 0.02)
    state["sums"] = torch.rand(batch, hkv, width * page, generator=g, device=dev) if case["sums"] else None
    return state


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


def _own(s):
    import pytorch_amd as pa
    if s["op"] == "norm":
        if s["int8"]:
            codes, scale, x = pa.npu_add_rms_norm_dynamic_quant(s["x1"], s["x2"], s["gamma"], epsilon=_EPS)
            values = torch.empty(codes.shape, dtype=s["dtype"], device=codes.device)
            return torch.mul(codes, scale[..., None], out=values), scale, x      # (without a residual x has no elements)
        return pa.npu_add_rms_norm(s["x1"], s["x2"], s["gamma"], _EPS)
    if s["op"] == "rotate":
        return pa.npu_mrope(s["positions"], s["query"], s["key"], s["table"], s["head"], mrope_section=s["sections"], rotary_mode=s["mode"])
    params = {name: s[name] for name in ("key_scale", "value_scale", "key_offset", "value_offset")}
    if s["op"] == "store":
        pa.npu_paged_cache_write(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"], **params)
        return pa.npu_paged_cache_read(s["key_cache"], s["value_cache"], s["slots"], **params, dtype=s["dtype"])
    out, lse = pa.npu_paged_decode_attention(s["query"], s["key_cache"], s["value_cache"], s["block_table"], s["lens"], **params,
                                             atten_mask=s["mask"], attn_sums=s["sums"], softmax_lse=True)
    return (out, lse) if s["sums"] is None else (out, lse, s["sums"])


def _plain_norm(s):
    x = s["x1"].float()
    if s["x2"] is not None:
        x = x + s["x2"].float()
    out = x.to(s["dtype"]) if s["x2"] is not None else s["x1"].new_empty(0)
    rstd = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS)
    gamma = s["gamma"].float()
    if not s["int8"]:
        return (x * rstd * gamma).to(s["dtype"]), rstd, out
    u = x * gamma                                               # the factor 1 / rms cancels in the codes
    step = u.abs().amax(-1, keepdim=True)
    step = step / torch.full_like(step, 127.0)                  # (divided, not multiplied by a reciprocal)
    codes = torch.where(step > 0, torch.round(u / step), 0.0).to(torch.int8)
    scale = step * rstd
    return (codes * scale).to(s["dtype"]), scale[..., 0], out


def _plain_rotate(s):
    half = s["table"].shape[1] // 2
    at = s["positions"]
    if s["sections"] is None:
        cos, sin = s["table"][at].float().split(half, 1)        # [tokens, half]
    else:
        cos, sin = s["table"][at].float().split(half, 2)        # [axes, tokens, half]
        cos = torch.cat([c[i] for i, c in enumerate(cos.split(s["sections"], 2))], 1)
        sin = torch.cat([c[i] for i, c in enumerate(sin.split(s["sections"], 2))], 1)
    return tuple(_turn(x, cos[:, None], sin[:, None], s["mode"]) for x in (s["query"], s["key"]))


def _turn(x, cos, sin, mode):
    half = cos.shape[-1]
    f = x[..., : 2 * half].float()
    a, b = f.split(half, -1) if mode == "half" else (f[..., ::2], f[..., 1::2])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((p, q), -1) if mode == "half" else torch.stack((p, q), -1).flatten(-2)
    return torch.cat((turned.to(x.dtype), x[..., 2 * half:]), -1)


def _unpack(words, scale, offset):
    """float32 values [..., 8 * words] of a cache's rows."""
    code = (words[..., None] >> torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)) & 15
    return (((code ^ 8) - 8).flatten(-2).float() + offset[..., None]) * scale[..., None]


def _plain_store(s):
    page = s["key_cache"].shape[1]
    block, spot = s["slots"] // page, s["slots"] % page
    _plain_write(s["key"].float(), s["key_cache"], s["key_scale"], s["key_offset"], block, spot)
    _plain_write(s["value"].float(), s["value_cache"], s["value_scale"], s["value_offset"], block, spot)
    return (_unpack(s["key_cache"][block, spot], s["key_scale"][block, spot], s["key_offset"][block, spot]).to(s["dtype"]),
            _unpack(s["value_cache"][block, spot], s["value_scale"][block, spot], s["value_offset"][block, spot]).to(s["dtype"]))


def _plain_write(x, cache, scales, offsets, block, spot):
    lo, hi = x.amin(-1), x.amax(-1)
    span = hi - lo
    flat = span <= 2.0 ** -120                                  # all values of the row are the same
    steps = torch.full_like(span, 15.0)
    scale = torch.where(flat, 1.0, span / steps)
    offset = torch.where(flat, lo, lo / scale + 8.0)
    code = torch.where(flat[..., None], 0.0, torch.round((x - lo[..., None]) * 15.0 / span[..., None]) - 8.0).to(torch.int32) & 15
    cache[block, spot] = (code.unflatten(-1, (-1, 8)) << torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)).sum(-1, dtype=torch.int32)
    scales[block, spot] = scale
    offsets[block, spot] = offset


def _plain_attend(s):
    q, lens, pages = s["query"], s["lens"], s["block_table"].long()
    batch, heads, d = q.shape
    hkv = s["key_cache"].shape[2]
    k = _unpack(s["key_cache"][pages], s["key_scale"][pages], s["key_offset"][pages]).flatten(1, 2)                   # [B, S, Hkv, D]
    score = torch.matmul(q.float().reshape(batch, hkv, heads // hkv, d), k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    seen = torch.arange(k.shape[1], device=q.device) < lens[:, None]
    if s["mask"] is not None:
        seen = seen & ~s["mask"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    v = _unpack(s["value_cache"][pages], s["value_scale"][pages], s["value_offset"][pages]).flatten(1, 2)
    out = torch.matmul(p, v.transpose(1, 2)).reshape(batch, heads, d).to(q.dtype)
    lse = (top + torch.log(total)).reshape(batch, heads)
    if s["sums"] is None:
        return out, lse
    s["sums"] += p.sum(2)
    return out, lse, s["sums"]


_PLAIN = {"norm": _plain_norm, "rotate": _plain_rotate, "store": _plain_store, "attend": _plain_attend}


def work(case):
    op = case["op"]
    if op == "norm":
        t, n = case["T"], case["N"]
        element = (2 + 2 + 2 if case["residual"] else 2) + (1 + 1 + 2 if case["int8"] else 2)      # codes are written, read and returned as values
        return {"bytes": t * n * element + 4 * t + 2 * n, "flops": t * n * 6}
    hkv, d = case["Hkv"], case["D"]
    if op == "rotate":
        t, r = case["T"], case["R"]
        axes = 3 if case["h"] else 1
        # of the table every row that occurs, of the positions each
        return {"bytes": t * ((case["H"] + hkv) * d * 4 + axes * 8) + min(t, 32768) * r * (4 if case["table"] == "fp32" else 2),
                "flops": t * (case["H"] + hkv) * r * 3}
    row = 2 * hkv * (d // 2 + 8)                                # one token's codes, scales and offsets
    if op == "store":
        return {"bytes": case["T"] * (2 * row + 2 * 2 * hkv * d * 2 + 2 * 8), "flops": case["T"] * hkv * d * 2 * 6}
    tokens, h = sum(_lengths(case)), case["H"]
    return {"bytes": tokens * (row + 4 / case["page"] + (8 * hkv if case["sums"] else 0) + (1 if case["mask"] else 0)) + case["B"] * h * (4 * d + 4),
            "flops": tokens * h * d * 4}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x1"].double() if s["x2"] is None else s["x1"].double() + s["x2"].double()
        out = s["x1"].new_empty(0).double() if s["x2"] is None else x
        y = s["gamma"].double() * x
        norm = (x.pow(2).sum(1, keepdim=True) / case["N"] + _EPS).pow(-0.5)
        y.mul_(norm)
        if not case["int8"]:
            return y, norm, out
        scale = y.abs().max(1, keepdim=True).values / 127.0
        y.div_(scale.clamp(min=1e-300)).round_().mul_(scale)
        return y, scale[:, 0], out
    if case["op"] == "rotate":
        half = case["R"] // 2
        axis = torch.zeros(half, dtype=torch.long) if not case["h"] else torch.tensor([0] * case["t"] + [1] * case["h"] + [2] * case["w"])
        at = s["positions"].reshape(-1, case["T"])[axis.to(s["positions"].device)].t()          # [tokens, half]
        f = torch.arange(half, device=at.device)
        turn = torch.complex(s["table"][at, f].double(), s["table"][at, f + half].double())[:, None]
        outs = []
        for x in (s["query"], s["key"]):
            y = x.double()
            first = f if case["mode"] == "half" else 2 * f
            second = f + half if case["mode"] == "half" else 2 * f + 1
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    if case["op"] == "store":
        outs = []
        for new in (s["key"], s["value"]):
            x = new.double()
            lo = x.min(-1, keepdim=True).values
            span = x.max(-1, keepdim=True).values - lo
            code = (15.0 * (x - lo) / span.clamp(min=1e-300)).round()              # (a value between two codes: the even one)
            outs.append(code * (span / 15.0) + lo)
        return tuple(outs)
    hkv, d, page = case["Hkv"], case["D"], case["page"]
    group = case["H"] // hkv
    table = s["block_table"].long()

    def rows(name, slots):                                      # [heads, n, d] in 64 bits
        block, spot = slots.div(page, rounding_mode="floor"), slots.remainder(page)
        words = s[name + "_cache"][block, spot]                 # [n, heads, words]
        codes = torch.stack([((words << (28 - 4 * i)) >> 28) for i in range(8)], -1).reshape(len(slots), hkv, d).double()
        return ((codes + s[name + "_offset"][block, spot].double()[..., None]) * s[name + "_scale"][block, spot].double()[..., None]).transpose(0, 1).contiguous()

    outs, lses, sums = [], [], None if s["sums"] is None else s["sums"].double()
    for b, n in enumerate(s["lens"].tolist()):
        at = torch.arange(n, device=table.device)
        if s["mask"] is not None:
            at = at[~s["mask"][b, :n]]
        slots = table[b][at.div(page, rounding_mode="floor")] * page + at.remainder(page)
        q = s["query"][b].double().view(hkv, group, d)
        z = torch.bmm(rows("key", slots), q.transpose(1, 2).contiguous()) / math.sqrt(d)        # [heads, n, group]
        lse = torch.logsumexp(z, 1)
        w = torch.exp(z - lse[:, None])
        outs.append(torch.bmm(w.transpose(1, 2).contiguous(), rows("value", slots)).view(-1, d))
        lses.append(lse.reshape(-1))
        if sums is not None:
            sums[b].index_add_(1, at, w.sum(-1))
    got = (torch.stack(outs), torch.stack(lses))
    return got if sums is None else (*got, sums)
