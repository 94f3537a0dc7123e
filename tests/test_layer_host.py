"""npu_add_rms_norm, npu_add_rms_norm_dynamic_quant and npu_mrope without a GPU: names, schemas, shapes and what they refuse."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, HF, F, I8, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32, torch.int64


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


def m(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_names_and_schemas(pa):
    for name in ("npu_add_rms_norm", "npu_add_rms_norm_dynamic_quant", "npu_mrope"):
        assert name in pa.__all__ and getattr(pa, name) is getattr(torch.ops.npu, name)
    assert "Tensor x1, Tensor? x2, Tensor gamma, float epsilon=" in str(torch.ops.npu.npu_add_rms_norm.default._schema)
    assert "Tensor x1, Tensor? x2, Tensor gamma, *, float epsilon=" in str(torch.ops.npu.npu_add_rms_norm_dynamic_quant.default._schema)
    s = str(torch.ops.npu.npu_mrope.default._schema)
    assert "Tensor positions, Tensor query, Tensor key, Tensor cos_sin_cache, int head_size, *, int[]? mrope_section=None" in s


@pytest.mark.parametrize("shape", [(5, 64), (2, 3, 64), (64,), (0, 64)])
def test_norm_shapes(pa, shape):
    for x2 in (m(*shape), None):
        y, rstd, x = pa.npu_add_rms_norm(m(*shape), x2, m(64))
        assert y.shape == shape and y.dtype == BF and rstd.shape == (*shape[:-1], 1) and rstd.dtype == F
        assert x.dtype == BF and x.shape == (shape if x2 is not None else (0,))
        y, scale, x = pa.npu_add_rms_norm_dynamic_quant(m(*shape), x2, m(64, dtype=F), epsilon=1e-5)
        assert y.shape == shape and y.dtype == I8 and scale.shape == shape[:-1] and scale.dtype == F
        assert x.dtype == BF and x.shape == (shape if x2 is not None else (0,))


ROPE = dict(positions=m(7, dtype=I64), query=m(7, 8, 64), key=m(7, 2, 64), cos_sin_cache=m(100, 64, dtype=F), head_size=64)


def test_rope_shapes(pa):
    q, k = pa.npu_mrope(**ROPE)
    assert q.shape == (7, 8, 64) and k.shape == (7, 2, 64) and q.dtype == k.dtype == BF
    q, k = pa.npu_mrope(m(3, 7, dtype=I32), m(7, 512), m(7, 128), m(100, 32), 64, mrope_section=[4, 6, 6], rotary_mode="interleave")
    assert q.shape == (7, 512) and k.shape == (7, 128)
    q, k = pa.npu_mrope(**{**ROPE, "positions": m(1, 7, dtype=I64), "mrope_section": (32,)})
    assert q.shape == (7, 8, 64)


def test_no_cpu_implementation(pa):
    x = torch.zeros(4, 8, dtype=BF)
    with pytest.raises(NotImplementedError, match="CPU"):
        pa.npu_add_rms_norm(x, x, torch.ones(8, dtype=BF))
    with pytest.raises(NotImplementedError, match="CPU"):
        pa.npu_mrope(torch.zeros(4, dtype=I64), x, x, torch.zeros(4, 8), 8)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("change,text", [
    (dict(x1=m(5, 64, dtype=F)), "x1 must be bfloat16 or float16"),
    (dict(x1=m(5, 0), x2=None, gamma=m(0)), "not empty"),
    (dict(x2=m(5, 64, dtype=HF)), "the same dtype"),
    (dict(x2=m(5, 32)), "the same shape"),
    (dict(x2=m(1, 64)), "the same shape"),
    (dict(gamma=m(64, dtype=HF)), "gamma must be float32 or have the dtype of x1"),
    (dict(gamma=m(32)), "gamma must have shape"),
    (dict(gamma=m(1, 64)), "gamma must have shape"),
    (dict(epsilon=-1.0), "epsilon must not be negative"),
    (dict(epsilon=float("nan")), "epsilon must not be negative"),
])
def test_norm_refusals(pa, int8, change, text):
    fn = pa.npu_add_rms_norm_dynamic_quant if int8 else pa.npu_add_rms_norm
    with pytest.raises(RuntimeError, match=text):
        fn(**{**dict(x1=m(5, 64), x2=m(5, 64), gamma=m(64)), **change})


@pytest.mark.parametrize("change,text", [
    (dict(query=m(7, 8, 64, dtype=F)), "both be bfloat16 or both float16"),
    (dict(key=m(7, 2, 64, dtype=HF)), "both be bfloat16 or both float16"),
    (dict(query=m(7, 8, 32)), "query must have shape"),
    (dict(key=m(7, 100)), "key must have shape"),
    (dict(key=m(6, 2, 64)), "the same number of tokens"),
    (dict(query=m(7, 65536, 1), key=m(7, 2, 1), head_size=1), "at most 65535 heads"),
    (dict(head_size=0), "head_size must be"),
    (dict(cos_sin_cache=m(100, 64, dtype=HF)), "cos_sin_cache must be float32"),
    (dict(cos_sin_cache=m(100, 66, dtype=F)), "cos_sin_cache must have shape"),
    (dict(cos_sin_cache=m(100, 63, dtype=F)), "cos_sin_cache must have shape"),
    (dict(cos_sin_cache=m(100, 0, dtype=F)), "cos_sin_cache must have shape"),
    (dict(rotary_mode="quarter"), "rotary_mode must be"),
    (dict(positions=m(7, dtype=F)), "positions must be int32 or int64"),
    (dict(positions=m(6, dtype=I64)), "positions must have shape"),
    (dict(positions=m(3, 7, dtype=I64)), "mrope_section says"),
    (dict(positions=m(3, 7, dtype=I64), mrope_section=[16, 16]), "positions must have shape"),
    (dict(positions=m(3, 7, dtype=I64), mrope_section=[8, 8, 8]), "add up to half"),
    (dict(positions=m(3, 7, dtype=I64), mrope_section=[40, -16, 8]), "must be between 0"),
    (dict(positions=m(3, 7, dtype=I64), mrope_section=[]), "between 1 and 4 axes"),
    (dict(positions=m(5, 7, dtype=I64), mrope_section=[8, 8, 8, 4, 4]), "between 1 and 4 axes"),
])
def test_rope_refusals(pa, change, text):
    with pytest.raises(RuntimeError, match=text):
        pa.npu_mrope(**{**ROPE, **change})


def test_c_entries_refuse_before_they_launch():
    """Arguments that no kernel may see come back as a status; nothing here needs a GPU."""
    lib = ctypes.CDLL(os.path.join(ROOT, "pytorch_amd", "csrc", "libmi355_quant.so"))
    p, i, f = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
    ok, bad, unsupported, alignment = 0, -1, -2, -3

    def norm(fn=lib.mi355_add_rms_norm, x1=64, x2=64, dtype=0, gamma=64, gamma_dtype=0, y=64, stat=64, x=64, rows=1, cols=64, eps=1e-6):
        return fn(p(x1), p(x2), dtype, p(gamma), gamma_dtype, p(y), p(stat), p(x), i(rows), i(cols), i(cols), i(cols), f(eps), None)

    quant = lib.mi355_add_rms_norm_dynamic_quant
    assert norm(rows=0) == ok and norm(cols=0) == ok and norm(quant, rows=0) == ok
    for change in (dict(x1=None), dict(gamma=None), dict(y=None), dict(x=None), dict(x2=None), dict(dtype=2), dict(gamma_dtype=1), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(rows=-1), dict(cols=-1), dict(fn=quant, stat=None)):
        assert norm(**change) == bad, change
    assert norm(cols=1 << 31) == unsupported
    for change in (dict(x1=65), dict(x2=65), dict(x=65), dict(gamma=65), dict(gamma=66, gamma_dtype=2), dict(y=65), dict(stat=66)):
        assert norm(**change) == alignment, change

    def rope(pos=64, pos_type=5, axes=1, sections=None, q=64, heads=2, k=64, kv=1, dtype=0, table=64, table_type=2, positions=10, tokens=3, dim=64, rot=64,
             qo=64, ko=64):
        stride = (i * 2)(256, 64)
        sections = None if sections is None else (i * len(sections))(*sections)
        return lib.mi355_mrope(p(pos), pos_type, i(3), i(1), i(axes), sections, p(q), stride, i(heads), p(k), stride, i(kv), dtype, p(table), table_type,
                               i(64), i(positions), i(tokens), i(dim), i(rot), 0, p(qo), p(ko), None)

    assert rope(tokens=0) == ok and rope(heads=0, kv=0) == ok
    for change in (dict(pos=None), dict(pos_type=0), dict(axes=0), dict(axes=2), dict(axes=2, sections=(16, 15)), dict(axes=2, sections=(40, -8)),
                   dict(axes=2, sections=(1 << 62, 1 << 62)), dict(q=None), dict(k=None), dict(dtype=2), dict(table=None), dict(table_type=1), dict(tokens=-1),
                   dict(dim=32), dict(rot=63), dict(rot=0), dict(qo=None), dict(ko=None), dict(positions=-1)):
        assert rope(**change) == bad, change
    for change in (dict(axes=5, sections=(8, 8, 8, 4, 4)), dict(heads=65536), dict(dim=65552)):
        assert rope(**change) == unsupported, change
    for change in (dict(pos=68), dict(q=65), dict(k=65), dict(table=66), dict(qo=65), dict(ko=65)):
        assert rope(**change) == alignment, change


# ------------------------------------------------------------------------------------------------ the 4-bit paged cache

def cache4(blocks=10, page=16, heads=2, dim=64):
    c = {name: m(blocks, page, heads, dim // 8, dtype=I32) for name in ("key_cache", "value_cache")}
    return c | {name: m(blocks, page, heads, dtype=F) for name in ("key_scale", "value_scale", "key_offset", "value_offset")}


SLOTS = m(5, dtype=I64)
TABLE = dict(block_table=m(3, 4, dtype=I32), context_lens=m(3, dtype=I32))


def test_cache4_shapes(pa):
    pa.npu_paged_cache_write(m(5, 2, 64), m(5, 2, 64), slots=SLOTS, **cache4())
    k, v = pa.npu_paged_cache_read(slots=SLOTS, **cache4())
    assert k.shape == v.shape == (5, 2, 64) and k.dtype == v.dtype == BF
    assert pa.npu_paged_cache_read(slots=SLOTS, dtype=HF, **cache4())[0].dtype == HF
    out, lse = pa.npu_paged_decode_attention(m(3, 8, 64, dtype=HF), **cache4(), **TABLE, softmax_lse=True)
    assert out.shape == (3, 8, 64) and out.dtype == HF and lse.shape == (3, 8)
    lens, sums, pos = pa.npu_paged_cache_evict(**cache4(), **TABLE, attn_sums=m(3, 2, 64, dtype=F), positions=m(3, 2, 64, dtype=I32), keep=40, recent=8)
    assert lens.shape == (3,) and sums.shape == pos.shape == (3, 2, 64)


@pytest.mark.parametrize("op", ["write", "read", "attend", "evict"])
@pytest.mark.parametrize("change,text", [
    (dict(key_offset=None), "needs key_scale, value_scale, key_offset and value_offset"),
    (dict(value_scale=None), "needs key_scale, value_scale, key_offset and value_offset"),
    (dict(key_offset=m(10, 16, 2, dtype=BF)), "key_offset and value_offset must be float32"),
    (dict(value_offset=m(10, 16, 2, 1, dtype=F)), "key_offset and value_offset must be float32"),
    (dict(value_scale=m(10, 16, 3, dtype=F)), "key_scale and value_scale must be float32"),
    (dict(value_cache=m(10, 16, 2, 8, dtype=I8)), "the same dtype"),
    (dict(key_cache=m(10, 16, 2, 64), value_cache=m(10, 16, 2, 64)), "belong to an int8 cache or a 4-bit one"),
    (dict(key_cache=m(10, 16, 2, 64), value_cache=m(10, 16, 2, 64), key_scale=None, value_scale=None), "belong to a 4-bit cache"),
    (dict(key_cache=m(10, 16, 2, 64, dtype=I8), value_cache=m(10, 16, 2, 64, dtype=I8)), "belong to a 4-bit cache"),
    (dict(key_cache=m(10, 16, 2, 8, dtype=I64), value_cache=m(10, 16, 2, 8, dtype=I64)), "4-bit codes"),
])
def test_cache4_refusals(pa, op, change, text):
    fn, more = {"write": (pa.npu_paged_cache_write, dict(key=m(5, 2, 64), value=m(5, 2, 64), slots=SLOTS)), "read": (pa.npu_paged_cache_read, dict(slots=SLOTS)),
                "attend": (pa.npu_paged_decode_attention, dict(query=m(3, 8, 64), **TABLE)),
                "evict": (pa.npu_paged_cache_evict, dict(attn_sums=m(3, 2, 64, dtype=F), positions=m(3, 2, 64, dtype=I32), keep=40, recent=8, **TABLE))}[op]
    with pytest.raises(RuntimeError, match=text):
        fn(**{**cache4(), **more, **change})


def test_cache4_widths_and_memory(pa):
    with pytest.raises(RuntimeError, match="key must have shape"):
        pa.npu_paged_cache_write(m(5, 2, 8), m(5, 2, 8), slots=SLOTS, **cache4())
    with pytest.raises(RuntimeError, match="query must have shape"):
        pa.npu_paged_decode_attention(m(3, 8, 8), **cache4(), **TABLE)
    with pytest.raises(RuntimeError, match="at most 256"):
        pa.npu_paged_decode_attention(m(3, 8, 264), **cache4(dim=264), **TABLE)
    with pytest.raises(RuntimeError, match="share memory"):
        pa.npu_paged_cache_write(m(5, 2, 64), m(5, 2, 64), slots=SLOTS, **{**cache4(), "value_offset": m(1, 16, 2, dtype=F).expand(10, 16, 2)})


class Descriptor4(ctypes.Structure):
    _fields_ = [("key", ctypes.c_void_p), ("value", ctypes.c_void_p), ("key_scale", ctypes.c_void_p), ("value_scale", ctypes.c_void_p),
                ("dtype", ctypes.c_int), ("num_blocks", ctypes.c_int64), ("block_size", ctypes.c_int64), ("kv_heads", ctypes.c_int64),
                ("head_dim", ctypes.c_int64), ("key_stride", ctypes.c_int64 * 3), ("value_stride", ctypes.c_int64 * 3),
                ("key_scale_stride", ctypes.c_int64 * 3), ("value_scale_stride", ctypes.c_int64 * 3), ("key_offset", ctypes.c_void_p),
                ("value_offset", ctypes.c_void_p), ("key_offset_stride", ctypes.c_int64 * 3), ("value_offset_stride", ctypes.c_int64 * 3)]


@pytest.mark.parametrize("change,status", [
    (dict(), 0), (dict(key_offset=None), -1), (dict(value_offset=None), -1), (dict(key_scale=None), -1), (dict(head_dim=60), -1), (dict(dtype=5), -1),
    (dict(key=66), -3), (dict(value_offset=66), -3), (dict(key_scale=65), -3), (dict(num_blocks=1 << 30), -2)])
def test_cache4_descriptor(change, status):
    """Without tokens nothing is launched, so that the descriptor's own checks answer."""
    lib = ctypes.CDLL(os.path.join(ROOT, "pytorch_amd", "csrc", "libmi355_quant.so"))
    three = (ctypes.c_int64 * 3)(16 * 2 * 8, 2 * 8, 8)
    one = (ctypes.c_int64 * 3)(32, 1, 16)
    d = Descriptor4(**{**dict(key=64, value=64, key_scale=64, value_scale=64, dtype=6, num_blocks=10, block_size=16, kv_heads=2, head_dim=64, key_stride=three,
                              value_stride=three, key_scale_stride=one, value_scale_stride=one, key_offset=64, value_offset=64, key_offset_stride=one,
                              value_offset_stride=one), **change})
    got = lib.mi355_paged_cache_write(ctypes.byref(d), None, None, None, None, 0, None, 5, ctypes.c_int64(0), None)
    assert got == status


def test_module_refusals():
    from pytorch_amd.contrib.module import PagedKVCache
    for more, text in ((dict(bits=4), "quantized=True"), (dict(bits=3, quantized=True), "bits should be"), (dict(bits=4, quantized=True, head_dim=60), "multiple of 8")):
        with pytest.raises(ValueError, match=text):
            PagedKVCache(**{**dict(batch=1, max_tokens=8, kv_heads=1, head_dim=64), **more})
