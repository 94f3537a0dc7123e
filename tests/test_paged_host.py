"""The paged cache's operators without a GPU: names, schemas, shapes of their results and what they refuse."""
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


def cache(dtype=BF, blocks=10, page=16, heads=2, dim=64):
    c = {"key_cache": m(blocks, page, heads, dim, dtype=dtype), "value_cache": m(blocks, page, heads, dim, dtype=dtype)}
    if dtype == I8:
        c |= {"key_scale": m(blocks, page, heads, dtype=F), "value_scale": m(blocks, page, heads, dtype=F)}
    return c


def test_names_and_schemas(pa):
    for name in ("npu_paged_cache_write", "npu_paged_cache_read", "npu_paged_decode_attention", "npu_paged_cache_evict"):
        assert name in pa.__all__ and getattr(pa, name) is getattr(torch.ops.npu, name)
    s = str(torch.ops.npu.npu_paged_cache_write.default._schema)
    assert "Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slots" in s and s.endswith("-> ()")
    s = str(torch.ops.npu.npu_paged_decode_attention.default._schema)
    assert "Tensor block_table, Tensor context_lens, *" in s and "Tensor(a!)? attn_sums=None, bool softmax_lse=False" in s


def test_shapes(pa):
    pa.npu_paged_cache_write(m(5, 2, 64), m(5, 2, 64), **cache(), slots=m(5, dtype=I64))
    k, v = pa.npu_paged_cache_read(**cache(), slots=m(7, dtype=I32))
    assert k.shape == v.shape == (7, 2, 64) and k.dtype == v.dtype == BF
    k, v = pa.npu_paged_cache_read(**cache(I8), slots=m(7, dtype=I32), dtype=HF)
    assert k.dtype == v.dtype == HF
    assert pa.npu_paged_cache_read(**cache(I8), slots=m(0, dtype=I32))[0].dtype == BF
    args = {"block_table": m(3, 4, dtype=I32), "context_lens": m(3, dtype=I64)}
    out, lse = pa.npu_paged_decode_attention(m(3, 8, 64, dtype=HF), **cache(I8), **args, softmax_lse=True)
    assert out.shape == (3, 8, 64) and out.dtype == HF and lse.shape == (3, 8) and lse.dtype == F
    out, lse = pa.npu_paged_decode_attention(m(3, 8, 64), **cache(), **args, atten_mask=m(3, 64, dtype=torch.bool), attn_sums=m(3, 2, 64, dtype=F))
    assert out.shape == (3, 8, 64) and lse.shape == (0,)
    lens, sums, pos = pa.npu_paged_cache_evict(**cache(), **args, attn_sums=m(3, 2, 64, dtype=F), positions=m(3, 2, 64, dtype=I32), keep=40, recent=8)
    assert lens.shape == (3,) and lens.dtype == I32 and sums.shape == pos.shape == (3, 2, 64) and sums.dtype == F and pos.dtype == I32


def test_no_cpu_implementation(pa):
    c = torch.zeros(2, 16, 1, 8, dtype=BF)
    with pytest.raises(NotImplementedError, match="CPU"):
        pa.npu_paged_cache_read(c, c, torch.zeros(1, dtype=I64))


WRITE = dict(key=m(5, 2, 64), value=m(5, 2, 64), slots=m(5, dtype=I64))
ATTEND = dict(query=m(3, 8, 64), block_table=m(3, 4, dtype=I32), context_lens=m(3, dtype=I32))
EVICT = dict(block_table=m(3, 4, dtype=I32), context_lens=m(3, dtype=I32), attn_sums=m(3, 2, 64, dtype=F), positions=m(3, 2, 64, dtype=I32), keep=40,
             recent=8)


@pytest.mark.parametrize("op,change,text", [
    ("write", dict(key_cache=m(10, 16, 2, dtype=BF)), "num_blocks, block_size, kv_heads, head_dim"),
    ("write", dict(value_cache=m(10, 16, 2, 63)), "the same shape"),
    ("write", dict(value_cache=m(10, 16, 2, 64, dtype=HF)), "the same dtype"),
    ("write", dict(key_cache=m(10, 16, 2, 64, dtype=F), value_cache=m(10, 16, 2, 64, dtype=F)), "bfloat16, float16 or int8"),
    ("write", dict(key_cache=m(10, 16, 2, 64, dtype=I8), value_cache=m(10, 16, 2, 64, dtype=I8)), "needs key_scale and value_scale"),
    ("write", dict(key_scale=m(10, 16, 2, dtype=F), value_scale=m(10, 16, 2, dtype=F)), "belong to an int8 cache"),
    ("write", dict(cache(I8), key_scale=m(10, 16, 3, dtype=F)), "must be float32 of shape"),
    ("write", dict(cache(I8), value_scale=m(10, 16, 2, dtype=BF)), "must be float32 of shape"),
    ("write", dict(key_cache=m(10, 16, 64, 2).transpose(2, 3)), "last dimension of key_cache"),
    ("write", dict(key_cache=m(1, 16, 2, 64).expand(10, 16, 2, 64)), "share memory"),
    ("write", dict(key_cache=m(0, 16, 2, 64), value_cache=m(0, 16, 2, 64)), "the cache is empty"),
    ("write", dict(slots=m(5, 1, dtype=I64)), "slots must be"),
    ("write", dict(slots=m(5, dtype=F)), "slots must be"),
    ("write", dict(slots=m(4, dtype=I64)), "key must have shape"),
    ("write", dict(key=m(5, 2, 64, dtype=HF)), "both be bfloat16 or both float16"),
    ("write", dict(key=m(5, 2, 64, dtype=HF), value=m(5, 2, 64, dtype=HF)), "the cache is"),
    ("write", dict(key=m(5, 3, 64)), "key must have shape"),
    ("write", dict(value=m(5, 2, 32)), "key and value must have the same shape"),
    ("read", dict(dtype=HF), "dtype must be that of the cache"),
    ("read", dict(cache(I8), dtype=F), "torch.bfloat16 or torch.float16"),
    ("attend", dict(query=m(3, 8, 64, dtype=F)), "query must be bfloat16 or float16"),
    ("attend", dict(query=m(3, 8, 64, dtype=HF)), "the cache is"),
    ("attend", dict(query=m(3, 8, 32)), "query must have shape"),
    ("attend", dict(query=m(3, 7, 64)), "not a multiple"),
    ("attend", dict(cache(dim=264), query=m(3, 8, 264)), "at most 256"),
    ("attend", dict(block_table=m(2, 4, dtype=I32)), "block_table must be"),
    ("attend", dict(block_table=m(3, 4, dtype=F)), "block_table must be"),
    ("attend", dict(context_lens=m(4, dtype=I32)), "context_lens must be"),
    ("attend", dict(atten_mask=m(3, 63, dtype=torch.bool)), "atten_mask must be bool"),
    ("attend", dict(atten_mask=m(3, 64, dtype=F)), "atten_mask must be bool"),
    ("attend", dict(attn_sums=m(3, 8, 64, dtype=F)), "attn_sums must be float32"),
    ("attend", dict(attn_sums=m(3, 64, 2, dtype=F).transpose(1, 2)), "last dimension of attn_sums"),
    ("attend", dict(attn_sums=m(1, 2, 64, dtype=F).expand(3, 2, 64)), "share memory"),
    ("evict", dict(attn_sums=m(3, 2, 60, dtype=F)), "attn_sums must be float32"),
    ("evict", dict(positions=m(3, 2, 64, dtype=I64)), "positions must be int32"),
    ("evict", dict(keep=4), "recent <= keep"),
    ("evict", dict(recent=-1), "recent <= keep"),
])
def test_refusals(pa, op, change, text):
    fn, base = {"write": (pa.npu_paged_cache_write, WRITE), "read": (pa.npu_paged_cache_read, dict(slots=m(5, dtype=I64))),
                "attend": (pa.npu_paged_decode_attention, ATTEND), "evict": (pa.npu_paged_cache_evict, EVICT)}[op]
    with pytest.raises(RuntimeError, match=text):
        fn(**{**cache(), **base, **change})


class Descriptor(ctypes.Structure):
    _fields_ = [("key", ctypes.c_void_p), ("value", ctypes.c_void_p), ("key_scale", ctypes.c_void_p), ("value_scale", ctypes.c_void_p),
                ("dtype", ctypes.c_int), ("num_blocks", ctypes.c_int64), ("block_size", ctypes.c_int64), ("kv_heads", ctypes.c_int64),
                ("head_dim", ctypes.c_int64), ("key_stride", ctypes.c_int64 * 3), ("value_stride", ctypes.c_int64 * 3),
                ("key_scale_stride", ctypes.c_int64 * 3), ("value_scale_stride", ctypes.c_int64 * 3)]


def descriptor(**change):
    s = (ctypes.c_int64 * 3)(16 * 2 * 64, 2 * 64, 64)
    f = dict(key=4096, value=8192, dtype=0, num_blocks=10, block_size=16, kv_heads=2, head_dim=64, key_stride=s, value_stride=s)
    return Descriptor(**{**f, **change})


def test_c_entries_refuse_on_the_host():
    """Every call here returns before it could launch anything."""
    lib = ctypes.CDLL(os.path.join(ROOT, "pytorch_amd", "csrc", "libmi355_quant.so"))
    vp, i64 = ctypes.c_void_p, ctypes.c_int64
    two = (i64 * 2)(128, 64)
    p = vp(4096)

    def write(d, key=p, dtype=0, slots=p, slots_dtype=5, tokens=3):
        return lib.mi355_paged_cache_write(ctypes.byref(d) if d is not None else None, key, two, p, two, dtype, slots, slots_dtype, i64(tokens), None)

    assert write(None) == -1
    assert write(descriptor(key=None)) == -1
    assert write(descriptor(dtype=2)) == -1                         # float32
    assert write(descriptor(dtype=4)) == -1                         # int8 without scales
    assert write(descriptor(key_scale=4096, value_scale=4096)) == -1
    assert write(descriptor(num_blocks=0)) == -1
    assert write(descriptor(num_blocks=2 ** 31)) == -2
    assert write(descriptor(key=4097)) == -3
    assert write(descriptor(), dtype=1) == -1                       # another type than the cache's
    assert write(descriptor(), key=None) == -1
    assert write(descriptor(), slots_dtype=0) == -1
    assert write(descriptor(), slots=vp(4100)) == -3
    assert write(descriptor(), tokens=-1) == -1
    assert write(descriptor(), tokens=2 ** 31) == -2
    assert write(descriptor(), tokens=0) == 0

    lib.mi355_paged_decode_attention_workspace.restype = ctypes.c_size_t
    need = lib.mi355_paged_decode_attention_workspace(i64(3), i64(8), i64(2), i64(64), i64(4), i64(16), 0)
    assert 0 < need < lib.mi355_paged_decode_attention_workspace(i64(3), i64(8), i64(2), i64(64), i64(4), i64(16), 1)
    assert lib.mi355_paged_decode_attention_workspace(i64(3), i64(7), i64(2), i64(64), i64(4), i64(16), 0) == 0

    def attend(d, q=p, q_dtype=0, batch=3, heads=8, table=p, ws=p, bytes_=need, lens=p, dims=4):
        return lib.mi355_paged_decode_attention(ctypes.byref(d), q, q_dtype, i64(512), i64(64), p, None, i64(batch), i64(heads), table, i64(4), i64(dims),
                                                lens, ctypes.c_float(0.125), None, i64(0), None, i64(0), i64(0), ws, ctypes.c_size_t(bytes_), None)

    assert attend(descriptor(), q=None) == -1 and attend(descriptor(), table=None) == -1 and attend(descriptor(), lens=None) == -1
    assert attend(descriptor(), heads=7) == -1 and attend(descriptor(), q_dtype=1) == -1 and attend(descriptor(), batch=-1) == -1
    assert attend(descriptor(), bytes_=need - 1) == -4 and attend(descriptor(), ws=None) == -4
    assert attend(descriptor(), ws=vp(4104)) == -3 and attend(descriptor(), q=vp(4097)) == -3
    assert attend(descriptor(head_dim=257)) == -2 and attend(descriptor(), dims=2 ** 28) == -2
    assert attend(descriptor(), batch=0) == 0

    lib.mi355_paged_cache_evict_workspace.restype = ctypes.c_size_t
    need = lib.mi355_paged_cache_evict_workspace(i64(3), i64(2), i64(4), i64(16), i64(40))

    def evict(d, keep=40, recent=8, batch=3, sums=p, ws=p, bytes_=need):
        return lib.mi355_paged_cache_evict(ctypes.byref(d), p, i64(4), i64(4), p, i64(batch), sums, i64(128), i64(64), p, i64(128), i64(64), i64(keep),
                                           i64(recent), p, p, p, ws, ctypes.c_size_t(bytes_), None)

    assert evict(descriptor(), keep=-1) == -1 and evict(descriptor(), recent=41) == -1 and evict(descriptor(), sums=None) == -1
    assert evict(descriptor(), bytes_=need - 1) == -4 and evict(descriptor(), sums=vp(4098)) == -3
    assert evict(descriptor(), batch=0) == 0


def test_paged_kv_cache_arguments_and_shapes():
    from pytorch_amd.contrib.module import PagedKVCache

    c = PagedKVCache(3, 100, 2, 64, block_size=16, budget=90, quantized=True)
    assert c.capacity == 112 and c.recent == 22
    assert c.key_cache.shape == (21, 16, 2, 64) and c.key_cache.dtype == torch.int8 and c.key_cache.stride() == (2048, 64, 1024, 1)
    assert c.key_scale.shape == (21, 16, 2) and c.value_scale.dtype == torch.float32
    assert c.block_table.shape == (3, 7) and c.attn_sums.shape == c.positions.shape == (3, 2, 112)
    c = PagedKVCache(1, 5, 1, 8, dtype=torch.float16)
    assert c.attn_sums is None and c.key_scale is None and c.value_cache.dtype == torch.float16 and c.capacity == 64
    for wrong in (dict(batch=0), dict(dtype=torch.float32), dict(budget=112), dict(budget=0), dict(recent=5), dict(budget=50, recent=51)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(batch=3, max_tokens=100, kv_heads=2, head_dim=64, block_size=16), **wrong})
