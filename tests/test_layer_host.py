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
