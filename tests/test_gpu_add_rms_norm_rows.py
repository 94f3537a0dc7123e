"""The norms of a row do not depend on what else is in the call, to the last bit: not on the number of rows (a prompt in one piece or in several),
not on where the rows lie."""
import pytest
import torch

from test_gpu_add_rms_norm import EPS, check8, check16, make, pa  # noqa: F401

pytestmark = pytest.mark.gpu


def norms(pa, a, b, g):  # noqa: F811
    return (*pa.npu_add_rms_norm(a, b, g, EPS), *pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=EPS))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [5, 8, 128, 200, 256, 257, 264, 300, 384, 391, 400, 509, 512, 520, 1000, 2048, 4104])
def test_rows_by_themselves(pa, cols, dt):  # noqa: F811
    rows = 4097 if cols <= 1000 else 600
    x1, x2, gamma = make(rows, cols, dt, seed=cols)
    a, b, g = x1.cuda(), x2.cuda(), gamma.cuda()
    whole = norms(pa, a, b, g)
    check16(tuple(t[:50] for t in whole[:3]), x1[:50], x2[:50], gamma)
    check8(tuple(t[:50] for t in whole[3:]), x1[:50], x2[:50], gamma)
    for start, stop in ((0, 1), (0, 17), (3, 600), (1, 4096), (0, 4095), (4, 4096)):
        part = norms(pa, a[start:stop], b[start:stop], g)
        for got, want in zip(part, whole):
            assert torch.equal(got, want[start:stop]), (start, stop)
    apart = torch.cat((a[:, :1], a), 1)[:, 1:]             # rows on odd addresses
    for got, want in zip(norms(pa, apart, b, g), whole):
        assert torch.equal(got, want)
