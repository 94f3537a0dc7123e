"""npu_add_rms_norm and npu_add_rms_norm_dynamic_quant on the GPU against their formulas in 64 bits on the CPU.

Tolerances.  u is half a step of the 16-bit type (2^-8 bfloat16, 2^-11 float16).  A float32 sum of N squares, added in parts of at
most 48 terms a thread (rows of up to 32768) and 22 partial sums, is off by at most 70 * 2^-24 of itself; its root halves that, and
division, addition, root and reciprocal add 4 * 2^-24: rstd is off by less than 2^-18 of itself.  y has 3 more roundings in float32 and one
to 16 bits.  The sum x is one float32 addition and one rounding, which the CPU does the same way: equal bits.  Codes follow
float32 operations that the CPU does the same way (an addition, a product, a maximum and two divisions): equal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}            # the step of subnormal numbers
EPS = 1e-6


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


def make(rows, cols, dt, seed=0, gamma=None, residual=True):
    g = torch.Generator().manual_seed(seed)
    loud = torch.where(torch.rand(cols, generator=g) < 0.01, 30.0, 1.0)
    x1 = torch.randn(rows, cols, generator=g).to(dt)
    x2 = (torch.randn(rows, cols, generator=g) * loud).to(dt) if residual else None
    return x1, x2, (1 + 0.3 * torch.randn(cols, generator=g)).to(gamma or dt)


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def check16(got, x1, x2, gamma, eps=EPS):
    y, rstd, x = (t.cpu() for t in got)
    dt = x1.dtype
    s = x1.double() if x2 is None else x1.double() + x2.double()
    want = 1 / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    assert rstd.shape == (*x1.shape[:-1], 1)
    assert bool(((rstd.double() - want).abs() <= 2.0 ** -18 * want).all())
    ref = s * want * gamma.double()
    assert y.dtype == dt and y.shape == x1.shape
    assert bool(((y.double() - ref).abs() <= (U[dt] + 2.0 ** -17) * ref.abs() + TINY[dt]).all())
    check_sum(x, x1, x2)


def check_sum(x, x1, x2):
    if x2 is None:
        assert x.shape == (0,) and x.dtype == x1.dtype
    else:
        assert torch.equal(x.cpu(), (x1.float() + x2.float()).to(x1.dtype))


def codes_of(x1, x2, gamma):
    u = x1.float() if x2 is None else x1.float() + x2.float()
    u = u * gamma.float()
    step = u.abs().amax(-1, keepdim=True)
    step = step / torch.full_like(step, 127.0)
    return torch.where(step > 0, torch.round(u / step), 0.0).to(torch.int8), step[..., 0]


def check8(got, x1, x2, gamma, eps=EPS):
    y, scale, x = (t.cpu() for t in got)
    codes, step = codes_of(x1, x2, gamma)
    assert y.dtype == torch.int8 and torch.equal(y, codes)
    s = x1.double() if x2 is None else x1.double() + x2.double()
    want = step.double() / (s.square().mean(-1) + eps).sqrt()
    assert scale.shape == x1.shape[:-1] and bool(((scale.double() - want).abs() <= 2.0 ** -18 * want).all())
    check_sum(x, x1, x2)


def check(pa, x1, x2, gamma, eps=EPS):
    a, b, g = cuda(x1, x2, gamma)
    check16(pa.npu_add_rms_norm(a, b, g, eps), x1, x2, gamma, eps)
    check8(pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=eps), x1, x2, gamma, eps)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 63, 64, 65, 511, 512, 520, 1000, 2047, 2048, 2056, 4095, 4096, 4097, 5128, 8191, 8192, 8200, 16384, 16392, 16385,
                                  32768])
def test_widths(pa, cols, dt):
    for rows, residual in ((1, True), (5, True), (6, False)):
        check(pa, *make(rows, cols, dt, seed=cols, residual=residual))


@pytest.mark.parametrize("cols", [32769, 40000, 70001])
def test_rows_longer_than_the_registers(pa, cols):
    # 72 terms a thread at 70001 columns: 100 * 2^-24 of the sum, still below 2^-17 and 2^-18 of its root
    for dt in U:
        check(pa, *make(3, cols, dt, seed=cols))
        check(pa, *make(2, cols, dt, seed=cols, residual=False))


@pytest.mark.parametrize("rows", [1, 3, 4, 64, 255, 256, 257, 1000, 3001])
@pytest.mark.parametrize("cols", [128, 1024, 4096])
def test_rows(pa, rows, cols):
    check(pa, *make(rows, cols, torch.bfloat16, seed=rows))


@pytest.mark.parametrize("rows", [5, 17, 4095, 4099])
@pytest.mark.parametrize("cols", [3, 8, 72, 100, 128, 129, 250, 256, 257, 300, 511, 512])
def test_rows_that_share_a_wavefront(pa, rows, cols):
    check(pa, *make(rows, cols, torch.bfloat16 if cols % 3 else torch.float16, seed=rows + cols))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [77, 512, 4096])
def test_float32_gamma(pa, cols, dt):
    """Products of any significand: their quotients by the step are rounded once."""
    check(pa, *make(200, cols, dt, seed=cols, gamma=torch.float32))


@pytest.mark.parametrize("magnitude", [2.0 ** -120, 1e-30, 2.0 ** -60, 1e-3, 1e4, 1e15])
def test_magnitudes(pa, magnitude):
    """Steps inside and outside the range in which codes go by the reciprocal."""
    x1, x2, gamma = make(16, 640, torch.bfloat16, seed=3)
    x1, x2 = x1 * magnitude, x2 * magnitude
    check(pa, x1, x2, gamma, eps=0.0 if 1e-12 < magnitude else EPS)


def test_ties(pa):
    """Quotients that lie exactly between two codes go to the even one."""
    x1 = torch.zeros(2, 256)
    x1[:, 0] = 254.0                                       # a step of 2
    x1[0, 1:] = torch.arange(255.0) - 127.0
    x1[1, 1:] = -x1[0, 1:]
    for dt in U:
        x, gamma = x1.to(dt), torch.ones(256, dtype=dt)
        check(pa, x, None, gamma)
        check(pa, x, torch.zeros_like(x), gamma)


@pytest.mark.parametrize("view", ["rows apart", "odd start", "odd pitch", "columns", "batches", "expanded"])
def test_views(pa, view):
    rows, cols = 12, 520
    x1, x2, gamma = make(rows, cols, torch.bfloat16)
    a, b, g = cuda(x1, x2, gamma)
    if view == "rows apart":
        a = torch.cat((a, a), 1)[:, :cols]
    elif view == "odd start":
        a = torch.cat((a[:, :1], a), 1)[:, 1:]
    elif view == "odd pitch":
        a, b = torch.cat((a, a[:, :3]), 1)[:, :cols], torch.cat((b, b[:, :5]), 1)[:, :cols]
    elif view == "columns":
        a = a.t().contiguous().t()
    elif view == "batches":
        x1, x2 = x1.view(3, 4, cols), x2.view(3, 4, cols)
        a, b = a.view(3, 4, cols), b.view(3, 4, cols).transpose(0, 1).contiguous().transpose(0, 1)
    else:
        x1, a = x1[:1].expand(rows, cols), a[:1].expand(rows, cols)
    check16(pa.npu_add_rms_norm(a, b, g, EPS), x1, x2, gamma)
    check8(pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=EPS), x1, x2, gamma)
    g = torch.cat((g, g))[1::2][: cols // 2]
    a, b = a[..., : cols // 2], b[..., : cols // 2]
    check16(pa.npu_add_rms_norm(a, b, g, EPS), x1[..., : cols // 2], x2[..., : cols // 2], torch.cat((gamma, gamma))[1::2][: cols // 2])


def test_shapes_without_rows(pa):
    for shape in ((0, 64), (3, 0, 64)):
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        y, rstd, s = pa.npu_add_rms_norm(x, x, torch.ones(64, dtype=torch.bfloat16, device="cuda"))
        assert y.shape == s.shape == shape and rstd.shape == (*shape[:-1], 1)
        y, scale, s = pa.npu_add_rms_norm_dynamic_quant(x, None, torch.ones(64, dtype=torch.bfloat16, device="cuda"))
        assert y.shape == shape and scale.shape == shape[:-1] and s.shape == (0,)
    check(pa, *[t if t is None or t.dim() == 1 else t[0] for t in make(1, 96, torch.float16)])             # one dimension


@pytest.mark.parametrize("cols", [64, 1000, 4096, 40000])
def test_rows_that_are_not_finite(pa, cols):
    """NaN and infinity stay in their row; a row of zeros gives zeros."""
    x1, x2, gamma = make(6, cols, torch.bfloat16)
    x1[1, cols // 2], x1[2, 3], x2[3, 5] = float("nan"), float("inf"), float("-inf")
    x1[4], x2[4] = 0, 0
    a, b, g = cuda(x1, x2, gamma)
    y, rstd, x = pa.npu_add_rms_norm(a, b, g, EPS)
    fine = [0, 4, 5]
    check16((y[fine], rstd[fine], x[fine]), x1[fine], x2[fine], gamma)
    assert bool(y[1].isnan().all()) and bool((y[4] == 0).all()) and bool((rstd[2:4] == 0).all())
    assert bool(y[2, 3].isnan()) and bool(y[3, 5].isnan()) and int(y[2:4].isnan().sum()) == 2 and bool((y[2:4].nan_to_num(0.0) == 0).all())
    y, scale, x = pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=EPS)
    check8((y[fine], scale[fine], x[fine]), x1[fine], x2[fine], gamma)
    assert bool(scale[1:4].isnan().all()) and float(scale[4]) == 0.0


def test_more_rows_than_one_launch_takes(pa):
    """2^21 rows are a launch; the rest go into a second one."""
    rows, cols = (1 << 21) + 3, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(torch.bfloat16)
    gamma = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    for at in (0, (1 << 21) - 2, 1 << 21):
        part = slice(at, at + 3)
        y, rstd, s = pa.npu_add_rms_norm(x, x, gamma, EPS)
        check16((y[part], rstd[part], s[part]), x[part].cpu(), x[part].cpu(), gamma.cpu())
        y, scale, s = pa.npu_add_rms_norm_dynamic_quant(x, x, gamma, epsilon=EPS)
        check8((y[part], scale[part], s[part]), x[part].cpu(), x[part].cpu(), gamma.cpu())


def test_offsets_beyond_32_bits(pa):
    """Rows that start behind 2^32 bytes."""
    cols, pitch = 256, 1 << 26
    big = torch.empty(40 * pitch, dtype=torch.bfloat16, device="cuda")
    x1, x2, gamma = make(40, cols, torch.bfloat16)
    a = big.view(40, pitch)[:, :cols]
    a.copy_(x1)
    b, g = cuda(x2, gamma)
    check16(pa.npu_add_rms_norm(a, b, g, EPS), x1, x2, gamma)
    check8(pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=EPS), x1, x2, gamma)


def test_streams_and_graphs(pa):
    """On a stream of its own, and captured: every replay sees the inputs of the moment."""
    x1, x2, gamma = make(33, 4096, torch.bfloat16)
    a, b, g = cuda(x1, x2, gamma)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=EPS)
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    check8(got, x1, x2, gamma)
    with torch.cuda.graph(graph, stream=side):
        codes = pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=EPS)
        rows = pa.npu_add_rms_norm(a, b, g, EPS)
    for seed in (1, 2, 3):
        x1, x2, _ = make(33, 4096, torch.bfloat16, seed=seed)
        a.copy_(x1), b.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        check8(codes, x1, x2, gamma)
        check16(rows, x1, x2, gamma)


def test_into_the_projection(pa):
    """Codes and scales as npu_quant_matmul takes them: the norm and the product against 64 bits."""
    x1, x2, gamma = make(48, 1024, torch.bfloat16, seed=9)
    a, b, g = cuda(x1, x2, gamma)
    gen = torch.Generator().manual_seed(1)
    w = torch.randint(-127, 128, (512, 1024), generator=gen, dtype=torch.int8)
    ws = torch.rand(512, generator=gen) * 0.01 + 0.001
    codes, scale, _ = pa.npu_add_rms_norm_dynamic_quant(a, b, g, epsilon=EPS)
    out = pa.npu_quant_matmul(codes, w.cuda().t(), ws.cuda(), pertoken_scale=scale, output_dtype=torch.bfloat16)
    want_codes, step = codes_of(x1, x2, gamma)
    rstd = 1 / ((x1.double() + x2.double()).square().mean(-1) + EPS).sqrt()
    want = (want_codes.double() @ w.double().t()) * (step.double() * rstd)[:, None] * ws.double()
    assert bool(((out.cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -17) * want.abs()).all())
