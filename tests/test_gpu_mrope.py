"""npu_mrope on the GPU against its formula in 64 bits on the CPU.

Tolerance: two float32 products and their sum, 2^-24 of each product and of the sum, and one rounding to 16 bits, half a step
(2^-8 bfloat16, 2^-11 float16) of the result.  Elements that are not turned are copied: equal bits.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
POSITIONS = 300


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


def make_table(rot, dtype, positions=POSITIONS):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    return torch.cat((angle.cos(), angle.sin()), 1).to(dtype)


def make(tokens, heads, kv, dim, dt, seed=0, axes=1):
    g = torch.Generator().manual_seed(seed)
    at = torch.randint(0, POSITIONS, (axes, tokens), generator=g)
    return at, torch.randn(tokens, heads, dim, generator=g).to(dt), torch.randn(tokens, kv, dim, generator=g).to(dt)


def check(got, positions, x, table, sections, mode):
    """positions [axes, tokens]; x [tokens, heads, dim]"""
    rot, dt = table.shape[1], x.dtype
    half = rot // 2
    f = torch.arange(half)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    at = positions[axis].t()                               # [tokens, half]
    there = (at >= 0) & (at < table.shape[0])
    row = at.clamp(0, table.shape[0] - 1)
    c = torch.where(there, table[row, f].double(), 0.0)[:, None]
    s = torch.where(there, table[row, half + f].double(), 0.0)[:, None]
    first, second = (f, half + f) if mode == "half" else (2 * f, 2 * f + 1)
    a, b = x[..., first].double(), x[..., second].double()
    got = got.cpu().reshape(x.shape)
    assert got.dtype == dt
    for place, want, size in ((first, a * c - b * s, (a * c).abs() + (b * s).abs()), (second, b * c + a * s, (b * c).abs() + (a * s).abs())):
        bound = U[dt] * want.abs() + 2.0 ** -23 * size + TINY[dt]
        assert bool(((got[..., place].double() - want).abs() <= bound).all())
    assert torch.equal(got[..., rot:], x[..., rot:])


def run(pa, at, q, k, table, sections, mode, dim):
    one = len(sections) == 1
    got = pa.npu_mrope((at[0] if one else at).cuda(), q.cuda(), k.cuda(), table.cuda(), dim, mrope_section=None if one else sections, rotary_mode=mode)
    for out, x in zip(got, (q, k)):
        assert out.shape == x.shape and out.is_contiguous()
        check(out, at, x, table, sections, mode)


@pytest.mark.parametrize("mode", ["half", "interleave"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,rot", [(2, 2), (8, 8), (16, 16), (64, 64), (80, 80), (96, 96), (128, 128), (256, 256), (128, 64), (80, 40), (96, 48), (100, 36), (129, 128),
                                     (128, 2)])
def test_widths(pa, dim, rot, dt, mode):
    for table_type in (dt, torch.float32):
        for heads, kv in ((8, 2), (5, 1), (1, 1)):
            at, q, k = make(9, heads, kv, dim, dt, seed=dim + heads)
            run(pa, at, q, k, make_table(rot, table_type), [rot // 2], mode, dim)


@pytest.mark.parametrize("mode", ["half", "interleave"])
@pytest.mark.parametrize("sections", [[64], [16, 24, 24], [32, 32], [8, 16, 16, 24], [11, 30, 23], [0, 40, 24], [64, 0, 0], [1, 1, 62], [0, 0, 0, 64], [3, 61]])
def test_axes(pa, sections, mode):
    for dt in U:
        at, q, k = make(33, 4, 2, 128, dt, seed=len(sections), axes=len(sections))
        run(pa, at, q, k, make_table(128, torch.float32), sections, mode, 128)


@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 1000, 4001])
@pytest.mark.parametrize("heads,kv", [(32, 8), (7, 7), (28, 4)])
def test_tokens(pa, tokens, heads, kv):
    at, q, k = make(tokens, heads, kv, 128, torch.bfloat16, seed=tokens, axes=3)
    run(pa, at, q, k, make_table(128, torch.float32), [16, 24, 24], "half", 128)


def test_one_section_is_one_axis(pa):
    at, q, k = make(20, 4, 2, 64, torch.bfloat16)
    table = make_table(64, torch.float32)
    a = pa.npu_mrope(at.cuda(), q.cuda(), k.cuda(), table.cuda(), 64, mrope_section=[32])
    b = pa.npu_mrope(at[0].cuda(), q.cuda(), k.cuda(), table.cuda(), 64)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dim", [128, 80, 100])
def test_views_of_a_projection(pa, dim):
    """Queries and keys as slices of [tokens, all heads, dim] and of [tokens, all heads * dim], at even and odd places; positions of 32 bits, of an
    expanded axis and with strides."""
    table = make_table(dim, torch.float32)
    at, qkv, _ = make(17, 14, 1, dim, torch.bfloat16, axes=3)
    sections = [dim // 2 - 20, 10, 10]
    full = qkv.cuda()
    got = pa.npu_mrope(at.cuda(), full[:, :8], full[:, 8:10], table.cuda(), dim, mrope_section=sections)
    check(got[0], at, qkv[:, :8], table, sections, "half")
    check(got[1], at, qkv[:, 8:10], table, sections, "half")
    wide = torch.cat((full.flatten(1)[:, :3], full.flatten(1)), 1)
    flat = wide[:, 3:]                                                     # rows that start at odd elements
    got = pa.npu_mrope(at.int().cuda(), flat[:, : 8 * dim], flat[:, 8 * dim:10 * dim], table.cuda(), dim, mrope_section=sections)
    assert got[0].shape == (17, 8 * dim) and got[1].shape == (17, 2 * dim)
    check(got[0], at, qkv[:, :8], table, sections, "half")
    check(got[1], at, qkv[:, 8:10], table, sections, "half")
    got = pa.npu_mrope(at[:1].cuda().expand(3, 17), full[:, :8].transpose(0, 1).contiguous().transpose(0, 1), full[:, 8:10].expand(17, 2, dim),
                       torch.cat((table, table), 1).cuda()[:, :dim], dim, mrope_section=sections)
    check(got[0], at[:1].expand(3, 17), qkv[:, :8], table, sections, "half")
    spread = torch.stack((at, at), -1).cuda()[..., 0]
    got = pa.npu_mrope(spread, full[:, :8], full[:, 8:10, :dim], table.cuda(), dim, mrope_section=sections)
    check(got[0], at, qkv[:, :8], table, sections, "half")
    columns = full.permute(2, 0, 1).contiguous().permute(1, 2, 0)          # the last dimension is not contiguous
    got = pa.npu_mrope(at.cuda(), columns[:, :8], columns[:, 8:10], table.cuda(), dim, mrope_section=sections)
    check(got[1], at, qkv[:, 8:10], table, sections, "half")


@pytest.mark.parametrize("sections", [[16, 24, 24], [17, 24, 23]])
@pytest.mark.parametrize("dim", [128, 130])
def test_positions_outside_the_table(pa, sections, dim):
    at, q, k = make(12, 4, 2, dim, torch.bfloat16, axes=3)
    at[0, 1], at[1, 2], at[2, 3], at[:, 4] = -1, POSITIONS, 1 << 40, -(1 << 62)
    table = make_table(128, torch.float32)
    run(pa, at, q, k, table, sections, "half", dim)
    run(pa, at, q, k, table, sections, "interleave", dim)
    empty = pa.npu_mrope(at.cuda(), q.cuda(), k.cuda(), table[:0].cuda(), dim, mrope_section=sections)
    assert bool((empty[0][..., :128] == 0).all()) and torch.equal(empty[0][..., 128:].cpu(), q[..., 128:])


def test_nothing_to_turn(pa):
    table = make_table(64, torch.float32).cuda()
    q, k = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    got = pa.npu_mrope(torch.empty(0, dtype=torch.int64, device="cuda"), q, k, table, 64)
    assert got[0].shape == q.shape and got[1].shape == k.shape
    at, q, k = make(5, 4, 2, 64, torch.bfloat16)
    got = pa.npu_mrope(at[0].cuda(), q.cuda(), k.cuda()[:, :0], table, 64)
    check(got[0], at, q, table.cpu(), [32], "half")
    assert got[1].shape == (5, 0, 64)
    got = pa.npu_mrope(at[0].cuda(), q.cuda()[:, :0], k.cuda(), table, 64)
    check(got[1], at, k, table.cpu(), [32], "half")


def test_values_that_are_not_finite(pa):
    """They reach their own pair only."""
    at, q, k = make(6, 4, 2, 64, torch.bfloat16)
    table = make_table(64, torch.float32)
    clean, _ = pa.npu_mrope(at[0].cuda(), q.cuda(), k.cuda(), table.cuda(), 64)
    q[2, 1, 5] = float("nan")
    got, _ = pa.npu_mrope(at[0].cuda(), q.cuda(), k.cuda(), table.cuda(), 64)
    assert bool(got[2, 1, 5].isnan()) and bool(got[2, 1, 37].isnan()) and int(got.isnan().sum()) == 2
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[2, 1, 5] = keep[2, 1, 37] = False
    assert torch.equal(got[keep], clean[keep])


def test_more_threads_than_one_launch_takes(pa):
    """2^30 threads are a launch: tokens of one wide head each, on the element-wise path."""
    tokens, dim = (1 << 30) // 1025 + 5, 1026 * 2 - 2                      # 1025 pairs a token
    q = torch.zeros(tokens, 1, dim, dtype=torch.bfloat16, device="cuda")
    k = q[:, :0]
    q[-3:, 0, 0], q[0, 0, 0] = torch.tensor([1.0, 2.0, 3.0], dtype=torch.bfloat16, device="cuda"), 4.0
    table = torch.cat((torch.full((2, dim // 2), 2.0), torch.full((2, dim // 2), 3.0)), 1).cuda()
    got, _ = pa.npu_mrope(torch.ones(tokens, dtype=torch.int32, device="cuda"), q, k, table, dim)
    assert got[-3:, 0, 0].tolist() == [2.0, 4.0, 6.0] and got[-3:, 0, dim // 2].tolist() == [3.0, 6.0, 9.0] and got[0, 0, [0, dim // 2]].tolist() == [8.0, 12.0]
    assert int((got[:, 0, 0] != 0).sum()) == 4 and int((got[:, 0, dim // 2] != 0).sum()) == 4


def test_streams_and_graphs(pa):
    at, q, k = make(64, 32, 8, 128, torch.bfloat16, axes=3)
    table, sections = make_table(128, torch.float32), [16, 24, 24]
    p, a, b, t = at.cuda(), q.cuda(), k.cuda(), table.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pa.npu_mrope(p, a, b, t, 128, mrope_section=sections)
    side.synchronize()
    check(got[0], at, q, table, sections, "half")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = pa.npu_mrope(p, a, b, t, 128, mrope_section=sections)
    for seed in (1, 2, 3):
        at, q, k = make(64, 32, 8, 128, torch.bfloat16, seed=seed, axes=3)
        p.copy_(at), a.copy_(q), b.copy_(k)
        graph.replay()
        torch.cuda.synchronize()
        check(got[0], at, q, table, sections, "half")
        check(got[1], at, k, table, sections, "half")
