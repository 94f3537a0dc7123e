"""Two host threads that call operators on one stream: an operator of several launches keeps the stream's workspace to itself
until the last of them is enqueued, so every call gives the bits that it gives alone."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

CALLS = 60


@pytest.fixture(scope="module")
def pa():
    import pytorch_amd
    return pytorch_amd


def side_by_side(*calls):
    """calls[i](j) for j < CALLS in thread i, all on the default stream; what they returned."""
    start, got, errors = threading.Barrier(len(calls)), [[] for _ in calls], []

    def work(i):
        try:
            start.wait(30)
            for j in range(CALLS):
                got[i].append(calls[i](j))
        except Exception as e:                                      # the test's thread raises it
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads)
    if errors:
        raise errors[0]
    torch.cuda.synchronize()
    return got


def same(results, want):
    return all(torch.equal(x, y) for got in results for x, y in zip(got, want))


class Cache:
    """A batch of equally long sequences, and as many copies of what a call changes as there are calls."""

    def __init__(self, seed, batch, n, hkv, d):
        g = torch.Generator().manual_seed(seed)
        width = -(-n // 16)
        self.table = torch.randperm(batch * width, generator=g).reshape(batch, width).to(torch.int32).cuda()
        self.lens = torch.full((batch,), n, dtype=torch.int32).cuda()
        self.key, self.value = (torch.randn(batch * width, 16, hkv, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        self.sums = torch.rand(batch, hkv, width * 16, generator=g).cuda()
        self.positions = torch.argsort(torch.rand(batch, hkv, width * 16, generator=g), -1).to(torch.int32).cuda()
        self.query = torch.randn(batch, hkv * 4, d, generator=g).to(torch.bfloat16).cuda()


def test_eviction(pa):
    """Lists of moves of different lengths and pitches, for caches of different sizes."""
    caches = [Cache(1, 2, 1200, 2, 64), Cache(2, 5, 330, 1, 128)]
    keep = [600, 200]
    assert all(k * c.key.shape[3] * 2 > 16384 for c, k in zip(caches, (600, 130)))       # rows are moved by a second launch
    copies = [[(c.key.clone(), c.value.clone()) for _ in range(CALLS + 1)] for c in caches]

    def call(i):
        def one(j):
            c, (key, value) = caches[i], copies[i][j]
            return (*pa.npu_paged_cache_evict(key, value, c.table, c.lens, c.sums, c.positions, keep[i], 20), key, value)
        return one

    want = [call(i)(CALLS) for i in range(2)]
    for results, alone in zip(side_by_side(call(0), call(1)), want):
        assert same(results, alone)


def test_attention_with_summed_weights(pa):
    caches = [Cache(3, 3, 900, 2, 128), Cache(4, 7, 333, 1, 64)]
    sums = [[c.sums.clone() for _ in range(CALLS + 1)] for c in caches]

    def call(i):
        def one(j):
            c = caches[i]
            return (*pa.npu_paged_decode_attention(c.query, c.key, c.value, c.table, c.lens, attn_sums=sums[i][j], softmax_lse=True), sums[i][j])
        return one

    want = [call(i)(CALLS) for i in range(2)]
    for results, alone in zip(side_by_side(call(0), call(1)), want):
        assert same(results, alone)


def test_quant_matmul_whose_weight_is_transposed_per_call(pa):
    g = torch.Generator().manual_seed(5)
    calls, want = [], []
    for m, k, n in ((96, 1024, 1536), (200, 512, 2048)):
        x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8).cuda()
        w = torch.randint(-127, 128, (k, n), generator=g, dtype=torch.int8).cuda()       # [K, N], contiguous
        scale, per_token = torch.rand(n, generator=g).cuda() * 1e-3, torch.rand(m, generator=g).cuda()
        calls.append(lambda j, x=x, w=w, s=scale, p=per_token: (pa.npu_quant_matmul(x, w, s, pertoken_scale=p, output_dtype=torch.bfloat16),))
        want.append(calls[-1](0))
    for results, alone in zip(side_by_side(*calls), want):
        assert same(results, alone)


def test_weight_quant_matmul_whose_weight_is_repacked_per_call(pa):
    g = torch.Generator().manual_seed(6)
    calls, want = [], []
    for m, k, n in ((256, 1024, 512), (300, 512, 1024)):
        x = torch.randn(m, k, generator=g).to(torch.bfloat16).cuda()
        w = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, k // 8), generator=g).to(torch.int32).cuda().t()      # words along K
        scale = (torch.rand(k // 128, n, generator=g) * 1e-2).to(torch.bfloat16).cuda()
        calls.append(lambda j, x=x, w=w, s=scale: (pa.npu_weight_quant_batchmatmul(x, w, s, None, None, None, None, 128),))
        want.append(calls[-1](0))
    for results, alone in zip(side_by_side(*calls), want):
        assert same(results, alone)
