"""PagedKVCache on the GPU where replays of a captured step bring more tokens than a sequence holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quantized", [False, True])
def test_replayed_append_past_the_capacity(quantized):
    """Against a cache that was given the tokens that fit and no more: the same tensors, before and after an eviction."""
    from pytorch_amd.contrib.module import PagedKVCache

    g = torch.Generator().manual_seed(4)
    batch, kv, d = 3, 2, 64
    full, exact = (PagedKVCache(batch, 32, kv, d, block_size=16, budget=12, recent=5, quantized=quantized, device="cuda") for _ in range(2))
    held = (27, 3, 32)
    for b, n in enumerate(held):
        k, v = (torch.randn(n, kv, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        full.prefill(b, k, v), exact.prefill(b, k, v)
    full._held = exact._held = [0] * batch                      # as replays leave the host's count
    new_k, new_v = (torch.zeros(batch, kv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        full.append(new_k, new_v)
    for step in range(9):
        for t in (new_k, new_v):
            t.copy_(torch.randn(batch, kv, d, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate(held):
            if n + step < 32:
                exact.prefill(b, new_k[b:b + 1], new_v[b:b + 1])
    assert full.context_lens.tolist() == full.next_position.tolist() == [32, 12, 32]
    sums = torch.rand(batch, kv, full.capacity, generator=g).cuda()
    for c in (full, exact):
        c.attn_sums.copy_(sums)
    for _ in range(2):
        for name in ("key_cache", "value_cache", "key_scale", "value_scale", "context_lens", "positions", "attn_sums", "next_position"):
            mine, want = getattr(full, name), getattr(exact, name)
            assert mine is want is None or torch.equal(mine, want), name
        full.evict(), exact.evict()
    newest = full.positions[0, :, :12].max(-1).values
    assert newest.tolist() == [31] * kv and all(set(range(27, 32)) <= set(row) for row in full.positions[0, :, :12].tolist())
