"""A captured call that was given no shard keeps the cached one's scratch, also when a larger batch outgrows it."""
import pytest
import torch

from prompt_cases import D

pytestmark = pytest.mark.gpu


def test_an_outgrown_shard_outlives_the_graphs_captured_with_it():
    from peerkv_b200 import ops
    dev, hq, hkv = torch.device("cuda", 0), 6, 2
    gen = torch.Generator(device=dev).manual_seed(1)
    pool = torch.randn(2, 8, 16, hkv, D, generator=gen, device=dev).bfloat16()
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)

    def call(B):
        q = torch.randn(B, hq, D, generator=torch.Generator(device=dev).manual_seed(B), device=dev).bfloat16()
        a = (q, pool[0], pool[1], i(1, 2)[None], i(20), i(3, 4, 5)[None].expand(B, -1).contiguous(), i(*[40] * B))
        return a, lambda: ops.decode_shared_prefix(*a, group_offsets=go)
    go = i(0, 4)
    _, small = call(4)
    want = small()
    key = (0, hq)
    shard = ops._shards[key]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    a, small = call(4)
    with torch.cuda.graph(graph):
        got = small()
    go_big = i(0, shard.max_batch + 1)
    B = shard.max_batch + 1
    q = torch.randn(B, hq, D, device=dev).bfloat16()
    ops.decode_shared_prefix(q, pool[0], pool[1], i(1, 2)[None], i(20), i(3, 4, 5)[None].expand(B, -1).contiguous(), i(*[40] * B),
                             group_offsets=go_big)
    assert ops._shards[key] is not shard
    torch.cuda.synchronize()
    ops.get_shard(dev, 1, hq)                             # frees what was retired and is done
    assert shard._h, "the scratch of a captured launch was freed"
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del graph
