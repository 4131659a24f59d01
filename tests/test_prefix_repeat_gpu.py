"""Shared-prefix decode gives the same bits for the same inputs, whatever ran on its shard before: with enough own
tokens that the decode kernel, left alone, would place its cuts by how long the last launch took."""
import pytest
import torch

from prompt_cases import D

pytestmark = pytest.mark.gpu


def inputs(dev, B, own, prefix, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    hq, hkv, page = 32, 8, 16
    n_own, n_pre = -(-own // page), -(-prefix // page)
    total = B * n_own + n_pre
    pool = torch.randn(2, total, page, hkv, D, generator=gen, device=dev, dtype=torch.float32).bfloat16()
    ids = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    lens = torch.randint(own // 2, own + 1, (B,), generator=gen, device=dev).to(torch.int32)
    q = torch.randn(B, hq, D, generator=gen, device=dev).bfloat16()
    return (q, pool[0], pool[1], ids[:n_pre][None], torch.tensor([prefix], dtype=torch.int32, device=dev),
            ids[n_pre:].view(B, n_own), lens)


def test_same_bits_whatever_ran_before():
    from peerkv_b200 import ops
    dev = torch.device("cuda", 0)
    a, b = inputs(dev, 64, 1024, 3000, 1), inputs(dev, 40, 2500, 500, 2)
    assert int(a[6].sum()) > 20000
    shard = ops.Shard(dev, 64, 32)
    want = ops.decode_shared_prefix(*a, return_lse=True, shard=shard)
    got = []
    for n in range(6):
        for _ in range(n):
            ops.decode_shared_prefix(*b, shard=shard)
            ops.decode_paged(b[0], b[1], b[2], b[5], b[6], shard=shard)
        got.append(ops.decode_shared_prefix(*a, return_lse=True, shard=shard))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = ops.decode_shared_prefix(*a, return_lse=True, shard=shard)
    for n in range(6):
        ops.decode_paged(b[0], b[1], b[2], b[5], b[6], shard=shard)
        graph.replay()
        got.append([x.clone() for x in res])
    torch.cuda.synchronize()
    for n, (out, lse) in enumerate(got):
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), f"call {n} differs"
    del graph
