"""Offsets behind 2^31 elements: rows at the end of a long packed batch, pages at the end of a large pool."""
import math

import pytest
import torch

from prompt_cases import D, assert_close, attend64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def test_rows_and_keys_at_the_end_of_a_long_batch(dev):
    """560000 packed tokens of 32 + 8 heads (2.3e9 values of q): the last sequences, against 64 bits."""
    from peerkv_b200 import ops
    hq, hkv, n, L = 32, 8, 8750, 64
    T = n * L
    assert T * hq * D > 2 ** 31
    q = torch.zeros(T, hq, D, dtype=torch.bfloat16, device=dev)
    k, v = torch.zeros(T, hkv, D, dtype=torch.bfloat16, device=dev), torch.zeros(T, hkv, D, dtype=torch.bfloat16, device=dev)
    gen = torch.Generator().manual_seed(1)
    tail = [torch.randn(2 * L, h, D, generator=gen).bfloat16() for h in (hq, hkv, hkv)]
    for x, t in zip((q, k, v), tail):
        x[-2 * L:] = t.to(dev)
    cu = torch.arange(0, T + 1, L, dtype=torch.int32, device=dev)
    out, lse = ops.prefill_packed(q, k, v, cu, return_lse=True)
    for i in range(2):
        at = slice(i * L, (i + 1) * L)
        ref = attend64(*[t[at] for t in tail], 1 / math.sqrt(D), 1 + torch.arange(L))
        rows = slice(T - (2 - i) * L, T - (1 - i) * L)
        assert_close(out[rows], lse[rows], *ref, torch.bfloat16, L)
    assert (out[:L] == 0).all()


@pytest.mark.parametrize("kv", ["16", "int8"])
def test_append_and_attend_in_the_last_pages_of_a_large_pool(dev, kv):
    """A pool of 2.2e9 values a side; tokens are appended to its last page and to its first, and (16 bits) attended
    over and decoded behind."""
    from peerkv_b200 import ops
    hq, hkv, page, n_pages, T = 8, 8, 16, 135000, 21
    assert n_pages * page * hkv * D > 2 ** 31
    gen = torch.Generator().manual_seed(2)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=gen).bfloat16().to(dev)
    pos, table = torch.arange(T, device=dev), torch.tensor([[n_pages - 1, 0]], dtype=torch.int32, device=dev)
    slots = table[0].long()[pos // page] * page + pos % page
    dt = torch.bfloat16 if kv == "16" else torch.int8
    k, v = torch.zeros(n_pages, page, hkv, D, dtype=dt, device=dev), torch.zeros(n_pages, page, hkv, D, dtype=dt, device=dev)
    small = [torch.zeros(2, page, hkv, D, dtype=dt, device=dev) for _ in range(2)]
    sc = [torch.zeros(p, page, hkv, dtype=torch.float16, device=dev) for p in (n_pages, n_pages, 2, 2)] if kv == "int8" else [None] * 4
    q = ops.norm_rope_append(qkv, pos, None, hq, hkv, None, k, v, slots, sc[0], sc[1])
    ops.norm_rope_append(qkv, pos, None, hq, hkv, None, *small, pos, sc[2], sc[3])
    for a, b in zip((k, v), small):
        assert torch.equal(a[table[0].long()], b)
    if kv == "int8":
        assert torch.equal(sc[0][table[0].long()], sc[2]) and torch.equal(sc[1][table[0].long()], sc[3])
        return
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    near = i(0, 1)[None]
    assert torch.equal(ops.prefill_paged(q, k, v, table, i(T), i(0, T)), ops.prefill_paged(q, *small, near, i(T), i(0, T)))
    one = q[-1:].contiguous()
    assert torch.equal(ops.decode_shared_prefix(one, k, v, table[:, :1], i(page), table[:, 1:], i(T - page)),
                       ops.decode_shared_prefix(one, *small, near[:, :1], i(page), near[:, 1:], i(T - page)))
