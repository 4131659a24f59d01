"""Tensors that are contiguous but start in the middle of a 16-byte word are copied, as anything else is that
the kernels cannot read in place."""
import math

import pytest
import torch

from prompt_cases import D

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def shifted(t, by=1):
    """The same values, contiguous, `by` elements behind an aligned address."""
    buf = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    out = buf[by:].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_contiguous_but_misaligned(dev, dt):
    from peerkv_b200 import ops
    gen = torch.Generator(device=dev).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev).to(dt)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    hq, hkv = 8, 2
    cu = i(0, 30, 77)
    q, k, v = r(77, hq, D), r(77, hkv, D), r(77, hkv, D)
    want = ops.prefill_packed(q, k, v, cu)
    for a in ((shifted(q), k, v), (q, shifted(k, 3), v), (q, k, shifted(v, 4)), (shifted(q, 2), shifted(k), shifted(v))):
        assert torch.equal(ops.prefill_packed(*a, cu), want)
    pool = r(2, 6, 16, hkv, D)
    table, lens = i(0, 1, 2, 3, 4, 5).view(2, 3), i(33, 48)
    assert torch.equal(ops.prefill_paged(shifted(q), pool[0], pool[1], table, lens, cu),
                       ops.prefill_paged(q, pool[0], pool[1], table, lens, cu))
    two = q[:2].contiguous()
    a = (pool[0], pool[1], table[:1], i(40), table[1:].expand(2, -1), i(5, 0))
    assert torch.equal(ops.decode_shared_prefix(shifted(two), *a), ops.decode_shared_prefix(two, *a))
    qkv, pos = r(5, (hq + 2 * hkv) * D), torch.arange(5, device=dev)
    inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, device=dev) / D))
    assert torch.equal(ops.norm_rope_append(shifted(qkv), pos, inv, hq, hkv), ops.norm_rope_append(qkv, pos, inv, hq, hkv))
