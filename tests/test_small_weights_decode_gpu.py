"""As test_small_weights_gpu, for decode attention, own tokens behind a prefix and the dense prefill partial: one
dominant key whose V is 0, and many others that are the output."""
import math

import pytest
import torch

from prompt_cases import D, attend64, fill_pool
from test_small_weights_gpu import bounds

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(D)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def sink_rows(gap, at, k, v):
    k[..., 0] = 0
    k[at] = 0
    k[at, :, 0] = gap / (SCALE * 16)
    v[at] = 0
    return k, v


def queries(shape, dt, gen):
    q = (torch.randn(*shape, generator=gen) * 0.25).to(dt)
    q[..., 0] = 16
    return q


def reference(q, k, v):
    """One row: attend64's results and what bounds() needs besides."""
    hq, hkv, L = q.shape[0], k.shape[1], k.shape[0]
    r = attend64(q[None], k, v, SCALE, torch.tensor([L]))
    v_sum = v.double().abs().sum(0).repeat_interleave(hq // hkv, 0)[None]
    top = torch.stack([torch.softmax((k[:, h // (hq // hkv)].double() @ q[h].double()) * SCALE, 0).max() for h in range(hq)])[None]
    return (*r, v_sum, top)


def check(out, lse, refs, dt, n_keys):
    ref, lse_ref, mag, big, v_sum, top = [torch.cat(x) for x in zip(*refs)]
    o_tol, l_tol = bounds(ref, lse_ref, mag, big, dt, n_keys, v_sum, top)
    worst = ((out.double().cpu() - ref).abs() / o_tol).max().item()
    assert worst <= 1.0, f"output off by {worst:.3g} of its bound"
    assert (((lse.double().cpu() - lse_ref).abs() / l_tol).max() <= 1.0)


# 30 sequences of 500 keys: a sequence per few CTAs; 250: several tiles a CTA; 2 of 9000: over all of them
@pytest.mark.parametrize("n_seq,L", [(30, 500), (250, 500), (2, 9000)])
@pytest.mark.parametrize("gap", [10, 14, 17, 20])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_decode_and_own_tokens(dev, dt, gap, n_seq, L):
    from peerkv_b200 import ops
    hq, hkv = 4, 2
    gen = torch.Generator().manual_seed(gap * L + n_seq)
    k, v, table, ks, vs = fill_pool([L] * n_seq, 16, hkv, dt, gen, lambda i, k, v: sink_rows(gap, i % 3, k, v))
    q = queries((n_seq, hq, D), dt, gen)
    refs = [reference(q[i], ks[i], vs[i]) for i in range(n_seq)]
    lens = torch.full((n_seq,), L, dtype=torch.int32, device=dev)
    a = [x.to(dev) for x in (q, k, v, table.clamp(min=0))]
    out, lse = ops.partial_paged(*a, lens)
    check(out, lse, refs, dt, L)
    none = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    out, lse = ops.decode_shared_prefix(*a[:3], none, none[0], a[3], lens, return_lse=True, out=torch.empty(q.shape, device=dev))
    check(out, lse, refs, dt, L)


@pytest.mark.parametrize("gap", [10, 17])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_dense_partial(dev, dt, gap):
    from peerkv_b200 import peer_parallel_attn as ppa
    gen = torch.Generator().manual_seed(gap)
    hq, hkv, L, n = 4, 2, 700, 70
    k, v = torch.randn(L, hkv, D, generator=gen).to(dt), torch.randn(L, hkv, D, generator=gen).to(dt)
    k, v = sink_rows(gap, 1, k, v)
    q = queries((n, hq, D), dt, gen)
    t = lambda x: x.transpose(0, 1)[None].contiguous().to(dev)
    o, l = ppa._partial_f32(t(q), t(k), t(v), SCALE)
    check(o[0].transpose(0, 1), l[0].T, [reference(q[i], k, v) for i in range(n)], dt, L)
