"""Weights far below the largest of their row.  P is rounded to the 16-bit type of V before it meets V, and
fp16 ends at 2^-24: behind one dominant key (an attention sink) whose V is small, the many others
are the output."""
import math

import pytest
import torch

from prompt_cases import D, attend64, fill_pool, tolerances

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def bounds(ref, lse, mag, big, dt, n_keys, v_sum, top):
    """prompt_cases.tolerances, and in fp16 what the smallest weights lose: the row's largest weight is held
    as at least 2^7 (with the running reference up to 2^15), subnormals are 2^-24 apart, so a weight is
    off by at most 2^-25 / 2^7 of the largest one: 2^-32 top sum_j |v_j| in all."""
    o_tol, l_tol = tolerances(ref, lse, mag, big, dt, n_keys)
    if dt == torch.float16:
        o_tol = o_tol + 2.0 ** -32 * top[..., None] * v_sum
    return o_tol, l_tol


# 300 sequences of 500 keys: whole items and items cut between two CTAs; 2 of 9000: items cut over many
@pytest.mark.parametrize("n_seq,L", [(300, 500), (2, 9000)])
@pytest.mark.parametrize("gap", [10, 14, 17, 20])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_one_dominant_key(dev, dt, gap, n_seq, L):
    from peerkv_b200 import ops
    hq, hkv, scale = 2, 1, 1 / math.sqrt(D)
    gen = torch.Generator().manual_seed(gap * L)

    def sink(i, k, v):
        k[..., 0] = 0
        k[i % 3] = 0                                    # the sink stands at key 0, 1 or 2
        k[i % 3, :, 0] = gap / (scale * 16)
        v[i % 3] = 0
        return k, v
    k, v, table, ks, vs = fill_pool([L] * n_seq, 16, hkv, dt, gen, sink)
    q = (torch.randn(n_seq, hq, D, generator=gen) * 0.25).to(dt)
    q[..., 0] = 16
    parts, v_sum, top = [], [], []
    for i in range(n_seq):
        parts.append(attend64(q[i:i + 1], ks[i], vs[i], scale, torch.tensor([L])))
        v_sum.append(vs[i].double().abs().sum(0)[:, None].expand(hkv, hq, D).reshape(1, hq, D))
        s = (q[i].double() @ ks[i][:, 0].double().T) * scale
        top.append(torch.softmax(s, -1).amax(-1)[None])
    ref, lse_ref, mag, big = [torch.cat(x) for x in zip(*parts)]
    o_tol, l_tol = bounds(ref, lse_ref, mag, big, dt, L, torch.cat(v_sum), torch.cat(top))
    cu = torch.arange(n_seq + 1, dtype=torch.int32, device=dev)
    lens = torch.full((n_seq,), L, dtype=torch.int32, device=dev)
    out, lse = ops.prefill_paged(q.to(dev), k.to(dev), v.to(dev), table.clamp(min=0).to(dev), lens, cu, return_lse=True,
                                 out=torch.empty(q.shape, device=dev))
    worst = ((out.double().cpu() - ref).abs() / o_tol).max().item()
    assert worst <= 1.0, f"output off by {worst:.3g} of its bound"
    worst = ((lse.double().cpu() - lse_ref).abs() / l_tol).max().item()
    assert worst <= 1.0, f"lse off by {worst:.3g} of its bound"
