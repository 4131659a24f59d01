"""NaN on its way through prompt attention: a row that has met one says so in its output and in its lse,
wherever the work was cut and whatever is folded in."""
import pytest
import torch

from prompt_cases import D, assert_close
from test_prompt_gpu import prefix_case

pytestmark = pytest.mark.gpu
HQ, HKV = 8, 2


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def decode_prefix(dev, q, k, v, pt, pl, bt, sl, go):
    from peerkv_b200 import ops
    out, lse = ops.decode_shared_prefix(*[x.to(dev) for x in (q, k, v, pt, pl, bt, sl)], group_offsets=go.to(dev),
                                        return_lse=True, shard=ops.Shard(dev, q.shape[0], HQ))
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def check(out, lse, nan, ref, dt, most):
    """nan [B, Hq]: rows that met a NaN; the others are the reference's."""
    assert torch.isnan(out[nan]).all() and torch.isnan(lse[nan]).all(), "a NaN was lost"
    keep = ~nan
    assert_close(out[keep], lse[keep], *[r[keep] for r in ref], dt, most)


# a prefix of one tile is never cut; one of 20000 tokens is cut over most of the CTAs
@pytest.mark.parametrize("plen", [40, 20000])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_nan_query_behind_a_prefix(dev, dt, plen):
    q, k, v, pt, pl, bt, sl, go, ref, most = prefix_case([(6, plen)], 70, HQ, HKV, 16, dt, 5 + plen)
    nan = torch.zeros(6, HQ, dtype=torch.bool)
    for b, h in ((0, 3), (2, 0), (2, 7), (5, 4)):
        q[b, h, 17] = float("nan")
        nan[b, h] = True
    out, lse = decode_prefix(dev, q, k, v, pt, pl, bt, sl, go)
    check(out, lse, nan, ref, dt, most)


@pytest.mark.parametrize("plen", [40, 20000])
def test_nan_key_in_a_prefix(dev, plen):
    """Every row of that group and kv-head; the other group and the other kv-head keep theirs."""
    dt = torch.float16
    q, k, v, pt, pl, bt, sl, go, ref, most = prefix_case([(3, plen), (4, 300)], 40, HQ, HKV, 16, dt, 3 + plen)
    k[pt[0, (plen - 5) // 16].long(), (plen - 5) % 16, 0, 100] = float("nan")
    nan = torch.zeros(7, HQ, dtype=torch.bool)
    nan[:3, :HQ // HKV] = True
    check(*decode_prefix(dev, q, k, v, pt, pl, bt, sl, go), nan, ref, dt, most)


@pytest.mark.parametrize("n_new,L", [(3, 100), (5, 20000)])
def test_nan_query_of_a_prompt(dev, n_new, L):
    from peerkv_b200 import ops
    from test_prompt_gpu import paged_case
    dt = torch.bfloat16
    q, k, v, table, sl, cu, ref, most = paged_case([(n_new, L), (2, 50)], HQ, HKV, 16, dt, L, extra_rows=0)
    nan = torch.zeros(q.shape[0], HQ, dtype=torch.bool)
    q[1, 2, 127] = float("nan")
    nan[1, 2] = True
    out, lse = ops.prefill_paged(*[x.to(dev) for x in (q, k, v, table, sl, cu)], return_lse=True)
    check(out.cpu(), lse.cpu(), nan, ref, dt, most)
