"""NaN and infinities on their way through decode attention, its merges and the fold behind it: a row that has met a
NaN says so in its output and in its lse; a score of -inf weighs nothing."""
import math

import pytest
import torch

from prompt_cases import D, assert_close, attend64
from test_nonfinite_prompt_gpu import HKV, HQ, check, decode_prefix
from test_prompt_gpu import prefix_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def test_nan_query_without_a_prefix(dev):
    """As behind one; a row that sees no key at all stays 0 with lse -inf."""
    q, k, v, pt, pl, bt, sl, go, ref, most = prefix_case([(6, 0)], 70, HQ, HKV, 16, torch.bfloat16, 5)
    sl[5] = 0
    ref[0][5], ref[1][5], ref[2][5], ref[3][5] = 0, -math.inf, 0, 0
    nan = torch.zeros(6, HQ, dtype=torch.bool)
    for b, h in ((0, 3), (2, 0), (2, 7), (5, 4)):
        q[b, h, 17] = float("nan")
        nan[b, h] = int(sl[b]) > 0
    assert nan.sum() == 3
    check(*decode_prefix(dev, q, k, v, pt, pl, bt, sl, go), nan, ref, torch.bfloat16, most)


@pytest.mark.parametrize("plen", [0, 40, 20000])
def test_nan_key_among_the_own_tokens(dev, plen):
    dt = torch.bfloat16
    q, k, v, pt, pl, bt, sl, go, ref, most = prefix_case([(5, plen)], 70, HQ, HKV, 16, dt, 11 + plen)
    nan = torch.zeros(5, HQ, dtype=torch.bool)
    for b in (1, 3):
        n = int(sl[b])
        assert n > 0
        k[bt[b, (n - 1) // 16].long(), (n - 1) % 16, 1, 9] = float("nan")          # its last token, kv-head 1
        nan[b, HQ // HKV:] = True
    check(*decode_prefix(dev, q, k, v, pt, pl, bt, sl, go), nan, ref, dt, most)


@pytest.mark.parametrize("L", [1, 16, 500, 30000])
def test_nan_query_and_nan_key_in_plain_decode(dev, L):
    """decode_paged and partial_paged: the same rule, for sequences in one CTA and over all of them."""
    from peerkv_b200 import ops
    dt = torch.bfloat16
    q, k, v, pt, pl, bt, sl, go, ref, most = prefix_case([(1, L)] * 3, 0, HQ, HKV, 16, dt, L)
    q[0, 5, 0] = float("nan")
    k[pt[1, (L - 1) // 16].long(), (L - 1) % 16, 0, 1] = float("nan")
    nan = torch.zeros(3, HQ, dtype=torch.bool)
    nan[0, 5], nan[1, :HQ // HKV] = True, True
    a = [x.to(dev) for x in (q, k, v, pt, pl)]
    out, lse = ops.decode_paged(*a, return_lse=True)
    check(out.cpu(), lse.cpu(), nan, ref, dt, most)
    o, l = ops.partial_paged(*a)
    check(o.cpu(), l.cpu(), nan, ref, dt, most)


def test_merging_nan_partials(dev):
    """A NaN partial survives beside finite ones, beside empty ones and alone."""
    from peerkv_b200 import ops
    o = torch.randn(3, 4, D, device=dev)
    l = torch.tensor([[0.5, float("nan"), -math.inf, float("nan")], [1.0, 2.0, -math.inf, -math.inf],
                      [-math.inf, -1.0, -math.inf, -math.inf]], device=dev)
    o[torch.isnan(l)] = float("nan")
    o[torch.isinf(l)] = 0.0
    out, lse = ops.merge_partials(o, l, return_lse=True)
    for r in (1, 3):
        assert torch.isnan(out[r]).all() and torch.isnan(lse[r])
    assert (out[2] == 0).all() and lse[2] == -math.inf
    w = torch.softmax(l[:2, 0].double(), 0)
    # three roundings of fp32 per value and the exponentials' 2^-20
    assert torch.allclose(out[0].double(), (w[:, None] * o[:2, 0].double()).sum(0), atol=1e-5, rtol=1e-5)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hidden,B", [(16, 3), (40, 3), (200, 3), (40, 250)])
def test_scores_of_minus_infinity_weigh_nothing(dev, dt, hidden, B):
    """The first `hidden` keys of 200 hold -inf where every query is positive: their scores are -inf, in
    the first tiles of a decode, of a prompt and of own tokens behind a prefix alike."""
    from peerkv_b200 import ops
    L = 200
    q, k, v, pt, pl, bt, sl, go, _, most = prefix_case([(1, L)] * B, 0, HQ, HKV, 16, dt, hidden)        # 250 sequences: several tiles a CTA
    q[..., 0] = q[..., 0].abs() + 0.5
    refs = []
    for b in range(B):
        at = torch.arange(L)
        page, tok = pt[b, at // 16].long(), at % 16
        k[page[:hidden], tok[:hidden], :, 0] = -math.inf
        kk, vv = k[page[hidden:], tok[hidden:]], v[page[hidden:], tok[hidden:]]
        refs.append(attend64(q[b:b + 1], kk, vv, 1 / math.sqrt(D), torch.tensor([L - hidden])))
    ref = [torch.cat(x) for x in zip(*refs)]
    a = [x.to(dev) for x in (q, k, v, pt, pl)]
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    none = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    for out, lse in (ops.decode_paged(*a, return_lse=True), ops.prefill_paged(*a, cu, return_lse=True),
                     ops.decode_shared_prefix(a[0], a[1], a[2], none, none[0], a[3], a[4], return_lse=True)):
        assert_close(out, lse, *ref, dt, most)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_nan_query_of_a_dense_shard(dev, dt):
    """The ring prefill's partial: the row's lse is NaN, the others' are finite."""
    from peerkv_b200 import peer_parallel_attn as ppa
    gen = torch.Generator().manual_seed(4)
    q, K, V = [torch.randn(1, h, 70, D, generator=gen).to(dt).to(dev) for h in (4, 2, 2)]
    want = ppa._partial_f32(q, K, V, 0.1, causal_diagonal=True)
    q[0, 1, 33, 5] = float("nan")
    o, l = ppa._partial_f32(q, K, V, 0.1, causal_diagonal=True)
    assert torch.isnan(o[0, 1, 33]).all() and torch.isnan(l[0, 1, 33])
    rest = torch.ones(1, 4, 70, dtype=torch.bool, device=dev)
    rest[0, 1, 33] = False
    assert torch.equal(o[rest], want[0][rest]) and torch.equal(l[rest], want[1][rest])
