"""Block tables without columns hold no tokens, whatever the lengths say."""
import pytest
import torch

from test_prompt_gpu import prefix_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def test_tables_without_columns(dev):
    """As in the C interface: lengths are clamped to what a block-table row has room for."""
    from peerkv_b200 import ops
    q, k, v, pt, pl, bt, sl, go, _, _ = [x.to(dev) if torch.is_tensor(x) else x for x in
                                         prefix_case([(4, 40)], 12, 8, 2, 16, torch.bfloat16, 7)]
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    zero, status = torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    only_own = ops.decode_shared_prefix(q, k, v, pt, torch.zeros_like(pl), bt, sl, return_lse=True)
    got = ops.decode_shared_prefix(q, k, v, pt[:, :0], pl, bt, sl, return_lse=True, status=status)
    assert torch.equal(got[0], only_own[0]) and torch.equal(got[1], only_own[1])
    only_prefix = ops.decode_shared_prefix(q, k, v, pt, pl, bt, zero, return_lse=True)
    got = ops.decode_shared_prefix(q, k, v, pt, pl, bt[:, :0], sl, return_lse=True, status=status)
    assert torch.equal(got[0], only_prefix[0]) and torch.equal(got[1], only_prefix[1])
    cu = torch.tensor([0, 1, 4], dtype=torch.int32, device=dev)
    o, l = ops.prefill_paged(q, k, v, bt[:2, :0], sl[:2], cu, return_lse=True, status=status)
    assert (o == 0).all() and torch.isneginf(l).all() and status.item() == 0
