"""Offsets of a shared-prefix batch that describe no group are refused."""
import pytest
import torch

from test_prompt_gpu import prefix_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def test_offsets_without_groups_are_refused(dev):
    """[0] describes no group, so no row of the batch would be written."""
    from peerkv_b200 import PeerKVError, ops
    q, k, v, pt, pl, bt, sl, go, _, _ = [x.to(dev) if torch.is_tensor(x) else x for x in
                                         prefix_case([(4, 40)], 12, 8, 2, 16, torch.bfloat16, 7)]
    with pytest.raises(PeerKVError, match="group_offsets"):
        ops.decode_shared_prefix(q, k, v, pt[:0], pl[:0], bt, sl, group_offsets=go[:1])
