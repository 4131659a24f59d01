"""Groups of query heads that do not divide a row tile (128 = 25 x 5 + 3): the tile's last rows belong to no token.
They hold what an earlier call left in shared memory, and nothing of it may reach the rows beside them."""
import pytest
import torch

from prompt_cases import D
from test_prompt_gpu import run_paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


@pytest.mark.parametrize("group", [3, 5, 7, 12])
def test_unused_rows_do_not_reach_the_others(dev, group):
    """The same call behind calls whose queries, in the same places of shared memory, were zero, ordinary and
    fifty times as large."""
    from peerkv_b200 import ops
    gen = torch.Generator(device=dev).manual_seed(group)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev).half()
    lens = [700, 1, 52, 9, 333]
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=dev)
    T, hkv = sum(lens), 4
    q, k, v = r(T, hkv * group, D), r(T, hkv, D), r(T, hkv, D)
    other, ok, ov = r(4096, 32, D), r(4096, 8, D), r(4096, 8, D)
    oc = torch.tensor([0, 4096], dtype=torch.int32, device=dev)
    got = []
    for size in (0.0, 1.0, 50.0, 0.0, 50.0):
        ops.prefill_packed(other * size, ok, ov, oc)
        got.append(ops.prefill_packed(q, k, v, cu, return_lse=True))
    torch.cuda.synchronize()
    for out, lse in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])


@pytest.mark.parametrize("hq,hkv", [(9, 3), (20, 4), (7, 1), (24, 2)])
def test_such_groups_against_64_bits(dev, hq, hkv):
    run_paged(dev, [(60, 300), (1, 1500), (26, 26), (130, 700)], hq, hkv, 16, torch.float16, hq)
