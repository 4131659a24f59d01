"""What the kernels of a model step report reaches its caller: slots and page ids outside the pools, from
PromptStep and from DecodeStep, eager and captured."""
import pytest
import torch

from test_prompt_step_gpu import caches, model, packed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def test_prompt_step_reports_bad_slots_and_pages(dev):
    from peerkv_b200 import PeerKVError
    from peerkv_b200.decoder import PromptStep
    g, w = model(dev)
    lens = [21, 40]
    seqs = [torch.arange(n) % g.vocab for n in lens]
    kv, tab = caches(g, lens, 0, dev)
    ps = PromptStep(g, w, kv, dev)
    args = packed(seqs, [0, 0], lens, tab, dev)
    ps.step(*args)
    assert ps.status() == 0
    ps.raise_on_status()
    for l in kv:                                        # every page readable, whatever the tables say below
        l.pool.nan_to_num_(0.0)
    bad = [x.clone() for x in args]
    bad[2][3] = kv[0].pool.shape[1] * 16 + 5            # a slot behind the last page: not stored
    ps.step(*bad)
    with pytest.raises(PeerKVError, match="outside the pool"):
        ps.raise_on_status()
    assert ps.status() == 0                             # read and cleared
    kv[1].table[0, 1] = 1 << 20                         # a page id outside the pool: read as page 0
    ps.step(*args)
    assert ps.status() == 2 and ps.status() == 0


@pytest.mark.parametrize("where", ["prefix", "own", "slot"])
def test_decode_step_reports_bad_pages_and_slots(dev, where):
    from peerkv_b200 import PeerKVError
    from peerkv_b200.decoder import DecodeStep, ShardedKVLayer
    g, w = model(dev, qk_norm=True)
    kv, tab = caches(g, [32, 5, 9], 1, dev)             # row 0: the prefix
    for l in kv:
        l.pool.nan_to_num_(0.0)
    i = lambda *x: torch.tensor(x, device=dev)
    own = [ShardedKVLayer(l.pool, l.table[1:].clone(), i(6, 10).to(torch.int32)) for l in kv]
    pt = tab[:1].to(dev)
    pages, slots = tab[1:, 0].long().to(dev), i(5, 9)
    ds = DecodeStep(g, w, own, 2, dev, append_slots=(pages, slots), prefix=(pt, i(32).to(torch.int32), i(0, 2).to(torch.int32)))
    tok, pos = i(1, 2), i(37, 41)
    good_pages, good_pt, good_own = pages.clone(), pt.clone(), own[1].table.clone()
    for captured in (False, True):
        if captured:
            ds.capture()
        ds.step(tok, pos)
        assert ds.status() == 0
        if where == "prefix":
            pt[0, 1] = -3
        elif where == "own":
            own[1].table[1, 0] = 1 << 20
        else:
            pages[1] = 1 << 20
        ds.step(tok, pos)
        with pytest.raises(PeerKVError, match="outside the pool"):
            ds.raise_on_status()
        assert ds.status() == 0
        pt.copy_(good_pt); pages.copy_(good_pages); own[1].table.copy_(good_own)
