"""Appends, prompt attention and shared-prefix decode run together, as a server runs them: a model
of two layers takes prompts, whole and in chunks, then decodes behind them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def model(dev, **kw):
    from peerkv_b200.decoder import LlamaGeometry, ModelWeights
    torch.manual_seed(3)
    g = LlamaGeometry(n_layers=2, hidden=512, n_q_heads=8, n_kv_heads=2, head_dim=128, ffn=768, vocab=256, **kw)
    w = ModelWeights(g, dev)
    for l in w.layers:
        for n in (l.q_norm, l.k_norm):
            if n is not None:
                n.copy_(1 + 0.2 * torch.randn_like(n))
    return g, w


def caches(g, lens, extra, dev, bs=16):
    """Per layer a pool and a shuffled table that has room for lens[i] + extra tokens."""
    from peerkv_b200.decoder import ShardedKVLayer
    need = [-(-(n + extra) // bs) for n in lens]
    ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(7))
    tab = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tab[i, :n] = ids[at:at + n].to(torch.int32)
        at += n
    layers = [ShardedKVLayer(torch.full((2, sum(need), bs, g.n_kv_heads, g.head_dim), float("nan"), dtype=torch.bfloat16, device=dev),
                             tab.to(dev), torch.zeros(len(lens), dtype=torch.int32, device=dev)) for _ in range(g.n_layers)]
    return layers, tab


def packed(seqs, start, end, tab, dev, bs=16):
    """Arguments of PromptStep.step for tokens start[i] .. end[i] - 1 of every sequence."""
    pos = [torch.arange(a, b) for a, b in zip(start, end)]
    tok = torch.cat([s[a:b] for s, a, b in zip(seqs, start, end)])
    slot = torch.cat([tab[i, p // bs].long() * bs + p % bs for i, p in enumerate(pos)])
    cu = torch.tensor([0] + list(torch.tensor([b - a for a, b in zip(start, end)]).cumsum(0)), dtype=torch.int32)
    return [x.to(dev) for x in (tok, torch.cat(pos), slot, cu, torch.tensor(end, dtype=torch.int32))]


def close(a, b):
    """Logits of the same tokens by two routes: the routes round activations to bf16 at different
    values of O (one half step each), so they agree to a few steps of the largest logit."""
    a, b = a.float(), b.float()
    assert torch.isfinite(a).all() and (a - b).abs().max() <= 8 * 2.0 ** -8 * b.abs().max()


@pytest.mark.parametrize("kw", [{}, {"qk_norm": True}, {"qk_norm": True, "rotary_dim": 64, "rope_interleaved": True}])
def test_chunks_and_decode_agree_with_whole_prompts(dev, kw):
    """Whole prompts at once; the same in three chunks; and prompt + decode steps: the same logits
    and the same cache."""
    from peerkv_b200.decoder import DecodeStep, PromptStep
    g, w = model(dev, **kw)
    lens = [37, 200, 5]
    gen = torch.Generator().manual_seed(11)
    seqs = [torch.randint(0, g.vocab, (n + 3,), generator=gen) for n in lens]
    full = [n + 3 for n in lens]
    whole, tab = caches(g, lens, 3, dev)
    ref = PromptStep(g, w, whole, dev).step(*packed(seqs, [0] * 3, full, tab, dev))

    parts, _ = caches(g, lens, 3, dev)
    ps = PromptStep(g, w, parts, dev)
    cuts = [[0, 10, 37, 40], [0, 128, 129, 203], [0, 1, 2, 8]]
    for k in range(3):
        got = ps.step(*packed(seqs, [c[k] for c in cuts], [c[k + 1] for c in cuts], tab, dev))
    close(got, ref)
    for a, b in zip(whole, parts):
        used = ~torch.isnan(a.pool)
        assert torch.equal(used, ~torch.isnan(b.pool))
        assert torch.allclose(a.pool[used].float(), b.pool[used].float(), atol=0.06, rtol=2.0 ** -5)

    step, _ = caches(g, lens, 3, dev)
    PromptStep(g, w, step, dev).step(*packed(seqs, [0] * 3, lens, tab, dev))
    pages, slots = torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for l in step:
        l.pool.nan_to_num_(0.0)
    ds = DecodeStep(g, w, step, 3, dev, append_slots=(pages, slots))
    for k in range(3):
        p = torch.tensor([n + k for n in lens])
        pages.copy_(tab[torch.arange(3), p // 16].long())
        slots.copy_(p % 16)
        for l in step:
            l.lens.copy_((p + 1).to(torch.int32))
        ds.step(torch.stack([s[q] for s, q in zip(seqs, p)]).to(dev), p.to(dev))
    torch.cuda.synchronize()
    assert ds.shard.status() == 0
    close(ds.logits, ref)


def test_decode_behind_a_shared_prefix(dev):
    """One prompt prefilled once, four requests that share it, each with some tokens of its own: the
    same logits as four full sequences, eagerly and as a graph."""
    from peerkv_b200.decoder import DecodeStep, PromptStep, ShardedKVLayer
    g, w = model(dev, qk_norm=True)
    gen = torch.Generator().manual_seed(13)
    P, own = 96, [1, 16, 17, 40]                      # a prefix of whole pages; own tokens behind it, the new one included
    prefix = torch.randint(0, g.vocab, (P,), generator=gen)
    seqs = [torch.cat([prefix, torch.randint(0, g.vocab, (n,), generator=gen)]) for n in own]
    full = [P + n for n in own]
    sep, tab = caches(g, full, 0, dev)
    ref = PromptStep(g, w, sep, dev).step(*packed(seqs, [0] * 4, full, tab, dev))

    lay, ptab = caches(g, [P] + own, 0, dev)          # row 0: the prefix; rows 1..: own pages
    PromptStep(g, w, [ShardedKVLayer(l.pool, l.table[:1], l.lens[:1]) for l in lay], dev).step(
        *packed([prefix], [0], [P], ptab[:1], dev))
    # own tokens but the last one, as a chunk behind the prefix: tables = prefix pages, then own pages
    joint = torch.cat([ptab[:1, :P // 16].expand(4, -1), ptab[1:]], 1)
    most = [P + n - 1 for n in own]
    rows = [i for i in range(4) if own[i] > 1]
    ps = PromptStep(g, w, [ShardedKVLayer(l.pool, joint[rows].to(dev), l.lens[:3]) for l in lay], dev)
    ps.step(*packed([seqs[i] for i in rows], [P] * 3, [most[i] for i in rows], joint[rows], dev))
    for l in lay:
        l.pool.nan_to_num_(0.0)
    p = torch.tensor([n - 1 for n in own])
    dec = [ShardedKVLayer(l.pool, l.table[1:].contiguous(), torch.tensor(own, dtype=torch.int32, device=dev)) for l in lay]
    ds = DecodeStep(g, w, dec, 4, dev, append_slots=(ptab[1:][torch.arange(4), p // 16].long().to(dev), (p % 16).to(dev)),
                    prefix=(lay[0].table[:1].contiguous(), torch.tensor([P], dtype=torch.int32, device=dev),
                            torch.tensor([0, 4], dtype=torch.int32, device=dev)))
    tok, pos = torch.stack([s[-1] for s in seqs]).to(dev), (p + P).to(dev)
    ds.step(tok, pos)
    close(ds.logits, ref)
    eager = ds.logits.clone()
    ds.capture()
    for _ in range(2):
        ds.step(tok, pos)
        torch.cuda.synchronize()
        assert torch.equal(ds.logits, eager)
    assert ds.shard.status() == 0


def test_sequences_without_new_tokens(dev):
    """A padded batch: first, middle and last sequences that add nothing give logits 0 and leave the
    others' as they are; a batch that adds nothing at all gives 0 everywhere."""
    from peerkv_b200.decoder import PromptStep
    g, w = model(dev)
    gen = torch.Generator().manual_seed(17)
    lens = [0, 21, 0, 0, 5, 0]
    seqs = [torch.randint(0, g.vocab, (n,), generator=gen) for n in lens]
    kept = [1, 4]
    some, tab = caches(g, [lens[i] for i in kept], 0, dev)
    ref = PromptStep(g, w, some, dev).step(*packed([seqs[i] for i in kept], [0, 0], [lens[i] for i in kept], tab, dev))
    every, tab = caches(g, lens, 0, dev)
    got = PromptStep(g, w, every, dev).step(*packed(seqs, [0] * 6, lens, tab, dev))
    close(got[kept], ref)
    assert (got[[0, 2, 3, 5]] == 0).all()
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    zero = torch.zeros(7, dtype=torch.int32, device=dev)
    out = PromptStep(g, w, every, dev).step(none, none, none, zero, zero[1:])
    assert out.shape == (6, g.vocab) and (out == 0).all()


def test_a_group_and_a_prefix_are_refused(dev):
    from peerkv_b200 import PeerKVError
    from peerkv_b200.decoder import DecodeStep
    g, w = model(dev)
    layers, _ = caches(g, [16], 0, dev)
    with pytest.raises(PeerKVError, match="one GPU"):
        DecodeStep(g, w, layers, 1, dev, group=object(), prefix=(None, None, None))
