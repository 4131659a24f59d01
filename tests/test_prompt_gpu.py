"""Prompt attention (paged and packed) and shared-prefix decode against 64-bit references, with
bounds derived in prompt_cases.tolerances; refusals; streams, graphs and repeated calls."""
import math

import pytest
import torch

from prompt_cases import D, assert_close, attend64, fill_pool

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def offsets(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)


def paged_case(lens, hq, hkv, page, dt, seed, causal=True, make=None, extra_rows=3):
    gen = torch.Generator().manual_seed(seed)
    new, full = [p[0] for p in lens], [p[1] for p in lens]
    k, v, table, ks, vs = fill_pool(full, page, hkv, dt, gen, make)
    q = torch.randn(sum(new) + extra_rows, hq, D, generator=gen).to(dt)
    scale = 1.0 / math.sqrt(D)
    parts = []
    at = 0
    for i, (n, L) in enumerate(lens):
        first = (L - n + 1 + torch.arange(n)).clamp(min=0) if causal else torch.full((n,), L)
        parts.append(attend64(q[at:at + n], ks[i], vs[i], scale, first))
        at += n
    ref = [torch.cat(x) for x in zip(*parts)]
    return q, k, v, table.clamp(min=0), torch.tensor(full, dtype=torch.int32), offsets(new), ref, max(full)


def run_paged(dev, lens, hq, hkv, page, dt, seed, causal=True, make=None):
    from peerkv_b200 import ops
    q, k, v, table, sl, cu, ref, most = paged_case(lens, hq, hkv, page, dt, seed, causal, make)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.full(q.shape, 7.0, dtype=dt, device=dev)
    got, lse = ops.prefill_paged(q.to(dev), k.to(dev), v.to(dev), table.to(dev), sl.to(dev), cu.to(dev), causal=causal,
                                 out=out, return_lse=True, status=status)
    torch.cuda.synchronize()
    rows = int(cu[-1])
    assert status.item() == 0
    assert got.data_ptr() == out.data_ptr() and (out[rows:] == 7.0).all(), "rows behind the last sequence were written"
    assert_close(out[:rows], lse[:rows], *ref, dt, most)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,L", [(1, 1), (64, 64), (128, 128), (65, 65), (129, 129), (300, 300), (1, 1000), (7, 130),
                                 (200, 1111)])
def test_one_sequence(dev, dt, n, L):
    run_paged(dev, [(n, L)], 8, 2, 16, dt, n * 7 + L)


@pytest.mark.parametrize("hq,hkv", [(8, 8), (4, 2), (6, 2), (8, 2), (5, 1), (14, 2), (16, 2), (32, 1), (128, 1)])
def test_head_layouts(dev, hq, hkv):
    run_paged(dev, [(37, 37), (1, 200), (150, 400)], hq, hkv, 16, torch.bfloat16, hq * 10 + hkv)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 256])
def test_page_sizes(dev, page):
    run_paged(dev, [(130, 259), (3, 17), (64, 512)], 8, 2, page, torch.bfloat16, page)


@pytest.mark.parametrize("causal", [True, False])
def test_ragged_batch_with_empty_and_short_sequences(dev, causal):
    """Sequences without new tokens, without keys, and with fewer keys than new tokens (rows that
    see nothing), between ordinary ones."""
    lens = [(5, 5), (0, 40), (4, 0), (9, 3), (1, 1), (128, 90), (257, 700), (1, 3000), (0, 0), (31, 64)]
    run_paged(dev, lens, 8, 2, 16, torch.bfloat16, 5, causal)


def test_many_sequences(dev):
    run_paged(dev, [(1 + (i % 3 == 0), 1 + i % 23) for i in range(900)], 2, 1, 16, torch.float16, 9)


def test_long_cache_is_cut_over_the_ctas(dev):
    run_paged(dev, [(2, 40000)], 4, 1, 64, torch.bfloat16, 3)
    run_paged(dev, [(70, 9000), (1, 17)], 2, 2, 16, torch.float16, 4)


def test_growing_maxima(dev):
    """Scores that grow from tile to tile, so that the reference of the exponentials moves every
    time, and a first tile that towers above the rest."""
    def grow(i, k, v):
        f = torch.arange(k.shape[0]).float()[:, None, None] / 128
        return ((k.float() * 0 + 1) * f * 0.05).to(k.dtype) if i == 0 else (k.float() * (1 + 20 * (f < 1))).to(k.dtype), v
    for dt in (torch.bfloat16, torch.float16):
        run_paged(dev, [(200, 2500), (130, 1300)], 4, 2, 16, dt, 12, make=grow)


def test_strided_inputs_and_head_major_pools(dev):
    from peerkv_b200 import ops
    dt, hq, hkv = torch.bfloat16, 8, 2
    q, k, v, table, sl, cu, ref, most = paged_case([(70, 300), (33, 33)], hq, hkv, 16, dt, 21, extra_rows=0)
    qkv = torch.randn(q.shape[0], (hq + 2 * hkv) * D).to(dt).to(dev)
    qv = qkv[:, :hq * D].view(-1, hq, D)
    qv.copy_(q)
    kh = k.transpose(1, 2).contiguous().transpose(1, 2).to(dev)
    vh = v.transpose(1, 2).contiguous().transpose(1, 2).to(dev)
    assert kh.stride(2) > kh.stride(1)
    wide = torch.zeros(2, table.shape[1] + 5, dtype=torch.int64)
    wide[:, :table.shape[1]] = table
    out, lse = ops.prefill_paged(qv, kh, vh, wide.to(dev)[:, :table.shape[1] + 2], sl.to(torch.int64), cu.to(dev), return_lse=True)
    assert_close(out, lse, *ref, dt, most)
    o32 = ops.prefill_paged(qv, kh, vh, table.to(dev), sl.to(dev), cu.to(dev), out=torch.empty(q.shape, device=dev))
    assert torch.equal(o32.to(dt), out)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,lens", [
    (8, 2, [1, 17, 0, 130, 64, 300]), (4, 1, [200, 3, 129]), (4, 4, [5, 260]),
    (8, 4, [1]), (2, 1, [1]), (5, 1, [1, 1, 40])])       # strides of a dimension of one are anything
def test_packed_keys(dev, dt, hq, hkv, lens):
    from peerkv_b200 import ops
    gen = torch.Generator().manual_seed(31)
    total = sum(lens)
    qkv = torch.randn(total, (hq + 2 * hkv) * D, generator=gen).to(dt)
    heads = qkv.view(total, hq + 2 * hkv, D)
    cu = offsets(lens)
    parts = []
    for i, n in enumerate(lens):
        x = heads[int(cu[i]):int(cu[i + 1])]
        parts.append(attend64(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], 1 / math.sqrt(D), 1 + torch.arange(n)))
    ref = [torch.cat(x) for x in zip(*parts)]
    g = qkv.to(dev).view(total, hq + 2 * hkv, D)
    q, k, v = g[:, :hq], g[:, hq:hq + hkv], g[:, hq + hkv:]
    out, lse = ops.prefill_packed(q, k, v, cu.to(dev), return_lse=True)
    assert_close(out, lse, *ref, dt, max(lens))
    # the same values laid out on their own, and head by head
    assert torch.equal(ops.prefill_packed(q.contiguous(), k.contiguous(), v.contiguous(), cu.to(dev)), out)
    by_head = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.prefill_packed(by_head(q), by_head(k), by_head(v), cu.to(dev)), out)


def test_packed_keys_of_other_lengths(dev):
    """Cross lengths, not causal; NaN in a neighbour's V stays with the neighbour."""
    from peerkv_b200 import ops
    gen = torch.Generator().manual_seed(33)
    dt, nq, nk = torch.float16, [3, 100, 20], [50, 129, 77]
    q = torch.randn(sum(nq), 4, D, generator=gen).to(dt)
    k, v = torch.randn(sum(nk), 4, D, generator=gen).to(dt), torch.randn(sum(nk), 4, D, generator=gen).to(dt)
    cq, ck = offsets(nq), offsets(nk)
    v[int(ck[1]):int(ck[2])] = float("nan")
    out, lse = ops.prefill_packed(q.to(dev), k.to(dev), v.to(dev), cq.to(dev), ck.to(dev), causal=False, return_lse=True)
    for i in (0, 2):
        r, c = slice(int(cq[i]), int(cq[i + 1])), slice(int(ck[i]), int(ck[i + 1]))
        ref = attend64(q[r], k[c], v[c], 1 / math.sqrt(D), torch.full((nq[i],), nk[i]))
        assert_close(out[r], lse[r], *ref, dt, max(nk))


def prefix_case(groups, suffix, hq, hkv, page, dt, seed):
    gen = torch.Generator().manual_seed(seed)
    size, plen = [g[0] for g in groups], [g[1] for g in groups]
    B = sum(size)
    slen = torch.randint(0, suffix + 1, (B,), generator=gen).tolist()
    k, v, table, ks, vs = fill_pool(plen + slen, page, hkv, dt, gen)
    q = torch.randn(B, hq, D, generator=gen).to(dt)
    parts, b = [], 0
    for g, n in enumerate(size):
        for _ in range(n):
            kk, vv = torch.cat([ks[g], ks[len(size) + b]]), torch.cat([vs[g], vs[len(size) + b]])
            parts.append(attend64(q[b:b + 1], kk, vv, 1 / math.sqrt(D), torch.tensor([kk.shape[0]])))
            b += 1
    ref = [torch.cat(x) for x in zip(*parts)]
    table = table.clamp(min=0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    return q, k, v, table[:len(size)], i32(plen), table[len(size):], i32(slen), offsets(size), ref, max(plen) + suffix


@pytest.mark.parametrize("dt,hq,hkv,groups,suffix", [
    (torch.bfloat16, 8, 2, [(1, 1)], 1), (torch.bfloat16, 8, 2, [(4, 2048)], 40), (torch.float16, 8, 2, [(33, 1000)], 300),
    (torch.bfloat16, 16, 2, [(70, 513)], 17), (torch.float16, 6, 2, [(5, 100), (1, 0), (40, 3001), (2, 16)], 64),
    (torch.bfloat16, 2, 2, [(150, 700), (130, 1)], 20), (torch.bfloat16, 32, 8, [(3, 20000)], 0)])
def test_shared_prefix(dev, dt, hq, hkv, groups, suffix):
    from peerkv_b200 import ops
    q, k, v, pt, pl, bt, sl, go, ref, most = prefix_case(groups, suffix, hq, hkv, 16, dt, hq + suffix)
    g = [x.to(dev) for x in (q, k, v, pt, pl, bt, sl, go)]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out, lse = ops.decode_shared_prefix(*g[:7], group_offsets=g[7], return_lse=True, status=status)
    # the own tokens' 16-bit-free partial is folded in fp32: same bounds
    assert_close(out, lse, *ref, dt, most)
    assert status.item() == 0
    if len(groups) == 1:
        again = ops.decode_shared_prefix(*g[:3], g[3][0], g[4], *g[5:7])
        assert torch.equal(again, out)


def test_same_result_every_time_and_on_any_stream(dev):
    """No result depends on what ran before, on the stream or on calls in flight beside it."""
    from peerkv_b200 import ops
    a = [x.to(dev) if torch.is_tensor(x) else x for x in paged_case([(90, 700), (1, 5000), (200, 200)], 8, 2, 16, torch.bfloat16, 41)[:6]]
    b = [x.to(dev) if torch.is_tensor(x) else x for x in paged_case([(400, 1400)], 8, 2, 16, torch.bfloat16, 42)[:6]]
    ra, rb = ops.prefill_paged(*a, return_lse=True), ops.prefill_paged(*b, return_lse=True)
    torch.cuda.synchronize()
    n_a, n_b = int(a[5][-1]), int(b[5][-1])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            got.append((ra, n_a, ops.prefill_paged(*a, return_lse=True)))
        with torch.cuda.stream(s2):
            got.append((rb, n_b, ops.prefill_paged(*b, return_lse=True)))
    torch.cuda.synchronize()
    for want, n, g in got:
        assert torch.equal(g[0][:n], want[0][:n]) and torch.equal(g[1][:n], want[1][:n])


def test_captured_and_replayed(dev):
    """Two graphs captured from one state, replayed in turn with new lengths and contents."""
    from peerkv_b200 import ops
    q, k, v, table, sl, cu, _, _ = [x.to(dev) if torch.is_tensor(x) else x for x in
                                    paged_case([(90, 700), (4, 2000)], 8, 2, 16, torch.bfloat16, 51)]
    pt, pl = table[:1].clone(), torch.tensor([640], dtype=torch.int32, device=dev)
    qd = q[:6].contiguous()
    bt, own = table[1:2].expand(6, -1).contiguous(), torch.arange(6, dtype=torch.int32, device=dev)
    shard = ops.Shard(dev, 8, 8)
    ops.prefill_paged(q, k, v, table, sl, cu)
    ops.decode_shared_prefix(qd, k, v, pt, pl, bt, own, shard=shard,
                             group_offsets=torch.tensor([0, 6], dtype=torch.int32, device=dev))
    go = torch.tensor([0, 6], dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = ops.prefill_paged(q, k, v, table, sl, cu)
    with torch.cuda.graph(g2):
        o2 = ops.decode_shared_prefix(qd, k, v, pt, pl, bt, own, shard=shard, group_offsets=go)
    rows = int(cu[-1])
    for step in range(3):
        sl[0] = 700 - 100 * step
        own.add_(step)
        q.mul_(1.0 if step == 0 else 0.5)
        g1.replay(); g2.replay()
        w1, w2 = ops.prefill_paged(q, k, v, table, sl, cu), ops.decode_shared_prefix(
            qd, k, v, pt, pl, bt, own, shard=shard, group_offsets=go)
        torch.cuda.synchronize()
        assert torch.equal(o1[:rows], w1[:rows]) and torch.equal(o2, w2)
    del g1, g2


def test_shared_prefix_sees_what_was_written_right_before(dev):
    """Every input is overwritten in place right before each call, eagerly and in a replayed graph:
    the prefix kernel, which starts before the decode kernel has ended, reads none of the old values."""
    from peerkv_b200 import ops
    cases = [prefix_case([(size, plen)], 40, 8, 2, 16, torch.bfloat16, 60 + i)
             for i, (size, plen) in enumerate([(9, 1500), (9, 700), (9, 1501), (9, 33)])]
    pages = max(c[1].shape[0] for c in cases)
    cols = [max(c[j].shape[1] for c in cases) for j in (3, 5)]

    def pad(x, shape):
        y = torch.zeros(shape, dtype=x.dtype)
        y[tuple(slice(n) for n in x.shape)] = torch.nan_to_num(x) if x.is_floating_point() else x
        return y.to(dev)
    sets = [[c[0].to(dev), pad(c[1], (pages, *c[1].shape[1:])), pad(c[2], (pages, *c[2].shape[1:])),
             pad(c[3], (1, cols[0])), c[4].to(dev), pad(c[5], (9, cols[1])), c[6].to(dev)] for c in cases]
    live = [x.clone() for x in sets[0]]
    go = cases[0][7].to(dev)
    shard = ops.Shard(dev, 9, 8)

    def refill(i):
        for x, y in zip(live, sets[i % 4]):
            x.copy_(y)

    def call():
        return ops.decode_shared_prefix(*live, group_offsets=go, return_lse=True, shard=shard)
    got = []
    for i in range(24):
        refill(i)
        got.append(call())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = call()
    for i in range(24):
        refill(i)
        graph.replay()
        got.append([x.clone() for x in res])
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        assert_close(out, lse, *cases[i % 4][8], torch.bfloat16, cases[i % 4][9])
    del graph


def test_bad_pages_set_the_status_bit(dev):
    from peerkv_b200 import ops
    q, k, v, table, sl, cu, ref, most = paged_case([(40, 300), (16, 64)], 8, 2, 16, torch.bfloat16, 61)
    table[0, 3], table[0, 5] = -4, 1 << 20
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out, lse = ops.prefill_paged(q.to(dev), torch.nan_to_num(k).to(dev), torch.nan_to_num(v).to(dev), table.to(dev), sl.to(dev), cu.to(dev), return_lse=True,
                                 status=status)
    assert status.item() == 2
    assert_close(out[40:56], lse[40:56], *[r[40:56] for r in ref], torch.bfloat16, most)


def test_nothing_to_do(dev):
    from peerkv_b200 import ops
    pool = torch.zeros(4, 16, 2, D, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(0, 8, D, dtype=torch.bfloat16, device=dev)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    assert ops.prefill_paged(q, pool, pool, i(0)[None], i(5), i(0, 0)).shape == (0, 8, D)
    q = torch.randn(3, 8, D, device=dev).bfloat16()
    out = torch.full_like(q, 5.0)
    ops.prefill_paged(q, pool, pool, i(0)[None], i(5), i(0, 0), out=out)         # no row belongs to a sequence
    assert (out == 5.0).all()
    o, l = ops.prefill_paged(q, pool[:0], pool[:0], i(0)[None], i(0), i(0, 3), return_lse=True)   # an empty pool
    assert (o == 0).all() and torch.isneginf(l).all()
    e = torch.zeros(0, 2, D, dtype=torch.bfloat16, device=dev)
    o, l = ops.prefill_packed(q, e, e, i(0, 3), i(0, 0), return_lse=True)
    assert (o == 0).all() and torch.isneginf(l).all()
    z = torch.zeros(0, 8, D, dtype=torch.bfloat16, device=dev)
    assert ops.decode_shared_prefix(z, pool, pool, i(0)[None], i(5), i()[None].view(0, 1), i()).shape == (0, 8, D)
