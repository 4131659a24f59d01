"""The work split as the kernel makes it: the records and pieces that prompt_attn_kernel leaves in its workspace,
against the host's restatement of the cost axis and against 64-bit sums over the keys of each piece."""
import math

import numpy as np
import pytest
import torch

from prompt_cases import D, attend64, fill_pool, tolerances
from test_prompt_gpu import offsets
from test_prompt_schedule import KEYS, MIN_PIECE, ROWS, cut, items, piece

pytestmark = pytest.mark.gpu
REC = np.dtype([("a", "<i8"), ("mid", "<i4"), ("kt0", "<i4"), ("kt1", "<i4"), ("n", "<i4"), ("q0", "<i4"), ("n_tok", "<i4"),
                ("h", "<i4"), ("pad", "<i4")])


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def run(dev, lens, hq, hkv, dt, causal, seed):
    """Outputs, the workspace's records (of the CTAs in use) and (m, l) pieces [2 * CTAs, 256, 2], NaN where
    nothing was written, and the inputs."""
    from peerkv_b200 import ops
    gen = torch.Generator().manual_seed(seed)
    new, full = [p[0] for p in lens], [p[1] for p in lens]
    k, v, table, ks, vs = fill_pool(full, 16, hkv, dt, gen)
    q = torch.randn(sum(new), hq, D, generator=gen).to(dt)
    g = [x.to(dev) for x in (q, k, v, table.clamp(min=0), torch.tensor(full, dtype=torch.int32), offsets(new))]
    ws = ops._prompt_workspace(dev)
    ws.fill_(255)
    out = torch.empty_like(g[0])
    ops._prompt_call(g[0], ops.paged_view(g[1], g[2]), 1 / math.sqrt(D), causal, out, None, g[5], len(lens), None,
                     block_table=g[3], seq_lens=g[4], ws=ws)
    torch.cuda.synchronize()
    grid = torch.cuda.get_device_properties(dev).multi_processor_count
    o_bytes, ml_bytes = 2 * grid * 32 * 256 * 16, 2 * grid * 256 * 8
    ml = ws[o_bytes:o_bytes + ml_bytes].view(torch.float32).view(2 * grid, 256, 2).cpu()
    raw = ws[o_bytes + ml_bytes:o_bytes + ml_bytes + (grid + 1) * REC.itemsize].cpu().numpy()
    rec = raw.view(REC)
    return rec[:rec[grid]["kt0"]], ml, q, ks, vs, grid


def item_rows(lens, hkv, group):
    """(sequence, kv-head, first token, first packed row) of every item, in the order of the cost axis."""
    tt, out, row = 2 * (ROWS // group), [], 0
    for s, (n, _) in enumerate(lens):
        out += [(s, h, t * tt, row + t * tt) for h in range(hkv) for t in range(-(-n // tt))]
        row += n
    return out


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,hq,hkv,causal", [
    ([(300, 1500), (1, 20000), (70, 70), (0, 9), (5, 3), (1, 1)], 8, 2, True), ([(6, 9000), (40, 130)], 8, 2, False),
    ([(3, 5000)] * 3, 5, 1, True), ([(1 + 37 * i % 60, 30 + 211 * i % 900) for i in range(60)], 4, 4, True),
    ([(2000, 2000)], 2, 2, True), ([(9, 9)], 8, 8, True)])
def test_records_and_pieces(dev, dt, lens, hq, hkv, causal):
    group = hq // hkv
    rec, ml, q, ks, vs, grid = run(dev, lens, hq, hkv, dt, causal, len(lens) * 7 + hq)
    its, total = items(lens, hkv, group, causal)
    where = item_rows(lens, hkv, group)
    assert len(its) == len(where) and len(rec) == min(grid, -(-total // MIN_PIECE))
    starts = np.array([a for a, *_ in its])

    def firsts(size):                                   # index of each CTA's first item
        return [int(np.searchsorted(starts, c * size, side="right")) - 1 for c in range(len(rec))]
    # the length of a piece is one of the three that the approximate quotient allows
    fits = []
    for size in piece(total, len(rec)):
        first = firsts(size)
        if all(starts[i] == r["a"] and (c * size > starts[i]) == bool(r["mid"]) for c, (i, r) in enumerate(zip(first, rec))):
            fits.append((size, first))
    assert fits, "the CTAs do not start where the cost axis says"
    size, first = fits[0]
    chain = {}                                          # item -> [(slot, kt0, kt1)]
    for c, (i, r) in enumerate(zip(first, rec)):
        a, cost, n, n_tok = its[i]
        assert (r["n"], r["n_tok"], r["h"], r["q0"]) == (n, n_tok, where[i][1], where[i][3])
        # the kernel's own quotient, in single precision, may fall a tile beside the host's
        assert abs(int(r["kt0"]) - cut(c * size - a, cost, n)) <= 1 and abs(int(r["kt1"]) - cut((c + 1) * size - a, cost, n)) <= 1
        assert 0 <= r["kt0"] <= r["kt1"] <= n
        chain.setdefault(i, []).append((2 * c + (0 if r["mid"] else 1), int(r["kt0"]), int(r["kt1"])))
        # a CTA's last item goes on in the next one's record
        if c + 1 < len(rec) and rec[c + 1]["mid"] and first[c + 1] != i:
            chain.setdefault(first[c + 1], []).append((2 * c + 1, 0, int(rec[c + 1]["kt0"])))
    for i, parts in chain.items():
        parts.sort(key=lambda x: (x[1], x[2]))
        at = 0
        for _, k0, k1 in parts:
            assert k0 == at, "a tile twice or not at all"
            at = k1
        assert at == its[i][2]
    written = (~torch.isnan(ml[..., 1])).any(1)
    expected = {s: (i, k0, k1) for i, parts in chain.items() for s, k0, k1 in parts
                if k1 > k0 and not (k0 == 0 and k1 == its[i][2])}
    assert set(expected) <= set(written.nonzero()[:, 0].tolist()), "a piece that the join reads was not written"
    scale, tok_tile = 1 / math.sqrt(D), ROWS // group
    for s, (i, k0, k1) in expected.items():
        seq, h, t0, row0 = where[i]
        n_new, L = lens[seq]
        n_tok = its[i][3]
        toks = torch.arange(n_tok)
        see = (L - n_new + 1 + t0 + toks if causal else torch.full((n_tok,), L)).clamp(min=0)
        lo, hi = k0 * KEYS, min(k1 * KEYS, L)
        rows = q[row0:row0 + n_tok, h * group:(h + 1) * group]
        _, lse, mag, big = attend64(rows, ks[seq][lo:hi, h:h + 1], vs[seq][lo:hi, h:h + 1], scale, (see - lo).clamp(0, hi - lo))
        at = (toks // tok_tile * ROWS)[:, None] + (toks % tok_tile)[:, None] * group + torch.arange(group)
        m, l = ml[s][at].double().unbind(-1)
        got = torch.where(l > 0, (m + l.log2()) * math.log(2), torch.full_like(l, -math.inf))
        seen = torch.isfinite(lse)
        assert torch.equal(torch.isfinite(got), seen)
        _, l_tol = tolerances(mag, lse, mag, big, dt, hi - lo)
        # (m carries the scale's rounding in base 2: one more half step of fp32)
        assert ((got - lse).abs() <= l_tol + 2.0 ** -23 * lse.abs())[seen].all()
