"""The work split of the prompt-attention kernel, restated on the host: every KV tile of every
item is done exactly once, a CTA's pieces never share a workspace slot, the join finds exactly
the pieces that were written, and the two streams of products never wait for a tile that waits
for them."""
import os
import random
import re

import numpy as np
import pytest

SRC = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "peerkv_b200", "csrc",
                        "prompt_kernel.cuh")).read()


def const(name):
    return int(re.search(r"constexpr int [^;]*?\b%s = (\d+)" % name, SRC).group(1))


ITEM_COST, MIN_PIECE, KEYS, ROWS, K_SLOTS, V_SLOTS = (
    const(n) for n in ("kPaItemCost", "kPaMinPiece", "kPaKeys", "kPaRows", "kPaKSlots", "kPaVSlots"))


def items(seqs, hkv, group, causal):
    """(name on the cost axis, cost, KV tiles, tokens) of every item in order."""
    tt, a, out = 2 * (ROWS // group), 0, []
    for n, length in seqs:
        tiles = -(-n // tt)
        for _ in range(hkv):
            for t in range(tiles):
                w = 3 if n > tt // 2 else 2
                cost = w * (max(length - n, 0) if causal else length) + ITEM_COST + (w * tt * (t + 1) if causal else 0)
                n_tok = min(tt, n - t * tt)
                vis = max(0, min(length, length - n + t * tt + n_tok)) if causal else length
                out.append((a, cost, -(-vis // KEYS), n_tok))
                a += cost
    return out, a


def cut(y, cost, n):
    """As the kernel rounds it: single precision (its quotient may differ in the last bits; what
    has to hold is that all CTAs use the same ascending function)."""
    if y <= 0 or n == 0:
        return 0
    return n if y >= cost else min(n, int(np.float32(y) * (np.float32(n) / np.float32(cost))))


def piece(total, n_cta):
    """As the kernel rounds it, with the quotient taken 2 steps of fp32 too low or too high (the bound
    of its approximate division)."""
    q = np.float32(total) * (np.float32(1.0) / np.float32(n_cta))
    return [int(q * np.float32(1 + e * 2.0 ** -22)) + (total >> 20) + 1 for e in (-1, 0, 1)]


def pieces(its, total, grid, which):
    """Per CTA: list of (item index, kt0, kt1, slot or None when written directly), and its record."""
    n_cta = min(grid, -(-total // MIN_PIECE))
    size = piece(total, n_cta)[which]
    assert size * n_cta >= total
    work, rec = [], []
    for c in range(n_cta):
        x0, x1 = c * size, min(total, c * size + size)
        assert x1 > x0
        mine, first = [], None
        for i, (a, cost, n, _) in enumerate(its):
            if a + cost <= x0 or a >= x1:
                continue
            k0, k1 = cut(x0 - a, cost, n), cut(x1 - a, cost, n)
            if first is None:
                first = (i, x0 > a, k0, k1, n)
            if k1 > k0 or (n == 0 and x0 <= a):
                whole = k0 == 0 and k1 == n
                mine.append((i, k0, k1, None if whole else 2 * c + (0 if x0 > a else 1)))
        work.append(mine)
        rec.append(first)
    return work, rec


def join(rec, c):
    """Slots block c adds up and the item, or None."""
    i, mid, k0, k1, n = rec[c]
    if not mid or k0 >= n or (c > 1 and rec[c - 1][1] and rec[c - 1][0] == i) or (k0 == 0 and k1 == n):
        return None
    last = c
    while last + 1 < len(rec):
        j, jmid, j0, j1, jn = rec[last + 1]
        if not jmid or j != i:
            break
        if j0 == 0 and j1 == jn:
            return None
        last += 1
    slots = [2 * (c - 1) + 1] if k0 > 0 else []
    return i, slots + [2 * d for d in range(c, last + 1) if rec[d][3] > rec[d][2]]


def check(seqs, hkv, group, causal, grid):
    its, total = items(seqs, hkv, group, causal)
    if total == 0:
        return
    for which in range(3):
        check_split(its, *pieces(its, total, grid, which))


def check_split(its, work, rec):
    done = {i: [] for i in range(len(its))}
    written = {}
    for c, mine in enumerate(work):
        slots = [s for *_, s in mine if s is not None]
        assert len(set(slots)) == len(slots)
        for i, k0, k1, s in mine:
            done[i].append((k0, k1))
            if s is not None:
                written.setdefault(i, []).append(s)
    for i, (_, _, n, _) in enumerate(its):
        at = 0
        for k0, k1 in done[i]:
            assert k0 == at
            at = k1
        assert at == n and done[i], (i, n, done[i])
    joined = {}
    for c in range(1, len(rec)):
        j = join(rec, c)
        if j is not None:
            assert j[0] not in joined
            joined[j[0]] = j[1]
    assert {i: sorted(s) for i, s in joined.items()} == {i: sorted(s) for i, s in written.items()}
    assert all(len(s) > 1 for s in joined.values())


@pytest.mark.parametrize("seed", range(60))
def test_every_tile_once(seed):
    rng = random.Random(seed)
    seqs = []
    for _ in range(rng.choice([1, 1, 2, 5, 20])):
        n = rng.choice([0, 1, 1, 2, 63, 64, 65, rng.randint(1, 3000)])
        seqs.append((n, rng.choice([0, n, n // 2, n + rng.randint(0, 20000)])))
    check(seqs, rng.choice([1, 2, 8]), rng.choice([1, 3, 4, 8, 128]), rng.random() < 0.6, rng.choice([1, 7, 148]))


def test_pieces_cover_the_axis():
    rng = random.Random(1)
    for n_cta in list(range(1, 150)) + [256]:
        for total in [1, 768 * n_cta + 1, MIN_PIECE * n_cta - 5] + [int(MIN_PIECE * n_cta * 10 ** rng.uniform(0, 8)) for _ in range(20)]:
            n = min(n_cta, -(-total // MIN_PIECE))
            for size in piece(total, n):
                assert size * n >= total > size * (n - 1)


def test_edge_lengths():
    for n, length in [(1, 1), (1, 0), (3, 0), (64, 1), (300, 7), (1, 1 << 20), (4, 2048), (257, 257)]:
        for causal in (False, True):
            check([(n, length)], 8, 4, causal, 148)


def program(items, w):
    """What the matrix warp of stream w does, in order: ("K" | "V", tile, used by this stream)."""
    out, base = [], 0
    for n, two in items:
        mine = lambda i: two or (i & 1) == w
        ahead = 1 if two else 2
        out += [("K", base + i, mine(i)) for i in range(min(ahead, n))]
        for i in range(n):
            out.append(("V", base + i, mine(i)))
            if i + ahead < n:
                out.append(("K", base + i + ahead, mine(i + ahead)))
        base += n
    return out


@pytest.mark.parametrize("seed", range(40))
def test_the_two_streams_never_wait_for_each_other_for_good(seed):
    """Loads fill K slots and V slots in order; both streams give every tile back; a V product
    waits for its stream's scores, which are there once they were issued.  Steps are taken in
    random order: everything has to end, whoever runs ahead."""
    rng = random.Random(seed)
    its = [(rng.choice([1, 2, 3, 4, 5, 9]), rng.random() < 0.5) for _ in range(rng.randint(1, 6))]
    total = sum(n for n, _ in its)
    progs, at = [program(its, w) for w in range(2)], [0, 0]
    loaded, given = {"K": 0, "V": 0}, {"K": [0] * total, "V": [0] * total}
    slots = {"K": K_SLOTS, "V": V_SLOTS}
    while at[0] < len(progs[0]) or at[1] < len(progs[1]):
        moves = []
        for kind in "KV":
            f = loaded[kind]
            if f < total and (f < slots[kind] or given[kind][f - slots[kind]] == 2):
                moves.append(("load", kind))
        for w in range(2):
            if at[w] < len(progs[w]):
                kind, tile, _ = progs[w][at[w]]
                if tile < loaded[kind]:
                    moves.append(("step", w))
        assert moves, (its, at, loaded)
        what, x = rng.choice(moves)
        if what == "load":
            loaded[x] += 1
        else:
            kind, tile, _ = progs[x][at[x]]
            given[kind][tile] += 1
            at[x] += 1
    assert all(g == 2 for k in given.values() for g in k)
    for w in range(2):                                   # every tile a stream owns: scores before values, once
        for i in range(total):
            steps = [j for j, (k, t, use) in enumerate(progs[w]) if t == i and use]
            assert len(steps) in (0, 2) and (not steps or progs[w][steps[0]][0] == "K")
    assert all(any(t == i and use for pr in progs for _, t, use in pr) for i in range(total))
