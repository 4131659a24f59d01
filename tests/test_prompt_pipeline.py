"""The barriers of the prompt-attention kernel, warp by warp, on the host: loaders, the two matrix warps with their
turns, the two softmax warpgroups with the hand-over of P, and copies and products that end when they
like.  Whatever the order in which they get on, everything ends, and no wait takes one round of a
barrier for another."""
import random

import pytest

from test_prompt_schedule import K_SLOTS, V_SLOTS

WORK_RING = 4


class Barrier:
    """An mbarrier: `count` arrivals complete a phase; a wait names the parity of the phase it wants."""

    def __init__(self, count):
        self.count, self.pending, self.done = count, count, 0

    def arrive(self, n=1):
        for _ in range(n):
            self.pending -= 1
            if self.pending == 0:
                self.pending, self.done = self.count, self.done + 1

    def passes(self, parity):
        return (self.done & 1) != parity


class Machine:
    def __init__(self):
        self.b = {"q_full": Barrier(1), "q_empty": Barrier(2), "x_ready": Barrier(4), "x_done": Barrier(4)}
        for kv, n in (("K", K_SLOTS), ("V", V_SLOTS)):
            for s in range(n):
                self.b["full", kv, s], self.b["empty", kv, s] = Barrier(1), Barrier(2)
        for w in range(2):
            self.b["s_full", w], self.b["o_full", w], self.b["turn", w] = Barrier(1), Barrier(1), Barrier(1)
            self.b["p_full", w, 0], self.b["p_full", w, 1] = Barrier(4), Barrier(4)
        for i in range(WORK_RING):
            self.b["w_full", i], self.b["w_empty", i] = Barrier(1), Barrier(11)
        # copies end in any order; the products of one warp in order, and its commits behind them
        self.copies, self.products = [], [[], []]
        self.ring = [None] * WORK_RING
        # what stands in S_w; halves of P written into it; products into O_w under way; O_w is being read
        self.s, self.p, self.o_busy, self.o_read = ["idle", "idle"], [0, 0], [0, 0], [False, False]


def wait(bar, parity, nth):
    """`nth`: which completion (from 1; 0: none needed) this wait is for."""
    return ("wait", bar, parity & 1, nth)


def slot(kv, i):
    n = K_SLOTS if kv == "K" else V_SLOTS
    return i % n, i // n


def take(m, n, arrivals):
    """Every reader warp of the work list; returns the item."""
    yield wait(("w_full", n % WORK_RING), n // WORK_RING, n // WORK_RING + 1)
    item = m.ring[n % WORK_RING]
    m.b["w_empty", n % WORK_RING].arrive(arrivals)
    return item


def loader(m, kv, items):
    n_tile = n_q = n = 0
    while True:
        if kv == "K":
            yield wait(("w_empty", n % WORK_RING), (n // WORK_RING) ^ 1, n // WORK_RING)
            item = items[n]
            m.ring[n % WORK_RING] = item
            m.b["w_full", n % WORK_RING].arrive()
        else:
            item = yield from take(m, n, 1)
        n += 1
        if item is None:
            return
        if item[0] == 0:
            continue
        if kv == "K":
            yield wait("q_empty", n_q ^ 1, n_q)
            n_q += 1
            m.copies.append("q_full")
        for _ in range(item[0]):
            s, r = slot(kv, n_tile)
            yield wait(("empty", kv, s), r ^ 1, r)
            m.copies.append(("full", kv, s))
            n_tile += 1


def matrix(m, w):
    n = n_tile = n_q = n_p = n_turn = 0

    def full(kv, i):
        s, r = slot(kv, i)
        return wait(("full", kv, s), r, r + 1)

    def give_back(kv, i):
        return ("empty", kv, slot(kv, i)[0])
    while True:
        item = yield from take(m, n, 1)
        n += 1
        if item is None:
            return
        n_tiles, two = item
        if n_tiles == 0:
            continue
        yield wait("q_full", n_q, n_q + 1)
        n_q += 1
        base, n_tile = n_tile, n_tile + n_tiles
        ahead = 1 if two else 2
        for t in range(n_tiles + ahead):
            i = t - ahead
            mine = two or (t & 1) == w
            if i >= 0:
                yield full("V", base + i)
                if mine:
                    for half in range(2):
                        yield wait(("p_full", w, half), n_p, n_p + 1)
                        if two and half == 0:
                            yield wait(("turn", w), n_turn ^ (1 if w == 0 else 0), n_turn + w)
                            n_turn += 1
                        assert m.s[w] == "scores" and m.p[w] > half, "a product before its half of P"
                        assert not m.o_read[w], "a product into O while the epilogue reads it"
                        m.products[w].append(("pv", half))
                        m.o_busy[w] += 1
                    n_p += 1
                    m.s[w] = "idle"                      # the next scores follow the products that read P
                    m.products[w].append(("commit", give_back("V", base + i)))
                    if i + (1 if two else 2) >= n_tiles:
                        m.products[w].append(("commit", ("o_full", w)))
                else:
                    m.b[give_back("V", base + i)].arrive()
            if t < n_tiles:
                yield full("K", base + t)
                if mine:
                    assert m.s[w] == "idle", "scores over a P that is still needed"
                    m.s[w], m.p[w] = "scores", 0
                    m.products[w].append(("qk", None))
                    m.products[w].append(("commit", ("s_full", w)))
                    m.products[w].append(("commit", give_back("K", base + t)))
                else:
                    m.b[give_back("K", base + t)].arrive()
                if t + 1 == n_tiles:
                    m.products[w].append(("commit", "q_empty"))
            if two and i >= 0:
                m.b["turn", w ^ 1].arrive()


def softmax(m, w):
    n = n_s = n_o = n_x = 0
    while True:
        item = yield from take(m, n, 4)
        n += 1
        if item is None:
            return
        n_tiles, two = item
        steps = n_tiles if two else (n_tiles + 1 - w) >> 1
        for _ in range(steps):
            yield wait(("s_full", w), n_s, n_s + 1)
            n_s += 1
            assert m.s[w] == "scores" and m.p[w] == 0 and m.o_busy[w] == 0, "O is rescaled while a product writes it"
            for half in range(2):
                yield ("step",)
                m.p[w] += 1
                m.b["p_full", w, half].arrive(4)
        if steps:
            yield wait(("o_full", w), n_o, n_o + 1)
            n_o += 1
        assert m.o_busy[w] == 0
        m.o_read[w] = True
        yield ("step",)
        if not two and n_tiles > 1:                       # stream 0 adds up the accumulators of both
            if w == 1:
                m.b["x_ready"].arrive(4)
                yield wait("x_done", n_x, n_x + 1)
            else:
                yield wait("x_ready", n_x, n_x + 1)
                assert m.o_read[1] and m.o_busy[1] == 0
                yield ("step",)
                assert m.o_read[1]
                m.b["x_done"].arrive(4)
            n_x += 1
        m.o_read[w] = False


def simulate(items, rng):
    m = Machine()
    work = list(items) + [None]
    actors = [loader(m, "K", work), loader(m, "V", work), matrix(m, 0), matrix(m, 1), softmax(m, 0), softmax(m, 1)]
    # some warps run far ahead of others, differently in every run
    speed = [rng.choice([1, 1, 5, 50]) for _ in range(len(actors) + 3)]
    at = [next(a, None) for a in actors]

    def ready(x):
        if x is None:
            return False
        if x[0] == "wait":
            return m.b[x[1]].passes(x[2])
        return True
    while any(x is not None for x in at):
        moves = [i for i in range(len(actors)) if ready(at[i])]
        if m.copies:
            moves.append(len(actors))
        moves += [len(actors) + 1 + w for w in range(2) if m.products[w]]
        assert moves, ("nothing can move", items, at)
        i = rng.choices(moves, [speed[j] for j in moves])[0]
        if i < len(actors):
            if at[i][0] == "wait":
                assert m.b[at[i][1]].done == at[i][3], ("a wait took another round for its own", at[i], m.b[at[i][1]].done)
            at[i] = next(actors[i], None)
        elif i == len(actors):
            m.b[m.copies.pop(rng.randrange(len(m.copies)))].arrive()
        else:
            w = i - len(actors) - 1
            kind, what = m.products[w].pop(0)
            if kind == "pv":
                m.o_busy[w] -= 1
            elif kind == "commit":
                m.b[what].arrive()
    assert not m.copies and not m.products[0] and not m.products[1] or all(k == "commit" for p in m.products for k, _ in p)


@pytest.mark.parametrize("seed", range(150))
def test_everything_ends_and_no_round_is_mistaken(seed):
    rng = random.Random(seed)
    items = [(rng.choice([0, 1, 1, 2, 3, 4, 5, 9]), rng.random() < 0.5) for _ in range(rng.randint(1, 9))]
    simulate(items, rng)


@pytest.mark.parametrize("two", [False, True])
def test_runs_of_one_kind(two):
    for n in range(7):
        simulate([(n, two)] * 12, random.Random(n))


@pytest.mark.parametrize("break_it", ["a reader short", "slots of one reader", "half of the turns"])
def test_the_model_is_not_blind(monkeypatch, break_it):
    """Planted mistakes in the model: a work ring that waits for a reader that is not there, V slots that are filled
    again once one of the two streams has given them back, a stream that gets every other turn only."""
    init = Machine.__init__

    def broken(self):
        init(self)
        if break_it == "a reader short":
            for i in range(WORK_RING):
                self.b["w_empty", i] = Barrier(12)
        elif break_it == "slots of one reader":
            for s in range(V_SLOTS):
                self.b["empty", "V", s] = Barrier(1)
        else:
            self.b["turn", 1] = Barrier(2)
    monkeypatch.setattr(Machine, "__init__", broken)
    with pytest.raises(AssertionError):
        for seed in range(20):
            simulate([(5, True)] * 8, random.Random(seed))
