"""The decode kernel's split of the tiles of own tokens, restated on the host: every tile in one CTA, in order, and no
CTA with much more than its share of what tiles and sequences cost."""
import os
import random
import re

SRC = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "peerkv_b200", "csrc",
                        "decode_kernel.cuh")).read()
SEQ_COST = int(re.search(r"constexpr int kSeqCost = (\d+)", SRC).group(1))


def bounds(tiles, n_cta):
    prefix = [0]
    for t in tiles:
        prefix.append(prefix[-1] + t)
    total, batch, out = prefix[-1], len(tiles), []
    for c in range(n_cta + 1):
        if total <= n_cta or c == n_cta:
            out.append(total if c == n_cta else min(c, total))
            continue
        x = (total + SEQ_COST * batch) * c // n_cta
        lo, hi = 0, batch
        while hi - lo > 1:
            mid = (lo + hi) >> 1
            if prefix[mid] + SEQ_COST * mid <= x:
                lo = mid
            else:
                hi = mid
        out.append(min(prefix[lo + 1], max(prefix[lo], x - SEQ_COST * (lo + 1))))
    return out, prefix


def test_bounds_ascend_and_cover():
    rng = random.Random(1)
    for _ in range(400):
        n_cta = rng.choice([1, 2, 37, 74, 148])
        batch = rng.choice([1, 2, 3, 64, 500, 4096])
        tiles = [rng.choice([0, 0, 1, 2, rng.randint(0, 70), rng.randint(0, 3000)]) for _ in range(batch)]
        b, prefix = bounds(tiles, n_cta)
        assert b[0] == 0 and b[-1] == prefix[-1] and all(x <= y for x, y in zip(b, b[1:]))
        if prefix[-1] <= n_cta:
            continue
        share = (prefix[-1] + SEQ_COST * batch) / n_cta
        for lo, hi in zip(b, b[1:]):
            # whole sequences inside, and the two that are cut
            inside = sum(1 for s in range(batch) if prefix[s] >= lo and prefix[s + 1] <= hi and tiles[s])
            assert hi - lo + SEQ_COST * inside <= share + 2 * SEQ_COST + 1
