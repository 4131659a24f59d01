"""The serving operators around the sharded cache, as they are timed: prompt attention over
packed sequences, decode attention for batches that share a long prefix, and the append that
norms, rotates and stores new tokens.

`own` selects what `run` does: False computes the operator from elementary torch operations
in fp32 (angles in fp64), True makes the library's calls.  Every case is a dict of plain
values; lengths are written "new:cached" per sequence (new tokens, tokens in the cache with
the new ones counted), joined by commas.
"""
import math

import numpy as np
import torch

own = False
D = 128


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def listed():
    return [
        # A prefill batch of short prompts, one of a single token, straight from the projection (no pages yet).
        {"name": "prompt-packed-short", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 0,
         "lens": "1:1,17:17,100:100,128:128,250:250,333:333,64:64,500:500"},
        # A server's usual prefill step: prompts of different lengths into a paged cache.
        {"name": "prompt-ragged", "op": "prompt", "dtype": "fp16", "hq": 32, "hkv": 8, "page": 16,
         "lens": "4096:4096,2900:2900,1777:1777,1024:1024,600:600,333:333,129:129,2048:2048"},
        # One long prompt at once.
        {"name": "prompt-8k", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 16, "lens": "8192:8192"},
        # A chunk of a very long prompt: 2048 new tokens behind 63488 that are in the cache already.
        {"name": "prompt-chunk-64k", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 16, "lens": "2048:65536"},
        # Continuous batching: one chunk rides with sequences that decode one token each.
        {"name": "prompt-mixed", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 32,
         "lens": "512:1536," + ",".join("1:%d" % (97 + 173 * i) for i in range(23))},
        # A handful of requests behind one system prompt.
        {"name": "prefix-b4", "op": "prefix", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 16, "groups": "4:2048",
         "suffix": 128},
        # Many samples of one long document.
        {"name": "prefix-b64-32k", "op": "prefix", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 16, "groups": "64:32768",
         "suffix": 1024},
        # Several prompts in one batch, each with its own set of requests; one request shares nothing.
        {"name": "prefix-groups", "op": "prefix", "dtype": "fp16", "hq": 64, "hkv": 8, "page": 16,
         "groups": "17:4097,40:12000,1:0,70:8192", "suffix": 300},
        # The append of one decode step, small batch (latency).
        {"name": "append-decode-b4", "op": "append", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 16, "tokens": 4,
         "rot": 128, "interleaved": False, "norm": True, "far": 1048575, "kv": "16"},
        # A large decode batch: half of each head rotated, interleaved pairs, no norm.
        {"name": "append-decode-b256", "op": "append", "dtype": "fp16", "hq": 32, "hkv": 8, "page": 16, "tokens": 256,
         "rot": 64, "interleaved": True, "norm": False, "far": 131071, "kv": "16"},
        # The append of a prefill step.
        {"name": "append-prompt-8k", "op": "append", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 16, "tokens": 8192,
         "rot": 128, "interleaved": False, "norm": True, "far": 131071, "kv": "16"},
        # The same into an 8-bit cache; what the codes stand for is returned.
        {"name": "append-prompt-fp8", "op": "append", "dtype": "bf16", "hq": 32, "hkv": 8, "page": 16, "tokens": 2047,
         "rot": 128, "interleaved": False, "norm": True, "far": 65535, "kv": "fp8"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prefix", "append"])
    hkv = rng.choice([1, 2, 4, 8, 8])
    c = {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "hq": hkv * rng.choice([1, 2, 4, 4, 5, 8]), "hkv": hkv,
         "page": rng.choice([16, 16, 32, 64])}
    if op == "prompt":
        n = _spread(rng, 1, 24)
        most = min(8192, int(math.sqrt(2.0e9 / (n * c["hq"]))))
        lens = []
        for _ in range(n):
            new = _spread(rng, 1, most) if rng.random() < 0.7 else 1
            lens.append((new, new + (_spread(rng, 1, most) if rng.random() < 0.4 else 0)))
        if rng.random() < 0.3:
            c["page"] = 0
            lens = [(new, new) for new, _ in lens]
        c["lens"] = ",".join("%d:%d" % p for p in lens)
    elif op == "prefix":
        groups = [(_spread(rng, 1, 96), _spread(rng, 64, 32768) if rng.random() < 0.9 else 0)
                  for _ in range(rng.choice([1, 1, 2, 3]))]
        c["groups"] = ",".join("%d:%d" % p for p in groups)
        c["suffix"] = _spread(rng, 1, 1024)
    else:
        c.update(tokens=_spread(rng, 1, 8192), rot=rng.choice([32, 64, 96, 128, 128]),
                 interleaved=rng.random() < 0.4, norm=rng.random() < 0.6, far=_spread(rng, 1000, 1048575),
                 kv=rng.choice(["16", "16", "fp8"]))
    return c


def _pairs(text):
    return [tuple(int(x) for x in p.split(":")) for p in text.split(",")]


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def _pages(rng, lens, page, spare=3):
    """Page ids of sequences of `lens` tokens: a shuffled table [n, most pages] and the pool's page count."""
    need = [(n + page - 1) // page for n in lens]
    ids = rng.permutation(sum(need) + spare)
    table = np.zeros((len(lens), max(1, max(need))), dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, sum(need) + spare


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.RandomState(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
    hq, hkv, page = case["hq"], case["hkv"], case["page"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dt)

    def ints(x, kind=torch.int32):
        return torch.as_tensor(np.asarray(x), dtype=kind, device=dev)

    s = {"op": case["op"], "hq": hq, "hkv": hkv, "scale": 1.0 / math.sqrt(D)}
    if case["op"] == "prompt":
        lens = _pairs(case["lens"])
        new, full = [p[0] for p in lens], [p[1] for p in lens]
        total = sum(new)
        s["q"] = normal(total, hq, D)
        s["cu"] = ints(np.concatenate([[0], np.cumsum(new)]))
        s["seq_lens"] = ints(full)
        # where every packed row lies in the padded batch
        s["row_seq"] = ints(np.repeat(np.arange(len(new)), new), torch.int64)
        s["row_pos"] = ints(np.concatenate([np.arange(n) for n in new]), torch.int64)
        s["most_new"], s["most_full"] = max(new), max(full)
        s["page"] = page
        if page:
            table, n_pages = _pages(rng, full, page)
            s["table"] = ints(table)
            s["k"], s["v"] = normal(n_pages, page, hkv, D), normal(n_pages, page, hkv, D)
        else:
            s["k"], s["v"] = normal(total, hkv, D), normal(total, hkv, D)
    elif case["op"] == "prefix":
        groups = _pairs(case["groups"])
        size, plen = [g[0] for g in groups], [g[1] for g in groups]
        batch = sum(size)
        suf = rng.randint(0, case["suffix"] + 1, batch)
        suf[rng.randint(0, batch)] = case["suffix"]
        table, n_pages = _pages(rng, list(plen) + list(suf), page)
        s["prefix_table"], s["table"] = ints(table[:len(size)]), ints(table[len(size):, :max(1, -(-case["suffix"] // page))])
        s["prefix_lens"], s["seq_lens"] = ints(plen), ints(suf)
        s["offsets"] = ints(np.concatenate([[0], np.cumsum(size)]))
        s["row_group"] = ints(np.repeat(np.arange(len(size)), size), torch.int64)
        s["row_pos"] = ints(np.concatenate([np.arange(n) for n in size]), torch.int64)
        s["most_size"], s["most_prefix"], s["most_suffix"] = max(size), max(plen), int(max(suf))
        s["page"] = page
        s["q"] = normal(batch, hq, D)
        s["k"], s["v"] = normal(n_pages, page, hkv, D), normal(n_pages, page, hkv, D)
    else:
        t, rot = case["tokens"], case["rot"]
        s["qkv"] = normal(t, (hq + 2 * hkv) * D)
        s["positions"] = ints(rng.randint(0, case["far"] + 1, t), torch.int64)
        s["inv_freq"] = (1.0 / (500000.0 ** (torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot))).float()
        s["interleaved"], s["eps"] = bool(case["interleaved"]), 1e-6
        s["wq"], s["wk"] = ((1 + 0.1 * normal(D).float()).to(dt), (1 + 0.1 * normal(D).float()).to(dt)) \
            if case["norm"] else (None, None)
        n_pages = -(-t // page) + 2
        s["slots"] = ints(rng.permutation(n_pages * page)[:t], torch.int64)
        s["q_out"] = torch.zeros(t, hq, D, dtype=dt, device=dev)
        s["kv"] = case["kv"]
        if case["kv"] == "16":
            s["k"], s["v"] = normal(n_pages, page, hkv, D), normal(n_pages, page, hkv, D)
            s["k_scale"] = s["v_scale"] = None
        else:
            for n in ("k", "v"):
                s[n] = torch.zeros(n_pages, page, hkv, D, dtype=torch.float8_e4m3fn, device=dev)
                s[n + "_scale"] = torch.ones(n_pages, page, hkv, dtype=torch.float16, device=dev)
    return s


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def run(s):
    if own:
        from peerkv_b200 import ops
        if s["op"] == "prompt":
            if s["page"]:
                return ops.prefill_paged(s["q"], s["k"], s["v"], s["table"], s["seq_lens"], s["cu"], scale=s["scale"],
                                         return_lse=True)
            return ops.prefill_packed(s["q"], s["k"], s["v"], s["cu"], scale=s["scale"], return_lse=True)
        if s["op"] == "prefix":
            return ops.decode_shared_prefix(s["q"], s["k"], s["v"], s["prefix_table"], s["prefix_lens"], s["table"],
                                            s["seq_lens"], group_offsets=s["offsets"], scale=s["scale"])
        ops.norm_rope_append(s["qkv"], s["positions"], s["inv_freq"], s["hq"], s["hkv"], s["q_out"], s["k"], s["v"],
                             s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"], q_weight=s["wq"],
                             k_weight=s["wk"], eps=s["eps"], interleaved=s["interleaved"])
        return _append_out(s)
    return {"prompt": _plain_prompt, "prefix": _plain_prefix, "append": _plain_append}[s["op"]](s)


def _append_out(s):
    if s["kv"] == "16":
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    t = s["q_out"].dtype
    return {"q": s["q_out"], "k": (s["k"].float() * s["k_scale"].float()[..., None]).to(t),
            "v": (s["v"].float() * s["v_scale"].float()[..., None]).to(t)}


def _plain_prompt(s):
    q, hq, hkv = s["q"], s["hq"], s["hkv"]
    cu, full = s["cu"].long(), s["seq_lens"].long()
    new = cu[1:] - cu[:-1]
    n, mq, mk = new.numel(), s["most_new"], s["most_full"]
    at = torch.arange(mq, device=q.device)
    qp = q[(cu[:-1, None] + at).clamp(max=q.shape[0] - 1)].float().view(n, mq, hkv, hq // hkv, D)
    if s["page"]:
        k = s["k"][s["table"].long()].flatten(1, 2)[:, :mk].float()
        v = s["v"][s["table"].long()].flatten(1, 2)[:, :mk].float()
    else:
        rows = (cu[:-1, None] + torch.arange(mk, device=q.device)).clamp(max=q.shape[0] - 1)
        k, v = s["k"][rows].float(), s["v"][rows].float()
    x = torch.einsum("nqhgd,nkhd->nhgqk", qp * s["scale"], k)
    keys = torch.arange(mk, device=q.device)
    seen = keys[None, None, :] <= (full - new)[:, None, None] + at[None, :, None]        # [n, mq, mk]
    seen &= keys[None, None, :] < full[:, None, None]
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    o = torch.einsum("nhgqk,nkhd->nhgqd", x, v) / torch.where(l > 0, l, torch.ones_like(l))
    lse = (m + l.log())[..., 0]
    b, p = s["row_seq"], s["row_pos"]
    return o[b, :, :, p].reshape(-1, hq, D).to(q.dtype), lse[b, :, :, p].reshape(-1, hq)


def _plain_prefix(s):
    q, hq, hkv = s["q"], s["hq"], s["hkv"]
    batch, grp = q.shape[0], hq // hkv
    off = s["offsets"].long()
    qf = (q.float() * s["scale"]).view(batch, hkv, grp, D)
    # the suffixes, one row of queries each
    ks = s["k"][s["table"].long()].flatten(1, 2)[:, :max(1, s["most_suffix"])].float()
    vs = s["v"][s["table"].long()].flatten(1, 2)[:, :max(1, s["most_suffix"])].float()
    xs = torch.einsum("bhgd,bkhd->bhgk", qf, ks)
    gone = torch.arange(xs.shape[-1], device=q.device)[None] >= s["seq_lens"].long()[:, None]
    xs.masked_fill_(gone[:, None, None], float("-inf"))
    # the prefixes, each read once for its group
    at = torch.arange(s["most_size"], device=q.device)
    qg = qf[(off[:-1, None] + at).clamp(max=batch - 1)]
    kp = s["k"][s["prefix_table"].long()].flatten(1, 2)[:, :max(1, s["most_prefix"])].float()
    vp = s["v"][s["prefix_table"].long()].flatten(1, 2)[:, :max(1, s["most_prefix"])].float()
    xp = torch.einsum("nbhgd,nkhd->nbhgk", qg, kp)
    gone = torch.arange(xp.shape[-1], device=q.device)[None] >= s["prefix_lens"].long()[:, None]
    xp.masked_fill_(gone[:, None, None, None], float("-inf"))
    mp = xp.amax(-1)[s["row_group"], s["row_pos"]]
    m = torch.maximum(xs.amax(-1), mp)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    mg = m[(off[:-1, None] + at).clamp(max=batch - 1)]
    es, ep = (xs - m[..., None]).exp(), (xp - mg[..., None]).exp()
    op = torch.einsum("nbhgk,nkhd->nbhgd", ep, vp)[s["row_group"], s["row_pos"]]
    l = es.sum(-1) + ep.sum(-1)[s["row_group"], s["row_pos"]]
    o = (torch.einsum("bhgk,bkhd->bhgd", es, vs) + op) / torch.where(l > 0, l, torch.ones_like(l))[..., None]
    return o.reshape(batch, hq, D).to(q.dtype)


def _plain_append(s):
    qkv, hq, hkv = s["qkv"], s["hq"], s["hkv"]
    t = qkv.shape[0]
    x = qkv.view(t, hq + 2 * hkv, D).float()

    def normed(y, w):
        return y if w is None else y * (y.square().mean(-1, keepdim=True) + s["eps"]).rsqrt() * w.float()

    y = torch.cat([normed(x[:, :hq], s["wq"]), normed(x[:, hq:hq + hkv], s["wk"])], 1)
    ang = s["positions"].double()[:, None] * s["inv_freq"].double()[None]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    half = s["inv_freq"].numel()
    if s["interleaved"]:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    y = torch.cat([turned, y[..., 2 * half:]], -1).to(qkv.dtype)
    s["q_out"].copy_(y[:, :hq])
    page = s["slots"] // s["k"].shape[1], s["slots"] % s["k"].shape[1]
    new = {"k": y[:, hq:], "v": qkv.view(t, hq + 2 * hkv, D)[:, hq + hkv:]}
    if s["kv"] == "16":
        s["k"][page], s["v"][page] = new["k"], new["v"]
    else:
        for n in ("k", "v"):
            r = new[n].float()
            a = r.abs().amax(-1)
            sc = torch.where(a == 0, torch.ones_like(a), a / 448.0).half()
            sc = torch.where(sc == 0, torch.full_like(sc, 2.0 ** -24), sc)
            codes = (r / sc.float()[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            s[n].view(torch.uint8)[page] = codes.view(torch.uint8)
            s[n + "_scale"][page] = sc
    return _append_out(s)


# --------------------------------------------------------------------------- #
# the definition, in 64 bits
# --------------------------------------------------------------------------- #
def _attend64(q, k, v, scale, first):
    """softmax(q k^T scale) v of one sequence and kv-head: q [rows, D], row i sees keys < first[i]."""
    w = (q @ k.T) * scale
    hidden = torch.arange(k.shape[0], device=q.device)[None] >= first[:, None]
    w[hidden] = float("-inf")
    lse = torch.logsumexp(w, -1)
    p = torch.exp(w - torch.where(lse == float("-inf"), torch.zeros_like(lse), lse)[:, None])
    return p @ v, lse


def _cached64(pool, row, n, head):
    page = pool.shape[1]
    ids = row[:-(-n // page)].long()
    return pool[ids, :, head].reshape(-1, D)[:n].double()


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv = s["hq"], s["hkv"]
    g = hq // hkv
    if s["op"] == "prompt":
        q, cu, full = s["q"], s["cu"].tolist(), s["seq_lens"].tolist()
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
        for i, n in enumerate(full):
            new = cu[i + 1] - cu[i]
            first = (n - new) + 1 + torch.arange(new, device=q.device)
            for h in range(hkv):
                if s["page"]:
                    k, v = _cached64(s["k"], s["table"][i], n, h), _cached64(s["v"], s["table"][i], n, h)
                else:
                    k, v = s["k"][cu[i]:cu[i + 1], h].double(), s["v"][cu[i]:cu[i + 1], h].double()
                for j in range(h * g, h * g + g):
                    out[cu[i]:cu[i + 1], j], lse[cu[i]:cu[i + 1], j] = _attend64(
                        q[cu[i]:cu[i + 1], j].double(), k, v, s["scale"], first)
        return out, lse
    if s["op"] == "prefix":
        q, off, plen, slen = s["q"], s["offsets"].tolist(), s["prefix_lens"].tolist(), s["seq_lens"].tolist()
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        for i, n in enumerate(plen):
            for h in range(hkv):
                kp, vp = _cached64(s["k"], s["prefix_table"][i], n, h), _cached64(s["v"], s["prefix_table"][i], n, h)
                for b in range(off[i], off[i + 1]):
                    k = torch.cat([kp, _cached64(s["k"], s["table"][b], slen[b], h)])
                    v = torch.cat([vp, _cached64(s["v"], s["table"][b], slen[b], h)])
                    all_ = torch.full((g,), k.shape[0], device=q.device)
                    out[b, h * g:h * g + g] = _attend64(q[b, h * g:h * g + g].double(), k, v, s["scale"], all_)[0]
        return out
    x = s["qkv"].double().view(-1, hq + 2 * hkv, D)
    heads = x[:, :hq + hkv].clone()
    for lo, hi, w in ((0, hq, s["wq"]), (hq, hq + hkv, s["wk"])):
        if w is not None:
            z = heads[:, lo:hi]
            heads[:, lo:hi] = z / torch.sqrt((z * z).sum(-1, keepdim=True) / D + s["eps"]) * w.double()
    half = s["inv_freq"].numel()
    turn = torch.polar(torch.ones(x.shape[0], half, dtype=torch.float64, device=x.device),
                       torch.outer(s["positions"].double(), s["inv_freq"].double()))[:, None]
    if s["interleaved"]:
        z = torch.view_as_real(torch.view_as_complex(heads[..., :2 * half].reshape(*heads.shape[:2], half, 2).contiguous()) * turn)
        heads[..., :2 * half] = z.flatten(-2)
    else:
        z = torch.complex(heads[..., :half].contiguous(), heads[..., half:2 * half].contiguous()) * turn
        heads[..., :half], heads[..., half:2 * half] = z.real, z.imag
    if s["kv"] != "16":
        return {"q": heads[:, :hq], "k": None, "v": None}
    res = {"q": heads[:, :hq], "k": s["k"].double(), "v": s["v"].double()}
    where = s["slots"] // s["k"].shape[1], s["slots"] % s["k"].shape[1]
    res["k"][where], res["v"][where] = heads[:, hq:], x[:, hq + hkv:]
    return res


# --------------------------------------------------------------------------- #
# what a pass cannot do without
# --------------------------------------------------------------------------- #
def work(case):
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] == "prompt":
        lens = _pairs(case["lens"])
        rows, keys = sum(p[0] for p in lens), sum(p[1] for p in lens)
        seen = sum(n * (f - n) + n * (n + 1) // 2 for n, f in lens)      # (query, key) pairs under the diagonal
        table = sum(-(-f // case["page"]) for _, f in lens) * 4 if case["page"] else 0
        return {"bytes": rows * hq * (D * 2 * 2 + 4) + keys * hkv * D * 2 * 2 + table + len(lens) * 8,
                "flops": 4 * D * hq * seen}
    if case["op"] == "prefix":
        groups, page = _pairs(case["groups"]), case["page"]
        batch = sum(n for n, _ in groups)
        suffix = batch * case["suffix"] // 2                             # lengths are uniform on [0, suffix]
        keys = sum(p for _, p in groups) + suffix
        return {"bytes": batch * hq * D * 2 * 2 + keys * (hkv * D * 2 * 2) + keys // page * 4 + batch * 4,
                "flops": 4 * D * hq * (sum(n * p for n, p in groups) + suffix)}
    t = case["tokens"]
    kv = D * 2 if case["kv"] == "16" else D + 2
    return {"bytes": t * ((hq + 2 * hkv) * D * 2 + hq * D * 2 + 2 * hkv * kv + 16),
            "flops": t * (hq + hkv) * (4 * D + 3 * case["rot"])}
