"""norm_rope_append against the formulas in 64 bits, its quantised pools against quantize_kv
bit for bit, and its edges: slots that are skipped, in-place q, strides, several pools."""
import pytest
import torch

from prompt_cases import D

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def reference(qkv, pos, freq, hq, hkv, wq, wk, eps, interleaved, gain):
    """q, k, v in 64 bits and, per value, the sum of magnitudes a rounding error can scale with."""
    x = qkv.double().view(qkv.shape[0], hq + 2 * hkv, D)
    qk = x[:, :hq + hkv].clone()
    for lo, hi, w in ((0, hq, wq), (hq, hq + hkv, wk)):
        if w is not None:
            z = qk[:, lo:hi]
            qk[:, lo:hi] = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * w.double()
    mag = qk.abs()
    if freq is not None:
        half = freq.numel()
        ang = pos.double()[:, None] * freq.double()[None]
        c, s = (ang.cos() * gain)[:, None], (ang.sin() * gain)[:, None]
        ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
        ib = ia + (1 if interleaved else half)
        a, b = qk[..., ia].clone(), qk[..., ib].clone()
        qk[..., ia], qk[..., ib] = a * c - b * s, b * c + a * s
        both = (a.abs() + b.abs()) * abs(gain)
        mag[..., ia], mag[..., ib] = both, both
    return qk[:, :hq], qk[:, hq:], x[:, hq + hkv:], mag[:, :hq], mag[:, hq:]


def bound(ref, mag, dt):
    """Half a step of the 16-bit type on the result (and the subnormal step of fp16), and fp32 on
    the way: 72 half steps cover the sum of 128 squares added 8 + 4 deep (the root halves its
    part), root, division and the products; the rotation adds sincospi's few steps: 2^-24 * 90."""
    half = torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).tiny * torch.finfo(dt).eps
    return half * ref.abs() + 90 * 2.0 ** -24 * (1 + half) * mag + tiny


def close(got, ref, mag, dt, what):
    err = (got.double().cpu() - ref).abs() / bound(ref, mag, dt)
    assert torch.isfinite(got.float()).all() and err.max() <= 1.0, f"{what} off by {err.max():.3g} of its bound"


def case(T, hq, hkv, rot, dt, seed, norm=True, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=g).to(dt)
    pos = torch.randint(0, far, (T,), generator=g)
    if T > 1:
        pos[0], pos[-1] = 0, far - 1
    freq = (1.0 / (500000.0 ** (torch.arange(0, rot, 2).double() / rot))).float() if rot else None
    wq, wk = [(1 + 0.2 * torch.randn(D, generator=g)).to(dt) for _ in range(2)] if norm else (None, None)
    return qkv, pos, freq, wq, wk, g


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,hq,hkv,rot,inter,norm,gain", [
    (1, 32, 8, 128, False, True, 1.0), (5, 8, 2, 128, True, True, 1.0), (3, 5, 1, 64, False, False, 1.0),
    (7, 14, 2, 96, False, True, 1.25), (130, 4, 4, 32, True, False, 1.0), (2, 1, 1, 16, False, True, 0.5),
    (9, 16, 2, 112, False, True, 1.0), (4, 8, 8, 0, False, True, 1.0), (1000, 8, 2, 128, False, True, 1.0)])
def test_against_the_formulas(dev, dt, T, hq, hkv, rot, inter, norm, gain):
    from peerkv_b200 import ops
    qkv, pos, freq, wq, wk, g = case(T, hq, hkv, rot, dt, T * 31 + rot, norm)
    page, eps = 16, 1e-6
    n_pages = -(-T // page) + 2
    slots = torch.randperm(n_pages * page, generator=g)[:T]
    to = lambda t: t.to(dev) if t is not None else None
    pool = torch.full((2, n_pages, page, hkv, D), 3.0, dtype=dt, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    q = ops.norm_rope_append(to(qkv), to(pos), to(freq), hq, hkv, None, pool[0], pool[1], to(slots), q_weight=to(wq),
                             k_weight=to(wk), eps=eps, interleaved=inter, gain=gain, status=status)
    rq, rk, rv, mq, mk = reference(qkv, pos, freq, hq, hkv, wq, wk, eps, inter, gain)
    close(q, rq, mq, dt, "q")
    flat = pool.view(2, n_pages * page, hkv, D)
    close(flat[0, to(slots)], rk, mk, dt, "k")
    assert torch.equal(flat[1, to(slots)].cpu(), rv.to(dt))
    rest = torch.ones(n_pages * page, dtype=torch.bool)
    rest[slots] = False
    assert (flat[:, to(rest)] == 3.0).all() and status.item() == 0
    # no append: the same q
    assert torch.equal(ops.norm_rope_append(to(qkv), to(pos), to(freq), hq, hkv, q_weight=to(wq), k_weight=to(wk), eps=eps,
                                            interleaved=inter, gain=gain), q)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_quantised_pools_hold_what_quantize_kv_makes(dev, fmt, dt):
    from peerkv_b200 import ops
    hq, hkv, T, page, n_pages = 8, 2, 37, 16, 5
    qkv, pos, freq, wq, wk, g = case(T, hq, hkv, 128, dt, 77)
    qkv[3] = 0
    qkv[4] *= 300 if dt == torch.bfloat16 else 30
    slots = torch.randperm(n_pages * page, generator=g)[:T].to(dev)
    args = [t.to(dev) for t in (qkv, pos, freq)]
    kw = dict(q_weight=wq.to(dev), k_weight=wk.to(dev))
    pool = torch.zeros(2, n_pages, page, hkv, D, dtype=dt, device=dev)
    q = ops.norm_rope_append(*args, hq, hkv, None, pool[0], pool[1], slots, **kw)
    codes = torch.zeros(2, n_pages, page, hkv, D, dtype=torch.int8 if fmt == "int8" else torch.float8_e4m3fn, device=dev)
    scales = torch.zeros(2, n_pages, page, hkv, dtype=torch.float16, device=dev)
    q8 = ops.norm_rope_append(*args, hq, hkv, None, codes[0], codes[1], slots, scales[0], scales[1], **kw)
    assert torch.equal(q8, q)
    at = (slots // page, slots % page)
    for i in range(2):
        c, s = ops.quantize_kv(pool[i][at], fmt)
        assert torch.equal(codes[i][at].view(torch.uint8), c.view(torch.uint8)) and torch.equal(scales[i][at], s)
    rest = torch.ones(n_pages * page, dtype=torch.bool, device=dev)
    rest[slots] = False
    assert (codes.view(torch.uint8).view(2, -1, hkv, D)[:, rest] == 0).all() and (scales.view(2, -1, hkv)[:, rest] == 0).all()


def test_skipped_and_bad_slots(dev):
    from peerkv_b200 import ops
    hq, hkv, T = 4, 2, 6
    qkv, pos, freq, wq, wk, _ = case(T, hq, hkv, 64, torch.bfloat16, 5)
    pool = torch.zeros(2, 3, 16, hkv, D, dtype=torch.bfloat16, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    a = [t.to(dev) for t in (qkv, pos, freq)]
    slots = torch.tensor([0, -1, 47, -7, 20, 3], device=dev)
    q = ops.norm_rope_append(*a, hq, hkv, None, pool[0], pool[1], slots, status=status)
    assert status.item() == 0
    wrote = (pool[1].view(48, hkv, D) != 0).any(-1).any(-1).nonzero()[:, 0].tolist()
    assert wrote == [0, 3, 20, 47]
    before = pool.clone()
    bad = torch.tensor([0, 48, 47, 1 << 40, 20, 3], device=dev)
    assert torch.equal(ops.norm_rope_append(*a, hq, hkv, None, pool[0], pool[1], bad, status=status), q)
    assert status.item() == 2 and torch.equal(pool, before)


def test_two_pools_in_place_and_strided(dev):
    """Page ids from 3 on live in a second pool (here on the same GPU); q is turned where it lies
    inside a wider row; the pools are head-major views."""
    from peerkv_b200 import ops
    hq, hkv, T, dt = 8, 2, 21, torch.float16
    qkv, pos, freq, wq, wk, g = case(T, hq, hkv, 128, dt, 91)
    wide = torch.zeros(T, qkv.shape[1] + 64, dtype=dt, device=dev)
    view = wide[:, :qkv.shape[1]]
    view.copy_(qkv)
    slots = torch.randperm(7 * 16, generator=g)[:T].to(dev)
    one = torch.zeros(2, 7, 16, hkv, D, dtype=dt, device=dev)
    want = ops.norm_rope_append(qkv.to(dev), pos.to(dev), freq.to(dev), hq, hkv, None, one[0], one[1], slots, q_weight=wq.to(dev),
                                k_weight=wk.to(dev))
    a = torch.zeros(2, 3, hkv, 16, D, dtype=dt, device=dev).transpose(2, 3)
    b = torch.zeros(2, 4, hkv, 16, D, dtype=dt, device=dev).transpose(2, 3)
    q = view[:, :hq * D].view(T, hq, D)
    got = ops.norm_rope_append(view, pos.to(dev), freq.to(dev), hq, hkv, q, a[0], a[1], slots, q_weight=wq.to(dev),
                               k_weight=wk.to(dev), peers=[(b[0], b[1])], bases=[3])
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got, want)
    assert torch.equal(view[:, hq * D:].cpu(), qkv[:, hq * D:]) and (wide[:, qkv.shape[1]:] == 0).all()
    assert torch.equal(torch.cat([a, b], 1), one)


def test_captured(dev):
    from peerkv_b200 import ops
    hq, hkv, T = 8, 2, 4
    qkv, pos, freq, wq, wk, _ = case(T, hq, hkv, 128, torch.bfloat16, 15)
    pool = torch.zeros(2, 3, 16, hkv, D, dtype=torch.bfloat16, device=dev)
    a = [t.to(dev) for t in (qkv, pos, freq)]
    slots, q = torch.arange(T, device=dev), torch.zeros(T, hq, D, dtype=torch.bfloat16, device=dev)
    ops.norm_rope_append(*a, hq, hkv, q, pool[0], pool[1], slots)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.norm_rope_append(*a, hq, hkv, q, pool[0], pool[1], slots)
    for step in range(3):
        a[1].add_(step)
        slots.add_(4)
        gr.replay()
        other = torch.zeros_like(pool)
        want = ops.norm_rope_append(*a, hq, hkv, None, other[0], other[1], slots)
        torch.cuda.synchronize()
        at = (slots // 16, slots % 16)
        assert torch.equal(q, want) and torch.equal(pool[0][at], other[0][at])
    del gr


def test_agrees_with_rope_append(dev):
    """Without norms, at positions that fp32 angles still resolve, the decode step's rope_append
    rounds to the same values up to a step."""
    from peerkv_b200 import ops
    from peerkv_b200.decoder import rope_append, rope_inv_freq
    B, hq, hkv = 5, 8, 2
    qkv = torch.randn(B, (hq + 2 * hkv) * D, device=dev).bfloat16()
    pos = torch.tensor([0, 1, 2, 60, 100], device=dev)
    inv = rope_inv_freq(D, 500000.0, dev)
    pa, pb = [torch.zeros(2, 2, 16, hkv, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    pages, slots = torch.tensor([1, 0, 1, 1, 0], device=dev), torch.tensor([3, 15, 0, 7, 4], device=dev)
    qa = torch.empty(B, hq, D, dtype=torch.bfloat16, device=dev)
    rope_append(qkv, pos, inv, qa, hq, hkv, pa, pages, slots)
    qb = ops.norm_rope_append(qkv, pos, inv, hq, hkv, None, pb[0], pb[1], pages * 16 + slots)
    assert torch.allclose(qa.float(), qb.float(), rtol=2.0 ** -7, atol=1e-4)
    assert torch.allclose(pa.float(), pb.float(), rtol=2.0 ** -7, atol=1e-4)


@pytest.mark.multigpu
def test_peer_pool(dev):
    from peerkv_b200 import ops
    hq, hkv, T = 8, 2, 9
    qkv, pos, freq, wq, wk, _ = case(T, hq, hkv, 128, torch.bfloat16, 19)
    a = [t.to(dev) for t in (qkv, pos, freq)]
    one = torch.zeros(2, 4, 16, hkv, D, dtype=torch.bfloat16, device=dev)
    home = torch.zeros(2, 2, 16, hkv, D, dtype=torch.bfloat16, device=dev)
    away = torch.zeros(2, 2, 16, hkv, D, dtype=torch.bfloat16, device=torch.device("cuda", 1))
    slots = torch.tensor([0, 63, 31, 32, 40, 5, 17, 48, 2], device=dev)
    want = ops.norm_rope_append(*a, hq, hkv, None, one[0], one[1], slots)
    got = ops.norm_rope_append(*a, hq, hkv, None, home[0], home[1], slots, peers=[(away[0], away[1])], bases=[2])
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(home, one[:, :2]) and torch.equal(away.to(dev), one[:, 2:])
