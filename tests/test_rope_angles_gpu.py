"""Far positions: the decode step's rope_append, norm_rope_append and the formula in 64 bits turn a row by the
same angle, so that keys a prompt left in the cache and the queries of later decode steps fit."""
import pytest
import torch

from prompt_cases import D
from test_append_gpu import close, reference
from test_prompt_step_gpu import caches, model

pytestmark = pytest.mark.gpu
FAR = [0, 1, 4097, 100003, 131071, 777777, 1048575]


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_rope_append_at_far_positions(dev, dt):
    from peerkv_b200.decoder import rope_append, rope_inv_freq
    hq, hkv, B = 8, 2, len(FAR)
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(B, (hq + 2 * hkv) * D, generator=gen).to(dt)
    pos, inv = torch.tensor(FAR), rope_inv_freq(D, 500000.0, dev)
    pool = torch.zeros(2, 2, 16, hkv, D, dtype=dt, device=dev)
    pages, slots = torch.arange(B, device=dev) % 2, torch.arange(B, device=dev) * 2
    q = torch.empty(B, hq, D, dtype=dt, device=dev)
    rope_append(qkv.to(dev), pos.to(dev), inv, q, hq, hkv, pool, pages, slots)
    rq, rk, _, mq, mk = reference(qkv, pos, inv.cpu(), hq, hkv, None, None, 0.0, False, 1.0)
    close(q, rq, mq, dt, "q")
    close(pool[0][pages, slots], rk, mk, dt, "k")


def test_prompt_and_decode_steps_store_the_same_keys(dev):
    """One new token per sequence at positions up to 2^20, through PromptStep and through DecodeStep: the
    first layer's keys and queries agree to a rounding of bf16."""
    from peerkv_b200.decoder import DecodeStep, PromptStep
    g, w = model(dev)
    B = len(FAR)
    tok, pos = torch.arange(B, device=dev) * 3, torch.tensor(FAR, device=dev)
    one = torch.ones(B, dtype=torch.int32, device=dev)
    a, tab = caches(g, [1] * B, 0, dev)
    pages = tab[:, 0].long().to(dev)
    PromptStep(g, w, a, dev).step(tok, pos, pages * 16, torch.arange(B + 1, dtype=torch.int32, device=dev), one)
    b, _ = caches(g, [1] * B, 0, dev)
    for l in b:
        l.lens.copy_(one)
        l.pool.nan_to_num_(0.0)
    DecodeStep(g, w, b, B, dev, append_slots=(pages, torch.zeros_like(pages))).step(tok, pos)
    ka, kb = a[0].pool[0][pages, 0].float(), b[0].pool[0][pages, 0].float()
    # one step of bf16 on either side, and fp32 on the way (see test_append_gpu.bound) scaled by a pair's size
    size = ka.abs() + ka.roll(D // 2, -1).abs()
    assert ((ka - kb).abs() <= 2.0 ** -7 * ka.abs() + 2.0 ** -17 * size).all()
