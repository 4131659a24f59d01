"""What the prompt, shared-prefix and append entry points refuse, at the C boundary and in Python, and
that the argument structs of the binding are the header's.  Runs without a GPU: every refusal
comes before the first CUDA call."""
import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20            # an aligned address that is never read


def lib():
    from peerkv_b200 import _lib
    return _lib.lib(), _lib


def prompt_args(_lib, **kw):
    a = _lib.PromptArgs()
    a.q, a.q_token_stride, a.q_head_stride, a.dtype = FAKE, 8 * 128, 128, 1
    a.n_q_heads, a.total_q, a.n_seqs, a.cu_seqlens_q = 8, 4, 1, FAKE
    a.kv = _lib.KvView(FAKE, FAKE, None, None, 1, 2, 128, 16, 4, 16 * 256, 256, 128)
    a.block_table, a.block_table_stride, a.block_table_cols, a.seq_lens = FAKE, 4, 4, FAKE
    a.scale, a.causal = 0.1, 1
    for k, v in kw.items():
        if k.startswith("kv_"):
            setattr(a.kv, k[3:], v)
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,word", [
    ({"kv_head_dim": 64}, -3, "head_dim"), ({"dtype": 4}, -1, "dtype"), ({"kv_dtype": 0}, -3, "share"),
    ({"kv_dtype": 2}, -3, "share"), ({"n_q_heads": 9}, -1, "multiple"), ({"n_q_heads": 512}, -3, "128 query heads"),
    ({"total_q": -1}, -1, "total_q"), ({"n_seqs": -2}, -1, "n_seqs"), ({"scale": 0.0}, -1, "scale"),
    ({"scale": -1.0}, -1, "scale"), ({"scale": float("nan")}, -1, "scale"), ({"scale": float("inf")}, -1, "scale"),
    ({"q": None}, -1, "null"), ({"cu_seqlens_q": None}, -1, "null"), ({"seq_lens": None}, -1, "either"),
    ({"block_table": None}, -1, "either"), ({"cu_seqlens_k": FAKE}, -1, "either"),
    ({"block_table": None, "seq_lens": None}, -1, "either"),
    ({"block_table": None, "seq_lens": None, "cu_seqlens_k": FAKE}, -1, "one page"),
    ({"kv_page_size": 8}, -3, "multiple of 16"), ({"kv_page_size": 0}, -3, "multiple of 16"),
    ({"kv_n_pages": -1}, -1, "n_pages"), ({"kv_k": None}, -1, "null k"), ({"kv_token_stride": 12}, -1, "stride"),
    ({"kv_page_stride": 0}, -1, "stride"), ({"kv_head_stride": -128}, -1, "stride"), ({"q_token_stride": 4}, -1, "stride"),
    ({"q_head_stride": 0}, -1, "stride"), ({"q": FAKE + 2}, -1, "aligned"), ({"kv_v": FAKE + 8}, -1, "aligned"),
    ({"o_more": FAKE}, -1, "together"), ({"lse_more": FAKE}, -1, "together")])
def test_prompt_attention_refuses(kw, code, word):
    L, _lib = lib()
    rc = L.pkv_prompt_attention(0, C.byref(prompt_args(_lib, **kw)), FAKE, 1, None, FAKE, 1 << 40, None, None)
    assert rc == code and word in L.pkv_last_error().decode()


def test_prompt_attention_refuses_its_outputs():
    L, _lib = lib()
    a = prompt_args(_lib)
    for out, dt, ws, word in ((None, 1, FAKE, "null"), (FAKE, 7, FAKE, "out_dtype"), (FAKE, 1, None, "null"),
                              (FAKE + 4, 1, FAKE, "aligned"), (FAKE, 1, FAKE + 16, "256-byte")):
        assert L.pkv_prompt_attention(0, C.byref(a), out, dt, None, ws, 1 << 40, None, None) == -1
        assert word in L.pkv_last_error().decode()
    assert L.pkv_prompt_attention(0, None, FAKE, 1, None, FAKE, 1 << 40, None, None) == -1
    assert L.pkv_prompt_workspace(0, None) == -1
    # nothing to do is not an error, whatever the pointers
    for kw in ({"total_q": 0, "q": None}, {"n_seqs": 0}):
        assert L.pkv_prompt_attention(0, C.byref(prompt_args(_lib, **kw)), None, 1, None, None, 0, None, None) == 0


def append_args(_lib, of=1, **kw):
    a = _lib.AppendArgs()
    a.qkv, a.qkv_stride, a.positions, a.inv_freq = FAKE, 12 * 128, FAKE, FAKE
    a.q_out, a.q_out_stride, a.slot_mapping = FAKE, 8 * 128, FAKE
    pools = (_lib.KvView * 2)(*[_lib.KvView(FAKE, FAKE, None, None, 1, 2, 128, 16, 4, 16 * 256, 256, 128)] * 2)
    a.pools, a.bases = pools, (C.c_int64 * 2)(0, 4)
    a.n_dev, a.n_tokens, a.n_q_heads, a.n_kv_heads, a.head_dim = of, 3, 8, 2, 128
    a.dtype, a.rot_dim, a.eps, a.gain = 1, 128, 1e-6, 1.0
    for k, v in kw.items():
        if k.startswith("pool_"):
            setattr(pools[of - 1], k[5:], v)
        elif k == "bases":
            a.bases = (C.c_int64 * 2)(*v)
        else:
            setattr(a, k, v)
    a._keep = pools
    return a


@pytest.mark.parametrize("kw,code,word", [
    ({"head_dim": 64}, -3, "head_dim"), ({"dtype": 2}, -1, "dtype"), ({"n_tokens": -1}, -1, "n_tokens"),
    ({"n_q_heads": 0}, -1, "heads"), ({"rot_dim": 136}, -3, "rot_dim"), ({"rot_dim": 24}, -3, "rot_dim"),
    ({"rot_dim": -16}, -3, "rot_dim"), ({"eps": -1.0}, -1, "eps"), ({"eps": float("nan")}, -1, "eps"),
    ({"qkv": None}, -1, "null"), ({"positions": None}, -1, "null"), ({"inv_freq": None}, -1, "null"),
    ({"qkv_stride": 1540}, -1, "strides"), ({"q_out_stride": 3}, -1, "strides"), ({"qkv": FAKE + 8}, -1, "aligned"),
    ({"q_weight": FAKE + 2}, -1, "aligned"), ({"n_dev": 0}, -1, "n_dev"), ({"n_dev": 99}, -1, "n_dev"),
    ({"pools": None}, -1, "pools"), ({"pool_dtype": 0}, -1, "dtype"), ({"pool_dtype": 3}, -1, "k_scale"),
    ({"pool_page_size": 0}, -1, "page_size"), ({"pool_n_kv_heads": 3}, -1, "must match"), ({"pool_k": None}, -1, "null pool"),
    ({"pool_head_stride": 4}, -1, "strides"), ({"pool_v": FAKE + 8}, -1, "aligned"),
    ({"of": 2, "pool_page_size": 32}, -1, "must match"), ({"of": 2, "bases": (4, 0)}, -1, "ascend")])
def test_norm_rope_append_refuses(kw, code, word):
    L, _lib = lib()
    rc = L.pkv_norm_rope_append(0, C.byref(append_args(_lib, **kw)), None, None)
    assert rc == code and word in L.pkv_last_error().decode()
    assert L.pkv_norm_rope_append(0, None, None, None) == -1
    assert L.pkv_norm_rope_append(0, C.byref(append_args(_lib, n_tokens=0, qkv=None)), None, None) == 0


def test_structs_are_the_header_s(tmp_path):
    """Size and every field's offset, as the C compiler lays them out."""
    _, _lib = lib()
    src = ['#include <stddef.h>', '#include <stdio.h>', '#include "peerkv.h"', 'int main(void) {']
    for name, cls in (("pkv_prompt_args", _lib.PromptArgs), ("pkv_append_args", _lib.AppendArgs), ("pkv_kv_view", _lib.KvView)):
        src.append(f'printf("{name} %zu\\n", sizeof({name}));')
        src += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "t.c").write_text("\n".join(src + ["return 0;", "}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "t"), str(tmp_path / "t.c")], check=True)
    got = dict(l.split() for l in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, cls in (("pkv_prompt_args", _lib.PromptArgs), ("pkv_append_args", _lib.AppendArgs), ("pkv_kv_view", _lib.KvView)):
        assert int(got[name]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset


def test_python_refuses_host_pools():
    """Every pool of an append goes through one check; a host pointer must not reach the kernel."""
    from peerkv_b200 import PeerKVError, ops
    pool = torch.zeros(3, 16, 2, 128).bfloat16()
    with pytest.raises(PeerKVError, match="CUDA"):
        ops._append_view(1, pool, pool, None, None, torch.bfloat16, 2)


def test_python_refuses_cpu_tensors():
    from peerkv_b200 import PeerKVError, ops
    q, pool = torch.zeros(2, 8, 128).bfloat16(), torch.zeros(3, 16, 2, 128).bfloat16()
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.prefill_paged(q, pool, pool, i[None], i, i), lambda: ops.prefill_packed(q, q, q, i),
                 lambda: ops.decode_shared_prefix(q, pool, pool, i[None], i[:1], i[:, None], i),
                 lambda: ops.norm_rope_append(torch.zeros(2, 12 * 128).bfloat16(), i, None, 8, 2)):
        with pytest.raises(PeerKVError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_python_refuses_on_the_gpu():
    from peerkv_b200 import PeerKVError, ops
    dev = torch.device("cuda", 0)
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device=dev)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    q, pool, cu, sl, bt = z(4, 8, 128), z(3, 16, 2, 128), i(0, 4), i(4), i(0)[None]
    bad = [
        (lambda: ops.prefill_paged(q.float(), pool, pool, bt, sl, cu), "fp16 or bf16"),
        (lambda: ops.prefill_paged(z(4, 8, 64), pool, pool, bt, sl, cu), "128"),
        (lambda: ops.prefill_paged(q, pool.half(), pool.half(), bt, sl, cu), "share a dtype"),
        (lambda: ops.prefill_paged(q, pool, pool.transpose(1, 2).contiguous().transpose(1, 2), bt, sl, cu), "equal strides"),
        (lambda: ops.prefill_paged(q, pool, pool, bt.expand(2, 1), sl, cu), "block_table"),
        (lambda: ops.prefill_paged(q, pool, pool, bt, i(4, 4), cu), "seq_lens"),
        (lambda: ops.prefill_paged(q, pool, pool, bt, sl, i(0, 4)[None]), "cu_seqlens_q"),
        (lambda: ops.prefill_paged(q, pool, pool, bt, sl, cu, out=z(4, 8, 256)[..., ::2]), "contiguous"),
        (lambda: ops.prefill_paged(q, pool, pool, bt, sl, cu, status=z(1)), "status"),
        (lambda: ops.prefill_paged(q, pool, pool, bt, sl, cu, scale=0.0), "scale"),
        (lambda: ops.prefill_paged(q, pool.cpu(), pool.cpu(), bt, sl, cu), "expected cuda"),
        (lambda: ops.prefill_paged(q, z(3, 8, 2, 128), z(3, 8, 2, 128), bt, sl, cu), "multiple of 16"),
        (lambda: ops.prefill_paged(q, z(3, 16, 3, 128), z(3, 16, 3, 128), bt, sl, cu), "multiple of n_kv_heads"),
        (lambda: ops.prefill_packed(q, z(4, 2, 128), z(5, 2, 128), cu), "one shape"),
        (lambda: ops.prefill_packed(q, z(4, 2, 128), z(4, 2, 128), cu, i(0, 2, 4)), "same number"),
        (lambda: ops.prefill_packed(q, z(4, 2, 128).half(), z(4, 2, 128), cu), "share a dtype"),
        (lambda: ops.decode_shared_prefix(q, pool, pool, bt, i(1, 2), bt.expand(4, 1), i(0, 0, 0, 0)), "prefix_lens"),
        (lambda: ops.decode_shared_prefix(q, pool, pool, bt, sl, bt, i(0, 0, 0, 0)), "block_table"),
        (lambda: ops.decode_shared_prefix(z(4, 18, 128), pool, pool, bt, sl, bt.expand(4, 1), i(0, 0, 0, 0)), "at most 8"),
        (lambda: ops.norm_rope_append(z(3, 128), i(0, 0, 0).long(), None, 8, 2), "qkv must be"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0).long(), None, 8, 2), "positions"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), z(64), 8, 2), "inv_freq"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), z(12, dt=torch.float32), 8, 2), "rot_dim"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, q_weight=z(64)), "q_weight"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, q_out=z(3, 8, 64)), "q_out"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, k_pool=pool, v_pool=pool), "slot_mapping"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, slot_mapping=i(0, 1, 2).long()), "k_pool"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, None, pool.half(), pool.half(), i(0, 1, 2).long()), "dtype"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, None, pool.to(torch.int8), pool.to(torch.int8),
                                      i(0, 1, 2).long()), "k_scale"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, None, z(3, 16, 4, 128), z(3, 16, 4, 128),
                                      i(0, 1, 2).long()), "n_pages"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, None, pool, pool, i(0, 1, 2).long(),
                                      peers=[(pool, pool)]), "bases"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, None, pool, pool, i(0, 1, 2).long(),
                                      peers=[(pool.cpu(), pool.cpu())], bases=[3]), "CUDA"),
        (lambda: ops.norm_rope_append(z(3, 1536), i(0, 0, 0).long(), None, 8, 2, None, pool.cpu(), pool.cpu(),
                                      i(0, 1, 2).long()), "expected cuda"),
    ]
    for n, (call, word) in enumerate(bad):
        with pytest.raises(PeerKVError, match=word):
            call()
