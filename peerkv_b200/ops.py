"""Tensor-level entry points over the C-ABI library: one GPU's shard context, the
paged / contiguous decode calls, the N-way merge and the KV quantiser.

torch is used for device memory and the current stream only; all device work is
done by libpeerkv.so.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import DecodeArgs, KvView, PeerKVError, check

_DT = {torch.float16: _lib.PKV_F16, torch.bfloat16: _lib.PKV_BF16, torch.float32: _lib.PKV_F32,
       torch.int8: _lib.PKV_INT8, torch.float8_e4m3fn: _lib.PKV_FP8_E4M3}
HEAD_DIM = 128


def _stream(device: torch.device) -> int:
    """Handle of torch's current stream on the device (without the Stream object, which costs 2 us)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if device.index is None else device.index)


def _require_cuda(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise PeerKVError(f"{name} must be a CUDA tensor (this package has no CPU path)")


def raise_on_bits(status: int):
    """PeerKVError that says what the bits of a device status word mean, if any is set."""
    if status:
        names = [n for b, n in ((1, "pipeline wait timed out"), (2, "block-table id outside the pool"),
                                (4, "query never arrived"), (8, "a peer partial never arrived")) if status & b]
        raise PeerKVError("device status 0x%x: %s" % (status, "; ".join(names)))


def read_status(word: torch.Tensor) -> int:
    """Reads and clears a status tensor (int32 [1]) that calls were given; synchronises the current stream."""
    bits = int(word[0])
    if bits:
        word.zero_()
    return bits


class Shard:
    """One GPU's attention context: persistent split-K scratch and status word
    (replaces the per-call scratch of PeerKV csrc/peer_fused_attn_ext.cu:56-63)."""

    def __init__(self, device, max_batch: int, n_q_heads: int):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise PeerKVError("Shard needs a CUDA device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.max_batch, self.n_q_heads = int(max_batch), int(n_q_heads)
        h = C.c_void_p()
        check(_lib.lib().pkv_shard_create(C.byref(h), self.device.index, self.max_batch, self.n_q_heads))
        self._h = h
        self.captured = False          # a CUDA graph may hold launches on this context (see get_shard)

    def close(self):
        if getattr(self, "_h", None):
            _lib.lib().pkv_shard_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def status(self) -> int:
        """Reads and clears the device status word (synchronises the current stream)."""
        v = C.c_uint32()
        check(_lib.lib().pkv_shard_status(self._h, _stream(self.device), C.byref(v)))
        return int(v.value)

    def stats(self, element_size: int = 2) -> dict:
        """Cumulative launches and KV bytes read by this shard's kernels (synchronises);
        also adds what is new since the last call to the package's counters."""
        from . import metrics
        a, b = C.c_uint64(), C.c_uint64()
        check(_lib.lib().pkv_shard_stats(self._h, _stream(self.device), C.byref(a), C.byref(b)))
        kv_bytes = int(b.value) * 16 * HEAD_DIM * 2 * element_size
        new = kv_bytes - getattr(self, "_bytes_seen", 0)
        self._bytes_seen = kv_bytes
        metrics.KV_BYTES_READ.labels(gpu=self.device.index).inc(new)
        return {"launches": int(a.value), "kv_bytes_read": kv_bytes}

    def raise_on_status(self):
        raise_on_bits(self.status())


_shards = {}
_retired = []          # (shard, event): outgrown contexts whose scratch queued kernels may still use
_kept = []             # outgrown contexts that graphs were captured with: those may be replayed at any time


def get_shard(device: torch.device, batch: int, n_q_heads: int) -> Shard:
    """Cached per (device, n_q_heads); regrown when a larger batch shows up.  The outgrown
    context is not freed under kernels that may still be queued on it, and the host does
    not wait for them either: it is retired with an event and freed once that has passed.  One
    that was handed out during a capture lives as long as the process."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    key = (device.index, n_q_heads)
    for item in list(_retired):
        if item[1].query():
            item[0].close()
            _retired.remove(item)
    s = _shards.get(key)
    if s is None or s.max_batch < batch:
        if s is not None and s.captured:
            _kept.append(s)
        elif s is not None:
            ev = torch.cuda.Event()
            with torch.cuda.device(device):
                ev.record(torch.cuda.current_stream(device))
            _retired.append((s, ev))
        cap = min(4096, max(64, 1 << max(0, batch - 1).bit_length()))   # next power of two, 64..4096
        s = Shard(device, max(cap, batch), n_q_heads)                    # > 4096: let the library refuse it
        _shards[key] = s
    if not s.captured and torch.cuda.is_current_stream_capturing():
        s.captured = True
    return s


def make_args(q: torch.Tensor, kv_view: KvView, block_table: Optional[torch.Tensor],
              bt_stride: int, seq_lens: torch.Tensor, scale: float, early_dependent: int = 0) -> DecodeArgs:
    return DecodeArgs(q.data_ptr(), _DT[q.dtype], q.shape[0], q.shape[1], 0, kv_view,
                      block_table.data_ptr() if block_table is not None else None, bt_stride, seq_lens.data_ptr(),
                      scale, early_dependent)


def paged_view(k_pool: torch.Tensor, v_pool: torch.Tensor,
               k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> KvView:
    """k_pool / v_pool: [n_pages, page_size, Hkv, D] (any strides with a unit last
    stride), e.g. cache[0] and cache[1] of vLLM's [2, nb, bs, Hkv, D]."""
    if k_pool.dim() != 4 or k_pool.shape != v_pool.shape or k_pool.stride() != v_pool.stride():
        raise PeerKVError("k_pool and v_pool must be [n_pages, page_size, Hkv, D] with equal strides")
    if k_pool.stride(3) != 1 and k_pool.numel() > 0:
        raise PeerKVError("the head dimension must be contiguous")
    if k_pool.dtype not in _DT or k_pool.dtype == torch.float32:
        raise PeerKVError(f"unsupported KV dtype {k_pool.dtype}")
    n_pages, page_size, n_kv_heads, head_dim = k_pool.shape
    st = k_pool.stride()
    return KvView(k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr() if k_scale is not None else None,
                  v_scale.data_ptr() if v_scale is not None else None, _DT[k_pool.dtype], n_kv_heads, head_dim,
                  page_size, n_pages, st[0], st[1], st[2])


def contiguous_view(K: torch.Tensor, V: torch.Tensor) -> KvView:
    """K / V: [B, Hkv, T, D] (the reference's shard layout, any batch/head/token
    strides with a unit last stride; slices along T are fine).  Each sequence is
    one page of T tokens."""
    if K.dim() != 4 or K.shape != V.shape:
        raise PeerKVError("K and V must both be [B, Hkv, T, D]")
    if K.stride() != V.stride() and K.numel() > 0:
        V = V.contiguous(); K = K.contiguous()
    if K.numel() > 0 and K.stride(3) != 1:
        K = K.contiguous(); V = V.contiguous()
    v = KvView()
    v.k, v.v = K.data_ptr(), V.data_ptr()
    v.dtype = _DT[K.dtype]
    B, Hkv, T, D = K.shape
    v.n_pages, v.n_kv_heads, v.page_size, v.head_dim = (B if T > 0 else 0), Hkv, max(T, 1), D
    v.page_stride, v.head_stride, v.token_stride = K.stride(0), K.stride(1), K.stride(2)
    v._keep = (K, V)
    return v


def _meta(t: torch.Tensor, device: torch.device, name: str) -> torch.Tensor:
    """Block tables and lengths as the kernels need them: int32, on `device`, rows
    contiguous.  The reference accepts host-side metadata (it calls .item() on it), so a
    CPU tensor or one on another GPU is moved here rather than refused; a pointer that is
    not valid on `device` must never reach a kernel."""
    if not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t)
    if t.dtype is not torch.int32:
        t = t.to(torch.int32)
    if t.device != device:
        t = t.to(device, non_blocking=True)
    st = t.stride()
    if st and st[-1] != 1:
        t = t.contiguous()
    return t


def _same_gpu(t: torch.Tensor, device: torch.device, name: str):
    if t is not None and t.device != device:
        raise PeerKVError(f"{name} lives on {t.device}, expected {device}")


def _check_q(q: torch.Tensor):
    _require_cuda(q, "q")
    if q.dim() != 3 or q.shape[2] != HEAD_DIM:
        raise PeerKVError(f"q must be [batch, n_q_heads, {HEAD_DIM}]; got {tuple(q.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise PeerKVError(f"q must be fp16 or bf16; got {q.dtype}")
    return q if q.is_contiguous() else q.contiguous()


def decode_paged(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 block_table: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None, return_lse: bool = False,
                 k_scale=None, v_scale=None, shard: Optional[Shard] = None):
    """Whole decode attention of one GPU over its paged pool -> out [B, Hq, D] in q.dtype."""
    q = _check_q(q)
    B, Hq, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    shard = shard or get_shard(q.device, B, Hq)
    bt, sl = _meta(block_table, q.device, "block_table"), _meta(seq_lens, q.device, "seq_lens")
    for t, n in ((k_pool, "k_pool"), (v_pool, "v_pool"), (k_scale, "k_scale"), (v_scale, "v_scale")):
        _same_gpu(t, q.device, n)
    if shard.device != q.device:
        raise PeerKVError(f"the shard context is on {shard.device}, q on {q.device}")
    view = paged_view(k_pool, v_pool, k_scale, v_scale)
    a = make_args(q, view, bt, bt.stride(0), sl, scale)
    if out is None:
        out = torch.empty_like(q)
    lse = torch.empty(B, Hq, dtype=torch.float32, device=q.device) if return_lse else None
    check(_lib.lib().pkv_decode(shard._h, C.byref(a), out.data_ptr(), _DT[out.dtype],
                                lse.data_ptr() if lse is not None else None, _stream(q.device)))
    return (out, lse) if return_lse else out


def partial_paged(q, k_pool, v_pool, block_table, seq_lens, scale=None, k_scale=None, v_scale=None,
                  shard: Optional[Shard] = None, o_part=None, lse_part=None):
    """One shard's (O fp32 [B,Hq,D] normalised, lse fp32 [B,Hq]) from a paged pool."""
    q = _check_q(q)
    B, Hq, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    shard = shard or get_shard(q.device, B, Hq)
    bt, sl = _meta(block_table, q.device, "block_table"), _meta(seq_lens, q.device, "seq_lens")
    for t, n in ((k_pool, "k_pool"), (v_pool, "v_pool"), (k_scale, "k_scale"), (v_scale, "v_scale")):
        _same_gpu(t, q.device, n)
    if shard.device != q.device:
        raise PeerKVError(f"the shard context is on {shard.device}, q on {q.device}")
    view = paged_view(k_pool, v_pool, k_scale, v_scale)
    a = make_args(q, view, bt, bt.stride(0), sl, scale)
    if o_part is None:
        o_part = torch.empty(B, Hq, D, dtype=torch.float32, device=q.device)
        lse_part = torch.empty(B, Hq, dtype=torch.float32, device=q.device)
    check(_lib.lib().pkv_decode_partial(shard._h, C.byref(a), o_part.data_ptr(), lse_part.data_ptr(),
                                        _stream(q.device)))
    return o_part, lse_part


def partial_contiguous(q, K, V, scale=None, shard: Optional[Shard] = None, o_part=None, lse_part=None):
    """One shard's partial from contiguous K/V [B, Hkv, T, D]; q [B, Hq, D]."""
    q = _check_q(q)
    _require_cuda(K, "K")
    _same_gpu(K, q.device, "K"); _same_gpu(V, q.device, "V")
    B, Hq, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    shard = shard or get_shard(q.device, B, Hq)
    view = contiguous_view(K, V)
    T = K.shape[2]
    sl = torch.full((B,), T, dtype=torch.int32, device=q.device)
    a = make_args(q, view, None, 1, sl, scale)
    if o_part is None:
        o_part = torch.empty(B, Hq, D, dtype=torch.float32, device=q.device)
        lse_part = torch.empty(B, Hq, dtype=torch.float32, device=q.device)
    check(_lib.lib().pkv_decode_partial(shard._h, C.byref(a), o_part.data_ptr(), lse_part.data_ptr(),
                                        _stream(q.device)))
    return o_part, lse_part


def decode_contiguous(q, K, V, scale=None, out=None, shard: Optional[Shard] = None):
    """Whole attention over contiguous K/V [B, Hkv, T, D] on one GPU -> [B, Hq, D]."""
    q = _check_q(q)
    _require_cuda(K, "K")
    _same_gpu(K, q.device, "K"); _same_gpu(V, q.device, "V")
    B, Hq, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    shard = shard or get_shard(q.device, B, Hq)
    view = contiguous_view(K, V)
    sl = torch.full((B,), K.shape[2], dtype=torch.int32, device=q.device)
    a = make_args(q, view, None, 1, sl, scale)
    if out is None:
        out = torch.empty_like(q)
    check(_lib.lib().pkv_decode(shard._h, C.byref(a), out.data_ptr(), _DT[out.dtype], None,
                                _stream(q.device)))
    return out


def merge_partials(o_parts: torch.Tensor, lse_parts: torch.Tensor, out_dtype=torch.float32,
                   return_lse: bool = False):
    """Single-pass N-way LSE merge.  o_parts [N, ..., D] fp32, lse_parts [N, ...] fp32
    (contiguous, same device) -> out [..., D] in out_dtype (and lse [...])."""
    _require_cuda(o_parts, "o_parts")
    if o_parts.dtype != torch.float32 or lse_parts.dtype != torch.float32:
        raise PeerKVError("partials must be fp32")
    o_parts, lse_parts = o_parts.contiguous(), lse_parts.contiguous()
    N, D = o_parts.shape[0], o_parts.shape[-1]
    rows = lse_parts[0].numel()
    out = torch.empty(o_parts.shape[1:], dtype=out_dtype, device=o_parts.device)
    lse = torch.empty(lse_parts.shape[1:], dtype=torch.float32, device=o_parts.device) if return_lse else None
    check(_lib.lib().pkv_merge_partials(o_parts.device.index, o_parts.data_ptr(), rows * D,
                                        lse_parts.data_ptr(), rows, N, rows, D, out.data_ptr(),
                                        _DT[out_dtype], lse.data_ptr() if lse is not None else None,
                                        _stream(o_parts.device)))
    return (out, lse) if return_lse else out


def quantize_kv(x: torch.Tensor, fmt: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-(token, kv-head) absmax quantiser: x [..., 128] fp16/bf16 ->
    (codes [..., 128] int8 or float8_e4m3fn, scales [...] fp16)."""
    _require_cuda(x, "x")
    if x.shape[-1] != HEAD_DIM or x.dtype not in (torch.float16, torch.bfloat16):
        raise PeerKVError("x must be [..., 128] fp16 or bf16")
    x = x.contiguous()
    rows = x.numel() // HEAD_DIM
    code_dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    if fmt not in ("int8", "fp8"):
        raise PeerKVError("fmt must be 'int8' or 'fp8'")
    codes = torch.empty(x.shape, dtype=code_dt, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float16, device=x.device)
    check(_lib.lib().pkv_quantize_kv(x.device.index, x.data_ptr(), _DT[x.dtype], rows, codes.data_ptr(),
                                     scales.data_ptr(), _DT[code_dt], _stream(x.device)))
    return codes, scales


# --------------------------------------------------------------------------- #
# prompts, shared prefixes, and the append in front of them
# --------------------------------------------------------------------------- #
_workspace_bytes = {}


def _prompt_workspace(device: torch.device, more: int = 0) -> torch.Tensor:
    """Workspace of one pkv_prompt_attention call and `more` bytes behind it, from torch's allocator:
    it belongs to the current stream (or to the graph being captured), so calls on other
    streams and other captured graphs have their own."""
    n = _workspace_bytes.get(device.index)
    if n is None:
        v = C.c_int64()
        check(_lib.lib().pkv_prompt_workspace(device.index, C.byref(v)))
        n = _workspace_bytes[device.index] = int(v.value)
    return torch.empty(n + more, dtype=torch.uint8, device=device)


def _rows_of_heads(t: torch.Tensor, name: str) -> torch.Tensor:
    """[tokens, heads, 128] as the kernels read it: unit last stride, the others positive
    multiples of 8 elements, 16-byte aligned; anything else is copied (contiguous() would return a
    contiguous tensor with a misaligned start as it is)."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM:
        raise PeerKVError(f"{name} must be [tokens, heads, {HEAD_DIM}]; got {tuple(shape)}")
    n0, n1, _ = shape
    s0, s1, s2 = t.stride()
    ok = s2 == 1 and t.data_ptr() % 16 == 0 and (n0 <= 1 or (s0 > 0 and s0 % 8 == 0)) and \
        (n1 <= 1 or (s1 > 0 and s1 % 8 == 0))
    return t if ok or t.numel() == 0 else t.clone(memory_format=torch.contiguous_format)


def _status_word(status: Optional[torch.Tensor], device: torch.device):
    if status is None:
        return None
    if status.device != device or status.dtype != torch.int32 or status.numel() < 1:
        raise PeerKVError("status must be an int32 tensor on the call's GPU")
    return status.data_ptr()


def _check_out(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)      # (1.8 us less than torch.empty)
    if out.shape != q.shape or out.device != q.device or not out.is_contiguous() or \
            out.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise PeerKVError("out must be a contiguous fp16 / bf16 / fp32 tensor of q's shape on q's GPU")
    return out


def _prompt_call(q, view, scale, causal, out, lse, cu_q, n_seqs, status, block_table=None, seq_lens=None, cu_k=None,
                 more=(None, None), ws=None):
    dev = q.device
    total_q, n_heads, _ = q.shape
    st = q.stride()
    paged = block_table is not None
    # (a table without columns has no memory; its rows have room for no token, and nothing is read)
    table = None if not paged else block_table.data_ptr() or cu_q.data_ptr()
    a = _lib.PromptArgs(q.data_ptr(), st[0], st[1], _DT[q.dtype], n_heads, total_q, n_seqs, cu_q.data_ptr(), view,
                        table, block_table.stride(0) if paged else 0,
                        block_table.shape[1] if paged else 0, 1 if causal else 0,
                        seq_lens.data_ptr() if paged else None, None if paged else cu_k.data_ptr(),
                        more[0], more[1], scale, 0 if more[0] is None else 1)
    if ws is None:
        ws = _prompt_workspace(dev)
    check(_lib.lib().pkv_prompt_attention(dev.index, C.byref(a), out.data_ptr(), _DT[out.dtype],
                                          lse.data_ptr() if lse is not None else None, ws.data_ptr(), ws.numel(),
                                          _status_word(status, dev), _stream(dev)))


def _check_prompt_q(q: torch.Tensor) -> torch.Tensor:
    _require_cuda(q, "q")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise PeerKVError(f"q must be fp16 or bf16; got {q.dtype}")
    return _rows_of_heads(q, "q")


def _cu(t, device, name) -> torch.Tensor:
    t = _meta(t, device, name)
    if t.dim() != 1 or t.numel() < 1:
        raise PeerKVError(f"{name} must be [n_seqs + 1]")
    return t


def _prompt_pool(q, k_pool, v_pool):
    dev, dt = q.device, q.dtype
    _same_gpu(k_pool, dev, "k_pool")
    _same_gpu(v_pool, dev, "v_pool")
    view = paged_view(k_pool, v_pool)
    if k_pool.dtype is not dt or v_pool.dtype is not dt:
        raise PeerKVError(f"k_pool ({k_pool.dtype}), v_pool ({v_pool.dtype}) and q ({q.dtype}) must share a dtype")
    return view


def _table(block_table, device, rows: int, name: str) -> torch.Tensor:
    bt = _meta(block_table, device, name)
    shape = bt.shape
    if len(shape) != 2 or shape[0] != rows:
        raise PeerKVError(f"{name} must be [{rows}, pages]; got {tuple(shape)}")
    return bt


def prefill_paged(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, cu_seqlens_q: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
                  out: Optional[torch.Tensor] = None, return_lse: bool = False,
                  status: Optional[torch.Tensor] = None):
    """Attention of whole prompts, chunks or single new tokens over the paged cache of one GPU.

    q [total_q, Hq, 128] fp16 / bf16, the new tokens of all sequences one behind the other:
    sequence i owns rows cu_seqlens_q[i] .. cu_seqlens_q[i+1] - 1 (possibly none).  seq_lens [n]
    counts every token of a sequence in the cache, the new ones included: append them first
    (norm_rope_append).  k_pool / v_pool, block_table as in decode_paged, 16-bit, page size a
    multiple of 16.  With `causal` row r of n new ones sees keys j <= seq_len - n + r.
    Returns out [total_q, Hq, 128] (q's dtype, or `out`'s), and with return_lse the natural-log lse
    [total_q, Hq] fp32, so that shards merge with merge_partials.  Rows that see nothing are 0 with
    lse -inf; rows behind the last sequence are not written.  V of every token of a sequence
    must be finite; what the pages hold behind a sequence does not matter.
    `status` (int32 [1] on q's GPU) gets the device status bits OR-ed in (read_status, raise_on_bits);
    without one a page id outside the pool, read as page 0, goes unreported."""
    q = _check_prompt_q(q)
    cu = _cu(cu_seqlens_q, q.device, "cu_seqlens_q")
    n = cu.numel() - 1
    bt = _table(block_table, q.device, n, "block_table")
    sl = _meta(seq_lens, q.device, "seq_lens")
    if sl.dim() != 1 or sl.numel() != n:
        raise PeerKVError(f"seq_lens must be [{n}]; got {tuple(sl.shape)}")
    view = _prompt_pool(q, k_pool, v_pool)
    out = _check_out(out, q)
    lse = q.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    _prompt_call(q, view, 1.0 / math.sqrt(HEAD_DIM) if scale is None else scale, causal, out, lse, cu, n, status,
                 block_table=bt, seq_lens=sl)
    return (out, lse) if return_lse else out


def prefill_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                   cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None, causal: bool = True,
                   out: Optional[torch.Tensor] = None, return_lse: bool = False,
                   status: Optional[torch.Tensor] = None):
    """prefill_paged for keys that are packed like the queries: k, v [total_k, Hkv, 128] (views
    into the fused projection are fine), sequence i owns keys cu_seqlens_k[i] ..
    cu_seqlens_k[i+1] - 1 (default: the queries' offsets)."""
    q = _check_prompt_q(q)
    _same_gpu(k, q.device, "k"); _same_gpu(v, q.device, "v")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise PeerKVError(f"k ({k.dtype}), v ({v.dtype}) and q ({q.dtype}) must share a dtype")
    if k.shape != v.shape:
        raise PeerKVError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
    k, v = _rows_of_heads(k, "k"), _rows_of_heads(v, "v")
    if k.stride() != v.stride():
        k, v = k.contiguous(), v.contiguous()
    cu = _cu(cu_seqlens_q, q.device, "cu_seqlens_q")
    ck = cu if cu_seqlens_k is None else _cu(cu_seqlens_k, q.device, "cu_seqlens_k")
    if ck.numel() != cu.numel():
        raise PeerKVError("cu_seqlens_q and cu_seqlens_k must describe the same number of sequences")
    total_k, n_kv, _ = k.shape
    view = KvView(k.data_ptr(), v.data_ptr(), None, None, _DT[k.dtype], n_kv, HEAD_DIM, total_k, 1 if total_k > 0 else 0,
                  HEAD_DIM, k.stride(0), k.stride(1))
    out = _check_out(out, q)
    lse = q.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    _prompt_call(q, view, 1.0 / math.sqrt(HEAD_DIM) if scale is None else scale, causal, out, lse, cu, cu.numel() - 1,
                 status, cu_k=ck)
    return (out, lse) if return_lse else out


def decode_shared_prefix(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, prefix_table: torch.Tensor,
                         prefix_lens: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         group_offsets: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None, return_lse: bool = False, shard: Optional[Shard] = None,
                         status: Optional[torch.Tensor] = None):
    """Decode attention (one token per sequence) of groups of sequences that share a prefix: the
    prefix is read once for its group instead of once per sequence.

    q [batch, Hq, 128]; group g owns sequences group_offsets[g] .. group_offsets[g+1] - 1 (default:
    one group of all; the offsets run from 0 to batch, rows of no group are not written) and the prefix of
    prefix_lens[g] tokens in the pages prefix_table[g] (any length, 0 allowed).  block_table / seq_lens
    describe what each sequence has of its own behind the prefix (0 tokens allowed; as in decode_paged
    every page of a length must stand in its row), e.g. the columns of a full table behind the shared pages.  Result as decode_paged over prefix
    and own tokens: out [batch, Hq, 128], with return_lse the lse [batch, Hq].  As decode_paged it takes
    at most 8 query heads per kv-head; pages hold a multiple of 16 tokens of q's type.
    The own tokens go through `shard` (see decode_paged), whose launches must not overlap and which
    reports their bad pages; `status` gets those of the prefixes."""
    q = _check_prompt_q(q)
    B, Hq, D = q.shape
    dev = q.device
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    pt = prefix_table if prefix_table.dim() == 2 else prefix_table[None]
    if group_offsets is not None:
        go = _cu(group_offsets, dev, "group_offsets")
    else:                                              # [0, B], made on the device: no copy, and capturable
        go = torch.arange(0, B + 1, B, dtype=torch.int32, device=dev) if B else \
            torch.zeros(2, dtype=torch.int32, device=dev)
    n = go.numel() - 1
    if n == 0 and B > 0:
        raise PeerKVError(f"group_offsets describe no group, and q has {B} rows")
    pt = _table(pt, dev, n, "prefix_table")
    pl = _meta(prefix_lens, dev, "prefix_lens").reshape(-1)
    if pl.numel() != n:
        raise PeerKVError(f"prefix_lens must be [{n}]; got {pl.numel()} of them")
    bt, sl = _table(block_table, dev, B, "block_table"), _meta(seq_lens, dev, "seq_lens")
    if sl.dim() != 1 or sl.numel() != B:
        raise PeerKVError(f"seq_lens must be [{B}]; got {tuple(sl.shape)}")
    if bt.shape[1] == 0:                               # no room for own tokens, whatever seq_lens says
        bt, sl = bt.new_zeros(B, 1), torch.zeros_like(sl)
    view = _prompt_pool(q, k_pool, v_pool)
    out = _check_out(out, q)
    lse = q.new_empty((B, Hq), dtype=torch.float32) if return_lse else None
    if B > 0:
        shard = shard or get_shard(dev, B, Hq)
        if shard.device != dev:
            raise PeerKVError(f"the shard context is on {shard.device}, q on {dev}")
        qd = q if q.is_contiguous() else q.contiguous()
        # one allocation: the join's workspace, then the own tokens' partial
        ws = _prompt_workspace(dev, B * Hq * (D + 1) * 4)
        o_own = ws.data_ptr() + _workspace_bytes[dev.index]
        l_own = o_own + B * Hq * D * 4
        # nothing comes between the two launches: the second starts while the first ends (graph of b4 / b64 with
        # a prefix of 2048 / 32768 tokens: 33.4 -> 25.4 us, 106.2 -> 99.7 us)
        a = make_args(qd, view, bt, bt.stride(0), sl, scale, 1)
        check(_lib.lib().pkv_decode_partial(shard._h, C.byref(a), o_own, l_own, _stream(dev)))
        _prompt_call(q, view, scale, False, out, lse, go, n, status, block_table=pt, seq_lens=pl, more=(o_own, l_own), ws=ws)
    return (out, lse) if return_lse else out


# The append of one decode step is a 4 us kernel behind these checks: attributes of a tensor cost 0.1 to
# 0.2 us each, so each is read once, and devices are compared by index.
_HALF_TYPES = (torch.float16, torch.bfloat16)
_CODE_TYPES = (torch.int8, torch.float8_e4m3fn)
_View1, _Base1 = KvView * 1, (C.c_int64 * 1)(0)


def _vector(t: torch.Tensor, n: int, dt, device: int, name: str) -> torch.Tensor:
    if t.dtype is not dt or t.get_device() != device or t.shape != (n,):
        raise PeerKVError(f"{name} must be {dt} [{n}] on cuda:{device}; got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _append_view(i: int, kp, vp, ks, vs, dtype, n_kv_heads: int) -> KvView:
    kdt = kp.dtype
    if kdt is not vp.dtype or (kdt is not dtype and kdt not in _CODE_TYPES):
        raise PeerKVError(f"pool {i}: {kdt} / {vp.dtype}; qkv's dtype, int8 or float8_e4m3fn")
    shape, st, dev = kp.shape, kp.stride(), kp.get_device()
    if len(shape) != 4 or shape[2] != n_kv_heads or shape[3] != HEAD_DIM or vp.shape != shape or vp.stride() != st:
        raise PeerKVError(f"pool {i}: k and v must be [n_pages, page, {n_kv_heads}, {HEAD_DIM}] with equal strides; got "
                          f"{tuple(shape)} and {tuple(vp.shape)}")
    if st[3] != 1 and kp.numel() > 0:
        raise PeerKVError("the head dimension must be contiguous")
    if dev < 0 or vp.get_device() != dev:
        raise PeerKVError(f"pool {i}: k and v must be CUDA tensors on one GPU; got {kp.device} and {vp.device}")
    if kdt is dtype:
        return KvView(kp.data_ptr(), vp.data_ptr(), None, None, _DT[kdt], n_kv_heads, HEAD_DIM, shape[1], shape[0], st[0],
                      st[1], st[2])
    for t in (ks, vs):
        if t is None or t.dtype is not torch.float16 or t.shape != shape[:3] or not t.is_contiguous() or t.get_device() != dev:
            raise PeerKVError("quantised pools need contiguous fp16 k_scale / v_scale [n_pages, page, Hkv] beside them")
    return KvView(kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr(), _DT[kdt], n_kv_heads, HEAD_DIM, shape[1],
                  shape[0], st[0], st[1], st[2])


def norm_rope_append(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: Optional[torch.Tensor], n_q_heads: int,
                     n_kv_heads: int, q_out: Optional[torch.Tensor] = None, k_pool: Optional[torch.Tensor] = None,
                     v_pool: Optional[torch.Tensor] = None, slot_mapping: Optional[torch.Tensor] = None, k_scale=None,
                     v_scale=None, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                     eps: float = 1e-6, interleaved: bool = False, gain: float = 1.0, peers=(), bases=(),
                     status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """New tokens on their way into the cache, one launch: per-head RMS norm of q and k (where
    q_weight / k_weight [128] are given), rotary positions, and the store of k and v by slot.

    qkv [T, (Hq + 2 Hkv) * 128] fp16 / bf16 (rows may be strided); positions [T] int64; inv_freq
    fp32 [rot / 2], which says how much of a head turns (rot a multiple of 16, at most 128;
    None: no rotation), halves against each other or, with `interleaved`, neighbours; `gain`
    multiplies cos and sin.  q goes to q_out [T, Hq, 128] (made if None; it may be the q part of qkv).
    slot_mapping [T] int64 = page * page_size + offset (negative: not stored); the slots of one
    call must differ.  k_pool / v_pool [n_pages, page, Hkv, 128] of qkv's dtype, int8 or
    float8_e4m3fn with k_scale / v_scale [n_pages, page, Hkv] fp16; `peers` = further (k_pool,
    v_pool[, k_scale, v_scale]) on other GPUs, holding the page ids from `bases` on.
    Returns q_out.  A slot outside every pool is skipped and sets bit 2 in `status`."""
    dev, dt, shape, st = qkv.get_device(), qkv.dtype, qkv.shape, qkv.stride()
    if dev < 0:
        _require_cuda(qkv, "qkv")
    if dt not in _HALF_TYPES:
        raise PeerKVError(f"qkv must be fp16 or bf16; got {dt}")
    if len(shape) != 2 or n_q_heads < 1 or n_kv_heads < 1 or shape[1] != (n_q_heads + 2 * n_kv_heads) * HEAD_DIM:
        raise PeerKVError(f"qkv must be [T, (n_q_heads + 2 n_kv_heads) * {HEAD_DIM}]; got {tuple(shape)}")
    T = shape[0]
    qkv_ptr = qkv.data_ptr()
    if T and (st[1] != 1 or st[0] % 8 or qkv_ptr % 16):
        qkv = qkv.clone(memory_format=torch.contiguous_format)        # (contiguous() keeps a misaligned start)
        qkv_ptr, st = qkv.data_ptr(), qkv.stride()
    if q_out is None:
        q_out = qkv.new_empty((T, n_q_heads, HEAD_DIM))
    qs = q_out.stride()
    if q_out.shape != (T, n_q_heads, HEAD_DIM) or q_out.dtype is not dt or q_out.get_device() != dev or \
            (T and (qs[2] != 1 or (n_q_heads > 1 and qs[1] != HEAD_DIM))):
        raise PeerKVError(f"q_out must be [T, n_q_heads, {HEAD_DIM}] of qkv's dtype and GPU with contiguous heads")
    if positions.dtype is not torch.int64:
        positions = positions.to(torch.int64)
    positions = _vector(positions, T, torch.int64, dev, "positions")
    half, freq_ptr, qw_ptr, kw_ptr, slot_ptr = 0, None, None, None, None
    if inv_freq is not None:
        half = inv_freq.numel()
        inv_freq = _vector(inv_freq, half, torch.float32, dev, "inv_freq")
        freq_ptr = inv_freq.data_ptr()
    if q_weight is not None:
        q_weight = _vector(q_weight, HEAD_DIM, dt, dev, "q_weight")
        qw_ptr = q_weight.data_ptr()
    if k_weight is not None:
        k_weight = _vector(k_weight, HEAD_DIM, dt, dev, "k_weight")
        kw_ptr = k_weight.data_ptr()
    views = first = None
    n_dev = 0
    if slot_mapping is not None:
        if k_pool is None or v_pool is None:
            raise PeerKVError("an append needs k_pool, v_pool and slot_mapping")
        if slot_mapping.dtype is not torch.int64:
            slot_mapping = slot_mapping.to(torch.int64)
        slot_mapping = _vector(slot_mapping, T, torch.int64, dev, "slot_mapping")
        slot_ptr = slot_mapping.data_ptr()
        if k_pool.get_device() != dev:
            raise PeerKVError(f"k_pool lives on {k_pool.device}, expected cuda:{dev}")
        if len(bases) != len(peers):
            raise PeerKVError("every peer pool needs its first page id in bases")
        n_dev = 1 + len(peers)
        home = _append_view(0, k_pool, v_pool, k_scale, v_scale, dt, n_kv_heads)
        if n_dev == 1:
            views, first = _View1(home), _Base1
        else:
            from .peerkv.kv_alloc import _enable_peer_access
            more = [_append_view(i + 1, *(tuple(p) + (None,) * (4 - len(p))), dt, n_kv_heads) for i, p in enumerate(peers)]
            _enable_peer_access(qkv.device, [p[0].device for p in peers])
            views = (KvView * n_dev)(home, *more)
            first = (C.c_int64 * n_dev)(0, *[int(b) for b in bases])
    elif k_pool is not None or v_pool is not None:
        raise PeerKVError("an append needs k_pool, v_pool and slot_mapping")
    a = _lib.AppendArgs(qkv_ptr, st[0] if T > 1 else shape[1], positions.data_ptr(), freq_ptr, qw_ptr, kw_ptr,
                        q_out.data_ptr(), qs[0] if T > 1 else n_q_heads * HEAD_DIM, slot_ptr, views, first, n_dev, T,
                        n_q_heads, n_kv_heads, HEAD_DIM, _DT[dt], 2 * half, 1 if interleaved else 0, eps, gain)
    check(_lib.lib().pkv_norm_rope_append(dev, C.byref(a), None if status is None else _status_word(status, qkv.device),
                                          torch._C._cuda_getCurrentRawStream(dev)))
    return q_out
