"""Paged KV cache and token log probabilities for callers that drive their own
batch (include/tl_api.h, the paged cache section).

Unlike the operators of :mod:`shim`, which mirror the reference's host
functions, these take and return CUDA tensors: a server's cache, activations
and logits stay on the device. Every call checks its arguments, enqueues one
kernel on the current stream of the tensors' device and returns without
synchronising; shapes, types, strides and devices that the library does not
take raise ``ValueError``, errors of the library :class:`shim.TLError`. There
is no CPU path.
"""

from __future__ import annotations

import ctypes as C
from struct import Struct
from typing import NamedTuple

from .shim import check, load_library

F32, BF16, F16, I8 = 0, 1, 2, 3  # tl_dtype
TOP_K_MAX = 32
HEAD_DIMS = (64, 128)

_FLOAT_CODES: dict = {}
_POOL_CODES: dict = {}


class PagedView(C.Structure):
    """tl_paged_kv"""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("dtype", C.c_int32), ("num_pages", C.c_int32), ("kv_heads", C.c_int32), ("page_size", C.c_int32),
                ("head_dim", C.c_int32)]


# tl_paged_append_args, tl_paged_read_args, tl_paged_attn_args, tl_token_logprobs_args
_APPEND = Struct("@9P4q6i")
_READ = Struct("@5Pq4i")
_ATTEND = Struct("@7PN2q5if")
_LOGPROBS = Struct("@6Pq4i")

# Imported by the first call that needs it (importing the package does not).
# Small calls are as long as their host side: what every call looks up is bound once.
torch = _Tensor = _INT32 = _FLOAT32 = _device = _stream = None


def _need_torch():
    global torch, _Tensor, _INT32, _FLOAT32, _device, _stream
    if torch is None:
        import torch as module
        _Tensor, _INT32, _FLOAT32 = module.Tensor, module.int32, module.float32
        _device = module.cuda.current_device
        _stream = getattr(module._C, "_cuda_getCurrentRawStream", None)  # (None without CUDA)
        torch = module
        _FLOAT_CODES.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})
        _POOL_CODES.update({torch.int8: I8, torch.bfloat16: BF16, torch.float16: F16})
    return torch


def _bad(name, t, want):
    got = (f"{t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}" if isinstance(t, _Tensor)
           else f"{type(t).__module__}.{type(t).__qualname__}")
    return ValueError(f"{name} must be {want}, got {got}")


def _index(name, t, n, gpu):
    """int32 vector of n entries on device ``gpu`` -> its address."""
    if (isinstance(t, _Tensor) and t.dtype is _INT32 and t.shape == (n,) and t.get_device() == gpu
            and t.is_contiguous()):
        return t.data_ptr()
    raise _bad(name, t, f"a contiguous int32 [{n}] tensor on cuda:{gpu}")


def _rows(name, t, n, heads, d, dtype, gpu):
    """[n, heads, d] activations with contiguous head rows, 16-byte aligned -> (address, row stride)."""
    if isinstance(t, _Tensor) and t.dtype is dtype and t.shape == (n, heads, d) and t.get_device() == gpu:
        s0, s1, s2 = t.stride()
        p = t.data_ptr()
        if n < 2:
            s0 = heads * d
        if s2 == 1 and (s1 == d or heads == 1) and s0 >= heads * d and not (p | s0 * dtype.itemsize) & 15:
            return p, s0
    raise _bad(name, t, f"a {dtype} [{n}, {heads}, {d}] tensor on cuda:{gpu}, head rows contiguous, tokens a multiple "
                        "of 16 bytes apart, 16-byte aligned")


def _angles(name, t, rows, d, gpu):
    if (isinstance(t, _Tensor) and t.dtype is _FLOAT32 and t.shape == (rows, d) and rows
            and t.get_device() == gpu and t.is_contiguous()):
        p = t.data_ptr()
        if not p & 15:
            return p
    raise _bad(name, t, f"a contiguous float32 [max_positions, {d}] tensor on cuda:{gpu}, 16-byte aligned")


def _out(name, t, like, shape, dtype):
    """``t`` checked as a contiguous output on ``like``'s device, or a new tensor."""
    if t is None:
        if like.dtype is dtype and like.shape == shape:
            return torch.empty_like(like, memory_format=torch.contiguous_format)
        return like.new_empty(*shape, dtype=dtype)  # (sizes one by one: 0.4 us less than a tuple)
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == like.device
            and t.is_contiguous() and not t.data_ptr() & 15):
        raise _bad(name, t, f"a contiguous {dtype} {list(shape)} tensor on {like.device}, 16-byte aligned")
    return t


def _enqueue(what, fn, gpu, *args):
    """Calls a library entry on the current stream of device ``gpu``, with that device current."""
    if _device() == gpu:
        code = fn(*args, _stream(gpu))
    else:
        with torch.cuda.device(gpu):
            code = fn(*args, _stream(gpu))
    if code:
        check(code, what)


def _not_captured(device):
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a paged cache cannot be made while the current stream is being captured: what clears "
                               "its memory would only be recorded")


class PagedKVCache:
    """One layer's pool of KV pages (tl_paged_kv).

    ``k`` and ``v`` are ``[num_pages, kv_heads, page_size, head_dim]`` tensors of
    int8, bfloat16 or float16; an int8 pool has float32 ``k_scale`` and
    ``v_scale`` ``[num_pages, kv_heads, page_size]``, one scale per stored row.
    ``head_dim`` is 64 or 128, ``page_size`` any positive number.

    The caller owns the page allocation: position ``p`` of sequence ``s`` is row
    ``p % page_size`` of page ``block_table[s, p // page_size]`` (int32 on the
    device). Entries that name no sequence, position or page are skipped (see
    each call), so a batch of fixed size is padded with ``seq = -1``. Calls on
    one cache are serialized by the caller, as on an engine: on one stream, or
    ordered by events. A cache may be dropped while its calls run on whichever
    stream: what it has allocated is kept until they end (tensors that the caller
    passed are the caller's to keep, and a cache lives as long as a graph with its
    calls). No call synchronises or allocates beyond its outputs (taken from
    torch's allocator), so with preallocated outputs calls can be captured in a
    CUDA graph, the first one too. Making a cache allocates the attention's
    scratch (2.5 or 5 MB), waits until the current stream has cleared it, and is
    refused (RuntimeError) while that stream is being captured.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=None, device="cuda"):
        """Allocates the pool, zeroed; ``dtype`` is torch.int8 (default), bfloat16 or float16."""
        _need_torch()
        dtype = torch.int8 if dtype is None else dtype
        if dtype not in _POOL_CODES:
            raise ValueError(f"dtype must be one of {[str(x) for x in _POOL_CODES]}, got {dtype}")
        if min(num_pages, page_size, kv_heads) < 1 or head_dim not in HEAD_DIMS:
            raise ValueError(f"num_pages, page_size and kv_heads must be positive and head_dim one of {HEAD_DIMS}")
        if not torch.cuda.is_available():
            raise RuntimeError("no CUDA device visible: the paged cache runs only on the GPU")
        _not_captured(device)
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        ks, vs = ((torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
                  if dtype == torch.int8 else (None, None))
        self._bind(k, v, ks, vs)
        self._owned += [t for t in (k, v, ks, vs) if t is not None]

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None) -> "PagedKVCache":
        """A cache over tensors the caller owns (one layer's slice of a larger pool, for instance)."""
        _need_torch()
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale):
        for name, t in (("k", k), ("v", v)):
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 4 and t.dtype in _POOL_CODES
                    and t.numel() and t.is_contiguous() and not t.data_ptr() & 15):
                raise _bad(name, t, "a contiguous, 16-byte aligned CUDA tensor [num_pages, kv_heads, page_size, "
                                    "head_dim] of int8, bfloat16 or float16")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must agree in shape, type and device")
        _not_captured(k.device)
        if k.shape[3] not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {k.shape[3]}")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if k.dtype != torch.int8:
                if t is not None:
                    raise ValueError(f"{name} is for int8 pools only")
            elif not (isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.shape == k.shape[:3]
                      and t.device == k.device and t.is_contiguous()):
                raise _bad(name, t, f"a contiguous float32 {list(k.shape[:3])} tensor on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self._gpu = k.device.index
        self._lib = lib = load_library()
        self._append, self._read, self._attend = lib.tl_paged_append, lib.tl_paged_read, lib.tl_paged_attn_decode
        ptr = [t.data_ptr() if t is not None else None for t in (k, v, k_scale, v_scale)]
        self._view = PagedView(*ptr, _POOL_CODES[k.dtype], *k.shape)
        self._ref = C.byref(self._view)
        self._scale = self.head_dim ** -0.5
        # The attention's scratch for any number of heads (its size depends on neither rows nor lengths). The
        # kernel needs it zeroed before the first call, whichever stream that runs on, and a call that is only
        # recorded in a graph clears nothing: so it is made here, and there when this returns.
        self._work_bytes = max(lib.tl_paged_attn_workspace_bytes(self.kv_heads * group, self.kv_heads, self.head_dim)
                               for group in (1, 16))
        self._work = torch.zeros(self._work_bytes, dtype=torch.uint8, device=self.device)
        torch.cuda.current_stream(self.device).synchronize()
        self._owned = [self._work]
        self._streams = {_stream(self._gpu)}  # raw handles of the streams that the allocator knows to use them

    def _enter_stream(self):
        """The current stream's first call: without this the allocator would hand the memory on as soon as the cache
        is dropped, ordered behind the stream that it was allocated on only."""
        for t in self._owned:
            t.record_stream(torch.cuda.current_stream(self.device))
        self._streams.add(_stream(self._gpu))

    # ---------------------------------------------------------------- calls
    def _table(self, t):
        if isinstance(t, _Tensor) and t.dtype is _INT32 and t.dim() == 2 and t.get_device() == self._gpu:
            n, m = t.shape
            stride, one = t.stride()
            if n < 2:
                stride = m
            if n and m and (one == 1 or m == 1) and stride >= m:
                return t.data_ptr(), n, m, stride
        raise _bad("block_table", t, f"an int32 [n_seqs, max_pages] tensor on {self.device} with contiguous rows that "
                                     "do not overlap")

    def append(self, k, v, block_table, seq, pos, cos=None, sin=None, q=None, q_out=None):
        """Stores key and value rows ``k``, ``v`` ``[tokens, kv_heads, head_dim]`` at
        ``(seq[t], pos[t])``, the keys rotated by their position on the way
        (tl_paged_append).

        ``cos`` and ``sin`` are :func:`shim.rope_tables`' float32 ``[max_positions,
        head_dim]`` on the device. ``q`` ``[tokens, heads, head_dim]`` is rotated too
        and returned (in ``q_out`` when given; ``q_out is q`` rotates a contiguous
        ``q`` in place); without ``q`` the result is None. Without ``cos`` and
        ``sin`` the keys are stored as they are. ``k``, ``v`` and ``q`` are float32,
        bfloat16 or float16 and may be columns of one fused projection. Tokens
        that name no row store nothing; a position beyond the angles stores
        nothing and gives a zero query row.
        """
        if not isinstance(k, torch.Tensor) or k.dim() != 3 or k.dtype not in _FLOAT_CODES:
            raise _bad("k", k, "a float32, bfloat16 or float16 [tokens, kv_heads, head_dim] tensor")
        n, dt, gpu, d = k.shape[0], k.dtype, self._gpu, self.head_dim
        kp, ks = _rows("k", k, n, self.kv_heads, d, dt, gpu)
        vp, vs = _rows("v", v, n, self.kv_heads, d, dt, gpu)
        tp, seqs, pages, ts = self._table(block_table)
        sp, pp = _index("seq", seq, n, gpu), _index("pos", pos, n, gpu)
        cp = np = angles = qp = qs = heads = op = 0
        if cos is not None or sin is not None:
            if cos is None or sin is None:
                raise ValueError("cos and sin go together")
            angles = cos.shape[0] if isinstance(cos, torch.Tensor) and cos.dim() else 0
            cp, np = _angles("cos", cos, angles, d, gpu), _angles("sin", sin, angles, d, gpu)
        if q is not None:
            if not angles:
                raise ValueError("q needs cos and sin")
            if not isinstance(q, torch.Tensor) or q.dim() != 3 or not q.shape[1]:
                raise _bad("q", q, "a [tokens, heads, head_dim] tensor")
            heads = q.shape[1]
            qp, qs = _rows("q", q, n, heads, d, dt, gpu)
            q_out = _out("q_out", q_out, q, (n, heads, d), dt)
            op = q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        if n:
            if _stream(gpu) not in self._streams:
                self._enter_stream()
            _enqueue("tl_paged_append", self._append, gpu, self._ref,
                     _APPEND.pack(qp, kp, vp, op, sp, pp, tp, cp, np, qs, ks, vs, ts, _FLOAT_CODES[dt], seqs, pages,
                                  angles, n, heads))
        return q_out

    def read(self, block_table, seq, pos, dtype=None, k_out=None, v_out=None):
        """Rows ``(seq[t], pos[t])`` as ``(k, v)``, each ``[tokens, kv_heads, head_dim]`` of
        ``dtype`` (float32 by default; tl_paged_read). Keys are as stored, rotated.
        Tokens that name no row give zeros."""
        dtype = torch.float32 if dtype is None else dtype
        if dtype not in _FLOAT_CODES:
            raise ValueError(f"dtype must be one of {[str(x) for x in _FLOAT_CODES]}, got {dtype}")
        if not isinstance(seq, torch.Tensor) or seq.dim() != 1:
            raise _bad("seq", seq, "an int32 vector")
        n, gpu = seq.shape[0], self._gpu
        tp, seqs, pages, ts = self._table(block_table)
        sp, pp = _index("seq", seq, n, gpu), _index("pos", pos, n, gpu)
        shape = (n, self.kv_heads, self.head_dim)
        k, v = _out("k_out", k_out, self.k, shape, dtype), _out("v_out", v_out, self.k, shape, dtype)
        if n:
            if _stream(gpu) not in self._streams:
                self._enter_stream()
            _enqueue("tl_paged_read", self._read, gpu, self._ref,
                     _READ.pack(sp, pp, tp, k.data_ptr(), v.data_ptr(), ts, seqs, pages, n, _FLOAT_CODES[dtype]))
        return k, v

    def attend(self, q, block_table, lengths, seq=None, sm_scale=None, out=None, return_lse=False, lse=None):
        """Attention of one new token of each row's sequence over its first
        ``lengths[r]`` positions (tl_paged_attn_decode).

        ``q`` ``[rows, heads, head_dim]`` is already rotated (:meth:`append` returns
        it), float32, bfloat16 or float16 whatever the pool's type; ``heads`` is any
        multiple of ``kv_heads``. Row ``r`` reads sequence ``seq[r]`` (default
        ``r``). ``sm_scale`` defaults to ``head_dim ** -0.5``. Returns ``out`` of
        ``q``'s shape and type, with ``return_lse`` also the float32 log-sum-exp
        ``[rows, heads]`` of the scores. A row without positions gives zeros and
        -inf.
        """
        if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in _FLOAT_CODES:
            raise _bad("q", q, "a float32, bfloat16 or float16 [rows, heads, head_dim] tensor")
        n, heads, d = q.shape
        dt, gpu = q.dtype, self._gpu
        if d != self.head_dim or not heads or heads % self.kv_heads:
            raise ValueError(f"q has {heads} heads of {d}: the pool has {self.kv_heads} heads of {self.head_dim}, and "
                             "q's must be a multiple")
        qp, qs = _rows("q", q, n, heads, d, dt, gpu)
        tp, seqs, pages, ts = self._table(block_table)
        lp = _index("lengths", lengths, n, gpu)
        sp = 0
        if seq is not None:
            sp = _index("seq", seq, n, gpu)
        elif n > seqs:
            raise ValueError(f"{n} rows but the table has {seqs} sequences: pass seq")
        out = _out("out", out, q, (n, heads, d), dt)
        if return_lse or lse is not None:
            lse = _out("lse", lse, q, (n, heads), torch.float32)
        if n:
            if _stream(gpu) not in self._streams:
                self._enter_stream()
            _enqueue("tl_paged_attn_decode", self._attend, gpu, self._ref,
                     _ATTEND.pack(qp, sp, lp, tp, out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                                  self._work.data_ptr(), self._work_bytes, qs, ts, _FLOAT_CODES[dt], seqs, pages, n,
                                  heads, self._scale if sm_scale is None else float(sm_scale)))
        return (out, lse) if return_lse else out


class TokenLogprobs(NamedTuple):
    logprob: object       # float32 [rows], None without tokens
    entropy: object       # float32 [rows]
    top_ids: object       # int32 [rows, top_k]
    top_logprobs: object  # float32 [rows, top_k]


def token_logprobs(logits, tokens=None, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` (int32 ``[rows]``), the entropy and the
    ``top_k`` (at most 32) most likely tokens of each row of ``logits``
    ``[rows, vocab]`` (float32, bfloat16 or float16; rows may be strided), in one
    pass over them (tl_token_logprobs). Equal logits are listed by the lowest
    id. Logits of -inf have probability 0 and are never listed (id -1, -inf).
    A negative token gives 0, one beyond the vocabulary NaN; a row with a NaN or
    +inf gives NaN everywhere."""
    _need_torch()
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dim() == 2 and logits.dtype in _FLOAT_CODES
            and logits.shape[1] and (logits.shape[1] == 1 or logits.stride(1) == 1)):
        raise _bad("logits", logits, "a CUDA tensor [rows, vocab] of float32, bfloat16 or float16 with contiguous rows")
    n, vocab = logits.shape
    dev = logits.device
    stride = logits.stride(0) if n > 1 else vocab
    if stride < vocab:
        raise _bad("logits", logits, "rows that do not overlap")
    if not 0 <= top_k <= TOP_K_MAX:
        raise ValueError(f"top_k must be in 0..{TOP_K_MAX}, got {top_k}")
    gpu = dev.index
    tp = 0 if tokens is None else _index("tokens", tokens, n, gpu)
    f32 = torch.float32
    # the float32 results share one allocation
    if tokens is None:
        lp = None
        ent, top = logits.new_empty(n * (1 + top_k), dtype=f32).split_with_sizes((n, n * top_k))
    else:
        lp, ent, top = logits.new_empty(n * (2 + top_k), dtype=f32).split_with_sizes((n, n, n * top_k))
    top = top.view(n, top_k)
    ids = logits.new_empty(n, top_k, dtype=_INT32)
    if n:
        _enqueue("tl_token_logprobs", load_library().tl_token_logprobs, gpu,
                 _LOGPROBS.pack(logits.data_ptr(), tp, 0 if lp is None else lp.data_ptr(), ent.data_ptr(),
                                ids.data_ptr(), top.data_ptr(), stride, _FLOAT_CODES[logits.dtype], n, vocab, top_k))
    return TokenLogprobs(lp, ent, ids, top)
