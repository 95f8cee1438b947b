"""Paged, quantised KV cache on torch tensors: the Python face of g4_op_page_store / page_read,
g4_op_paged_attention and g4_op_verify_drafts (include/g4.h states what each computes).

Calls launch on the current torch stream and wait for nothing. Workspaces are kept per (device,
stream) and grow as calls need them. What a call finds wrong in device data (a page outside the
pool, lengths past their bounds) is collected on the device and read by `errors()`.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _abi

F32, BF16 = 0, 1
_TYPES = {torch.float32: F32, torch.bfloat16: BF16}
_FORMATS = {torch.bfloat16: 0, torch.int8: 1, torch.float8_e4m3fn: 2}
_PAGE_TYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}

BAD_PAGE, BAD_LENGTH, TIMEOUT = 1, 2, 4

_workspaces: dict = {}
_needs: dict = {}


def _invalid(message: str):
    return _abi.G4Error(-1, message)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _type(t: torch.Tensor, what: str) -> int:
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise _invalid(f"{what} is f32 or bf16, got {t.dtype}") from None


def _ints(t: torch.Tensor, what: str, device, n: int) -> int:
    if t.dtype != torch.int32 or t.device != device or t.dim() != 1 or t.numel() < n or not t.is_contiguous():
        raise _invalid(f"{what} is a contiguous int32 vector of {n} or more on {device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, what: str, device, shape) -> int:
    """Stride between rows of t [n, heads, head_dim], whose rows are contiguous."""
    if t.device != device or tuple(t.shape) != shape:
        raise _invalid(f"{what} is {list(shape)} on {device}, got {list(t.shape)} on {t.device}")
    if t.numel() and (t.stride(2) != 1 or t.stride(1) != shape[2]):
        raise _invalid(f"{what}: one token's heads are contiguous")
    return t.stride(0) if shape[0] > 1 else shape[1] * shape[2]


def _workspace(device, stream: int, need: int) -> torch.Tensor:
    key = (device, stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


class PagePool:
    """A pool of pages over k, v [n_pages, kv_heads, page_size, head_dim] (bf16, int8 or e4m3) and,
    for 8-bit pages, k_scale, v_scale f32 [n_pages, kv_heads, page_size]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _FORMATS:
            raise _invalid("k and v are [n_pages, kv_heads, page_size, head_dim] of bf16, int8 or e4m3")
        if not k.is_cuda or k.device != v.device or not k.is_contiguous() or not v.is_contiguous():
            raise _invalid("k and v are contiguous on one CUDA device")
        fmt = _FORMATS[k.dtype]
        if fmt:
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or s.device != k.device \
                        or not s.is_contiguous():
                    raise _invalid("8-bit pages need f32 scales [n_pages, kv_heads, page_size]")
        elif k_scale is not None or v_scale is not None:
            raise _invalid("bf16 pages have no scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.struct = _abi.PagePool(k.data_ptr(), v.data_ptr(), _abi.ptr(k_scale), _abi.ptr(v_scale),
                                    self.n_pages, self.page_size, self.kv_heads, self.head_dim, fmt)
        self.ref = C.byref(self.struct)
        self.lib = _abi.load()

    @classmethod
    def create(cls, n_pages: int, page_size: int, kv_heads: int, head_dim: int, format: str = "int8",
               device="cuda") -> "PagePool":
        """A zeroed pool; `format` is "bf16", "int8" or "e4m3"."""
        if format not in _PAGE_TYPES:
            raise _invalid(f"page format {format!r}: bf16, int8 or e4m3")
        shape = (n_pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8 if format != "bf16" else torch.bfloat16,
                            device=device) for _ in range(2))
        if format == "bf16":
            return cls(k, v)
        t = _PAGE_TYPES[format]
        ks, vs = (torch.zeros(shape[:3], device=device) for _ in range(2))
        return cls(k.view(t), v.view(t), ks, vs)

    def store(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise rows k, v [tokens, kv_heads, head_dim] into the pages at `slots`."""
        n = k.shape[0]
        shape = (n, self.kv_heads, self.head_dim)
        ks, vs = _rows(k, "k", self.device, shape), _rows(v, "v", self.device, shape)
        if k.dtype != v.dtype:
            raise _invalid("k and v have one type")
        if n == 0:
            return
        with torch.cuda.device(self.device):
            _abi.check(self.lib.g4_op_page_store(
                self.ref, k.data_ptr(), v.data_ptr(), _type(k, "k"), ks, vs, n,
                _ints(slots, "slots", self.device, n), _stream(k)))

    def read(self, slots: torch.Tensor, dtype=torch.float32, k_out: torch.Tensor | None = None,
             v_out: torch.Tensor | None = None):
        """The rows at `slots`, dequantised: (k, v) [tokens, kv_heads, head_dim]."""
        n = slots.numel()
        shape = (n, self.kv_heads, self.head_dim)
        if k_out is None:
            k_out = torch.empty(shape, dtype=dtype, device=self.device)
        if v_out is None:
            v_out = torch.empty(shape, dtype=dtype, device=self.device)
        if k_out.dtype != v_out.dtype:
            raise _invalid("k_out and v_out have one type")
        ks, vs = _rows(k_out, "k_out", self.device, shape), _rows(v_out, "v_out", self.device, shape)
        if n:
            with torch.cuda.device(self.device):
                _abi.check(self.lib.g4_op_page_read(
                    self.ref, _ints(slots, "slots", self.device, n), n, _type(k_out, "dtype"),
                    k_out.data_ptr(), v_out.data_ptr(), ks, vs, _stream(k_out)))
        return k_out, v_out


def attention(pool: PagePool, q: torch.Tensor, q_begin: torch.Tensor, q_pos: torch.Tensor,
              kv_len: torch.Tensor, page_table: torch.Tensor, max_q: int, max_kv: int,
              window: int = 0, scale: float = 1.0, out: torch.Tensor | None = None,
              lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the ragged batch q [rows, heads, head_dim] over the pool's pages: sequence b's
    rows q_begin[b] .. are the positions q_pos[b] .., over kv_len[b] cached positions that lie in
    the pages page_table[b]. lse: optional f32 [rows, heads] output."""
    dev = pool.device
    if q.dim() != 3:
        raise _invalid("q is [rows, heads, head_dim]")
    rows, heads = q.shape[0], q.shape[1]
    shape = (rows, heads, pool.head_dim)
    qs = _rows(q, "q", dev, shape)
    kind = _type(q, "q")
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    elif out.dtype != q.dtype:
        raise _invalid("out has q's type")
    os = _rows(out, "out", dev, shape)
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != dev \
            or (page_table.numel() and page_table.stride(1) != 1):
        raise _invalid(f"page_table is int32 [batch, pages] on {dev}")
    batch, width = page_table.shape
    if lse is not None and (lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous()
                            or tuple(lse.shape) != (rows, heads)):
        raise _invalid("lse is f32 [rows, heads]")
    stride = page_table.stride(0) if batch > 1 else width
    if stride < width:
        raise _invalid("page_table's rows overlap")
    stream = _stream(q)
    with torch.cuda.device(dev):
        key = (pool.kv_heads, pool.page_size, pool.head_dim, pool.struct.format, kind, heads, rows,
               batch, max_q, max_kv, window)
        need = _needs.get(key)
        if need is None:
            n = C.c_uint64()
            _abi.check(pool.lib.g4_op_paged_attention_workspace(
                pool.ref, kind, heads, rows, batch, max_q, max_kv, window, C.byref(n)))
            if len(_needs) > 4096:
                _needs.clear()
            need = _needs[key] = n.value
        ws = _workspace(dev, stream, need)
        # Positions past the table's width are cut off by the stride only when it equals the width.
        _abi.check(pool.lib.g4_op_paged_attention(
            pool.ref, q.data_ptr(), qs, out.data_ptr(), os, _abi.ptr(lse), kind, heads, rows, batch,
            _ints(q_begin, "q_begin", dev, batch + 1), _ints(q_pos, "q_pos", dev, batch),
            _ints(kv_len, "kv_len", dev, batch), page_table.data_ptr(), stride, max_q,
            min(max_kv, width * pool.page_size), window, scale, ws.data_ptr(), ws.numel(), stream))
    return out


def verify_drafts(logits: torch.Tensor, row_begin: torch.Tensor, drafts: torch.Tensor,
                  uniforms: torch.Tensor, gumbel: torch.Tensor, temperature: torch.Tensor,
                  max_drafts: int, draft_probs: torch.Tensor | None = None):
    """Which drafted tokens stand, and the token each sequence emits after them: (tokens
    [batch, max_drafts + 1] padded with -1, their log probabilities, counts [batch])."""
    dev = logits.device
    if logits.dim() != 2 or not logits.is_cuda or logits.stride(1) != 1:
        raise _invalid("logits is [rows, vocab] on a CUDA device, rows contiguous")
    rows, vocab = logits.shape
    batch = row_begin.numel() - 1
    kind = _type(logits, "logits")
    for t, what, n in ((uniforms, "uniforms", rows), (temperature, "temperature", batch)):
        if t.dtype != torch.float32 or t.device != dev or t.numel() < n or not t.is_contiguous():
            raise _invalid(f"{what} is a contiguous f32 vector of {n} or more on {dev}")
    for t, what, n in ((gumbel, "gumbel", batch), (draft_probs, "draft_probs", rows)):
        if t is not None and (t.dtype != torch.float32 or t.device != dev or t.dim() != 2
                              or t.shape[0] < n or t.shape[1] != vocab or t.stride(1) != 1):
            raise _invalid(f"{what} is f32 [{n}, {vocab}] on {dev}, rows contiguous")
    lib = _abi.load()
    tokens = torch.empty((batch, max_drafts + 1), dtype=torch.int32, device=dev)
    logprobs = torch.empty((batch, max_drafts + 1), dtype=torch.float32, device=dev)
    counts = torch.empty(batch, dtype=torch.int32, device=dev)
    stream = _stream(logits)
    with torch.cuda.device(dev):
        key = (vocab, rows, batch, max_drafts)
        need = _needs.get(key)
        if need is None:
            n = C.c_uint64()
            _abi.check(lib.g4_op_verify_drafts_workspace(vocab, rows, batch, max_drafts, C.byref(n)))
            if len(_needs) > 4096:
                _needs.clear()
            need = _needs[key] = n.value
        ws = _workspace(dev, stream, need)
        _abi.check(lib.g4_op_verify_drafts(
            logits.data_ptr(), logits.stride(0), kind, vocab, rows, batch,
            _ints(row_begin, "row_begin", dev, batch + 1), _ints(drafts, "drafts", dev, rows),
            _abi.ptr(draft_probs), 0 if draft_probs is None else draft_probs.stride(0),
            uniforms.data_ptr(), gumbel.data_ptr(), gumbel.stride(0), temperature.data_ptr(),
            max_drafts, tokens.data_ptr(), logprobs.data_ptr(), counts.data_ptr(), ws.data_ptr(),
            ws.numel(), stream))
    return tokens, logprobs, counts


def errors(device=None) -> int:
    """The BAD_PAGE / BAD_LENGTH / TIMEOUT bits raised on `device` since the last call. Waits for
    the device."""
    flags = C.c_int32()
    with torch.cuda.device(device):
        _abi.check(_abi.load().g4_op_paged_errors(C.byref(flags)))
    return flags.value
