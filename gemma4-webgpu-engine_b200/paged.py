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

_I32, _FLOAT = torch.int32, torch.float32
_workspaces: dict = {}
_needs: dict = {}


def _invalid(message: str):
    return _abi.G4Error(-1, message)


_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(device):
    """(its index, the current stream there, the device that was current if another has to be)."""
    index, current = device.index, _current_device()
    if index == current:
        return index, _current_stream(index), None
    torch.cuda.set_device(index)
    return index, _current_stream(index), current


def _type(t: torch.Tensor, what: str) -> int:
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise _invalid(f"{what} is f32 or bf16, got {t.dtype}")
    return kind


def _ints(t: torch.Tensor, what: str, device, n: int) -> int:
    if t.dtype is not _I32 or t.device != device or t.dim() != 1 or t.shape[0] < n or not t.is_contiguous():
        raise _invalid(f"{what} is a contiguous int32 vector of {n} or more on {device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, what: str, device, shape) -> int:
    """Stride between rows of t [n, heads, head_dim], whose rows are contiguous."""
    if t.shape != shape or t.device != device:
        raise _invalid(f"{what} is {list(shape)} on {device}, got {list(t.shape)} on {t.device}")
    s = t.stride()
    if (s[2] != 1 or s[1] != shape[2]) and t.numel():
        raise _invalid(f"{what}: one token's heads are contiguous")
    return s[0] if shape[0] > 1 else shape[1] * shape[2]


def _workspace(device, index: int, stream: int, need: int) -> torch.Tensor:
    key = (index, stream)
    ws = _workspaces.get(key)
    if ws is None or ws.shape[0] < need:
        ws = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def _need(key, ask) -> int:
    need = _needs.get(key)
    if need is None:
        n = C.c_uint64()
        _abi.check(ask(C.byref(n)))
        if len(_needs) > 4096:
            _needs.clear()
        need = _needs[key] = n.value
    return need


class PagePool:
    """A pool of pages over k, v [n_pages, kv_heads, page_size, head_dim] (bf16, int8 or e4m3) and,
    for 8-bit pages, k_scale, v_scale f32 [n_pages, kv_heads, page_size]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        shape, device, fmt = k.shape, k.device, _FORMATS.get(k.dtype)
        if len(shape) != 4 or shape != v.shape or k.dtype != v.dtype or fmt is None:
            raise _invalid("k and v are [n_pages, kv_heads, page_size, head_dim] of bf16, int8 or e4m3")
        if not k.is_cuda or device != v.device or not k.is_contiguous() or not v.is_contiguous():
            raise _invalid("k and v are contiguous on one CUDA device")
        ks = vs = None
        if fmt:
            for s in (k_scale, v_scale):
                if s is None or s.dtype is not _FLOAT or s.shape != shape[:3] or s.device != device \
                        or not s.is_contiguous():
                    raise _invalid("8-bit pages need f32 scales [n_pages, kv_heads, page_size]")
            ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
        elif k_scale is not None or v_scale is not None:
            raise _invalid("bf16 pages have no scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = device
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = shape
        self.format = fmt
        self.struct = _abi.PagePool(k.data_ptr(), v.data_ptr(), ks, vs, *(shape[i] for i in (0, 2, 1, 3)), fmt)
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
        n, device = k.shape[0], self.device
        shape = (n, self.kv_heads, self.head_dim)
        ks, vs = _rows(k, "k", device, shape), _rows(v, "v", device, shape)
        if k.dtype is not v.dtype:
            raise _invalid("k and v have one type")
        kind, at = _type(k, "k"), _ints(slots, "slots", device, n)
        _, stream, back = _on(device)
        rc = self.lib.g4_op_page_store(self.ref, k.data_ptr(), v.data_ptr(), kind, ks, vs, n, at, stream) if n else 0
        if back is not None:
            torch.cuda.set_device(back)
        _abi.check(rc)

    def read(self, slots: torch.Tensor, dtype=torch.float32, k_out: torch.Tensor | None = None,
             v_out: torch.Tensor | None = None):
        """The rows at `slots`, dequantised: (k, v) [tokens, kv_heads, head_dim]."""
        n, device = slots.numel(), self.device
        shape = (n, self.kv_heads, self.head_dim)
        if k_out is None:
            k_out = torch.empty(shape, dtype=dtype, device=device)
        if v_out is None:
            v_out = torch.empty(shape, dtype=dtype, device=device)
        if k_out.dtype is not v_out.dtype:
            raise _invalid("k_out and v_out have one type")
        ks, vs = _rows(k_out, "k_out", device, shape), _rows(v_out, "v_out", device, shape)
        kind, at = _type(k_out, "dtype"), _ints(slots, "slots", device, n)
        _, stream, back = _on(device)
        rc = self.lib.g4_op_page_read(self.ref, at, n, kind, k_out.data_ptr(), v_out.data_ptr(), ks, vs, stream) if n else 0
        if back is not None:
            torch.cuda.set_device(back)
        _abi.check(rc)
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
    rows, heads, _ = q.shape
    shape = (rows, heads, pool.head_dim)
    qs = _rows(q, "q", dev, shape)
    kind = _type(q, "q")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os = heads * pool.head_dim
    elif out.dtype is not q.dtype:
        raise _invalid("out has q's type")
    else:
        os = _rows(out, "out", dev, shape)
    if page_table.dim() != 2 or page_table.dtype is not _I32 or page_table.device != dev:
        raise _invalid(f"page_table is int32 [batch, pages] on {dev}")
    batch, width = page_table.shape
    stride, step = page_table.stride()
    if batch < 2:
        stride = width
    if (step != 1 and width > 1) or stride < width:
        raise _invalid("page_table's rows are contiguous and do not overlap")
    if lse is not None and (lse.dtype is not _FLOAT or lse.device != dev or not lse.is_contiguous()
                            or lse.shape != (rows, heads)):
        raise _invalid("lse is f32 [rows, heads]")
    begin, pos, length = (_ints(q_begin, "q_begin", dev, batch + 1), _ints(q_pos, "q_pos", dev, batch),
                          _ints(kv_len, "kv_len", dev, batch))
    # Positions past the table's width are cut off, as those past max_kv are.
    max_kv = min(max_kv, width * pool.page_size)
    index, stream, back = _on(dev)
    try:
        lib = pool.lib
        need = _need((pool.kv_heads, pool.page_size, pool.head_dim, pool.format, kind, heads, rows, batch, max_q, max_kv,
                      window), lambda n: lib.g4_op_paged_attention_workspace(
                          pool.ref, kind, heads, rows, batch, max_q, max_kv, window, n))
        ws = _workspace(dev, index, stream, need)
        rc = lib.g4_op_paged_attention(
            pool.ref, q.data_ptr(), qs, out.data_ptr(), os, None if lse is None else lse.data_ptr(), kind, heads, rows,
            batch, begin, pos, length, page_table.data_ptr(), stride, max_q, max_kv, window, scale, ws.data_ptr(),
            ws.shape[0], stream)
    finally:
        if back is not None:
            torch.cuda.set_device(back)
    if rc:
        _abi.check(rc)
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
    batch = row_begin.shape[0] - 1
    kind = _type(logits, "logits")
    for t, what, n in ((uniforms, "uniforms", rows), (temperature, "temperature", batch)):
        if t.dtype is not _FLOAT or t.device != dev or t.numel() < n or not t.is_contiguous():
            raise _invalid(f"{what} is a contiguous f32 vector of {n} or more on {dev}")
    for t, what, n in ((gumbel, "gumbel", batch), (draft_probs, "draft_probs", rows)):
        if t is not None and (t.dtype is not _FLOAT or t.device != dev or t.dim() != 2
                              or t.shape[0] < n or t.shape[1] != vocab or t.stride(1) != 1):
            raise _invalid(f"{what} is f32 [{n}, {vocab}] on {dev}, rows contiguous")
    begin, at = _ints(row_begin, "row_begin", dev, batch + 1), _ints(drafts, "drafts", dev, rows)
    if max_drafts < 0 or batch < 0:
        raise _invalid("max_drafts is not negative, and row_begin holds one more than the sequences")
    lib = _abi.load()
    tokens = torch.empty((batch, max_drafts + 1), dtype=_I32, device=dev)
    logprobs = torch.empty((batch, max_drafts + 1), dtype=_FLOAT, device=dev)
    counts = torch.empty(batch, dtype=_I32, device=dev)
    index, stream, back = _on(dev)
    try:
        need = _need((vocab, rows, batch, max_drafts), lambda n: lib.g4_op_verify_drafts_workspace(
            vocab, rows, batch, max_drafts, n))
        ws = _workspace(dev, index, stream, need)
        rc = lib.g4_op_verify_drafts(
            logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, kind, vocab, rows, batch, begin, at,
            None if draft_probs is None else draft_probs.data_ptr(),
            0 if draft_probs is None else draft_probs.stride(0) if rows > 1 else vocab, uniforms.data_ptr(),
            gumbel.data_ptr(), gumbel.stride(0) if batch > 1 else vocab, temperature.data_ptr(), max_drafts,
            tokens.data_ptr(), logprobs.data_ptr(), counts.data_ptr(), ws.data_ptr(), ws.shape[0], stream)
    finally:
        if back is not None:
            torch.cuda.set_device(back)
    if rc:
        _abi.check(rc)
    return tokens, logprobs, counts


def errors(device=None) -> int:
    """The BAD_PAGE / BAD_LENGTH / TIMEOUT bits raised on `device` since the last call. Waits for
    the device."""
    flags = C.c_int32()
    with torch.cuda.device(device):
        _abi.check(_abi.load().g4_op_paged_errors(C.byref(flags)))
    return flags.value
