"""The paged 8-bit K/V cache of a serving batch (include/sepia_cuda.h,
SepiaKv8Cache; csrc/kv8_append.cu, csrc/kv8_attn.cu).

  Kv8Cache      one layer's blocks: e4m3 codes, a power-of-two scale per block
                and KV head, fp16 tails of the unfinished blocks
  Kv8Step       one step of a batch, shared by all layers: the block table,
                the tokens held, the new tokens of each sequence
  append        norms, rotates and stores new keys and values (and the queries
                beside them); attention reads them back

Tensors only carry device memory here; every computation is one of the
library's CUDA kernels. A step's lengths stay on the device: a caller that
replays a CUDA graph changes them in place.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from .lib import SepiaKv8Append, SepiaKv8Attn, SepiaKv8Cache, SepiaKv8Step, last_error, load

_F16 = {torch.float32: 0, torch.float16: 1}


def _fail(what):
    raise ValueError(f"sepia_b200: kv8: {what}")


def _check(t, name, dtype, shape):
    """The pointer of a contiguous CUDA tensor of this type and shape."""
    if t.dtype is not dtype or not t.is_cuda or not t.is_contiguous():
        _fail(f"{name} must be a contiguous CUDA tensor of {dtype}")
    if t.shape != shape:
        _fail(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t.data_ptr()


def _rows(t, name, dtype, heads, dim, n):
    """A [tokens, heads, dim] tensor whose heads lie side by side; returns (pointer, token stride)."""
    if t.dtype is not dtype or not t.is_cuda:
        _fail(f"{name} must be a CUDA tensor; q, k and v must have one type, float32 or float16")
    if t.shape != (n, heads, dim):
        _fail(f"{name} has shape {tuple(t.shape)}, expected {(n, heads, dim)}")
    s0, s1, s2 = t.stride()
    if n and (s2 != 1 or (heads > 1 and s1 != dim)):
        _fail(f"the heads of {name} must lie side by side")
    return t.data_ptr(), s0 if n > 1 else heads * dim


def _stream(index, stream):
    return torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream


def _empty_like(t, stream):
    """A result's memory belongs to the stream that fills it."""
    if stream is None:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return torch.empty_like(t, memory_format=torch.contiguous_format)


def rotation_table(n_positions: int, rot_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """Cosines and sines [n_positions, rot_dim/2, 2] of angle position * base^(-2i/rot_dim), from 64-bit angles."""
    freq = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    ang = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()


class Kv8Step:
    """One step of a batch. table int32 [n_seqs, columns], kv_len int32
    [n_seqs] (tokens held before the step; < 0: idle), start int32
    [n_seqs + 1] (None: one new token each), slot int32 [n_seqs] (None: row s
    of the tails). n_tokens, max_new and max_kv are host bounds; max_new
    defaults to n_tokens with start (a tighter bound is less work) and to 1
    without, max_kv to what the table can hold."""

    def __init__(self, table, kv_len, start=None, slot=None, n_tokens=None, max_new=None, max_kv=None):
        n = kv_len.shape[0]
        if table.dim() != 2:
            _fail("table must have two dimensions")
        st = SepiaKv8Step()
        st.table = _check(table, "table", torch.int32, (n, table.shape[1]))
        st.kv_len = _check(kv_len, "kv_len", torch.int32, (n,))
        st.start = _check(start, "start", torch.int32, (n + 1,)) if start is not None else None
        st.slot = _check(slot, "slot", torch.int32, (n,)) if slot is not None else None
        st.n_seqs, st.table_cols = n, table.shape[1]
        st.n_tokens = n if n_tokens is None else int(n_tokens)
        st.max_new = int(max_new) if max_new is not None else 1 if start is None else st.n_tokens
        st.max_kv = -1 if max_kv is None else int(max_kv)
        self.n_tokens, self.struct, self._keep = st.n_tokens, st, (table, kv_len, start, slot)
        self.device, self.index = kv_len.device, kv_len.device.index
        self._max_kv, self._bound, self._ws, self._lock = max_kv, {}, {}, threading.Lock()

    def _for(self, cache):
        """The address of the step's struct for this cache's block size."""
        b = cache.block
        r = self._bound.get(b)
        if r is None:
            st = SepiaKv8Step.from_buffer_copy(self.struct)
            if self._max_kv is None:
                st.max_kv = st.table_cols * b
            r = self._bound[b] = (C.addressof(st), st)
        return r[0]

    def workspace(self, cache, attn, key, stream):
        """The attention workspace for one shape and stream. It serves one call at a time, which takes
        two launches in a row: callers hold the step's lock from here to the call's end."""
        ws = self._ws.get(key)
        if ws is None:
            nb = load().sepia_cuda_kv8_attn_ws_bytes(cache._ref, self._for(cache), C.addressof(attn))
            if not nb:
                raise RuntimeError(f"sepia_b200: kv8_attn: {last_error()}")
            with torch.cuda.stream(stream):            # None: the current one
                t = torch.empty(nb, dtype=torch.uint8, device=self.device)
            ws = self._ws[key] = (t.data_ptr(), nb, t)
        return ws


class Kv8Cache:
    """One layer's cache over tensors of the caller: k, v float8_e4m3fn
    [n_blocks, n_kv_heads, block, head_dim], k_scale, v_scale float32
    [n_blocks, n_kv_heads], k_tail, v_tail float16 [n_slots, n_kv_heads,
    block, head_dim]."""

    def __init__(self, k, v, k_scale, v_scale, k_tail, v_tail):
        if k.dim() != 4 or k_tail.dim() != 4:
            _fail("k and k_tail must have four dimensions")
        n, hk, b, d = k.shape
        st = SepiaKv8Cache()
        st.n_blocks, st.n_slots, st.n_kv_heads, st.head_dim, st.block = n, k_tail.shape[0], hk, d, b
        for name, t in (("k", k), ("v", v)):
            setattr(st, name, _check(t, name, torch.float8_e4m3fn, (n, hk, b, d)))
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            setattr(st, name, _check(t, name, torch.float32, (n, hk)))
        for name, t in (("k_tail", k_tail), ("v_tail", v_tail)):
            setattr(st, name, _check(t, name, torch.float16, (k_tail.shape[0], hk, b, d)))
        self.struct, self.n_kv_heads, self.head_dim, self.block = st, hk, d, b
        self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail = k, v, k_scale, v_scale, k_tail, v_tail
        self._ref, lib = C.addressof(st), load()
        self._append, self._attn = lib.sepia_cuda_kv8_append, lib.sepia_cuda_kv8_attn

    @classmethod
    def allocate(cls, n_blocks, n_slots, n_kv_heads, head_dim, block=32, device="cuda"):
        def codes():
            return torch.zeros(n_blocks, n_kv_heads, block, head_dim, dtype=torch.uint8,
                               device=device).view(torch.float8_e4m3fn)

        def scales():
            return torch.ones(n_blocks, n_kv_heads, device=device)

        def tails():
            return torch.zeros(n_slots, n_kv_heads, block, head_dim, dtype=torch.float16, device=device)
        return cls(codes(), codes(), scales(), scales(), tails(), tails())

    def append(self, step, k, v, q=None, k_norm=None, q_norm=None, eps=1e-6, q_scale=None, rotation=None,
               adjacent=False, q_out=None, stream=None):
        """Stores the new tokens' keys and values (float32 or float16
        [n_tokens, heads, head_dim]; a token's heads side by side, any token
        stride): norm of each head, rotation by position, 8 bits. With q, also
        norms, rotates and scales (q_scale float32 [n_tokens]) the queries into
        q_out, which is returned."""
        d, hk, n, dt = self.head_dim, self.n_kv_heads, step.n_tokens, k.dtype
        if dt not in _F16:
            _fail("k must be float32 or float16")
        a = SepiaKv8Append()
        a.x_f16, a.eps = _F16[dt], eps
        a.k, a.k_stride = _rows(k, "k", dt, hk, d, n)
        a.v, a.v_stride = _rows(v, "v", dt, hk, d, n)
        if k_norm is not None:
            a.k_norm = _check(k_norm, "k_norm", torch.float32, (d,))
        if q is not None:
            a.n_heads = h = q.shape[1]
            a.q, a.q_stride = _rows(q, "q", dt, h, d, n)
            if q_out is None:
                q_out = _empty_like(q, stream)
                a.q_out = q_out.data_ptr()
            else:
                a.q_out = _check(q_out, "q_out", dt, (n, h, d))
            if q_norm is not None:
                a.q_norm = _check(q_norm, "q_norm", torch.float32, (d,))
            if q_scale is not None:
                a.q_scale = _check(q_scale, "q_scale", torch.float32, (n,))
        if rotation is not None:
            r = rotation.shape
            if len(r) != 3 or r[2] != 2:
                _fail("rotation must be [positions, rot_dim/2, 2]")
            a.rotation = _check(rotation, "rotation", torch.float32, r)
            a.rot_positions, a.rot_dim, a.rot_adjacent = r[0], 2 * r[1], adjacent
        if not self._append(self._ref, step._for(self), C.addressof(a), _stream(step.index, stream)):
            raise RuntimeError(f"sepia_b200: kv8_append failed: {last_error()}")
        return q_out

    def attention(self, step, q, scale, window=0, rel_logits=None, tau=None, out=None, stream=None):
        """Causal attention of the new tokens (after append) over what the
        cache holds of their sequences. rel_logits float32 [n_tokens, heads,
        extent] is added at distance 0 .. extent-1, times tau[token]."""
        d, n, dt = self.head_dim, step.n_tokens, q.dtype
        if dt not in _F16 or q.dim() != 3:
            _fail("q must be float32 or float16 [tokens, heads, head_dim]")
        a = SepiaKv8Attn()
        a.n_heads = h = q.shape[1]
        a.x_f16, a.scale, a.window = _F16[dt], scale, window
        a.q, a.q_stride = _rows(q, "q", dt, h, d, n)
        if out is None:
            out = _empty_like(q, stream)
            a.out = out.data_ptr()
        else:
            a.out = _check(out, "out", dt, (n, h, d))
        if rel_logits is not None:
            e = rel_logits.shape[-1]
            a.rel_logits = _check(rel_logits, "rel_logits", torch.float32, (n, h, e))
            a.rel_extent = e
        if tau is not None:
            a.tau = _check(tau, "tau", torch.float32, (n,))
        st = _stream(step.index, stream)
        with step._lock:                               # host threads that share a step take turns
            ws = step.workspace(self, a, (st, a.x_f16, h, self.n_kv_heads, d, self.block, window), stream)
            if not self._attn(self._ref, step._for(self), C.addressof(a), ws[0], ws[1], st):
                raise RuntimeError(f"sepia_b200: kv8_attn failed: {last_error()}")
        return out
