"""Python mirror of the 8-bit cache (shannon_prime_q8.h): rotary positions
with several axes, the quantising write, the read back and attention.  Every
method calls straight into the C-ABI; device buffers are torch CUDA tensors.
As everywhere in torch, tensors given to a call on another stream than the one
they were made on have to be ready there and to live until it has run."""
from __future__ import annotations

import ctypes as C

from . import (SP_DTYPE_BF16, SP_DTYPE_F16, SP_DTYPE_F32, SP_Q8_E4M3, SP_Q8_INT8, SP_ROPE_ADJACENT,
               SP_ROPE_AXIS_LADDER, SP_ROPE_HALVES, SP_ROPE_INTERLEAVED, SpConfig, SpQ8Batch, SpQ8Cache, SpRopeAxes,
               _ptr, _stream_ptr, check, lib)
from .cache import _wrap_device

_FORMATS = {"int8": SP_Q8_INT8, "e4m3": SP_Q8_E4M3}
_PAIRINGS = {"adjacent": SP_ROPE_ADJACENT, "halves": SP_ROPE_HALVES}
_DTYPES: dict = {}


def _dtype(t) -> int:
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float32: SP_DTYPE_F32, torch.float16: SP_DTYPE_F16, torch.bfloat16: SP_DTYPE_BF16})
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{t.dtype}: float32, float16 and bfloat16 are possible")
    return code


def _rows(t, heads, head_dim: int, what: str, device: int = 0) -> int:
    """The token stride of t [n_tokens][heads][head_dim] (0: dense), whose rows lie
    together in memory of `device`."""
    sh = t.shape
    if len(sh) != 3 or sh[2] != head_dim or (heads is not None and sh[1] != heads):
        raise ValueError(f"{what}: shape {tuple(sh)}, not [tokens][{heads or 'heads'}][{head_dim}]")
    if t.get_device() == device:
        if t.is_contiguous():
            return 0
        s = t.stride()
        # tokens that share memory (an expanded tensor's, whose stride is 0) have less than the shape says
        if s[2] == 1 and (sh[1] == 1 or s[1] == head_dim) and s[0] >= sh[1] * head_dim:
            return s[0]
    raise ValueError(f"{what}: a token's heads must lie together in memory of device {device}, and tokens apart from one another")


def _output(t, stream):
    """An output like t, to be written on `stream` (None: the default stream).
    Its memory is that stream's, so that whoever had it before, there, is done
    with it, and goes back to it only after the current stream's work as well:
    the output may be dropped while either still runs."""
    import torch
    now = torch.cuda.current_stream(t.device)
    at = _stream_ptr(stream)
    if now.cuda_stream == at:
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)
    with torch.cuda.stream(torch.cuda.ExternalStream(at, t.device) if at else torch.cuda.default_stream(t.device)):
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    out.record_stream(now)
    return out


_ROTATION = None


def _rotation():
    """The rotation as a function with a gradient, which is the rotation back."""
    global _ROTATION
    if _ROTATION is None:
        import torch

        class Rotation(torch.autograd.Function):
            @staticmethod
            def forward(ctx, plan, pos, q, k, inverse, stream):
                ctx.plan, ctx.inverse = plan, inverse
                ctx.save_for_backward(pos)
                out = plan.apply(pos, q, k, inverse=inverse, stream=stream)
                ctx.mark_non_differentiable(*(t for t, need in zip(out, ctx.needs_input_grad[2:4]) if t is not None and not need))
                return out

            @staticmethod
            def backward(ctx, gq, gk):
                pos, = ctx.saved_tensors
                gq, gk = (g.contiguous() if g is not None and need else None
                          for g, need in zip((gq, gk), ctx.needs_input_grad[2:4]))
                gq, gk = ctx.plan.apply(pos, gq, gk, inverse=not ctx.inverse, stream=torch.cuda.current_stream(pos.device))
                return None, None, gq, gk, None, None
        _ROTATION = Rotation
    return _ROTATION


class RopeAxes:
    """A rotation plan: `sections` pairs for each axis (together rot_dim / 2)."""

    def __init__(self, head_dim: int, sections, rot_dim: int | None = None, pairing: str = "adjacent",
                 interleave: bool = False, axis_ladder: bool = False, theta: float = 10000.0, freq_factors=None):
        sections = [int(n) for n in sections]
        rot_dim = 2 * sum(sections) if rot_dim is None else rot_dim
        self.plan = SpRopeAxes()
        flags = (SP_ROPE_INTERLEAVED if interleave else 0) | (SP_ROPE_AXIS_LADDER if axis_ladder else 0)
        ff = None if freq_factors is None else (C.c_float * (rot_dim // 2))(*freq_factors)
        check(lib().sp_rope_axes_init(C.byref(self.plan), head_dim, rot_dim, _PAIRINGS[pairing], len(sections),
                                      (C.c_int * len(sections))(*sections), flags, theta, ff), "sp_rope_axes_init")
        self.head_dim, self.n_axes = head_dim, len(sections)
        import torch
        self._ref, self._call = C.byref(self.plan), lib().sp_cuda_rope_axes
        # a step's call is host time
        self._int32, self._device, self._grad_enabled = torch.int32, torch.cuda.current_device, torch.is_grad_enabled

    def apply(self, pos, q=None, k=None, q_out=None, k_out=None, inverse: bool = False, stream=None):
        """Rotates q and k ([tokens][heads][head_dim] CUDA tensors; either may be
        None) at positions pos (int32 [axes][tokens]).  The outputs are new
        tensors unless given; an output may be its input.  Returns both.  Where
        gradients are wanted they flow back through it, and outputs cannot be given."""
        if (q is not None and q.requires_grad or k is not None and k.requires_grad) and self._grad_enabled():
            if q_out is not None or k_out is not None:
                raise RuntimeError("a rotation into a given output has no gradient: leave the output out, or use torch.no_grad()")
            return _rotation().apply(self, pos, q, k, inverse, stream)
        t = k if q is None else q
        n, dev = 0 if t is None else t.shape[0], pos.get_device()
        if pos.dtype is not self._int32 or pos.shape != (self.n_axes, n) or dev < 0 or not pos.is_contiguous():
            raise ValueError(f"pos must be a contiguous int32 CUDA tensor [{self.n_axes}][{n}]")
        if dev != self._device():
            raise ValueError(f"pos is on device {dev}, the current device is {self._device()}")
        hd = self.head_dim
        qp = qs = hq = qo = qos = kp = ks = hk = ko = kos = 0
        if q is not None:
            if q_out is None:
                q_out = _output(q, stream)
            qs, hq = _rows(q, None, hd, "q", dev), q.shape[1]
            qos = _rows(q_out, hq, hd, "q_out", dev)
            qp, qo = q.data_ptr(), q_out.data_ptr()
            if q_out.dtype is not q.dtype or q_out.shape[0] != n:
                raise ValueError("q and its output must have one type and number of tokens")
        if k is not None:
            if k_out is None:
                k_out = _output(k, stream)
            ks, (nk, hk, _) = _rows(k, None, hd, "k", dev), k.shape
            kos = _rows(k_out, hk, hd, "k_out", dev)
            kp, ko = k.data_ptr(), k_out.data_ptr()
            if k_out.dtype is not k.dtype or k_out.shape[0] != n or nk != n or k.dtype is not t.dtype:
                raise ValueError("q, k and their outputs must have one type and number of tokens")
        rc = self._call(self._ref, pos.data_ptr(), n, qp, qs, hq, qo, qos, kp, ks, hk, ko, kos,
                        0 if t is None else _dtype(t), 1 if inverse else 0, 0 if stream is None else stream.cuda_stream)
        if rc:
            check(rc, "sp_cuda_rope_axes")
        return q_out, k_out


class Q8Batch:
    """The new tokens of one step: cu [n + 1] and kv_len [n] (and seq [n], where
    the entries are not sequences 0, 1, ...), int32 CUDA tensors; n_tokens packed
    tokens, at most max_new of one entry, at most max_kv positions held."""

    def __init__(self, cu, kv_len, n_tokens: int, max_new: int, max_kv: int, seq=None):
        import torch
        n = kv_len.shape[0]
        for name, t, size in (("cu", cu, n + 1), ("kv_len", kv_len, n), ("seq", seq, n)):
            if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (size,) or not t.is_contiguous()
                                  or not t.is_cuda):
                raise ValueError(f"{name} must be a contiguous int32 CUDA tensor [{size}]")
            if t is not None and t.get_device() != cu.get_device():
                raise ValueError(f"{name} is on device {t.get_device()}, cu on {cu.get_device()}")
        self._keep, self.device = (cu, kv_len, seq), cu.get_device()
        self.n_tokens = n_tokens
        self.b = SpQ8Batch(n, n_tokens, max_new, max_kv, _ptr(seq), cu.data_ptr(), kv_len.data_ptr())
        self.ref = C.byref(self.b)


class Q8Cache:
    """A cache held in 8 bits (sp_cuda_q8_cache_t) on the current device.  Writes
    and reads are ordered on `stream`, attention on the stream it is given."""

    def __init__(self, head_dim: int, n_layers: int, n_heads_kv: int, max_seq_len: int, n_seqs: int = 1,
                 fmt: str = "int8", block_tokens: int = 64, stream=None):
        self.qc = SpQ8Cache()
        self.stream, self.fmt = stream, fmt
        cfg = SpConfig(head_dim=head_dim, n_layers=n_layers, n_heads_kv=n_heads_kv)
        check(lib().sp_cuda_q8_cache_init(C.byref(self.qc), C.byref(cfg), _FORMATS[fmt], block_tokens, n_seqs,
                                          max_seq_len, _stream_ptr(stream)), "sp_cuda_q8_cache_init")
        self.head_dim, self.n_layers, self.n_heads_kv, self.n_seqs = head_dim, n_layers, n_heads_kv, n_seqs
        self.block_tokens, self.max_seq_len, self.device = block_tokens, self.qc.max_seq_len, self.qc.device
        self._ref = C.byref(self.qc)
        self._write, self._read, self._attn = (lib().sp_cuda_q8_write_kv_tokens, lib().sp_cuda_q8_read_kv_tokens,
                                               lib().sp_cuda_q8_attn)

    def free(self) -> None:
        if self.qc.d_k_cache:
            lib().sp_cuda_q8_cache_free(C.byref(self.qc))

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def slab(self, which: int):
        """The K (0) or V (1) codes [layers][seqs][heads][max_seq_len][head_dim]
        (int8 or float8_e4m3fn; shares memory with the cache and keeps it)."""
        import torch
        shape = (self.n_layers, self.n_seqs, self.n_heads_kv, self.max_seq_len, self.head_dim)
        n = self.qc.n_slots * self.max_seq_len * self.head_dim
        t = torch.int8 if self.fmt == "int8" else torch.float8_e4m3fn
        return _wrap_device(self.qc.d_v_cache if which else self.qc.d_k_cache, n, t, self).view(shape)

    def scales(self, which: int):
        """The scales [layers][seqs][heads][blocks] (shares memory with the cache and keeps it)."""
        import torch
        shape = (self.n_layers, self.n_seqs, self.n_heads_kv, self.max_seq_len // self.block_tokens)
        n = self.qc.n_slots * shape[-1] * 4
        return _wrap_device(self.qc.d_v_scale if which else self.qc.d_k_scale, n, torch.float32, self).view(shape)

    def write_kv_tokens(self, layer: int, batch: Q8Batch, k, v) -> None:
        """k, v: [n_tokens][n_heads_kv][head_dim] (f32/f16/bf16, one token stride;
        either may be None)."""
        t = v if k is None else k
        if t is None:
            return
        stride = _rows(t, self.n_heads_kv, self.head_dim, "k", self.device)
        if k is not None and v is not None and (v.dtype is not k.dtype or v.shape[0] != k.shape[0]
                                                or _rows(v, self.n_heads_kv, self.head_dim, "v", self.device) != stride):
            raise ValueError("k and v must have one type, token stride and number of tokens")
        if t.shape[0] != batch.n_tokens:
            raise ValueError(f"{t.shape[0]} tokens, the batch has {batch.n_tokens}")
        if batch.device != self.device:
            raise ValueError(f"the batch is on device {batch.device}, the cache on {self.device}")
        rc = self._write(self._ref, layer, batch.ref, 0 if k is None else k.data_ptr(), 0 if v is None else v.data_ptr(),
                         stride, _dtype(t))
        if rc:
            check(rc, "sp_cuda_q8_write_kv_tokens")

    def read_kv_tokens(self, which: int, layer: int, seq: int, start_pos: int, out) -> None:
        """out: [n_tok][n_heads_kv][head_dim], contiguous (f32/f16/bf16)."""
        if _rows(out, self.n_heads_kv, self.head_dim, "out", self.device) != 0:
            raise ValueError(f"out must be contiguous [tokens][{self.n_heads_kv}][{self.head_dim}]")
        rc = self._read(self._ref, which, layer, seq, start_pos, out.shape[0], out.data_ptr(), _dtype(out))
        if rc:
            check(rc, "sp_cuda_q8_read_kv_tokens")

    def attn(self, layer: int, batch: Q8Batch, q, out=None, lse=None, logit_scale: float = 1.0, causal: bool = True,
             window: int = 0, stream=None):
        """q: [n_tokens][n_q_heads][head_dim] fp16 or bf16; out the same (new unless
        given); lse: fp32 [n_tokens][n_q_heads] or None.  Returns out, which has
        no gradient."""
        n, hq, hd = *q.shape[:2], self.head_dim
        if out is None:
            out = _output(q, stream)
        qs, os = _rows(q, None, hd, "q", self.device), _rows(out, hq, hd, "out", self.device)
        if n != batch.n_tokens or out.shape[0] != n or out.dtype is not q.dtype:
            raise ValueError(f"q and out must have one type and the batch's {batch.n_tokens} tokens")
        if batch.device != self.device:
            raise ValueError(f"the batch is on device {batch.device}, the cache on {self.device}")
        lp = 0
        if lse is not None:
            if lse.shape != (n, hq) or lse.element_size() != 4 or not (lse.is_floating_point() and lse.is_contiguous()
                                                                       and lse.get_device() == self.device):
                raise ValueError(f"lse must be a contiguous float32 tensor [{n}][{hq}] on device {self.device}")
            lp = lse.data_ptr()
        rc = self._attn(self._ref, layer, batch.ref, q.data_ptr(), qs, hq, _dtype(q), logit_scale, 1 if causal else 0, window,
                        out.data_ptr(), os, lp, 0 if stream is None else stream.cuda_stream)
        if rc:
            check(rc, "sp_cuda_q8_attn")
        return out

    def status(self, clear: bool = False, stream=None) -> int:
        """The device error word after the stream's work (synchronises)."""
        v = C.c_uint(0)
        check(lib().sp_cuda_q8_status(self._ref, C.byref(v), int(clear), _stream_ptr(stream)), "sp_cuda_q8_status")
        return v.value
