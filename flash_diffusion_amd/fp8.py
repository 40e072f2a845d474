"""Layers over the 8-bit products and the embedding lookup (csrc/fp8.hip, csrc/embed.hip): ``Fp8Linear``, a frozen linear map whose input
gradient flows, ``TokenEmbedding``, ``nn.Embedding``'s lookup and sparse-by-nature gradient on the HIP path, and ``PackedFp8``, the
cache through which a module keeps the 8-bit form of a parameter (the frozen text encoder of ``t5.py`` with precision="fp8").

A token table trains in front of a chain of frozen ``Fp8Linear`` layers: its gradient is the products' input gradient summed by token.  (The
text encoders themselves run without gradients.)  The weights are frozen: there is no weight gradient.  GPU only; there is no CPU
fallback."""
from __future__ import annotations

import threading

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable
from torch.multiprocessing.reductions import StorageWeakRef

from . import ops

BF16, F32 = torch.bfloat16, torch.float32


class PackedFp8:
    """The 8-bit form of ONE parameter, packed on first use and again when the parameter has changed (replaced, moved, or written in place:
    torch counts those, but for writes through .data).  It is packed again into the same memory where shape and device allow, so a
    captured graph that reads it sees the new weight.  The parameter itself is held, and its memory by a weak reference, so another one at
    the same address is not taken for it.  Packing has ended when the call returns (once per weight, the host waits for it): other
    streams and the replays of captured graphs may read the codes at once.  A capture cannot pack (run the layer once before).  Threads may share it."""

    def __init__(self, transposed=False):
        self.transposed, self._lock = transposed, threading.Lock()
        self._of = self._storage = self._key = self._packed = None

    def __deepcopy__(self, memo):
        return PackedFp8(self.transposed)          # (the copy's parameter is another one)

    def __reduce__(self):
        return PackedFp8, (self.transposed,)

    def __call__(self, w):
        with self._lock:
            return self._of_now(w)

    def _of_now(self, w):
        storage = w.untyped_storage()
        key = (w._version, storage._cdata, w.data_ptr(), w.device, w.dtype, w.shape, w.stride())
        if self._of is not w or self._key != key:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the weight has to be packed before a graph is captured: run the layer once")
            old, into = self._packed, None
            if old is not None:
                torch.cuda.synchronize(old.codes.device)   # (a stream may still read the codes that are overwritten or dropped here)
                into = old if (old.N, old.K, old.codes.device) == (*w.shape, w.device) else None
            packed = ops.pack_weight_fp8(w.detach().contiguous(), self.transposed, into)
            torch.cuda.current_stream().synchronize()
            # (while the weak reference is held, no other storage can have this one's _cdata)
            self._packed, self._key, self._of, self._storage = packed, key, w, StorageWeakRef(storage)
        return self._packed


def _rows_of(t):
    """[..., K] as the [M, K] that the products take: rows that are contiguous and do not overlap (a transposed, a broadcast tensor is copied)"""
    t = t.reshape(-1, t.shape[-1])
    apart = t.shape[0] <= 1 or t.stride(0) >= t.shape[1]
    return t if apart and (t.shape[1] <= 1 or t.stride(1) == 1) else t.contiguous()


def _versions(packed):
    """what a write to the weight's transposed codes changes (tensors made in inference mode count no writes)"""
    return [t._version for t in (packed.codes_t, packed.scales_t) if not t.is_inference()]


class _Fp8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, packed, bias, out_f32):
        ctx.packed, ctx.versions, ctx.shape, ctx.dtype = packed, _versions(packed), x.shape, x.dtype
        y = ops.gemm_fp8(_rows_of(x), packed, bias=bias, out_f32=out_f32)
        return y.view(*x.shape[:-1], packed.N)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if _versions(ctx.packed) != ctx.versions:
            raise RuntimeError("the weight of this Fp8Linear has been modified by an inplace operation since the forward")
        dx = ops.gemm_fp8_dgrad(_rows_of(dy), ctx.packed, out_f32=ctx.dtype == F32)
        return dx.view(ctx.shape), None, None, None


class Fp8Linear(nn.Module):
    """``nn.Linear`` with a frozen weight held in 8 bits (ops.pack_weight_fp8) and a frozen fp32 bias: y = x W^T + b for bf16 / fp32 inputs of
    any leading shape, in the input's dtype.  The gradient flows to the input; its dY is quantised like an activation."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor = None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        packed = ops.pack_weight_fp8(weight.detach(), transposed=True)
        for name in self._PARTS:
            self.register_buffer(name, getattr(packed, name))
        self.register_buffer("bias", None if bias is None else bias.detach().to(weight.device, F32).contiguous())

    _PARTS = ("codes", "scales", "codes_t", "scales_t")

    @classmethod
    def from_linear(cls, linear: nn.Linear):
        return cls(linear.weight, linear.bias)

    def packed(self):
        """the weight as the ops take it (the buffers move and are saved with the module)"""
        w = ops.Fp8Weight.__new__(ops.Fp8Weight)
        w.N, w.K = self.out_features, self.in_features
        for name in self._PARTS:
            setattr(w, name, getattr(self, name))
        return w

    def forward(self, x):
        return _Fp8LinearFn.apply(x, self.packed(), None if self.bias is None else self.bias.float(), x.dtype == F32)


class _LookupFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, pos, ids, scale, dtype):
        ctx.save_for_backward(ids)
        ctx.V, ctx.scale, ctx.wdtype = weight.shape[0], scale, weight.dtype
        ctx.pos_rows = None if pos is None else pos.shape[0]
        return ops.embed_fwd(weight, ids, scale=scale, pos=pos, dtype=dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        dy = dy.contiguous()
        dw = dp = None
        if ctx.needs_input_grad[0]:
            dw = ops.embed_bwd(dy, ids, ctx.V, scale=ctx.scale).to(ctx.wdtype)
        if ctx.needs_input_grad[1]:                # the position rows are a lookup too, by the last index of ids
            t = torch.arange(ids.shape[-1] if ids.dim() else 1, dtype=torch.int32, device=ids.device)
            t = t.expand(ids.shape).contiguous() if ids.dim() else t.view(())
            dp = ops.embed_bwd(dy, t, ctx.pos_rows)
        return dw, dp, None, None, None


class TokenEmbedding(nn.Embedding):
    """``nn.Embedding`` (same parameter, same state_dict) whose lookup is ops.embed_fwd -- scale * weight[ids] + pos[t] in one pass, rounded
    once to `dtype` -- and whose gradient is ops.embed_bwd's (fixed order of sums).  The options of nn.Embedding that change either
    (padding_idx, max_norm, scale_grad_by_freq, sparse) are refused.  An id outside the table gives a row of NaN."""

    def __init__(self, num_embeddings, embedding_dim, **kw):
        super().__init__(num_embeddings, embedding_dim, **kw)
        if self.padding_idx is not None or self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise NotImplementedError("TokenEmbedding: padding_idx, max_norm, scale_grad_by_freq and sparse are not implemented")

    def forward(self, ids, scale=1.0, pos=None, dtype=BF16):
        return _LookupFn.apply(self.weight, pos, ids, float(scale), dtype)
