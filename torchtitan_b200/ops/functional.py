"""Differentiable operators used by the models.

Every operator has one CUDA implementation (the in-tree sm_100a extension,
``torch.ops.tb200``) and one plain-PyTorch implementation used for CPU tensors.
If the extension is missing, a call with CUDA tensors raises.  Two library paths remain for
CUDA tensors and are counted in ``settings.library_fallbacks``: a bf16 GEMM whose inner
dimensions are not multiples of 8 elements (a TMA row must be a multiple of 16 bytes) runs on
``torch.mm``, as does any GEMM when ``kernels.gemm = "cublas"`` selects the library arm; and
attention shapes outside the flash kernel's instantiations run the blocked PyTorch fallback of
:func:`attention`.

Memory policy.  The fused functions below are where op-level selective
recomputation lives: ``norm_linear`` keeps only the un-normalised input and the
per-row ``rstd`` and recomputes the normalised activations for the weight
gradient; ``swiglu_linear`` keeps the gate/up GEMM output and recomputes the
activation.  GEMM and attention outputs are kept.  (The reference expresses the
same intent as a per-op save list, torchtitan/distributed/activation_checkpoint.py:31-94.)

Weight gradients.  When a weight carries a ``main_grad`` attribute (set by the
sharded-data-parallel engine, a view into the unit's flat gradient buffer) the
linear backward writes the weight gradient straight into it and reports no
gradient to autograd, which removes the extra zero-fill and accumulate passes
over the gradient buffer.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import ext, reference as ref

__all__ = [
    "settings", "rms_norm", "linear", "norm_linear", "swiglu", "swiglu_linear", "rope_qk_", "rope", "qk_norm_rope",
    "attention", "attention_packed", "linear_cross_entropy", "cross_entropy_sum", "gemm_nt", "gemm_nn", "gemm_tn", "embedding",
]


@dataclass
class _Settings:
    gemm: str = "tcgen05"  # "cublas" | "tcgen05"
    attention: str = "native"  # "sdpa" | "native"
    qk_norm_rope: str = "separate"  # "separate" | "fused": per-head norms and RoPE as kernels of their own, or in one pass
    recompute: bool = True  # fused functions recompute norm / SwiGLU activations in backward
    launches: int = 0  # count of launches of this package's own kernels
    count_launches: bool = False
    library_fallbacks: int = 0  # CUDA calls that went to a library / PyTorch path (see the module docstring)
    strict_native: bool = False  # batch-invariant mode: a CUDA call that would take a library path raises instead
    sac: object | None = None  # the SacSession of the checkpointed block whose forward (or recompute) is running


settings = _Settings()


class SacSession:
    """Per-op selective checkpointing inside a block that is otherwise recomputed in backward: the outputs of the
    ops the policy selects (attention, every second GEMM, ...) are kept from the first forward and handed back,
    in call order, when the block's forward runs again for the backward pass; everything else is recomputed.

    ``policy(kind, shape, session) -> bool`` decides at the first forward whether the output of the op is kept
    (``kind``: "mm" with ``shape = (in_features, out_features)``, or "attention").  Parity with the save-list
    policy of torchtitan/distributed/activation_checkpoint.py:186-287, acting on this package's own ops."""

    def __init__(self, policy):
        self.policy = policy
        self.store: dict[int, object] = {}
        self.kinds: dict[int, str] = {}
        self.replaying = False
        self.index = 0
        self.mm_count = 0
        self.saved = 0
        self.recomputed = 0

    def begin(self, replaying: bool) -> None:
        self.replaying = replaying
        self.index = 0

    @staticmethod
    def _tensors(out):
        return [t for t in (out if isinstance(out, (tuple, list)) else (out,)) if isinstance(t, torch.Tensor)]

    def run(self, kind: str, shape, compute):
        i = self.index
        self.index += 1
        if self.replaying:
            kept = self.store.pop(i, None)
            if kept is not None:
                out, versions = kept
                # an output that was written in place after it was kept no longer holds the op's result
                if [t._version for t in self._tensors(out)] == versions:
                    return out
            self.recomputed += 1
            return compute()
        out = compute()
        if self.policy(kind, shape, self):
            self.store[i] = (out, [t._version for t in self._tensors(out)])
            self.kinds[i] = kind
            self.saved += 1
        return out

    def written_in_place(self, t: torch.Tensor) -> None:
        """An op is about to overwrite ``t``: a kept output that shares its memory is given up (it will be
        recomputed), and a GEMM that is given up hands its place in the every-second count to the next one."""
        if self.replaying:
            return
        ptr = t.untyped_storage().data_ptr()
        for i in [i for i, (out, _) in self.store.items()
                  if any(x.untyped_storage().data_ptr() == ptr for x in self._tensors(out))]:
            del self.store[i]
            self.saved -= 1
            if self.kinds.pop(i, None) == "mm":
                self.mm_count -= 1


def _sac_run(kind: str, shape, compute):
    s = settings.sac
    return compute() if s is None else s.run(kind, shape, compute)


def _fwd_gemm_nt(a: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """The forward GEMM of a linear layer (``a @ w^T``), subject to the running per-op checkpoint session."""
    if settings.sac is None:
        return gemm_nt(a, w)
    return settings.sac.run("mm", (w.shape[1], w.shape[0]), lambda: gemm_nt(a, w))


def _count(n: int = 1) -> None:
    if settings.count_launches:
        settings.launches += n


def _library_fallback(what: str) -> None:
    """Book-keeping for a CUDA call that leaves the hand-written kernels."""
    settings.library_fallbacks += 1
    if settings.strict_native:
        raise RuntimeError(f"{what} would run on a library / PyTorch path, which is not batch-invariant "
                           "(debug.batch_invariant is on)")


def _cuda(t: torch.Tensor) -> bool:
    return t.is_cuda


# =====================================================================
# GEMM front-ends (bf16 in, fp32 accumulate)
# =====================================================================
def _tc_ok(*ts: torch.Tensor) -> bool:
    return (
        settings.gemm == "tcgen05"
        and all(t.is_cuda and t.dtype == torch.bfloat16 for t in ts)
    )


def gemm_nt(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """``a[M,K] @ b[N,K]^T``; with ``accumulate`` adds into ``out``."""
    if _tc_ok(a, b) and ext.available() and hasattr(torch.ops.tb200, "gemm_bf16"):
        r = _tc_gemm(a, b, 0, out, accumulate)
        if r is not None:
            return r
    if out is None:
        return torch.mm(a, b.t())
    if accumulate:
        return out.addmm_(a, b.t())
    return torch.mm(a, b.t(), out=out)


def gemm_nn(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """``a[M,K] @ b[K,N]``."""
    if _tc_ok(a, b) and ext.available() and hasattr(torch.ops.tb200, "gemm_bf16"):
        r = _tc_gemm(a, b, 1, out, accumulate)
        if r is not None:
            return r
    if out is None:
        return torch.mm(a, b)
    if accumulate:
        return out.addmm_(a, b)
    return torch.mm(a, b, out=out)


def gemm_tn(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """``a[K,M]^T @ b[K,N]`` (weight-gradient shape)."""
    if _tc_ok(a, b) and ext.available() and hasattr(torch.ops.tb200, "gemm_bf16"):
        r = _tc_gemm(a, b, 2, out, accumulate)
        if r is not None:
            return r
    if out is None:
        return torch.mm(a.t(), b)
    if accumulate:
        return out.addmm_(a.t(), b)
    return torch.mm(a.t(), b, out=out)


def _tc_gemm(a, b, mode, out, accumulate):
    """Hand-written tcgen05 GEMM; returns None (library path, counted) when a row is not a multiple of 16 bytes."""
    a, b = a.contiguous(), b.contiguous()
    if mode == 0:
        M, K = a.shape
        N = b.shape[0]
    elif mode == 1:
        M, K = a.shape
        N = b.shape[1]
    else:
        K, M = a.shape
        N = b.shape[1]
    if (N % 8) or K == 0 or ((M % 8) if mode == 2 else (K % 8)):
        _library_fallback(f"a bf16 GEMM with M={M} N={N} K={K}")
        return None
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=a.device)
        accumulate = False
    elif not (out.is_contiguous() and out.dtype == torch.bfloat16):
        _library_fallback("a bf16 GEMM into a strided or non-bf16 output")
        return None
    torch.ops.tb200.gemm_bf16(a, b, out, mode, accumulate)
    _count()
    return out


# =====================================================================
# RMSNorm
# =====================================================================
def _rms_fwd(x2, w, eps):
    if _cuda(x2):
        _count()
        return ext.require().rmsnorm_fwd(x2, w, eps)
    return ref.rms_norm_fwd(x2, w, eps)


def _rms_bwd(dy2, x2, w, rstd):
    if _cuda(x2):
        _count(2 if w is not None else 1)
        dx, dw = ext.require().rmsnorm_bwd(dy2, x2, w, rstd)
        return dx, (dw if w is not None else None)
    return ref.rms_norm_bwd(dy2, x2, w, rstd)


def _deliver_wgrad(weight: torch.Tensor, dw: torch.Tensor | None):
    """Route a weight gradient to ``main_grad`` when present; else return it for autograd."""
    if dw is None:
        return None
    mg = getattr(weight, "main_grad", None)
    if mg is None:
        return dw.to(weight.dtype) if dw.dtype != weight.dtype else dw
    dwv = dw.view_as(mg)
    if getattr(weight, "_main_grad_written", False):
        mg.add_(dwv)
    else:
        mg.copy_(dwv)
        weight._main_grad_written = True
    return None


class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        x2 = x.reshape(-1, x.shape[-1])
        if not x2.is_contiguous():
            x2 = x2.contiguous()
        y, rstd = _rms_fwd(x2, weight, eps)
        ctx.save_for_backward(x2, weight, rstd)
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, weight, rstd = ctx.saved_tensors
        dy2 = dy.reshape(x2.shape)
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dx, dw = _rms_bwd(dy2, x2, weight, rstd)
        dwr = _deliver_wgrad(weight, dw) if weight is not None else None
        return dx.view(ctx.shape), dwr, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-5) -> torch.Tensor:
    return _RMSNormFn.apply(x, weight, eps)


# =====================================================================
# Linear (+ fused prologues)
# =====================================================================
def _wgrad(dy2: torch.Tensor, x2: torch.Tensor, weight: torch.Tensor):
    """dW[N,K] = dy2[M,N]^T @ x2[M,K], delivered to main_grad when available."""
    mg = getattr(weight, "main_grad", None)
    if mg is not None and mg.dtype == dy2.dtype:
        acc = getattr(weight, "_main_grad_written", False)
        gemm_tn(dy2, x2, out=mg.view(weight.shape), accumulate=acc)
        weight._main_grad_written = True
        return None
    dw = gemm_tn(dy2, x2)
    return _deliver_wgrad(weight, dw)


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        x2 = x.reshape(-1, x.shape[-1])
        y = _fwd_gemm_nt(x2, weight)
        if bias is not None:
            y = y + bias
        ctx.save_for_backward(x2, weight)
        ctx.has_bias = bias is not None
        ctx.xshape = x.shape
        return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x2, weight = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dx = gemm_nn(dy2, weight).view(ctx.xshape) if ctx.needs_input_grad[0] else None
        dw = _wgrad(dy2, x2, weight) if weight.requires_grad else None
        db = dy2.sum(dim=0) if ctx.has_bias else None
        return dx, dw, db


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    if x.dtype != weight.dtype:
        x = x.to(weight.dtype)
    return _LinearFn.apply(x, weight, bias)


class _NormLinearFn(torch.autograd.Function):
    """``rms_norm(x) @ W^T`` keeping only ``x`` and ``rstd`` for backward."""

    @staticmethod
    def forward(ctx, x, norm_w, weight, eps):
        x2 = x.reshape(-1, x.shape[-1])
        xn, rstd = _rms_fwd(x2, norm_w, eps)
        y = _fwd_gemm_nt(xn, weight)
        ctx.save_for_backward(x2, norm_w, weight, rstd)
        ctx.eps = eps
        ctx.xshape = x.shape
        return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x2, norm_w, weight, rstd = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        xn, _ = _rms_fwd(x2, norm_w, ctx.eps)
        dw = _wgrad(dy2, xn, weight) if weight.requires_grad else None
        del xn
        dxn = gemm_nn(dy2, weight)
        dx, dnw = _rms_bwd(dxn, x2, norm_w, rstd)
        dnw = _deliver_wgrad(norm_w, dnw) if norm_w is not None else None
        return dx.view(ctx.xshape), dnw, dw, None


def norm_linear(x: torch.Tensor, norm_weight: torch.Tensor | None, weight: torch.Tensor, eps: float) -> torch.Tensor:
    if not settings.recompute:
        return linear(rms_norm(x, norm_weight, eps), weight)
    return _NormLinearFn.apply(x, norm_weight, weight, eps)


# =====================================================================
# SwiGLU
# =====================================================================
def _swiglu_fwd(gu2: torch.Tensor) -> torch.Tensor:
    if _cuda(gu2):
        _count()
        return ext.require().swiglu_fwd(gu2)
    f = gu2.shape[-1] // 2
    return ref.swiglu_fwd(gu2[:, :f], gu2[:, f:])


def _swiglu_bwd(gu2: torch.Tensor, da: torch.Tensor) -> torch.Tensor:
    if _cuda(gu2):
        _count()
        return ext.require().swiglu_bwd(gu2, da)
    f = gu2.shape[-1] // 2
    dg, du = ref.swiglu_bwd(gu2[:, :f], gu2[:, f:], da)
    return torch.cat([dg, du], dim=-1)


class _SwiGLUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        gu2 = gu.reshape(-1, gu.shape[-1])
        ctx.save_for_backward(gu2)
        ctx.shape = gu.shape
        return _swiglu_fwd(gu2).view(*gu.shape[:-1], gu.shape[-1] // 2)

    @staticmethod
    def backward(ctx, da):
        (gu2,) = ctx.saved_tensors
        da2 = da.reshape(gu2.shape[0], -1)
        if not da2.is_contiguous():
            da2 = da2.contiguous()
        return _swiglu_bwd(gu2, da2).view(ctx.shape)


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` where ``gate_up[..., :F]`` is the gate and ``[..., F:]`` the up projection."""
    return _SwiGLUFn.apply(gate_up)


class _SwiGLULinearFn(torch.autograd.Function):
    """``swiglu(gu) @ W^T`` keeping only ``gu``; the activation is recomputed in backward."""

    @staticmethod
    def forward(ctx, gu, weight):
        gu2 = gu.reshape(-1, gu.shape[-1])
        a = _swiglu_fwd(gu2)
        y = _fwd_gemm_nt(a, weight)
        ctx.save_for_backward(gu2, weight)
        ctx.shape = gu.shape
        return y if gu.dim() == 2 else y.view(*gu.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        gu2, weight = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        a = _swiglu_fwd(gu2)
        dw = _wgrad(dy2, a, weight) if weight.requires_grad else None
        del a
        da = gemm_nn(dy2, weight)
        dgu = _swiglu_bwd(gu2, da)
        return dgu.view(ctx.shape), dw


def swiglu_linear(gate_up: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    if not settings.recompute:
        return linear(swiglu(gate_up), weight)
    return _SwiGLULinearFn.apply(gate_up, weight)


# =====================================================================
# RoPE
# =====================================================================
def _rope_inplace(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool, inverse: bool):
    """Rotate ``x[T, H, D]`` (last dim contiguous, arbitrary row stride) in place."""
    if _cuda(x):
        _count()
        ext.require().rope_(x, table, positions, interleaved, inverse)
        return x
    x.copy_(ref.rope_apply(x, table, positions, interleaved, inverse))
    return x


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, positions, interleaved):
        ctx.save_for_backward(table, positions)
        ctx.interleaved = interleaved
        out = x.clone() if x.is_contiguous() else x.contiguous()
        return _rope_inplace(out, table, positions, interleaved, False)

    @staticmethod
    def backward(ctx, dy):
        table, positions = ctx.saved_tensors
        d = dy.clone() if dy.is_contiguous() else dy.contiguous()
        return _rope_inplace(d, table, positions, ctx.interleaved, True), None, None, None


def rope(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """Out-of-place RoPE on ``x[T, H, D]``."""
    return _RopeFn.apply(x, table, positions, interleaved)


class _RopeQKInplaceFn(torch.autograd.Function):
    """Rotate the first ``n_rot_heads`` heads of a packed ``[T, H_total * D]`` tensor in place."""

    @staticmethod
    def forward(ctx, qkv, table, positions, interleaved, n_rot_heads, head_dim):
        ctx.save_for_backward(table, positions)
        ctx.interleaved = interleaved
        ctx.n_rot, ctx.hd = n_rot_heads, head_dim
        ctx.mark_dirty(qkv)
        if settings.sac is not None:
            settings.sac.written_in_place(qkv)
        v = qkv.view(qkv.shape[0], -1, head_dim)
        _rope_inplace(v[:, :n_rot_heads], table, positions, interleaved, False)
        return qkv

    @staticmethod
    def backward(ctx, d):
        table, positions = ctx.saved_tensors
        d = d.contiguous() if not d.is_contiguous() else d.clone()
        v = d.view(d.shape[0], -1, ctx.hd)
        _rope_inplace(v[:, : ctx.n_rot], table, positions, ctx.interleaved, True)
        return d, None, None, None, None, None


def rope_qk_(qkv: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool, n_rot_heads: int,
             head_dim: int):
    """In-place RoPE on the q and k heads of a packed projection output ``[T, (Hq+2Hkv)*D]``."""
    return _RopeQKInplaceFn.apply(qkv, table, positions, interleaved, n_rot_heads, head_dim)


# =====================================================================
# Per-head norms of queries and keys + RoPE
# =====================================================================
class _QKNormRopeFn(torch.autograd.Function):
    """Keeps the projection output only: the backward reads it in any case and recomputes each head's rsqrt.  Runs on the
    CPU, where the weights' gradients go to ``main_grad``, and where launches are counted; else a node in C++ does the same."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, table, positions, axes, meta):
        q, k = _qk_norm_rope_fwd(qkv, q_weight, k_weight, table, positions, axes, meta)
        ctx.save_for_backward(qkv, q_weight, k_weight, table, positions, axes)
        ctx.meta = meta
        return q, k, qkv[:, meta[0] + meta[1]:]

    @staticmethod
    def backward(ctx, dq, dk, dv):
        x, q_weight, k_weight, table, positions, axes = ctx.saved_tensors
        args = (x, ctx.meta[0], ctx.meta[1], q_weight, k_weight, table, positions, axes, *ctx.meta[2:])
        if _cuda(x):
            weights = [w for w in (q_weight, k_weight) if w is not None]
            _count(2 if weights else 1)
            # the gradient is rounded once, to the type that receives it
            fp32 = any(w.main_grad.dtype == torch.float32 for w in weights if getattr(w, "main_grad", None) is not None)
            dx, dw = ext.require().qk_norm_rope_bwd(dq, dk, dv, *args, fp32)
        else:
            dx, dw = ref.qk_norm_rope_bwd(dq, dk, dv, *args)
        if q_weight is None and k_weight is None:
            return dx, None, None, None, None, None, None
        need = ctx.needs_input_grad
        dqw, dkw = dw.unbind(0)
        return (dx, _deliver_wgrad(q_weight, dqw) if need[1] else None, _deliver_wgrad(k_weight, dkw) if need[2] else None,
                None, None, None, None)


def _qk_norm_rope_fwd(qkv, q_weight, k_weight, table, positions, axes, meta):
    hq, hkv, *rest = meta
    if not _cuda(qkv):
        return ref.qk_norm_rope_fwd(qkv, hq, hkv, q_weight, k_weight, table, positions, axes, *rest)
    _count()
    return ext.require().qk_norm_rope_fwd(qkv, hq, hkv, q_weight, k_weight, table, positions, axes, *rest)


def qk_norm_rope(qkv: torch.Tensor, n_heads: int, n_kv_heads: int, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 table: torch.Tensor | None, positions: torch.Tensor | None, interleaved: bool, *, eps: float = 1e-6,
                 gain_center: float = 0.0, q_scale: float = 1.0, axes: torch.Tensor | None = None):
    """RMSNorm of every query and key head and the rotary embedding in one pass over a packed projection output.

    ``qkv [T, Hq + 2 Hkv, D]`` -> ``(q [T, Hq, D], k [T, Hkv, D], v)`` with ``v`` a view of ``qkv``: each head vector is
    scaled by its ``rsqrt(mean(x^2) + eps)`` and by ``weight + gain_center`` (nothing when the weight is None), queries
    also by ``q_scale``, and its first ``table.shape[1]`` elements are rotated (``table = None``: no rotation).
    ``positions [T]`` int64 index the fp32 ``table`` (``cos | sin``); with several position axes ``positions`` is
    ``[axes, T]`` and ``axes [rot / 2]`` (int32) names the axis that each frequency follows.  The result is rounded
    once.  bf16 or fp32, head dimensions up to 256 in multiples of 8, rotary widths in multiples of 16 (8 when
    ``interleaved``)."""
    if qkv.dim() != 3 or qkv.shape[1] != n_heads + 2 * n_kv_heads:
        raise ValueError(f"qk_norm_rope: expected [T, {n_heads} + 2 * {n_kv_heads}, D], got {tuple(qkv.shape)}")
    if table is not None:
        if positions is None:
            raise ValueError("qk_norm_rope: a rotation needs positions")
        want = (qkv.shape[0],) if axes is None else (positions.shape[0], qkv.shape[0])
        if tuple(positions.shape) != want:
            raise ValueError(f"qk_norm_rope: positions {tuple(positions.shape)} do not fit {qkv.shape[0]} tokens"
                             + ("" if axes is None else " on several axes"))
        if table.shape[1] > qkv.shape[2] or table.shape[1] % (8 if interleaved else 16):
            raise ValueError(f"qk_norm_rope: rotary width {table.shape[1]} for head dimension {qkv.shape[2]}")
        positions = positions.long().contiguous()
    else:
        positions = axes = None
    meta = (int(n_heads), int(n_kv_heads), bool(interleaved), float(eps), float(gain_center), float(q_scale))
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (qkv, q_weight, k_weight))):
        q, k = _qk_norm_rope_fwd(qkv, q_weight, k_weight, table, positions, axes, meta)
        return q, k, qkv[:, n_heads + n_kv_heads:]
    if _cuda(qkv) and not settings.count_launches and all(getattr(w, "main_grad", None) is None for w in (q_weight, k_weight)):
        return ext.require().qk_norm_rope(qkv, n_heads, n_kv_heads, q_weight, k_weight, table, positions, axes, *meta[2:])
    return _QKNormRopeFn.apply(qkv, q_weight, k_weight, table, positions, axes, meta)


# =====================================================================
# Attention
# =====================================================================
def _sdpa_causal(q, k, v, scale):
    """Library attention (cuDNN / flash) on ``[T,H,D]`` tensors: the baseline path."""
    qh, kh, vh = (t.transpose(0, 1).unsqueeze(0) for t in (q, k, v))
    gqa = q.shape[1] != k.shape[1]
    if q.is_cuda:
        from torch.nn.attention import SDPBackend, sdpa_kernel

        order = [SDPBackend.CUDNN_ATTENTION, SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION, SDPBackend.MATH]
        with sdpa_kernel(order, set_priority=True):
            out = F.scaled_dot_product_attention(qh, kh, vh, is_causal=True, scale=scale, enable_gqa=gqa)
    else:
        out = F.scaled_dot_product_attention(qh, kh, vh, is_causal=True, scale=scale, enable_gqa=gqa)
    return out.squeeze(0).transpose(0, 1)


def _native_attention_ok(q, k, v) -> bool:
    if not (_cuda(q) and settings.attention == "native"):
        return False
    from . import flash

    return flash.supported(q, k, v)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, causal: bool = True,
              doc_ids: torch.Tensor | None = None, window: int | None = None, sinks: torch.Tensor | None = None,
              q_pos: torch.Tensor | None = None, k_pos: torch.Tensor | None = None,
              kv_first: torch.Tensor | None = None) -> torch.Tensor:
    """Attention over folded tokens: ``q[T,Hq,D]``, ``k/v[T,Hkv,D]`` -> ``[T,Hq,Dv]``.

    Documents are separated with ``doc_ids`` (``None`` = one document); ``kv_first`` is the same
    information as the index of the first token of each query's document, the form the
    tcgen05 kernel consumes.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    simple = window is None and sinks is None and q_pos is None and k_pos is None and causal
    if (causal and q_pos is None and k_pos is None and (doc_ids is None or kv_first is not None)
            and _native_attention_ok(q, k, v)):
        from .flash import flash_attention

        _count(4)  # forward + (delta, backward, dq cast)
        return flash_attention(q, k, v, scale, causal=True, kv_first=kv_first, window=window, sinks=sinks)
    D = q.shape[-1]
    if (settings.attention == "native" and _cuda(q) and causal and q_pos is None and k_pos is None
            and (doc_ids is None or kv_first is not None) and D < 128 and v.shape[-1] == D
            and q.dtype == torch.bfloat16 and q.shape[1] % k.shape[1] == 0):
        # Smaller head dimensions run on the 128-wide kernels with zero-padded heads: the padded columns add
        # nothing to q . k and produce zero output columns, which are cut off again (twice the attention FLOPs of a
        # dedicated instantiation, still tensor-core attention without a T x T intermediate).
        from .flash import flash_attention

        pad = (0, 128 - D)
        _count(4)
        o = flash_attention(F.pad(q, pad), F.pad(k, pad), F.pad(v, pad), scale, causal=True, kv_first=kv_first,
                            window=window, sinks=sinks)
        return o[..., :D]
    if _cuda(q):
        _library_fallback(f"attention with head dimension {q.shape[-1]}")
    if simple and doc_ids is None and q.shape[-1] == v.shape[-1]:
        return _sdpa_causal(q, k, v, scale)
    return _masked_attention(q, k, v, scale, causal, doc_ids, window, sinks, q_pos, k_pos)


class _PackedFlashFn(torch.autograd.Function):
    """Causal attention on a packed projection output ``[T, Hq + 2 Hkv, 128]``; the gradient
    comes back as one packed tensor, written in place by the backward kernel."""

    @staticmethod
    def forward(ctx, qkv3, hq, hkv, scale, kv_first):
        ops = ext.require()
        q, k, v = qkv3[:, :hq], qkv3[:, hq:hq + hkv], qkv3[:, hq + hkv:]
        o, lse = _sac_run("attention", None, lambda: ops.flash_fwd(q, k, v, scale, True, 0, kv_first))
        ctx.save_for_backward(qkv3, o, lse, kv_first if kv_first is not None else torch.empty(0))
        ctx.meta = (hq, hkv, scale, kv_first is not None)
        return o

    @staticmethod
    def backward(ctx, d_o):
        qkv3, o, lse, kv_first = ctx.saved_tensors
        hq, hkv, scale, has_first = ctx.meta
        ops = ext.require()
        q, k, v = qkv3[:, :hq], qkv3[:, hq:hq + hkv], qkv3[:, hq + hkv:]
        g = torch.empty_like(qkv3)
        ops.flash_bwd(d_o.contiguous(), q, k, v, o, lse, scale, True, 0, kv_first if has_first else None,
                      g[:, :hq], g[:, hq:hq + hkv], g[:, hq + hkv:])
        return g, None, None, None, None


def attention_packed(qkv3: torch.Tensor, hq: int, hkv: int, scale: float, *, doc_ids: torch.Tensor | None = None,
                     kv_first: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention where q, k and v are head slices of one ``[T, Hq + 2 Hkv, D]`` tensor."""
    q, k, v = qkv3[:, :hq], qkv3[:, hq:hq + hkv], qkv3[:, hq + hkv:]
    if (doc_ids is None or kv_first is not None) and qkv3.is_contiguous() and _native_attention_ok(q, k, v):
        _count(4)
        return _PackedFlashFn.apply(qkv3, hq, hkv, float(scale), kv_first)
    return attention(q, k, v, scale=scale, causal=True, doc_ids=doc_ids, kv_first=kv_first)


_DENSE_SCORE_BYTES = 256 << 20   # largest fp32 score block the PyTorch fallback materialises at a time


def _mask_block(qp, kp, causal, window, qd, kd):
    mask = torch.ones(qp.numel(), kp.numel(), dtype=torch.bool, device=qp.device)
    if causal:
        mask &= qp[:, None] >= kp[None, :]
    if window is not None and window > 0:
        mask &= (qp[:, None] - kp[None, :]) < window
    if qd is not None:
        mask &= qd[:, None] == kd[None, :]
    return mask


class _ChunkedAttentionFn(torch.autograd.Function):
    """PyTorch fallback for shapes and masks outside the flash kernels (general masks through positions, documents,
    windows, sinks; any head dimension).  Queries are processed in blocks sized so that one fp32 score block
    ``[Hq, Bq, Tk]`` stays under ``_DENSE_SCORE_BYTES``; nothing of size ``T x T`` is kept for the backward, which
    recomputes each block's probabilities from the saved log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, sinks, scale, causal, window, qp, kp, qd, kd):
        Tq, Hq, _ = q.shape
        Tk, Hkv, Dv = v.shape
        rep = Hq // Hkv
        kf = k.float().transpose(0, 1)
        vf = v.float().transpose(0, 1)
        if rep > 1:
            kf, vf = kf.repeat_interleave(rep, 0), vf.repeat_interleave(rep, 0)
        bq = max(16, min(Tq, _DENSE_SCORE_BYTES // max(1, 4 * Hq * Tk)))
        out = torch.empty(Tq, Hq, Dv, dtype=q.dtype, device=q.device)
        lse = torch.empty(Hq, Tq, dtype=torch.float32, device=q.device)
        for a in range(0, Tq, bq):
            b = min(Tq, a + bq)
            s_ = torch.matmul(q[a:b].float().transpose(0, 1), kf.transpose(1, 2)) * scale
            mask = _mask_block(qp[a:b], kp, causal, window, None if qd is None else qd[a:b], kd)
            s_ = s_.masked_fill(~mask[None], float("-inf"))
            if sinks is not None:
                l = torch.logsumexp(torch.cat([s_, sinks.float()[:, None, None].expand(Hq, b - a, 1)], dim=-1), dim=-1)
            else:
                l = torch.logsumexp(s_, dim=-1)
            safe = torch.where(torch.isinf(l), torch.zeros_like(l), l)
            p = torch.where(mask[None], torch.exp(s_ - safe[..., None]), torch.zeros_like(s_))
            out[a:b] = torch.matmul(p, vf).transpose(0, 1).to(q.dtype)
            lse[:, a:b] = l
        ctx.save_for_backward(q, k, v, out, lse, qp, kp, *(t for t in (sinks, qd, kd) if t is not None))
        ctx.meta = (scale, causal, window, bq, sinks is not None, qd is not None)
        return out

    @staticmethod
    def backward(ctx, d_o):
        scale, causal, window, bq, has_sinks, has_docs = ctx.meta
        q, k, v, out, lse, qp, kp, *rest = ctx.saved_tensors
        sinks = rest.pop(0) if has_sinks else None
        qd, kd = (rest[0], rest[1]) if has_docs else (None, None)
        Tq, Hq, _ = q.shape
        Tk, Hkv, Dv = v.shape
        rep = Hq // Hkv
        kf = k.float().transpose(0, 1)
        vf = v.float().transpose(0, 1)
        if rep > 1:
            kf, vf = kf.repeat_interleave(rep, 0), vf.repeat_interleave(rep, 0)
        dq = torch.empty_like(q)
        dk = torch.zeros(Hq, Tk, k.shape[2], dtype=torch.float32, device=q.device)
        dv = torch.zeros(Hq, Tk, Dv, dtype=torch.float32, device=q.device)
        d_sinks = torch.zeros(Hq, dtype=torch.float32, device=q.device) if has_sinks else None
        for a in range(0, Tq, bq):
            b = min(Tq, a + bq)
            qf = q[a:b].float().transpose(0, 1)
            dof = d_o[a:b].float().transpose(0, 1)
            s_ = torch.matmul(qf, kf.transpose(1, 2)) * scale
            mask = _mask_block(qp[a:b], kp, causal, window, None if qd is None else qd[a:b], kd)
            l = lse[:, a:b]
            safe = torch.where(torch.isinf(l), torch.zeros_like(l), l)
            p = torch.where(mask[None], torch.exp(s_ - safe[..., None]), torch.zeros_like(s_))
            delta = (dof * out[a:b].float().transpose(0, 1)).sum(-1)                    # [Hq, Bq]
            ds = p * (torch.matmul(dof, vf.transpose(1, 2)) - delta[..., None]) * scale
            dq[a:b] = torch.matmul(ds, kf).transpose(0, 1).to(q.dtype)
            dk += torch.matmul(ds.transpose(1, 2), qf)
            dv += torch.matmul(p.transpose(1, 2), dof)
            if has_sinks:
                d_sinks -= (torch.exp(sinks.float()[:, None] - safe) * delta).masked_fill(torch.isinf(l), 0.0).sum(-1)
        dk = dk.view(Hkv, rep, Tk, -1).sum(1).transpose(0, 1).to(k.dtype)
        dv = dv.view(Hkv, rep, Tk, -1).sum(1).transpose(0, 1).to(v.dtype)
        return dq, dk, dv, (d_sinks.to(sinks.dtype) if has_sinks else None), None, None, None, None, None, None, None


def _masked_attention(q, k, v, scale, causal, doc_ids, window, sinks, q_pos, k_pos):
    """General masks (documents, windows, sinks, explicit positions): memory-bounded PyTorch fallback."""
    Tq, Tk = q.shape[0], k.shape[0]
    dev = q.device
    qp = torch.arange(Tq, device=dev) if q_pos is None else q_pos
    kp = torch.arange(Tk, device=dev) if k_pos is None else k_pos
    qd = kd = None
    if doc_ids is not None:
        qd, kd = doc_ids if isinstance(doc_ids, tuple) else (doc_ids, doc_ids)
    return _ChunkedAttentionFn.apply(q, k, v, sinks, float(scale), bool(causal), window, qp, kp, qd, kd)


# =====================================================================
# Embedding
# =====================================================================
class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight):
        ctx.save_for_backward(tokens, weight)
        return weight.index_select(0, tokens.reshape(-1)).view(*tokens.shape, weight.shape[1])

    @staticmethod
    def backward(ctx, dy):
        tokens, weight = ctx.saved_tensors
        mg = getattr(weight, "main_grad", None)
        flat = dy.reshape(-1, dy.shape[-1])
        if mg is not None:
            g = mg.view(weight.shape)
            if not getattr(weight, "_main_grad_written", False):
                g.zero_()
                weight._main_grad_written = True
            g.index_add_(0, tokens.reshape(-1), flat.to(g.dtype))
            return None, None
        dw = torch.zeros_like(weight)
        dw.index_add_(0, tokens.reshape(-1), flat.to(dw.dtype))
        return None, dw


def embedding(tokens: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    return _EmbeddingFn.apply(tokens, weight)


# =====================================================================
# Cross entropy
# =====================================================================
def _ce_inplace(logits: torch.Tensor, labels: torch.Tensor, grad_scale: torch.Tensor, loss_acc: torch.Tensor):
    """Turn ``logits`` into ``dlogits`` in place and add the summed loss into ``loss_acc``."""
    if _cuda(logits):
        _count()
        row_loss = ext.require().cross_entropy_(logits, labels, grad_scale)
        loss_acc.add_(row_loss.sum())
        return logits
    loss, dl, _ = ref.cross_entropy_fwd_bwd(logits, labels, grad_scale)
    loss_acc.add_(loss)
    logits.copy_(dl)
    return logits


class _LinearCrossEntropyFn(torch.autograd.Function):
    """Chunked ``lm_head`` GEMM + cross entropy with gradients produced in the forward.

    Each chunk of rows computes its logits, turns them into ``dlogits`` in place
    (scaled by ``1 / global_valid_tokens``), and immediately produces the hidden
    and weight gradients, so the ``[T, V]`` logits never exist.  Parity with the
    chunked loss wrapper of the reference: torchtitan/components/loss.py:501-809.
    """

    @staticmethod
    def forward(ctx, hidden, weight, labels, inv_tokens, num_chunks):
        h2 = hidden.reshape(-1, hidden.shape[-1])
        lab = labels.reshape(-1)
        T = h2.shape[0]
        loss_acc = torch.zeros(1, dtype=torch.float32, device=h2.device)
        need_grad = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        dh = torch.empty_like(h2) if need_grad else None
        mg = getattr(weight, "main_grad", None)
        direct = need_grad and mg is not None and mg.dtype == h2.dtype
        dw = None
        if need_grad and weight.requires_grad and not direct:
            dw = torch.zeros(weight.shape, dtype=torch.float32, device=h2.device)
        chunk = max(1, -(-T // max(1, num_chunks)))
        scale = inv_tokens.to(torch.float32).reshape(1)
        for s in range(0, T, chunk):
            e = min(T, s + chunk)
            logits = gemm_nt(h2[s:e], weight)
            _ce_inplace(logits, lab[s:e], scale, loss_acc)
            if need_grad:
                gemm_nn(logits, weight, out=dh[s:e])
                if weight.requires_grad:
                    if direct:
                        acc = getattr(weight, "_main_grad_written", False)
                        gemm_tn(logits, h2[s:e], out=mg.view(weight.shape), accumulate=acc)
                        weight._main_grad_written = True
                    else:
                        dw.addmm_(logits.t().float(), h2[s:e].float())
            del logits
        ctx.save_for_backward(dh, dw)
        ctx.weight = weight
        ctx.hshape = hidden.shape
        ctx.direct = direct
        return (loss_acc * scale).squeeze(0)

    @staticmethod
    def backward(ctx, dloss):
        dh, dw = ctx.saved_tensors
        weight = ctx.weight
        # Gradients were computed for d(loss)=1; the trainer calls backward on the loss
        # itself, so dloss is one.  A different upstream scale is applied here.
        dhid = (dh * dloss.to(dh.dtype)).view(ctx.hshape) if dh is not None else None
        dwr = None
        if dw is not None:
            dwr = _deliver_wgrad(weight, (dw * dloss).to(weight.dtype))
        return dhid, dwr, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                         inv_global_tokens: torch.Tensor, num_chunks: int = 8) -> torch.Tensor:
    """``sum(CE(hidden @ W^T, labels)) * inv_global_tokens`` without materialising the logits."""
    if hidden.dtype != weight.dtype:
        hidden = hidden.to(weight.dtype)
    return _LinearCrossEntropyFn.apply(hidden, weight, labels, inv_global_tokens, num_chunks)


class _CrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels):
        l2 = logits.reshape(-1, logits.shape[-1]).clone()
        loss_acc = torch.zeros(1, dtype=torch.float32, device=logits.device)
        one = torch.ones(1, dtype=torch.float32, device=logits.device)
        _ce_inplace(l2, labels.reshape(-1), one, loss_acc)
        ctx.save_for_backward(l2)
        ctx.shape = logits.shape
        return loss_acc.squeeze(0)

    @staticmethod
    def backward(ctx, dloss):
        (dl,) = ctx.saved_tensors
        return (dl * dloss.to(dl.dtype)).view(ctx.shape), None


def cross_entropy_sum(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Sum over non-ignored tokens of the fp32 cross entropy."""
    return _CrossEntropyFn.apply(logits, labels)
