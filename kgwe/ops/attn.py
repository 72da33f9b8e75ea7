"""Causal GQA attention for the Llama block.

Dispatch order on a GPU:
  1. ``kgwe_flash_attn_*`` — the hand-written gfx950 MFMA flash-attention
     kernels in ``native/ops/flash_attn.hip`` (when built into the library);
  2. otherwise (head_dim != 128, or forced) PyTorch SDPA (ROCm flash
     backend) with the GQA heads expanded.
On CPU the fp32 reference is used.

``attention_packed`` is the same for sequences of different lengths packed on
one token axis (``native/ops/packed_attn.hip``).
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import reference as ref
from ._lib import (HALF_TYPES, addr, check, dense16, has_symbol, launch, lib, no_tangents, ptr, rows16, stream,
                   token_view, use_hip)
from .packed import PackedBatch


class _FlashAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal):
        B, S, Hq, D = q.shape
        Hkv = k.shape[2]
        o = torch.empty_like(q)
        lse = torch.empty(B, Hq, S, device=q.device, dtype=torch.float32)
        scale = 1.0 / math.sqrt(D)
        check(lib().kgwe_flash_attn_fwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), B, S, Hq, Hkv,
                                        D, scale, int(causal), stream(q)), "flash_attn_fwd")
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        B, S, Hq, D = q.shape
        Hkv = k.shape[2]
        do = do.contiguous()
        dq = torch.empty_like(q)
        dk = torch.empty_like(k)
        dv = torch.empty_like(v)
        ws = lib().kgwe_flash_attn_bwd_workspace(B, S, Hq, Hkv, D)
        work = torch.empty(max(ws, 4) // 4, device=q.device, dtype=torch.float32)
        check(lib().kgwe_flash_attn_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(do),
                                        ptr(dq), ptr(dk), ptr(dv), ptr(work), None, B, S, Hq,
                                        Hkv, D, 1.0 / math.sqrt(D), int(ctx.causal),
                                        stream(q)), "flash_attn_bwd")
        return dq, dk, dv, None


_FORCE_SDPA = False


def set_force_sdpa(flag: bool) -> None:
    global _FORCE_SDPA
    _FORCE_SDPA = flag


def hip_flash_available() -> bool:
    return has_symbol("kgwe_flash_attn_fwd") and has_symbol("kgwe_flash_attn_bwd")


def flash_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True):
    """Forward only (inference / tests): returns (o, lse2) with lse2 in log2 units."""
    B, S, Hq, D = q.shape
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()
            and q.dtype == k.dtype == v.dtype == torch.bfloat16 and D == 128
            and k.shape == v.shape == (B, S, k.shape[2], D) and Hq % k.shape[2] == 0):
        raise ValueError("flash_fwd: contiguous bf16 [B,S,H,128] q/k/v with Hq % Hkv == 0")
    o = torch.empty_like(q)
    lse = torch.empty(B, Hq, S, device=q.device, dtype=torch.float32)
    check(lib().kgwe_flash_attn_fwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), B, S, Hq, k.shape[2],
                                    D, 1.0 / math.sqrt(D), int(causal), stream(q)), "flash_attn_fwd")
    return o, lse


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True):
    """q [B,S,Hq,D], k/v [B,S,Hkv,D] -> o [B,S,Hq,D]."""
    if not use_hip(q):
        return ref.attention(q, k, v, causal)
    if not _FORCE_SDPA and q.shape[-1] == 128 and hip_flash_available():
        return _FlashAttn.apply(q.contiguous(), k.contiguous(), v.contiguous(), causal)
    hq, hkv = q.shape[2], k.shape[2]
    qt, kt, vt = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    if hq != hkv:
        kt = kt.repeat_interleave(hq // hkv, dim=1)
        vt = vt.repeat_interleave(hq // hkv, dim=1)
    o = F.scaled_dot_product_attention(qt, kt, vt, is_causal=causal)
    return o.transpose(1, 2)


# --------------------------------------------------------------------------
# Packed sequences
# --------------------------------------------------------------------------
def _packed_fwd(qv, kv, vv, batch, causal, prefix, train):
    """qv, kv, vv: token_view of q, k, v."""
    (q, qp, qr, qh), (k, kp, kr, kh), (_, vp, vr, vh) = qv, kv, vv
    (T, Hq, D), device = q.shape, q.device
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    low = lse = None
    if train:
        lse = torch.empty((Hq, T), device=device, dtype=torch.float32)
        low = torch.empty_like(o)  # what the rounding of o drops
    if prefix is None:
        pk = pv = pkr = pkh = pvr = pvh = P = 0
    else:  # [Hkv, P, D]: row stride, head stride
        (pkh, pkr, _), (pvh, pvr, _), P = prefix[0].stride(), prefix[1].stride(), prefix[0].shape[1]
        pk, pv = prefix[0].data_ptr(), prefix[1].data_ptr()
    jobs, slots = batch.tables
    launch("kgwe_packed_attn_fwd", device, qp, kp, vp, pk, pv, o.data_ptr(), addr(low), addr(lse), jobs, qr, qh, kr, kh,
           vr, vh, pkr, pkh, pvr, pvh, P, slots, T, Hq, k.shape[1], D, causal, HALF_TYPES[q.dtype], D ** -0.5)
    return o, low, lse


class _PackedAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, batch, causal):
        views = token_view(q), token_view(k), token_view(v)
        o, low, lse = _packed_fwd(*views, batch, causal, None, True)
        q, k, v = (t[0] for t in views)
        ctx.save_for_backward(q, k, v, o, low, lse)
        ctx.batch, ctx.causal = batch, causal
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, low, lse = ctx.saved_tensors
        batch = ctx.batch
        T, Hq, D = q.shape
        Hkv = k.shape[1]
        do = dense16(do)
        dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
        delta = torch.empty_like(lse)
        (qr, qh, _), (kr, kh, _), (vr, vh, _) = q.stride(), k.stride(), v.stride()
        jobs, slots = batch.tables
        words = int(lib().kgwe_packed_attn_bwd_workspace(slots, T, Hq, Hkv, D))
        work = torch.empty(words, device=q.device, dtype=torch.float32) if words else None
        launch("kgwe_packed_attn_bwd", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), low.data_ptr(),
               lse.data_ptr(), do.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), addr(work),
               jobs, qr, qh, kr, kh, vr, vh, slots, T, Hq, Hkv, D, ctx.causal, HALF_TYPES[q.dtype], D ** -0.5)
        return dq, dk, dv, None, None


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: PackedBatch, causal: bool = True,
                     prefix: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
    """Attention of every sequence of a packed batch with itself: q [T, Hq, D],
    k / v [T, Hkv, D] -> [T, Hq, D], T = ``batch.total``; differentiable.

    prefix: (keys, values), each [Hkv, P, D], that every row sees before its
    own sequence (a prompt shared by the batch); forward only.  Padding rows
    (behind the last sequence) give zeros and get zero gradients, whatever they
    hold.  On a GPU: bf16 or fp16, D 64 or 128; q / k / v may be views with
    dense 16-byte aligned rows (slices of a fused projection), others are
    copied.  A call that will be differentiated keeps its inputs, the result,
    what the result's rounding dropped (a second [T, Hq, D]) and row sums (fp32
    [Hq, T]) for the gradient.  Forward-mode derivatives are refused on a GPU.

    How the work is split depends on the whole batch (its rows and its number of
    sequences), so a sequence may round differently in another batch; one call
    repeated gives the same bits.  Never does anything of one sequence enter
    another, NaN and infinities included.  Inside its own sequence a non-finite value (in v; for gradients
    also in q, k or the incoming gradient) reaches what depends on it, and may
    also reach up to 63 rows on its other side of the causal diagonal."""
    qs, ks = q.shape, k.shape
    if not (len(qs) == len(ks) == 3 and v.shape == ks and qs[0] == ks[0] == batch.total and qs[2] == ks[2]
            and qs[1] > 0 and ks[1] > 0 and qs[1] % ks[1] == 0):
        raise ValueError(f"attention_packed: q [T, Hq, D], k / v [T, Hkv, D] with T = {batch.total} and Hq % Hkv == 0, "
                         f"got {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    dtype, device = q.dtype, q.device
    if not (k.dtype == v.dtype == dtype and k.device == v.device == device == batch.device):
        raise ValueError("attention_packed: tensors and batch must share one type and device")
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if prefix is not None:
        pk, pv = prefix
        if not (pk.dim() == 3 and pk.shape == pv.shape and pk.shape[0] == ks[1] and pk.shape[2] == ks[2]
                and pk.dtype == pv.dtype == dtype and pk.device == pv.device == device):
            raise ValueError("attention_packed: prefix keys and values must be [Hkv, P, D] of k's type and device")
        if grad or (torch.is_grad_enabled() and (pk.requires_grad or pv.requires_grad)):
            raise ValueError("attention_packed: a shared prefix has no gradient; call it under torch.no_grad()")
    if not q.is_cuda:
        return ref.attention_packed(q, k, v, batch.lengths.tolist(), causal, prefix)
    if dtype not in HALF_TYPES or qs[2] not in (64, 128):
        raise ValueError("attention_packed: bf16 or fp16 with head_dim 64 or 128")
    no_tangents("attention_packed", q, k, v, *(prefix or ()))
    if batch.total == 0:
        return q.clone()
    if grad:
        return _PackedAttn.apply(q, k, v, batch, bool(causal))
    if prefix is not None:
        prefix = (rows16(pk), rows16(pv)) if pk.shape[1] else None
    return _packed_fwd(token_view(q), token_view(k), token_view(v), batch, bool(causal), prefix, False)[0]
