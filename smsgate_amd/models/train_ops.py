"""Fused training forward of the extractor LM (the bench trains it in-run, untimed).

:func:`~smsgate_amd.models.extractor.reference_forward` is the plain-PyTorch forward:
every RMSNorm, RoPE and SwiGLU is a chain of small elementwise kernels forward and
backward (~45 launches per layer), which at the bench recipe (128 sequences x ~60
tokens, 7.7 k rows) spent over half of a training step's GPU time re-reading the same
activations (scripts/train_step_profile.py).  :func:`fused_forward` is the same
network with those groups as single HIP kernels (ops/csrc/train_kernels.hip), each an
autograd Function with a hand-written backward:

* ``RMSNorm``: fp32 residual stream in, bf16 normalised rows out (the GEMM's input, so
  autocast's cast is folded in), rstd saved; backward dx in fp32 and dw from per-block
  partial sums;
* ``RopeSplit``: the QKV GEMM's bf16 output -> q / k / v in SDPA's [B, heads, T, D]
  layout with rotate-half RoPE on q and k (fp32 math, the caller's cos / sin tables);
  backward is the adjoint rotation straight into dqkv;
* ``SwiGLU``: silu(gate) * up from the fused gate/up GEMM output, and its backward;
* ``Attention`` (opt-in, ``SMSGATE_TRAIN_SDPA=own``): causal grouped-query attention over
  the batch (<= 192 rows) straight into the o-proj's [B, T, heads * 64] input and its
  backward -- correct (fp32-reference tests) but one thread per row is latency-bound:
  56 ms of a step against SDPA's ~6 (``r05_train_step_sdpa_ab.jsonl``), so SDPA (flash)
  stays the default.

Three operators of the whole step, on request (``hip_ops``; TrainConfig.hip_ops):

* :func:`embed_lookup`: both embedding rows of a position in one pass, the table's gradient
  by sorted ids in a fixed order (csrc/embed_kernels.hip);
* :func:`tiled_attention`: attention of any length in matrix instructions, its backward pass
  recomputing the probabilities (csrc/attn_grad_kernels.hip);
* :func:`lm_loss`: cross entropy over the embedding's rows without logits, for the copy and
  span answer formats (csrc/loss_kernels.hip).

Their autograd functions are C++ (csrc/train_autograd.cpp): one message's call is host time,
and a Python Function spends 1.3 to 1.7 times as much of it.  Forward and backward of 45
positions take 26 to 46 us (36 to 79 in Python), attention of 37 rows 40 to 70 (57 to 116),
the loss of 61 rows 47 to 76 (60 to 115): autograd hands a GPU backward to another thread and
back in about 16 us or in 40, for seconds at a time.  Through autograd, torch's own operators
take 46 us for the embedding, 104 for the attention and 170 for the loss where these take 45,
64 and 73.

Their forward and backward can be captured into a graph.  As with any torch operator, no
eager graph of the same leaves may be alive then: a leaf's accumulation node belongs to the
stream that it was first used on, and autograd would wait for that stream inside the capture.
Where such a leaf is an operator's own input, the captured call raises.

GEMMs stay hipBLASLt (autocast bf16), so the math is
reference_forward's up to bf16 rounding order (tests/test_train_ops_gpu.py compares
losses and gradients).  CPU / no-library: reference_forward.
"""
from __future__ import annotations

import contextlib
import functools
import math
import operator
import os
from typing import Optional

import torch
import torch.nn.functional as F

from .. import ops
from .extractor import ExtractorWeights, _rope_tables

__all__ = ["fused_forward", "rms_norm", "rope_split", "swiglu", "attention", "available", "ATTN_MAX_T",
           "embed_lookup", "tiled_attention", "lm_loss"]


def available(device) -> bool:
    return str(device).startswith("cuda") and torch.cuda.is_available()


def _lib():
    return ops.load_library()


def _st() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ok(rc: int, name: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{name} failed (rc={rc})")


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
        H = x.shape[-1]
        x2 = x.reshape(-1, H)
        if x2.dtype != torch.float32 or not x2.is_contiguous() or w.dtype != torch.float32:
            raise ValueError("rms_norm: contiguous fp32 rows and fp32 weight")
        R = x2.shape[0]
        y = torch.empty(R, H, dtype=torch.bfloat16, device=x.device)
        rstd = torch.empty(R, dtype=torch.float32, device=x.device)
        _ok(_lib().sg_rms_fwd(x2.data_ptr(), w.data_ptr(), y.data_ptr(), rstd.data_ptr(), R, H, float(eps), _st()),
            "rms_fwd")
        ctx.save_for_backward(x2, w, rstd)
        ctx.shape = x.shape
        return y.view(*x.shape[:-1], H)

    @staticmethod
    def backward(ctx, dy: torch.Tensor):
        x2, w, rstd = ctx.saved_tensors
        R, H = x2.shape
        dy = dy.reshape(R, H)
        if dy.dtype != torch.bfloat16:
            dy = dy.to(torch.bfloat16)
        dy = dy.contiguous()
        rpb = 64
        nb = (R + rpb - 1) // rpb
        dx = torch.empty(R, H, dtype=torch.float32, device=x2.device)
        part = torch.empty(nb, H, dtype=torch.float32, device=x2.device)
        _ok(_lib().sg_rms_bwd(dy.data_ptr(), x2.data_ptr(), w.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                              part.data_ptr(), R, H, rpb, _st()), "rms_bwd")
        return dx.view(ctx.shape), part.sum(0), None


class _RopeSplit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nh: int, nkv: int, rep: int):
        B, T, N = qkv.shape
        D = N // (nh + 2 * nkv)
        if qkv.dtype != torch.bfloat16 or D != 64 or N != (nh + 2 * nkv) * D:
            raise ValueError("rope_split: bf16 [B, T, (nh + 2 nkv) * 64]")
        qkv = qkv.contiguous()
        q = torch.empty(B, nh, T, D, dtype=qkv.dtype, device=qkv.device)
        k = torch.empty(B, nkv * rep, T, D, dtype=qkv.dtype, device=qkv.device)
        v = torch.empty(B, nkv * rep, T, D, dtype=qkv.dtype, device=qkv.device)
        _ok(_lib().sg_rope_split(1, qkv.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(),
                                 sin.data_ptr(), B, T, nh, nkv, D, rep, _st()), "rope_split")
        ctx.save_for_backward(cos, sin)
        ctx.dims = (B, T, nh, nkv, D, rep)
        return q, k, v

    @staticmethod
    def backward(ctx, dq, dk, dv):
        cos, sin = ctx.saved_tensors
        B, T, nh, nkv, D, rep = ctx.dims
        dev = cos.device

        def _g(t, h):
            if t is None:
                return torch.zeros(B, h, T, D, dtype=torch.bfloat16, device=dev)
            return t.to(torch.bfloat16).contiguous()

        dq, dk, dv = _g(dq, nh), _g(dk, nkv * rep), _g(dv, nkv * rep)
        dqkv = torch.empty(B, T, (nh + 2 * nkv) * D, dtype=torch.bfloat16, device=dev)
        _ok(_lib().sg_rope_split(-1, dqkv.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), cos.data_ptr(),
                                 sin.data_ptr(), B, T, nh, nkv, D, rep, _st()), "rope_split_bwd")
        return dqkv, None, None, None, None, None


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu: torch.Tensor) -> torch.Tensor:
        I2 = gu.shape[-1]
        if gu.dtype != torch.bfloat16 or I2 % 16:
            raise ValueError("swiglu: bf16 [..., 2 I] with I % 8 == 0")
        g2 = gu.reshape(-1, I2).contiguous()
        R, I = g2.shape[0], I2 // 2
        a = torch.empty(R, I, dtype=gu.dtype, device=gu.device)
        _ok(_lib().sg_swiglu_fwd(g2.data_ptr(), a.data_ptr(), R, I, _st()), "swiglu_fwd")
        ctx.save_for_backward(g2)
        ctx.shape = gu.shape
        return a.view(*gu.shape[:-1], I)

    @staticmethod
    def backward(ctx, da: torch.Tensor):
        (g2,) = ctx.saved_tensors
        R, I2 = g2.shape
        da = da.reshape(R, I2 // 2).to(torch.bfloat16).contiguous()
        dgu = torch.empty_like(g2)
        _ok(_lib().sg_swiglu_bwd(da.data_ptr(), g2.data_ptr(), dgu.data_ptr(), R, I2 // 2, _st()), "swiglu_bwd")
        return dgu.view(ctx.shape)


ATTN_MAX_T = 192  # csrc/train_kernels.hip AT_MAXT


class _Attention(torch.autograd.Function):
    """Causal grouped-query attention of one training batch (attn_train_* kernels):
    q [B, nh, T, 64], k / v [B, nkv, T, 64] -> out [B, T, nh * 64] (the o-proj input)."""

    @staticmethod
    def forward(ctx, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> torch.Tensor:
        B, nh, T, D = q.shape
        nkv = k.shape[1]
        if D != 64 or T > ATTN_MAX_T or nh % nkv or q.dtype != torch.bfloat16:
            raise ValueError("attention: bf16, head_dim 64, T <= 192, nh % nkv == 0")
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        out = torch.empty(B, T, nh * D, dtype=q.dtype, device=q.device)
        lse = torch.empty(B, nh, T, dtype=torch.float32, device=q.device)
        _ok(_lib().sg_attn_train_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), B, T,
                                     nh, nkv, float(scale), _st()), "attn_train_fwd")
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout: torch.Tensor):
        q, k, v, out, lse = ctx.saved_tensors
        B, nh, T, D = q.shape
        nkv = k.shape[1]
        dout = dout.to(torch.bfloat16).contiguous()
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dsum = torch.empty(B, nh, T, dtype=torch.float32, device=q.device)
        _ok(_lib().sg_attn_train_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                                     dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dsum.data_ptr(), B,
                                     T, nh, nkv, float(ctx.scale), _st()), "attn_train_bwd")
        return dq, dk, dv, None


_TABLES = (torch.float32, torch.bfloat16, torch.float16)


@functools.lru_cache(maxsize=1)
def _native():
    """The operators' autograd functions (csrc/train_autograd.cpp)."""
    return ops.load_train_autograd()


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, heads, T, D] itself when its rows can be read 16 bytes at a time, else a copy
    (what tiled_attention does with q, k and v)."""
    return _native().rows16(t)


def _on_gpu(name: str, *tensors: Optional[torch.Tensor]) -> None:
    first = tensors[0]
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device != first.device):
            raise ValueError(f"{name}: every tensor must be on the same GPU")


def embed_lookup(ids: torch.Tensor, table: torch.Tensor, add_ids: Optional[torch.Tensor] = None, *,
                 scale: float = 1.0) -> torch.Tensor:
    """``scale * (table[ids] + table[add_ids])`` as ``[*ids.shape, H]`` in the table's type
    (csrc/embed_kernels.hip), differentiable in ``table``.

    ``ids``: int32 or int64, any shape.  ``table`` [V, H]: fp32, bf16 or fp16.  ``add_ids``
    (``ids``' shape and type): a second row added to each position, negative = none (the
    span formats' pointer rows).  The sum is taken and scaled in fp32 and rounded once.  The
    table's gradient sums the positions of each id in fp32, in their order: the same bits
    every run.  An id outside [0, V) (``add_ids``: above it) makes its position NaN and has no row in
    the gradient."""
    if table.dim() != 2 or table.dtype not in _TABLES:
        raise TypeError("embed_lookup: table must be fp32, bf16 or fp16 [V, H]")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("embed_lookup: ids must be int32 or int64")
    if add_ids is not None and (add_ids.shape != ids.shape or add_ids.dtype != ids.dtype):
        raise ValueError("embed_lookup: add_ids must have the shape and type of ids")
    most = (1 << 26) - 4  # a wave a row, 4 a block, fewer than 2^32 threads
    if not (1 <= table.shape[0] <= most and 1 <= table.shape[1] <= 1 << 20) or ids.numel() > most:
        raise ValueError("embed_lookup: 1 <= V <= 2^26 - 4, 1 <= H <= 2^20, at most 2^26 - 4 ids")
    _on_gpu("embed_lookup", table, ids, add_ids)
    return _native().embed(table, ids, add_ids, float(scale))


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> torch.Tensor:
    return _Attention.apply(q, k, v, scale)


def tiled_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None, *,
                    causal: bool = True, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped-query attention of a batch in matrix instructions
    (csrc/attn_grad_kernels.hip), any length, differentiable in q, k and v.

    ``q`` [B, nh, T, D], ``k`` / ``v`` [B, nkv, T, D]: bf16 or fp16, D 64 or 128, nh a
    multiple of nkv (query head h reads key head ``h // (nh // nkv)``), any strides.
    ``scale``: > 0, default ``D ** -0.5``.  ``causal``: query i sees keys up to i.
    ``lengths`` (int32 [B]): sequence b is its first ``lengths[b]`` rows (clamped to 0..T);
    the rows behind are zero in the result and in every gradient, and what they hold in q,
    k, v and the incoming gradient has no effect, infinities and NaN included.  (Inside a
    sequence, an infinity or NaN may reach rows that a causal mask keeps from it, as 0 times
    it does in any product with masked probabilities; other sequences never.)  Returns
    [B, T, nh * D] (the o-projection's input).  Probabilities are recomputed in the
    backward pass and nothing of size T x T is stored; every sum has a fixed order."""
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("tiled_attention: q, k and v must all be bf16 or all fp16")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or min(q.shape) < 1 or min(k.shape) < 1:
        raise ValueError("tiled_attention: q [B, nh, T, D], k and v [B, nkv, T, D], none of them empty")
    B, nh, T, D = q.shape
    if k.shape[0] != B or k.shape[2:] != (T, D) or nh % k.shape[1] or D not in (64, 128):
        raise ValueError("tiled_attention: k and v need q's batch, length and width (64 or 128), and nh % nkv == 0")
    if T > 1 << 24 or B * nh > 1 << 20 or B * nh * ((T + 127) // 128) >= 1 << 24:
        raise ValueError("tiled_attention: T <= 2^24, B * nh <= 2^20, fewer than 2^24 tiles of 128 rows")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError("tiled_attention: scale must be finite and above 0 (1e-30 to 1e30)")
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != (B,)):
        raise ValueError("tiled_attention: lengths must be int32 [B]")
    _on_gpu("tiled_attention", q, k, v, lengths)
    return _native().attention(q, k, v, lengths, scale, bool(causal))


_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def lm_loss(h: torch.Tensor, table: torch.Tensor, labels: torch.Tensor, *, reduction: str = "mean",
            ignore_index: int = -100) -> torch.Tensor:
    """Softmax cross entropy of ``h @ table.T`` against ``labels`` (csrc/loss_kernels.hip),
    differentiable in ``h`` and ``table``, without a matrix of logits: the forward keeps
    tiles of them in registers, the backward recomputes them a piece of the vocabulary at a
    time.

    ``h`` [..., H] and ``table`` [V, H]: both bf16 or both fp16, H a multiple of 8 (masters
    in fp32 are cast by the caller, as autocast does).  ``labels`` [...]: int32 or int64.
    Rows of label ``ignore_index`` cost no product: they are left out by a list built on the
    GPU.  ``reduction``: ``mean`` over the labelled rows (none labelled: NaN, gradients 0),
    ``sum``, or ``none`` (fp32 per row, 0 where ignored).  A label outside [0, V) makes its
    row's loss NaN, and the gradients that take part in it.  Sums are fp32 in a fixed order."""
    if h.dtype not in (torch.bfloat16, torch.float16) or table.dtype != h.dtype:
        raise TypeError("lm_loss: h and table must both be bf16 or both fp16")
    if labels.dtype not in (torch.int32, torch.int64):
        raise TypeError("lm_loss: labels must be int32 or int64")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"lm_loss: reduction {reduction!r}: mean | sum | none")
    if h.dim() < 1 or table.dim() != 2 or h.shape[-1] != table.shape[1] or labels.shape != h.shape[:-1]:
        raise ValueError("lm_loss: h [..., H], table [V, H] and labels [...] do not fit")
    V, H = table.shape
    N = labels.numel()
    if not (1 <= N <= 1 << 24 and 1 <= V <= 1 << 24 and 8 <= H <= 1 << 14) or H % 8 \
            or ((N + 255) // 128) * ((V + 255) // 256) >= 1 << 24 or (N + V + 512) * (H + 63) >= 1 << 34:
        raise ValueError("lm_loss: 1 to 2^24 rows and ids, H a multiple of 8 up to 2^14, fewer than 2^24 tiles of "
                         "128 x 256, (rows + ids) * H under 2^34")
    try:
        ignore_index = operator.index(ignore_index)
    except TypeError:
        raise TypeError("lm_loss: ignore_index must be a whole number") from None
    if not -(1 << 31) <= ignore_index < 1 << 31:
        raise ValueError("lm_loss: ignore_index must fit 32 bits")
    _on_gpu("lm_loss", h, table, labels)
    return _native().loss(h, table, labels, _REDUCTIONS[reduction], ignore_index)


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    return _RMSNorm.apply(x, w, eps)


def rope_split(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nh: int, nkv: int, rep: int = 1):
    """q [B, nh, T, D], k / v [B, nkv * rep, T, D] (``rep`` copies of each kv head)."""
    return _RopeSplit.apply(qkv, cos, sin, nh, nkv, rep)


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    return _SwiGLU.apply(gu)


def fused_forward(w: ExtractorWeights, ids: torch.Tensor, add_ids: Optional[torch.Tensor] = None, *,
                  hip_ops: bool = False, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Final-normed hidden states [B, T, H] (bf16) of ``reference_forward(w, ids,
    return_hidden=True, add_ids=add_ids)``; call under ``torch.autocast(bf16)`` with fp32
    master weights (models/train.py).  ``hip_ops``: the embedding is :func:`embed_lookup` and
    the attention :func:`tiled_attention` (over the first ``lengths[b]`` positions of each
    row, int32; the states behind them are then not meant to be read) instead of
    F.embedding and SDPA."""
    cfg = w.cfg
    B, T = ids.shape
    nh, nkv, D = cfg.heads, cfg.kv_heads, cfg.head_dim
    if hip_ops:
        x = embed_lookup(ids, w.embed, add_ids)
    else:
        if lengths is not None:
            raise ValueError("fused_forward: lengths need hip_ops")
        x = F.embedding(ids, w.embed)
        if add_ids is not None:
            x = x + F.embedding(add_ids.clamp(min=0), w.embed) * (add_ids >= 0).unsqueeze(-1).to(x.dtype)
    x = x.float().contiguous()
    cos, sin = _rope_tables(T, D, cfg.rope_theta, ids.device)
    cos, sin = cos.reshape(T, D // 2).contiguous(), sin.reshape(T, D // 2).contiguous()
    scale = 1.0 / math.sqrt(D)
    # attention: SDPA (flash) by default; SMSGATE_TRAIN_SDPA=own runs the attn_train_*
    # kernels (<= 192 rows; correct, but 56 vs ~6 ms per step: one thread per row is
    # latency-bound, r05_train_step_sdpa_ab.jsonl); the efficient backend has no GQA
    # support, so it gets k / v expanded to nh heads by rope_split (its adjoint sums them)
    sdpa = os.environ.get("SMSGATE_TRAIN_SDPA", "")
    rep = nh // nkv if sdpa == "efficient" else 1
    own = sdpa == "own" and T <= ATTN_MAX_T
    if hip_ops:
        rep, own = 1, functools.partial(tiled_attention, lengths=lengths)
    else:
        own = attention if own else None
    with _sdpa_backend():
        for i in range(cfg.layers):
            x = _layer(w, i, x, cos, sin, scale, B, T, nh, nkv, D, rep, own)
    return rms_norm(x, w.ln_f, cfg.eps)


def _sdpa_backend():
    """SMSGATE_TRAIN_SDPA = flash | efficient | math pins SDPA's backend (A/B of the
    training step, scripts/train_step_profile.py); default: PyTorch's choice."""
    name = os.environ.get("SMSGATE_TRAIN_SDPA", "")
    if name in ("", "own"):
        return contextlib.nullcontext()
    from torch.nn.attention import SDPBackend, sdpa_kernel

    return sdpa_kernel({"flash": SDPBackend.FLASH_ATTENTION, "efficient": SDPBackend.EFFICIENT_ATTENTION,
                        "math": SDPBackend.MATH}[name])


def _layer(w, i, x, cos, sin, scale, B, T, nh, nkv, D, rep=1, own=None):
    """One decoder layer of the residual stream ``x`` (fp32); ``own``: an attention of
    (q, k, v, scale) in SDPA's place."""
    eps = w.cfg.eps
    h = rms_norm(x, w.ln1[i], eps)
    q, k, v = rope_split(h @ w.qkv[i].t(), cos, sin, nh, nkv, rep)
    if own is not None:
        a = own(q, k, v, scale)
    else:
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=scale,
                                           enable_gqa=nh != nkv * rep).transpose(1, 2).reshape(B, T, nh * D)
    x = x + a @ w.o[i].t()
    h = rms_norm(x, w.ln2[i], eps)
    return x + swiglu(h @ w.gate_up[i].t()) @ w.down[i].t()
