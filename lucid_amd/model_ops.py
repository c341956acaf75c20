"""Fused elementwise layers of the Llama-LUCID decoder on HIP kernels.

The reference model (``modeling_lucid.py:58-75`` RMSNorm, ``:112-145`` rotate_half /
apply_rotary_pos_emb, ``:155-167`` the SwiGLU MLP, ``:847-967`` the loss) writes these as
chains of torch elementwise ops, each a full pass over the activations in HBM.  Here each is
one kernel pass forward and one backward:

* :func:`rms_norm` -- y = w * bf16(x * rstd) with rstd = 1 / sqrt(mean(x^2) + eps) in fp32
  (the reference's statistics and rounding points); backward dx = rstd (g - xn mean(g xn)),
  g = bf16(dy w), and dw summed over row blocks in a fixed order (deterministic).
* :func:`apply_rope` -- x cos + rotate_half(x) sin on a ``[B, H, T, 64]`` view of the
  ``[B, T, H, 64]`` projection output (any strides that are multiples of 8), written as
  ``[B, T, H, 64]`` (returned as the same transposed view), rounded to bf16 once; backward
  applies the transposed rotation.

* :func:`swiglu` -- silu(g) * u of the MLP, one pass each way with fp32 inside (the
  reference rounds silu(g) to bf16 before the product).
* :func:`causal_lm_loss` -- the shifted cross entropy on bf16 logits, one read of the logits
  forward (per-row logsumexp) and one read + write backward, instead of fp32 copies of them.
* :func:`rotary` -- queries and keys turned by their positions in one pass: any head dim up to 256, the whole head or a
  part, in halves or interleaved, frequencies of :func:`rope_frequencies` (scaled for long contexts) or any others,
  angles in 64 bits (bf16 or fp32).
* :func:`constrain_logits` -- penalties of tokens that have occurred, biases and bit masks of allowed tokens on logit
  rows (bf16 or fp32, any vocabulary).
* :func:`token_logprobs` -- log probabilities of given tokens, entropy and the top alternatives of
  logit rows (bf16 or fp32, any vocabulary), and the gradient of all three.

The others take bf16 GPU tensors only (RMSNorm: hidden sizes 512, 1024, 2048 or 4096; RoPE: head
dim 64; the loss: a vocabulary that is a multiple of 8) and raise otherwise; the
``*_supported`` predicates tell the model which inputs they cover.
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_NORM_H = (512, 1024, 2048, 4096)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous with a 16-byte aligned base (the kernels load 8 bf16 at a time)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def rms_norm_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    return (x.is_cuda and x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16
            and x.shape[-1] in _NORM_H and weight.shape == (x.shape[-1],))


def rope_supported(x: torch.Tensor, cos: torch.Tensor) -> bool:
    return x.is_cuda and x.dtype == torch.bfloat16 and cos.dtype == torch.bfloat16 and x.dim() == 4 \
        and x.shape[-1] == 64


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: torch.Tensor, weight: torch.Tensor, eps: float):
        if not rms_norm_supported(x, weight):
            raise TypeError("lucid_amd.rms_norm: bf16 GPU input and weight with hidden size in "
                            f"{_NORM_H}, got {x.dtype} {tuple(x.shape)} / {weight.dtype}")
        H = x.shape[-1]
        x2 = _aligned(x.reshape(-1, H))
        w = _aligned(weight)
        N = x2.shape[0]
        y = torch.empty_like(x2)
        rstd = torch.empty(N, dtype=torch.float32, device=x.device)
        lib = _lib.load()
        rc = lib.lucid_rmsnorm_fwd(_lib.ptr(x2), _lib.ptr(w), _lib.ptr(y), _lib.ptr(rstd), N, H, float(eps),
                                   _lib.stream_handle(x.device))
        _lib.check(lib, rc, "lucid_rmsnorm_fwd")
        ctx.save_for_backward(x2, w, rstd)
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy: torch.Tensor):
        x2, w, rstd = ctx.saved_tensors
        N, H = x2.shape
        dy2 = _aligned(dy.reshape(N, H))
        dx = torch.empty_like(x2)
        dw = torch.empty_like(w)
        lib = _lib.load()
        nbytes = lib.lucid_rmsnorm_bwd_workspace_bytes(N, H)
        ws = torch.empty(max(nbytes // 4, 1), dtype=torch.float32, device=x2.device)
        rc = lib.lucid_rmsnorm_bwd(_lib.ptr(x2), _lib.ptr(w), _lib.ptr(dy2), _lib.ptr(rstd), _lib.ptr(dx),
                                   _lib.ptr(dw), _lib.ptr(ws), N, H, _lib.stream_handle(x2.device))
        _lib.check(lib, rc, "lucid_rmsnorm_bwd")
        return dx.view(ctx.shape), dw, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """RMSNorm over the last axis (``LlamaRMSNorm.forward``, modeling_lucid.py:58-75)."""
    return RMSNormFunction.apply(x, weight, eps)


def _strided(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, H, T, 64] as the kernel reads it: unit stride on the head axis, the other
    strides multiples of 8 elements, a 16-byte aligned base (copied otherwise)."""
    if t.stride(3) == 1 and all(s % 8 == 0 for s in t.stride()[:3]) and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous()


def _tokens(c: torch.Tensor, B: int, T: int) -> torch.Tensor:
    """cos / sin [B or 1, T, 64] as B*T contiguous token rows."""
    if c.dim() == 2:
        c = c.unsqueeze(0)
    return _aligned(c.expand(B, T, c.shape[-1]))


def _rope_launch(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, transpose: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """x [B, H, T, 64] rotated into ``out`` ([B, H, T, 64], strides multiples of 8; default: a
    new [B, T, H, 64] buffer seen as [B, H, T, 64])."""
    B, Hn, T, D = x.shape
    xr = _strided(x)
    if out is None:
        out = torch.empty(B, T, Hn, D, dtype=x.dtype, device=x.device).transpose(1, 2)
    lib = _lib.load()
    rc = lib.lucid_rope(_lib.ptr(xr), _lib.strides3(xr, (0, 1, 2)), B, Hn, T, _lib.ptr(cos), _lib.ptr(sin),
                        _lib.ptr(out), _lib.strides3(out, (0, 1, 2)), D, transpose, _lib.stream_handle(x.device))
    _lib.check(lib, rc, "lucid_rope")
    return out


class RopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
        if not rope_supported(x, cos) or sin.dtype != cos.dtype:
            raise TypeError(f"lucid_amd.apply_rope: bf16 GPU [B, H, T, 64] input, got {x.dtype} {tuple(x.shape)}")
        B, _, T, _ = x.shape
        c, s = _tokens(cos, B, T), _tokens(sin, B, T)
        ctx.save_for_backward(c, s)
        return _rope_launch(x, c, s, 0)

    @staticmethod
    def backward(ctx, g: torch.Tensor):
        c, s = ctx.saved_tensors
        return _rope_launch(g, c, s, 1), None, None


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x cos + rotate_half(x) sin for x [B, H, T, 64] and cos / sin [B or 1, T, 64]
    (modeling_lucid.py:118-145 with unsqueeze_dim 1)."""
    return RopeFunction.apply(x, cos, sin)


class QKVRopeFunction(torch.autograd.Function):
    """The stacked projection output qkv [B, T, (Hq + 2 Hkv) 64] split into q, k, v, with the
    rotary embedding applied to q and k.  Its backward writes the rotated-back dq, dk and dv
    straight into one [B, T, (Hq + 2 Hkv) 64] gradient, so that no concatenation of the three
    follows (the split's own backward would concatenate them)."""

    @staticmethod
    def forward(ctx, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nq: int, nk: int):
        B, T, N = qkv.shape
        if not (qkv.is_cuda and qkv.dtype == torch.bfloat16 and cos.dtype == torch.bfloat16
                and nq % 64 == 0 and nk % 64 == 0 and N == nq + 2 * nk):
            raise TypeError("lucid_amd.qkv_rope: bf16 GPU [B, T, (Hq + 2 Hkv) 64] projections")
        hq, hk = nq // 64, nk // 64

        def heads(t, h):
            return t.view(B, T, h, 64).transpose(1, 2)

        c, s = _tokens(cos, B, T), _tokens(sin, B, T)
        q = _rope_launch(heads(qkv[..., :nq], hq), c, s, 0)
        k = _rope_launch(heads(qkv[..., nq:nq + nk], hk), c, s, 0)
        v = heads(qkv[..., nq + nk:], hk)
        ctx.save_for_backward(c, s)
        ctx.dims = (B, T, N, nq, nk)
        return q, k, v

    @staticmethod
    def backward(ctx, dq, dk, dv):
        c, s = ctx.saved_tensors
        B, T, N, nq, nk = ctx.dims
        dev = c.device
        g = torch.empty(B, T, N, dtype=torch.bfloat16, device=dev)

        def heads(t, h):
            return t.view(B, T, h, 64).transpose(1, 2)

        for grad, lo, n in ((dq, 0, nq), (dk, nq, nk)):
            if grad is None:
                g[..., lo:lo + n].zero_()
            else:
                _rope_launch(grad, c, s, 1, out=heads(g[..., lo:lo + n], n // 64))
        if dv is None:
            g[..., nq + nk:].zero_()
        else:
            heads(g[..., nq + nk:], nk // 64).copy_(dv)
        return g, None, None, None, None


def qkv_rope(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nq: int, nk: int):
    """(q, k, v) [B, H, T, 64] from the stacked projection output, q and k rotated
    (apply_rotary_pos_emb, modeling_lucid.py:118-145)."""
    return QKVRopeFunction.apply(qkv, cos, sin, nq, nk)


# Entries of a scaling that its type knows, beside the type and the length trained on
_ROPE_ENTRIES = {"default": (), "linear": ("factor",), "ntk": ("factor",),
                 "llama3": ("factor", "low_freq_factor", "high_freq_factor"),
                 "yarn": ("factor", "beta_fast", "beta_slow", "attention_factor")}


def rope_frequencies(dim: int, theta: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """Inverse frequencies (float64 ``[dim / 2]``, on the CPU) of ``dim`` turning columns, and the factor of the turned
    values: ``theta^(-2 i / dim)`` and 1, or scaled for contexts longer than the model was trained on.

    ``scaling["rope_type"]``: ``"default"``; ``"linear"`` (positions divided by ``factor``); ``"ntk"`` (the base grows to
    theta factor^(dim / (dim - 2)): the slowest frequency is divided by ``factor``, the fastest stays); ``"llama3"``
    (wavelengths below ``original_max_position_embeddings / high_freq_factor`` stay, those above ``... / low_freq_factor`` are
    divided by ``factor``, those between are interpolated over the inverse wavelength); ``"yarn"`` (pairs that turn ``beta_fast`` (32) times
    or more in ``original_max_position_embeddings`` positions stay, those that turn ``beta_slow`` (1) times or less
    are divided by ``factor``, with a ramp over the pair's number between, and values are multiplied by ``attention_factor``,
    0.1 ln(factor) + 1 if it is not given).  An entry that is None is as if it were not there; entries that the type does not know are
    refused (``original_max_position_embeddings`` may go with any)."""
    if dim < 0 or dim % 2:
        raise ValueError(f"lucid_amd.rope_frequencies: an even number of columns, got {dim}")
    i = torch.arange(0, dim, 2, dtype=torch.float64, device="cpu")
    freq = theta ** (-i / max(dim, 1))
    scaling = {} if scaling is None else {name: x for name, x in scaling.items() if x is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _ROPE_ENTRIES:
        raise ValueError(f"lucid_amd.rope_frequencies: rope_type one of {tuple(_ROPE_ENTRIES)}, got {kind!r}")
    if scaling.get("type", kind) != kind:
        raise ValueError(f"lucid_amd.rope_frequencies: rope_type {kind!r} beside type {scaling['type']!r}")
    unknown = sorted(set(scaling) - {"rope_type", "type", "original_max_position_embeddings", *_ROPE_ENTRIES[kind]})
    if unknown:
        raise ValueError(f"lucid_amd.rope_frequencies: {kind} does not know {', '.join(map(repr, unknown))}")
    if kind == "default" or dim == 0:
        return freq, 1.0
    try:
        factor = float(scaling["factor"])
        length = float(scaling["original_max_position_embeddings"]) if kind in ("llama3", "yarn") else 0.0
    except KeyError as e:
        raise ValueError(f"lucid_amd.rope_frequencies: {kind} needs {e.args[0]!r}") from None
    if not factor > 0.0:
        raise ValueError(f"lucid_amd.rope_frequencies: the factor must be positive, got {factor}")
    if kind in ("llama3", "yarn") and not length > 0.0:
        raise ValueError(f"lucid_amd.rope_frequencies: {kind} needs positive original_max_position_embeddings, got {length}")
    if kind == "yarn" and not theta > 1.0:
        raise ValueError(f"lucid_amd.rope_frequencies: yarn needs a theta above 1, got {theta}")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        return (theta * factor ** (dim / max(dim - 2, 1))) ** (-i / dim), 1.0
    if kind == "llama3":
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        turns = length * freq / (2 * math.pi)
        keep = ((turns - low) / max(high - low, 1e-9)).clamp(0.0, 1.0)
        return freq * keep + freq / factor * (1 - keep), 1.0

    def pair(turns):  # the (fractional) number of the pair that turns so often
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))

    first = max(math.floor(pair(float(scaling.get("beta_fast", 32.0)))), 0)
    last = min(math.ceil(pair(float(scaling.get("beta_slow", 1.0)))), dim - 1)
    keep = 1 - ((torch.arange(dim // 2, dtype=torch.float64, device="cpu") - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
    scale = scaling.get("attention_factor")
    scale = (0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0) if scale is None else float(scale)
    return freq * keep + freq / factor * (1 - keep), scale


class RotaryPositions(NamedTuple):
    """What :func:`rotary` takes beside queries and keys (a decoder's layers share one)."""

    positions: torch.Tensor     # int32 or int64 [T], [1, T] or [B, T]
    inv_freq: torch.Tensor      # fp32 or fp64 [part / 2]
    interleaved: bool = False
    scale: float = 1.0


_ROTARY_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


@functools.lru_cache(maxsize=4096)
def _strides(stride: tuple):
    """The first three of a tensor's strides as the C entry points take them (they only read the array)."""
    return (ctypes.c_int64 * 3)(*stride[:3])


def _tracked(*tensors: torch.Tensor) -> bool:
    """Whether a result of these needs an autograd function: a gradient, or a tangent of forward-mode differentiation
    (which the functions refuse)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                return True
    # (the level first: 1 of the 2 us that asking two tensors for a tangent takes)
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _rotary(q, k, positions, inv_freq, interleaved, scale, inverse):
    """q and k (either may be None) turned, into new tensors [B, H, T, d] laid out as [B, T, H, d] (no views, which could not be
    changed in place behind an autograd function)."""
    some = k if q is None else q
    B, _, T, d = some.shape
    dtype, dev = some.dtype, some.device
    qo = ko = None
    qa = ka = (None, None, None, None, 0)
    if q is not None:
        if q.stride(3) != 1 and d > 1:
            q = q.contiguous()
        H = q.shape[1]
        by = (T * H * d, d, H * d, 1)
        qo = torch.empty_strided((B, H, T, d), by, dtype=dtype, device=dev)
        qa = (q.data_ptr(), _strides(q.stride()), qo.data_ptr(), _strides(by), H)
    if k is not None:
        if k.stride(3) != 1 and d > 1:
            k = k.contiguous()
        H = k.shape[1]
        by = (T * H * d, d, H * d, 1)
        ko = torch.empty_strided((B, H, T, d), by, dtype=dtype, device=dev)
        ka = (k.data_ptr(), _strides(k.stride()), ko.data_ptr(), _strides(by), H)
    ps = positions.stride()
    lib = _lib.load()
    with _lib.on(dev):
        rc = lib.lucid_rotary(*qa, *ka, positions.data_ptr(), positions.dtype is torch.int64,
                              0 if len(ps) == 1 or positions.shape[0] == 1 else ps[0], ps[-1], inv_freq.data_ptr(),
                              inv_freq.dtype is torch.float64, B, T, d, 2 * inv_freq.shape[0], scale, interleaved, inverse,
                              _ROTARY_DTYPES[dtype], _lib.stream_handle(dev))
    _lib.check(lib, rc, "lucid_rotary")
    return qo, ko


class RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved: bool, scale: float):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = interleaved, scale
        ctx.set_materialize_grads(False)
        return _rotary(q, k, positions, inv_freq, interleaved, scale, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        if dq is not None or dk is not None:
            dq, dk = _rotary(dq, dk, *ctx.saved_tensors, *ctx.how, True)
        return dq, dk, None, None, None, None


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
           interleaved: bool = False, scale: float = 1.0):
    """``(q, k)`` turned by their positions, in one pass; differentiable.

    ``q [B, Hq, T, d]`` and ``k [B, Hkv, T, d]`` (or None) bf16 or fp32 on the GPU, any strides; ``positions`` int32 or int64 ``[T]``,
    ``[1, T]`` or ``[B, T]``; ``inv_freq`` fp32 or fp64 ``[part / 2]`` (:func:`rope_frequencies`), part at most d.  With x =
    position inv_freq[i], the pair (a, b) number i of a row becomes scale (a cos x - b sin x, b cos x + a sin x): columns i and
    i + part / 2, or 2 i and 2 i + 1 where ``interleaved``; columns from part on stay as they are.  Angles are worked out in
    64 bits (good for positions up to 2^31 and beyond), values in 32, rounded once.  Results are ``[B, H, T, d]``, laid out
    as ``[B, T, H, d]`` as the projections leave them."""
    what = "lucid_amd.rotary"
    if not q.is_cuda:
        raise RuntimeError("lucid_amd: query must be a GPU tensor (no CPU path)")
    dev = q.device
    if q.dtype not in _ROTARY_DTYPES or (k is not None and (k.dtype != q.dtype or k.device != dev)):
        raise TypeError(f"{what}: bf16 or fp32 queries and keys of one dtype on one GPU, got {q.dtype}"
                        + (f" / {k.dtype} on {k.device}" if k is not None else ""))
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:])):
        raise ValueError(f"{what}: q [B, Hq, T, d] and k [B, Hkv, T, d], got {tuple(q.shape)}"
                         + (f" and {tuple(k.shape)}" if k is not None else ""))
    B, _, T, d = q.shape
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != dev \
            or tuple(positions.shape) not in ((T,), (1, T), (B, T)):
        raise ValueError(f"{what}: positions int32 or int64 [{T}] or [{B}, {T}] on {dev}, got {positions.dtype} "
                         f"{tuple(positions.shape)} on {positions.device}")
    if inv_freq.dtype not in (torch.float32, torch.float64) or inv_freq.dim() != 1 or inv_freq.device != dev \
            or 2 * inv_freq.numel() > d or not inv_freq.is_contiguous():
        raise ValueError(f"{what}: inv_freq contiguous fp32 or fp64 of at most {d // 2} on {dev}, got {inv_freq.dtype} "
                         f"{tuple(inv_freq.shape)} on {inv_freq.device}")
    if inv_freq.requires_grad:
        raise NotImplementedError(f"{what}: no gradient of the frequencies")
    if _tracked(q) or (k is not None and _tracked(k)):
        return RotaryFunction.apply(q, k, positions, inv_freq, bool(interleaved), float(scale))
    return _rotary(q, k, positions, inv_freq, bool(interleaved), float(scale), False)


def swiglu_supported(g: torch.Tensor, u: torch.Tensor) -> bool:
    return g.is_cuda and g.dtype == torch.bfloat16 and u.dtype == torch.bfloat16 and g.shape == u.shape


class SwiGLUFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g: torch.Tensor, u: torch.Tensor):
        if not swiglu_supported(g, u):
            raise TypeError(f"lucid_amd.swiglu: bf16 GPU gate and up of one shape, got {g.dtype} {tuple(g.shape)} / "
                            f"{u.dtype} {tuple(u.shape)}")
        g2, u2 = _aligned(g), _aligned(u)
        h = torch.empty_like(g2)
        lib = _lib.load()
        rc = lib.lucid_swiglu_fwd(_lib.ptr(g2), _lib.ptr(u2), _lib.ptr(h), g2.numel(), _lib.stream_handle(g.device))
        _lib.check(lib, rc, "lucid_swiglu_fwd")
        ctx.save_for_backward(g2, u2)
        return h

    @staticmethod
    def backward(ctx, dh: torch.Tensor):
        g2, u2 = ctx.saved_tensors
        dh2 = _aligned(dh)
        dg, du = torch.empty_like(g2), torch.empty_like(u2)
        lib = _lib.load()
        rc = lib.lucid_swiglu_bwd(_lib.ptr(g2), _lib.ptr(u2), _lib.ptr(dh2), _lib.ptr(dg), _lib.ptr(du), g2.numel(),
                                  _lib.stream_handle(g2.device))
        _lib.check(lib, rc, "lucid_swiglu_bwd")
        return dg, du


def swiglu(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    """silu(g) * u (the gated activation of ``LlamaMLP.forward``, modeling_lucid.py:155-167)."""
    return SwiGLUFunction.apply(g, u)


IGNORE_INDEX = -100


def causal_lm_loss_supported(logits: torch.Tensor, labels: torch.Tensor) -> bool:
    return (logits.is_cuda and logits.dtype == torch.bfloat16 and logits.dim() == 3 and logits.shape[-1] % 8 == 0
            and labels.shape == logits.shape[:2] and labels.dtype == torch.int64)


class CausalLMLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: torch.Tensor, labels: torch.Tensor):
        if not causal_lm_loss_supported(logits, labels):
            raise TypeError("lucid_amd.causal_lm_loss: bf16 GPU logits [B, T, V] (V a multiple of 8) and int64 "
                            f"labels [B, T], got {logits.dtype} {tuple(logits.shape)} / {labels.dtype}")
        B, T, V = logits.shape
        lg = _aligned(logits.reshape(B * T, V))
        lb = labels.reshape(-1).contiguous()
        R = B * T
        lse, per_row, valid = (torch.empty(R, dtype=torch.float32, device=logits.device) for _ in range(3))
        lib = _lib.load()
        rc = lib.lucid_causal_lm_loss_fwd(_lib.ptr(lg), V, _lib.ptr(lb), R, T, V, _lib.ptr(lse), _lib.ptr(per_row),
                                          _lib.ptr(valid), _lib.stream_handle(logits.device))
        _lib.check(lib, rc, "lucid_causal_lm_loss_fwd")
        count = valid.sum()
        ctx.save_for_backward(lg, lb, lse, valid, count)
        ctx.dims = (B, T, V)
        return per_row.sum() / count

    @staticmethod
    def backward(ctx, dloss: torch.Tensor):
        lg, lb, lse, valid, count = ctx.saved_tensors
        B, T, V = ctx.dims
        scale = (dloss.float() / count).reshape(1).contiguous()
        dlogits = torch.empty(B * T, V, dtype=torch.bfloat16, device=lg.device)
        lib = _lib.load()
        rc = lib.lucid_causal_lm_loss_bwd(_lib.ptr(lg), V, _lib.ptr(lb), B * T, T, V, _lib.ptr(lse), _lib.ptr(valid),
                                          _lib.ptr(scale), _lib.ptr(dlogits), _lib.stream_handle(lg.device))
        _lib.check(lib, rc, "lucid_causal_lm_loss_bwd")
        return dlogits.view(B, T, V), None


def causal_lm_loss(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Mean cross entropy of logits[:, :-1] against labels[:, 1:] with -100 ignored, computed in
    fp32 (``LlamaForCausalLM.forward``'s loss, modeling_lucid.py:847-967); a float32 scalar."""
    return CausalLMLossFunction.apply(logits, labels)


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` gives for logits ``[..., V]`` (fp32, indices int64)."""

    logprobs: torch.Tensor       # [...] log probability of the given token
    entropy: torch.Tensor        # [...] of the row's distribution
    top_logprobs: torch.Tensor   # [..., top] log probabilities of the most likely tokens
    top_indices: torch.Tensor    # [..., top] those tokens


_LP_DTYPES = {torch.bfloat16: 0, torch.float32: 1}
MAX_TOP = 64


def _logit_rows(logits: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """``logits`` as the kernels read them, with rows per batch entry and the two strides: [R, V] and
    [B, T, V] views with contiguous rows are read as they are, anything else as one run of rows."""
    if logits.stride(-1) == 1 or logits.shape[-1] == 1:
        if logits.dim() == 1:
            return logits, 1, 0, 0
        if logits.dim() == 2:
            return logits, max(logits.shape[0], 1), 0, logits.stride(0)
        if logits.dim() == 3:
            return logits, max(logits.shape[1], 1), logits.stride(0), logits.stride(1)
    rows = logits.reshape(-1, logits.shape[-1])
    rows = rows if rows.stride(1) == 1 or rows.shape[1] == 1 else rows.contiguous()
    return rows, max(rows.shape[0], 1), 0, rows.stride(0)


def _token_logprobs(logits: torch.Tensor, tok: torch.Tensor, top: int, temperature: float, backward: bool):
    """(logprobs, entropy, top_logprobs, top_indices) and, for a backward, the rows' state."""
    shape, V, dev = tok.shape, logits.shape[-1], logits.device
    rows, T, sb, st = _logit_rows(logits)
    R = tok.numel()
    lib = _lib.load()
    f32 = torch.float32
    logprobs = torch.empty_like(tok, dtype=f32)
    entropy = torch.empty_like(logprobs)
    stats = torch.empty((R, 3), dtype=f32, device=dev) if backward else None
    top_lp = torch.empty((*shape, top), dtype=f32, device=dev)
    top_idx = torch.empty((*shape, top), dtype=torch.int64, device=dev)
    nbytes = lib.lucid_token_logprobs_workspace_bytes(R, V, top)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _lib.on(dev):
        rc = lib.lucid_token_logprobs_fwd(
            rows.data_ptr(), sb, st, tok.data_ptr(), R, T, V, _LP_DTYPES[logits.dtype], temperature, top,
            logprobs.data_ptr(), entropy.data_ptr(), None if stats is None else stats.data_ptr(),
            top_lp.data_ptr(), top_idx.data_ptr(), None if ws is None else ws.data_ptr(), _lib.stream_handle(dev))
    _lib.check(lib, rc, "lucid_token_logprobs_fwd")
    return logprobs, entropy, top_lp, top_idx, stats


class TokenLogprobsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: torch.Tensor, tokens: torch.Tensor, top: int, temperature: float):
        tok = tokens.contiguous()
        logprobs, entropy, top_lp, top_idx, stats = _token_logprobs(logits, tok, top, temperature, True)
        ctx.save_for_backward(logits, tok, stats, top_idx)
        ctx.top, ctx.temperature = top, temperature
        ctx.mark_non_differentiable(top_idx)
        ctx.set_materialize_grads(False)
        return logprobs, entropy, top_lp, top_idx

    @staticmethod
    @once_differentiable
    def backward(ctx, dlp, dent, dtop, _didx):
        logits, tok, stats, top_idx = ctx.saved_tensors
        if dlp is None and dent is None and dtop is None:
            return None, None, None, None
        rows, T, sb, st = _logit_rows(logits)
        dlp, dent, dtop = (None if g is None else g.contiguous() for g in (dlp, dent, dtop))
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        lib = _lib.load()
        with _lib.on(logits.device):
            rc = lib.lucid_token_logprobs_bwd(
                rows.data_ptr(), sb, st, tok.data_ptr(), tok.numel(), T, logits.shape[-1], _LP_DTYPES[logits.dtype],
                ctx.temperature, ctx.top, stats.data_ptr(), top_idx.data_ptr(),
                *(None if g is None else g.data_ptr() for g in (dlp, dent, dtop)), dlogits.data_ptr(),
                _lib.stream_handle(logits.device))
        _lib.check(lib, rc, "lucid_token_logprobs_bwd")
        return dlogits, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` under ``softmax(logits / temperature)``, with the rows' entropy and their
    ``top`` most likely tokens (0 .. 64), from one read of the logits; differentiable w.r.t. ``logits`` through all
    three (one more read and one write).

    ``logits [..., V]`` bf16 or fp32 on the GPU, ``tokens [...]`` int64; results in fp32.  A token of -100 (the
    loss's ignore index) has the log probability 0 and no gradient, one outside ``[0, V)`` NaN.  The alternatives are
    ordered by their logits, equal ones by the lower index.  Logits of -inf have probability 0; a row of -inf
    alone, or with a NaN or +inf, gives NaN as torch's log_softmax does; in the gradient too, unless nothing comes
    in for it (an ignored row of a padded batch, say): zeros then.  Forward-mode differentiation is refused
    (NotImplementedError)."""
    if not logits.is_cuda:
        raise RuntimeError("lucid_amd: logits must be a GPU tensor (no CPU path)")
    if logits.dtype not in _LP_DTYPES or tokens.dtype != torch.int64 or tokens.device != logits.device:
        raise TypeError("lucid_amd.token_logprobs: bf16 or fp32 logits and int64 tokens on one GPU, got "
                        f"{logits.dtype} / {tokens.dtype} on {tokens.device}")
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape or logits.shape[-1] < 1:
        raise ValueError(f"lucid_amd.token_logprobs: logits [..., V] and tokens [...], got {tuple(logits.shape)} and "
                         f"{tuple(tokens.shape)}")
    top = operator.index(top)
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"lucid_amd.token_logprobs: top must be in [0, min({MAX_TOP}, V)], got {top}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"lucid_amd.token_logprobs: the temperature must be positive and finite, got {temperature}")
    # (a tangent of forward-mode differentiation takes the autograd function too, which refuses it)
    if logits.requires_grad and torch.is_grad_enabled() or forward_ad.unpack_dual(logits).tangent is not None:
        return TokenLogprobs(*TokenLogprobsFunction.apply(logits, tokens, top, float(temperature)))
    return TokenLogprobs(*_token_logprobs(logits.detach(), tokens.contiguous(), top, float(temperature), False)[:4])


class _Constraints(NamedTuple):
    """Checked arguments of :func:`constrain_logits`: tensors by rows of the logits, or None."""

    history: torch.Tensor | None
    prompt_lens: torch.Tensor | None
    repetition: torch.Tensor | float
    presence: torch.Tensor | float
    frequency: torch.Tensor | float
    bias: torch.Tensor | None
    allowed: torch.Tensor | None


def _rows_at(t: torch.Tensor | None) -> tuple:
    """(address, row stride) of the rows of a constraint; 0 for one row that all share, and no address for none."""
    if t is None or t.shape[1] == 0:
        return None, 0
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else 0


def _number(x) -> tuple:
    return (x.data_ptr(), 1.0) if isinstance(x, torch.Tensor) else (None, x)


def _constrain(logits: torch.Tensor, c: _Constraints) -> torch.Tensor:
    rows, T, sb, st = _logit_rows(logits)
    V, dev = logits.shape[-1], logits.device
    out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    lib = _lib.load()
    with _lib.on(dev):
        rc = lib.lucid_constrain_logits(
            rows.data_ptr(), sb, st, out.numel() // V, T, V, _LP_DTYPES[logits.dtype], *_rows_at(c.history),
            0 if c.history is None else c.history.shape[1], None if c.prompt_lens is None else c.prompt_lens.data_ptr(),
            *_number(c.repetition), *_number(c.presence), *_number(c.frequency), *_rows_at(c.bias), *_rows_at(c.allowed),
            out.data_ptr(), _lib.stream_handle(dev))
    _lib.check(lib, rc, "lucid_constrain_logits")
    return out


class ConstrainLogitsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: torch.Tensor, *constraints):
        c = _Constraints(*constraints)
        number = not isinstance(c.repetition, torch.Tensor)
        # (the gradient depends on the logits through their sign, where a repetition penalty applies, and on nothing else)
        if c.history is None or c.history.shape[1] == 0 or (number and c.repetition == 1.0):
            ctx.repetition = 1.0
            ctx.save_for_backward(None, None, None, c.allowed)
        else:
            ctx.repetition = c.repetition if number else None
            ctx.save_for_backward(logits, c.history, None if number else c.repetition, c.allowed)
        return _constrain(logits, c)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout: torch.Tensor):
        logits, history, repetition, allowed = ctx.saved_tensors
        rows, T, sb, st = (None, 1, 0, 0) if logits is None else _logit_rows(logits)
        V, dev = dout.shape[-1], dout.device
        g = dout.contiguous()
        dlogits = torch.empty(dout.shape, dtype=dout.dtype, device=dev)
        lib = _lib.load()
        with _lib.on(dev):
            rc = lib.lucid_constrain_logits_bwd(
                None if rows is None else rows.data_ptr(), sb, st, dlogits.numel() // V, T, V, _LP_DTYPES[dout.dtype], *_rows_at(history),
                0 if history is None else history.shape[1],
                *_number(ctx.repetition if repetition is None else repetition), *_rows_at(allowed), g.data_ptr(),
                dlogits.data_ptr(), _lib.stream_handle(dev))
        _lib.check(lib, rc, "lucid_constrain_logits_bwd")
        return (dlogits,) + (None,) * len(_Constraints._fields)


def constrain_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                     repetition: torch.Tensor | float = 1.0, presence: torch.Tensor | float = 0.0,
                     frequency: torch.Tensor | float = 0.0, bias: torch.Tensor | None = None,
                     allowed: torch.Tensor | None = None) -> torch.Tensor:
    """Logits under the constraints of a sampling step, in their own shape and dtype, in one pass; differentiable w.r.t.
    ``logits`` (what :func:`token_logprobs` makes of them included).

    ``logits [..., V]`` bf16 or fp32 on the GPU.  ``history [..., N]`` int64: the tokens so far of each row, values outside
    ``[0, V)`` (padding) ignored; its first ``prompt_lens [...]`` (int32) are the prompt.  In this order, in 32 bits, rounded
    once:

    * a token that occurs in the history: x / repetition where x > 0, x repetition where not;
    * one that occurs n > 0 times behind the prompt: x - presence - n frequency;
    * ``bias`` (fp32 ``[V]`` or ``[..., V]``) is added;
    * what ``allowed`` (int32 ``[words]`` or ``[..., words]``, words = ceil(V / 32): bit v % 32 of word v // 32) has no bit for
      becomes -inf, whatever it was (NaN too); its gradient is 0.

    The three penalties are numbers or fp32 tensors ``[...]`` (positive repetition)."""
    what = "lucid_amd.constrain_logits"
    if not logits.is_cuda:
        raise RuntimeError("lucid_amd: logits must be a GPU tensor (no CPU path)")
    if logits.dtype not in _LP_DTYPES:
        raise TypeError(f"{what}: bf16 or fp32 logits, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits [..., V], got {tuple(logits.shape)}")
    lead, V, dev = logits.shape[:-1], logits.shape[-1], logits.device

    def rows(name, t, dtype, last, shared):
        """t [..., last] as [R, last] with contiguous rows ([1, last] for one row that all share)."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != dev:
            raise TypeError(f"{what}: {name} must be a {dtype} tensor on {dev}")
        if t.requires_grad:
            raise NotImplementedError(f"{what}: no gradient of {name}")
        if t.dim() < 1 or (last is not None and t.shape[-1] != last) or not (t.shape[:-1] == lead or (shared and t.dim() == 1)):
            raise ValueError(f"{what}: {name} {tuple(t.shape)} does not fit logits {tuple(logits.shape)}")
        if t.shape[-1] >= 1 << 30:
            raise ValueError(f"{what}: {name} of fewer than 2^30 a row, got {t.shape[-1]}")
        if t.dim() != 2:
            t = t.reshape(1 if t.shape[:-1] != lead else lead.numel(), t.shape[-1])
        return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()

    def number(name, x):
        if not isinstance(x, torch.Tensor):
            return float(x)
        if x.dtype != torch.float32 or x.device != dev or x.shape != lead:
            raise ValueError(f"{what}: {name} must be a number or fp32 {tuple(lead)} on {dev}")
        if x.requires_grad:
            raise NotImplementedError(f"{what}: no gradient of {name}")
        return x.contiguous()

    if prompt_lens is not None:
        if history is None:
            raise ValueError(f"{what}: prompt_lens without a history")
        if not isinstance(prompt_lens, torch.Tensor) or prompt_lens.dtype != torch.int32 or prompt_lens.shape != lead \
                or prompt_lens.device != dev:
            raise ValueError(f"{what}: prompt_lens must be int32 {tuple(lead)} on {dev}")
        prompt_lens = prompt_lens.contiguous()
    c = _Constraints(rows("history", history, torch.int64, None, False), prompt_lens, number("repetition", repetition),
                     number("presence", presence), number("frequency", frequency), rows("bias", bias, torch.float32, V, True),
                     rows("allowed", allowed, torch.int32, -(-V // 32), True))
    if _tracked(logits):
        return ConstrainLogitsFunction.apply(logits, *c)
    return _constrain(logits, c)
