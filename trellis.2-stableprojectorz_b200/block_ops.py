"""Group norm and differential attention over concatenated sequences, with their gradients.

The operators of an attention block over sparse voxels beside
``layernorm_silu`` and ``sparse_attention``: rows (voxels, tokens) of the
sequences of a batch lie one after the other, and ``cu_seqlens`` gives the
``B + 1`` offsets, read on the host.  Both run on torch's current stream, may
be called from any thread and captured into a CUDA graph (pass the offsets as
host values then), and give the same bits on every run.  Errors from the
library surface as ``SparseConvError``.

Both support ``torch.autograd`` (first derivatives in reverse mode; forward
mode is refused).  A backward pass captured
into a graph goes through torch's own rules: use ``torch.autograd.grad``, and
let no eager graph of the same leaves live meanwhile.
"""
from __future__ import annotations

import ctypes
import math
import operator

import torch
from torch.autograd import forward_ad

from . import _lib as L
from .sparse_conv import _DTYPES, get_engine

__all__ = ["sparse_group_norm", "sparse_diff_attention"]


def _offsets(cu, rows, name):
    """``cu`` as a ctypes int32 array; it must end at ``rows``."""
    if not isinstance(cu, (list, tuple)):
        if isinstance(cu, torch.Tensor) and (cu.dim() != 1 or cu.is_floating_point() or cu.dtype == torch.bool):
            raise ValueError(f"{name} must be 1-D whole numbers")
        cu = cu.tolist() if hasattr(cu, "tolist") else list(cu)
    cu = list(map(operator.index, cu))
    if len(cu) < 2:
        raise ValueError(f"{name} must be 1-D with batch + 1 entries")
    if cu[-1] != rows:
        raise ValueError(f"{name} must end at the row count {rows}")
    if cu[0] != 0 or any(a > b for a, b in zip(cu, cu[1:])):
        raise ValueError(f"{name} must start at 0 and be non-decreasing")
    if rows > 0x7FFFFFFF:
        raise ValueError(f"{name} must be 32-bit offsets")
    return (ctypes.c_int32 * len(cu))(*cu)


def _same_device(x, *others):
    for t in others:
        if t is not None and t.device != x.device:
            raise ValueError(f"tensors on {x.device} and on {t.device}")


def _p(t):
    return None if t is None else t.data_ptr()


def _dense(t):
    """An uninitialised dense tensor like ``t``."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _wants_grad(*inputs):
    """Whether autograd takes part: an input requires grad, or is dual.  A dual one goes to the autograd function too,
    which has no forward-mode rule, so that torch says so instead of dropping the tangent."""
    tensors = [t for t in inputs if isinstance(t, torch.Tensor)]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _overlap(a, b):
    """Whether the bytes of two tensors' extents meet."""
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False

    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in
                                                                       zip(t.shape, t.stride())))
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _check_out(out, shape, like):
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device or \
            not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {tuple(shape)} {like.dtype} tensor on {like.device}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out= takes no part in autograd: out requires grad")


def _written(out):
    """``out`` after the library wrote it: autograd refuses a backward pass that saved what it held before."""
    torch.autograd.graph.increment_version(out)
    return out


def _rows_view(x):
    """``x`` (N, C) with dense channels: itself where only its rows are apart, else a copy."""
    n, c = x.shape
    if n <= 1:
        return x.contiguous(), c
    if (x.stride(1) == 1 or c == 1) and x.stride(0) >= c:
        return x, x.stride(0)
    return x.contiguous(), c


# ------------------------------------------------------------------ group norm
def _dense_vectors(*vectors):
    """The library reads ``(C,)`` consecutive values: strided and expanded vectors are copied."""
    return tuple(None if t is None else t.contiguous() for t in vectors)


def _gn_forward(x, groups, weight, bias, eps, cu, silu, out, want_stats):
    x, stride = _rows_view(x)
    weight, bias = _dense_vectors(weight, bias)
    wd = _DTYPES[(weight if weight is not None else bias if bias is not None else x).dtype]
    y = _dense(x) if out is None else out
    stats = torch.empty((len(cu) - 1, groups, 2), dtype=torch.float32, device=x.device) if want_stats else None
    get_engine(x.device).call("sc_group_norm", _p(x), stride, _p(weight), _p(bias), _p(y), _p(stats), cu, len(cu) - 1,
                              x.shape[1], groups, eps, int(silu), _DTYPES[x.dtype], wd)
    return y, stats


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, cu, silu):
        y, stats = _gn_forward(x, groups, weight, bias, eps, cu, silu, None, True)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.args = (groups, cu, silu)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        groups, cu, silu = ctx.args
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        x, stride = _rows_view(x)
        dy = dy.contiguous()
        dx = _dense(x) if need_x else None
        dw = _dense(weight) if need_w else None
        db = _dense(bias) if need_b else None
        wd = _DTYPES[(weight if weight is not None else bias if bias is not None else x).dtype]
        weight, bias = _dense_vectors(weight, bias)
        get_engine(x.device).call("sc_group_norm_backward", _p(x), stride, _p(dy), _p(weight), _p(bias), _p(stats),
                                  _p(dx), _p(dw), _p(db), cu, len(cu) - 1, x.shape[1], groups, int(silu),
                                  _DTYPES[x.dtype], wd)
        return dx, dw, db, None, None, None, None


def sparse_group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, cu_seqlens=None, silu=False, out=None):
    """Group norm of sparse rows, channels last, per sequence (``sc_group_norm``).

    ``x`` ``(N, C)`` (f32, bf16 or f16, CUDA; rows may be apart, as in a slice
    of wider rows).  Each of the ``num_groups`` groups of ``C / num_groups``
    channels is normalised with the mean and biased variance of one sequence's
    rows, as ``torch.nn.GroupNorm`` does for a batch item; then ``* weight +
    bias`` (``(C,)``, in x's dtype or f32, both the same; either may be None),
    then SiLU with ``silu=True``.  ``cu_seqlens`` defaults to one sequence of
    all rows.  Statistics and sums are f32.  Returns ``(N, C)`` in x's dtype.

    Differentiable in x, weight and bias.  ``out`` receives the result without
    autograd; it may be a contiguous ``x`` itself (in place)."""
    if x.dtype not in _DTYPES:
        raise TypeError(f"unsupported feature dtype {x.dtype}")
    if x.dim() != 2:
        raise ValueError("x must be (N, C)")
    n, c = x.shape
    groups = operator.index(num_groups)
    if groups < 1 or c < 1 or c % groups != 0:
        raise ValueError(f"{c} channels do not split into {num_groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (c,):
            raise ValueError(f"{name} must be ({c},)")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be {x.dtype} or float32")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one dtype")
    _same_device(x, weight, bias)
    eps = float(eps)
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError("eps must be positive and finite")
    cu = _offsets([0, n] if cu_seqlens is None else cu_seqlens, n, "cu_seqlens")
    if not x.is_cuda:
        raise ValueError("sparse_group_norm runs on CUDA tensors only")
    if _wants_grad(x, weight, bias):
        if out is not None:
            raise ValueError("out= takes no part in autograd: use it under torch.no_grad()")
        return _GroupNorm.apply(x, weight, bias, groups, eps, cu, bool(silu))
    if out is not None:
        _check_out(out, (n, c), x)
        same = out.data_ptr() == x.data_ptr() and x.is_contiguous()
        if (_overlap(out, x) and not same) or _overlap(out, weight) or _overlap(out, bias):
            raise ValueError("out overlaps an input (only a contiguous x itself may be written in place)")
    y, _ = _gn_forward(x, groups, weight, bias, eps, cu, silu, out, False)
    return y if out is None else _written(out)


# ------------------------------------------------------ differential attention
def _tokens(t):
    """``t`` (N, heads, D) with dense tokens 16-byte apart: itself, or a copy."""
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    if s2 == 1 and (h == 1 or s1 == d) and t.data_ptr() % 16 == 0:
        if n <= 1:
            return t, h * d
        if s0 >= h * d and s0 % 8 == 0:
            return t, s0
    t = t.contiguous()
    return (t if t.data_ptr() % 16 == 0 else t.clone()), h * d


def _da_args(q, k, v, lam, cu_q, cu_kv, scale, causal, out=None, lse=None, maps=None, dout=None,
             grads=(None, None, None, None)):
    (q, qs), (k, ks), (v, vs) = _tokens(q), _tokens(k), _tokens(v)
    dt, ldt, count, value = _DTYPES[q.dtype], L.SC_F32, 0, 0.0
    if isinstance(lam, torch.Tensor):
        lam = lam.contiguous()
        ldt, count, at = _DTYPES[lam.dtype], lam.numel(), lam.data_ptr()
    else:
        value, at = lam, None
    a = L.ScDiffAttentionArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), at, qs, ks, vs, ctypes.addressof(cu_q),
                              ctypes.addressof(cu_kv), len(cu_q) - 1, q.shape[1] // 2, v.shape[1], count, value, scale,
                              causal, dt, ldt, _p(out), _p(lse), _p(maps), _p(dout), *map(_p, grads))
    return a, (q, k, v, lam)  # the tensors the addresses belong to


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, cu_q, cu_kv, scale, causal):
        nq, heads = q.shape[0], q.shape[1] // 2
        out = torch.empty((nq, heads, 128), dtype=q.dtype, device=q.device)
        maps = torch.empty((nq, heads, 2, 128), dtype=torch.float32, device=q.device)
        lse = torch.empty((2, heads, nq), dtype=torch.float32, device=q.device)
        a, hold = _da_args(q, k, v, lam, cu_q, cu_kv, scale, causal, out=out, lse=lse, maps=maps)
        get_engine(q.device).call("sc_diff_attention", ctypes.byref(a))
        ctx.save_for_backward(q, k, v, lam if isinstance(lam, torch.Tensor) else None, maps, lse)
        ctx.args = (None if isinstance(lam, torch.Tensor) else lam, cu_q, cu_kv, scale, causal)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, lam, maps, lse = ctx.saved_tensors
        value, cu_q, cu_kv, scale, causal = ctx.args
        dense = [_dense(t) if need else None for t, need in zip((q, k, v, lam), ctx.needs_input_grad)]
        dout = dout.contiguous()
        dout = dout if dout.data_ptr() % 16 == 0 else dout.clone()
        a, hold = _da_args(q, k, v, value if lam is None else lam, cu_q, cu_kv, scale, causal, lse=lse,
                           maps=maps, dout=dout, grads=dense)
        get_engine(q.device).call("sc_diff_attention_backward", ctypes.byref(a))
        return (*dense, None, None, None, None)


def sparse_diff_attention(q, k, v, lam, cu_seqlens_q, cu_seqlens_kv=None, scale=None, causal=False, out=None):
    """Variable-length differential attention (``sc_diff_attention``): the
    difference of two softmax maps over one set of values.

    ``q`` ``(total_N, 2 H, 64)``: head h's two maps are rows ``2h`` and
    ``2h + 1``; ``k`` ``(total_N_kv, 2 H_kv, 64)`` and ``v`` ``(total_N_kv,
    H_kv, 128)`` likewise, with H a multiple of H_kv (head h reads key / value
    head ``h // (H / H_kv)``); bf16 or f16, CUDA; tokens may be apart, as in a
    slice of a fused projection.  ``lam`` is a number or a tensor of one or H
    values (f32 or q's dtype).  Per sequence::

        out[i, h] = softmax_j(scale q[i, 2h] . k[j, 2g]) v[j, g]
                    - lam_h softmax_j(scale q[i, 2h+1] . k[j, 2g+1]) v[j, g]

    ``cu_seqlens_q`` / ``cu_seqlens_kv`` as in ``sparse_attention`` (the latter
    defaults to the former); ``scale`` (2^-20 to 2^20) defaults to ``1 / sqrt(64)``.  With
    ``causal`` query i of a sequence sees the keys ``j <= i + len_kv - len_q``
    (a single new token sees the whole cache).  Rows that see no key are zero.
    A NaN or an infinity stays inside its sequence and makes the rows that see
    it non-finite as softmax does; it may reach rows that ``causal`` hides it
    from too (0 * NaN), as in any product with the weights.  Sums and softmax
    statistics are f32; weights and score gradients are rounded to q's dtype
    for the products.  Returns ``(total_N, H, 128)``.

    Differentiable in q, k, v and lam (f16: rows whose log-sum-exp over
    ``scale`` is beyond 6.7e7 get NaN gradients).  ``out`` receives the result without
    autograd and may not overlap an input."""
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("sparse_diff_attention takes bf16 or f16 tensors")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must have one dtype")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or q.shape[2] != 64 or k.shape[2] != 64 or v.shape[2] != 128:
        raise ValueError("q must be (N, 2H, 64), k (N_kv, 2H_kv, 64) and v (N_kv, H_kv, 128)")
    heads, kv_heads = q.shape[1] // 2, v.shape[1]
    if heads < 1 or q.shape[1] % 2 or k.shape[1] != 2 * kv_heads or k.shape[0] != v.shape[0] or kv_heads < 1 or \
            heads % kv_heads:
        raise ValueError("q must have 2H heads, k 2H_kv and v H_kv over the same rows, H a multiple of H_kv")
    if isinstance(lam, torch.Tensor):
        if lam.numel() not in (1, heads) or lam.dim() > 1:
            raise ValueError(f"lam must hold 1 or {heads} values")
        if lam.dtype not in (q.dtype, torch.float32):
            raise TypeError(f"lam must be {q.dtype} or float32")
        _same_device(q, lam)
    else:
        lam = float(lam)
    _same_device(q, k, v)
    cu_q = _offsets(cu_seqlens_q, q.shape[0], "cu_seqlens_q")
    if cu_seqlens_kv is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError("k and v have other rows than q: pass cu_seqlens_kv")
        cu_kv = cu_q
    else:
        cu_kv = _offsets(cu_seqlens_kv, k.shape[0], "cu_seqlens_kv")
    if len(cu_q) != len(cu_kv):
        raise ValueError("cu_seqlens_q and cu_seqlens_kv must have the same count")
    scale = 0.125 if scale is None else float(scale)
    if not 2.0 ** -20 <= scale <= 2.0 ** 20:
        raise ValueError("scale must lie in [2^-20, 2^20]")
    if not q.is_cuda:
        raise ValueError("sparse_diff_attention runs on CUDA tensors only")
    leaves = [t for t in (q, k, v, lam) if isinstance(t, torch.Tensor)]
    if _wants_grad(*leaves):
        if out is not None:
            raise ValueError("out= takes no part in autograd: use it under torch.no_grad()")
        return _DiffAttention.apply(q, k, v, lam, cu_q, cu_kv, scale, bool(causal))
    given = out is not None
    if not given:
        out = torch.empty((q.shape[0], heads, 128), dtype=q.dtype, device=q.device)
    else:
        _check_out(out, (q.shape[0], heads, 128), q)
        if out.data_ptr() % 16 or any(_overlap(out, t) for t in leaves):
            raise ValueError("out must be 16-byte aligned and overlap no input")
    a, hold = _da_args(q, k, v, lam, cu_q, cu_kv, scale, causal, out=out)
    get_engine(q.device).call("sc_diff_attention", ctypes.byref(a))
    return _written(out) if given else out
