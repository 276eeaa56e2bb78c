"""Operators of an encoder block over longer token rows than the reference's: attention in a sliding window whose first keys stay visible, and the norms
before and after a block with its gate and the residual scale (csrc/wattn.hip, csrc/gnorm.hip; include/dic_hip.h states the formulas).

As everywhere in this package there is no autograd: each forward call has a call that computes its gradients, and a tensor that asks for a gradient is refused.
Calls run on the current stream of the tensors' device, allocate what they return and their workspaces from torch's allocator, never synchronise, and can
be captured into a graph.  Errors of the arguments raise ValueError or TypeError before anything is launched."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DIC_F32, torch.bfloat16: _lib.DIC_BF16}
_RES_F32 = 0x200
_KINDS = {"none": 0, "layer": 1, "rms": 2}
_INT = 2 ** 31 - 1


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(cond, what):
    if not cond:
        raise ValueError(what)


def _on(t, like, name, dtypes, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {t.dtype} where {' or '.join(map(str, dtypes))} is needed")
    _need(t.device == like.device, f"{name} is on {t.device}, not on {like.device}")
    _need(shape is None or tuple(t.shape) == tuple(shape), f"{name} has shape {tuple(t.shape)}, not {shape and tuple(shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} asks for a gradient: this package has no autograd, call the operator's _grad function on detached tensors")
    return t


def _launch(fn, code, params, device, what):
    """One C call on the current stream of `device`."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _lib.check(fn(code, C.byref(params), torch.cuda.current_stream().cuda_stream), what)
    _lib.check(fn(code, C.byref(params), torch.cuda.current_stream().cuda_stream), what)


# ------------------------------------------------------------------------------------------------ attention
def _bound(x, name):
    if x is None:
        return -1
    x = int(x)
    _need(x >= 0, f"{name} must be None (no bound) or at least 0")
    return min(x, _INT)


def _attention(q, k, v, left, right, sinks, key_mask, kv_len, q_pos, scale, *rest):
    """The checked arguments as a parameter struct (outputs and what the backward pass adds are filled in by the caller)."""
    _lib.require_gpu()
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be a tensor [N, Tq, H, dh]")
    _need(q.is_cuda, "q must be on the GPU")
    types = (q.dtype,)
    if q.dtype not in _DTYPES:
        raise TypeError(f"q: {q.dtype} where float32 or bfloat16 is needed")
    N, Tq, H, dh = q.shape
    _on(q, q, "q", types)
    _on(k, q, "k", types)
    _need(k.dim() == 4 and k.shape[0] == N and k.shape[3] == dh, f"k has shape {tuple(k.shape)}, not [{N}, Tk, Hkv, {dh}]")
    Tk, Hkv = k.shape[1], k.shape[2]
    _on(v, q, "v", types, k.shape)
    _need(dh in (64, 128), "the head dimension must be 64 or 128")
    _need(Hkv > 0 and H % Hkv == 0 and H > 0, f"{H} query heads are no multiple of {Hkv} key heads")
    if key_mask is not None:
        _on(key_mask, q, "key_mask", (torch.bool, torch.uint8), (N, Tk))
        _need(key_mask.is_contiguous(), "key_mask must be contiguous")
    for t, name in ((kv_len, "kv_len"), (q_pos, "q_pos")):
        if t is not None:
            _on(t, q, name, (torch.int32,), (N,))
            _need(t.is_contiguous(), f"{name} must be contiguous")
    p = _lib.WinAttnParams(q.data_ptr(), k.data_ptr(), v.data_ptr())
    _strides(p, q=q, k=k, v=v)
    p.key_mask, p.kv_len, p.q_pos = _ptr(key_mask), _ptr(kv_len), _ptr(q_pos)
    p.N, p.Tq, p.Tk, p.H, p.Hkv, p.dh = N, Tq, Tk, H, Hkv, dh
    p.left, p.right, p.sinks = _bound(left, "left"), _bound(right, "right"), _bound(sinks, "sinks") if sinks is not None else 0
    p.scale = dh ** -0.5 if scale is None else float(scale)
    _need(0.0 < p.scale < float("inf"), "scale must be positive and finite")
    return p, _DTYPES[q.dtype]


def _strides(p, **tensors):
    for name, t in tensors.items():
        n, tk, h, d = t.stride()
        _need(d == 1 or t.shape[3] == 1, f"the rows of {name} must be contiguous")
        per = 16 // t.element_size()
        _need(t.numel() == 0 or not (t.data_ptr() % 16 or n % per and t.shape[0] > 1 or tk % per and t.shape[1] > 1 or h % per and t.shape[2] > 1),
              f"the rows of {name} must start at multiples of 16 bytes")
        # (the stride of a dimension of size 0 or 1 is arbitrary and unused)
        setattr(p, name + "_stride_n", n if t.shape[0] > 1 else 0)
        setattr(p, name + "_stride_t", tk if t.shape[1] > 1 else 0)
        setattr(p, name + "_stride_h", h if t.shape[2] > 1 else 0)


def window_attention(q, k, v, *, left=None, right=None, sinks=0, key_mask=None, kv_len=None, q_pos=None, scale=None, out=None):
    """softmax(scale q k^T) v over the keys each query row sees; returns (out like q, lse [N, H, Tq] fp32).

    q [N, Tq, H, dh]; k, v [N, Tk, Hkv, dh]: float32 or bfloat16, dh 64 or 128, any strides with contiguous 16-byte-aligned rows (views of a packed q|k|v
    tensor or of a longer cache); H a multiple of Hkv.  Row i of sequence n stands at position t = i + q_pos[n] (int32 [N]; 0 without).  It sees key j when
    j < kv_len[n] (int32 [N]; Tk without), key_mask[n, j] is true (bool or uint8 [N, Tk]), j <= t + right, and j >= t - left or j < sinks; left / right None:
    no bound.  A row that sees nothing gives zeros and lse = -inf.  `out`: write there instead of into a new tensor.

    One new token behind a cache: Tq = 1, kv_len = the cache's lengths with the new key in place, q_pos = kv_len - 1, right = 0."""
    p, code = _attention(q, k, v, left, right, sinks, key_mask, kv_len, q_pos, scale)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _on(out, q, "out", (q.dtype,), q.shape)
    lse = torch.empty((p.N, p.H, p.Tq), dtype=torch.float32, device=q.device)
    _strides(p, out=out)
    p.out, p.lse = out.data_ptr(), lse.data_ptr()
    L = _lib.lib()
    ws = _workspace(p, L.dic_win_attn_ws_bytes(code, 0, C.byref(p)), q.device)  # noqa: F841  (keeps the memory until the launch is queued)
    _launch(L.dic_win_attn_fwd, code, p, q.device, "window_attention")
    return out, lse


def window_attention_grad(dout, q, k, v, out, lse, *, left=None, right=None, sinks=0, key_mask=None, kv_len=None, q_pos=None, scale=None, grads=None):
    """(dq, dk, dv) of window_attention for the gradient `dout` of its output; the other arguments as they went into and came out of that call.
    `grads`: three tensors to write them into (views of a packed gradient, say).  dk and dv are summed over the query heads of each key head."""
    p, code = _attention(q, k, v, left, right, sinks, key_mask, kv_len, q_pos, scale)
    _on(dout, q, "dout", (q.dtype,), q.shape)
    _on(out, q, "out", (q.dtype,), q.shape)
    _on(lse, q, "lse", (torch.float32,), (p.N, p.H, p.Tq))
    _need(lse.is_contiguous(), "lse must be contiguous")
    if dout.stride(3) != 1 or any(s % (16 // dout.element_size()) for s in dout.stride()[:3]) or dout.data_ptr() % 16:
        dout = dout.contiguous()                 # an expanded or transposed gradient
    if grads is None:
        grads = [torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v)]
    else:
        for t, like, name in zip(grads, (q, k, v), ("dq", "dk", "dv")):
            _on(t, q, name, (q.dtype,), like.shape)
    dq, dk, dv = grads
    _strides(p, out=out, dout=dout, dq=dq, dk=dk, dv=dv)
    p.out, p.lse, p.dout, p.dq, p.dk, p.dv = out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    L = _lib.lib()
    ws = _workspace(p, L.dic_win_attn_ws_bytes(code, 1, C.byref(p)), q.device)  # noqa: F841
    _launch(L.dic_win_attn_bwd, code, p, q.device, "window_attention_grad")
    return dq, dk, dv


def _workspace(p, size, device):
    if not size:
        return None
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    p.ws, p.ws_bytes = ws.data_ptr(), size
    return ws


# ------------------------------------------------------------------------------------------------ norms
class NormParams(NamedTuple):
    """A norm over the last dimension: kind "layer" or "rms", weight and bias [D] float32 (None: 1 and 0)."""
    kind: str = "layer"
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-12


def _norms(x, like, post, pre, gate, residual_scale):
    """(params, rows): the checked part that forward and backward share; `like` gives rows and device."""
    D = like.shape[-1] if like.dim() else 0
    _need(like.dim() >= 2 and 1 <= D <= 8192, "rows of 1 to 8192 elements in at least two dimensions are needed")
    rows = like.numel() // D
    p = _lib.GatedNormParams()
    p.rows, p.rows_per_gate, p.D, p.residual_scale = rows, max(rows, 1), D, float(residual_scale)
    for norm, side in ((post, "post"), (pre, "pre")):
        if norm is None:
            continue
        _need(norm.kind in ("layer", "rms"), f"{side}: a norm is \"layer\" or \"rms\"")
        for t, name in ((norm.weight, "weight"), (norm.bias, "bias")):
            if t is not None:
                _on(t, like, f"{side} {name}", (torch.float32,), (D,))
                _need(t.is_contiguous(), f"{side} {name} must be contiguous")
                setattr(p, f"{side}_{name}", t.data_ptr())
        setattr(p, side + "_kind", _KINDS[norm.kind])
        setattr(p, side + "_eps", float(norm.eps))
    if gate is not None:
        _on(gate, like, "gate", (torch.float32,))
        _need(gate.is_contiguous() and gate.dim() in (1, 2) and gate.shape[-1] == D, f"gate must be contiguous, [{D}] or [sequences, {D}]")
        n = 1 if gate.dim() == 1 else gate.shape[0]
        _need(rows == 0 or (n > 0 and rows % n == 0), f"{rows} rows do not divide over {n} gates")
        p.gate, p.rows_per_gate = gate.data_ptr(), max(rows // max(n, 1), 1)
    return p


def _rows(t, like, name, dtypes, shape):
    _on(t, like, name, dtypes, shape)
    _need(t.is_contiguous(), f"{name} must be contiguous")
    return t


def _norm_code(stream, inner):
    if stream not in _DTYPES or inner not in _DTYPES or (stream, inner) == (torch.bfloat16, torch.float32):
        raise TypeError(f"a {stream} residual stream with {inner} blocks: float32 with float32 or bfloat16, or bfloat16 with bfloat16")
    return _DTYPES[inner] | (_RES_F32 if stream != inner else 0)


def gated_norm(x, y=None, *, post=None, gate=None, residual_scale=1.0, pre=None, dtype=None):
    """x_new = residual_scale x + gate * post(y) and a = pre(x_new), the next block's input, in one pass; returns (x_new, a, saved).

    y [..., D] is a block's output, x the residual stream in front of the block (x may be float32 beside a bfloat16 y).  post, pre: NormParams or None (no
    norm; without pre, a is None).  gate: float32 [D], [N, D] (one row for each of N equal runs of rows: the sequences of [N, T, D]), or None.  `saved`
    [4, rows] holds the rows' statistics for gated_norm_grad.  Without y it is a stack's first norm: a = pre(residual_scale x), of type `dtype` (x's)."""
    _lib.require_gpu()
    _need(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a tensor on the GPU")
    inner = y.dtype if isinstance(y, torch.Tensor) else (dtype or x.dtype)
    _need(y is None or dtype in (None, inner), "dtype is the type of a without y")
    code = _norm_code(x.dtype, inner)
    _rows(x, x, "x", (x.dtype,), x.shape)
    if y is not None:
        _rows(y, x, "y", (inner,), x.shape)
    else:
        _need(post is None and gate is None and pre is not None, "without y there is a pre norm and nothing else")
    p = _norms(x, x, post, pre, gate, residual_scale)
    x_new = x if y is None and residual_scale == 1.0 else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = torch.empty(x.shape, dtype=inner, device=x.device) if pre is not None else None
    saved = torch.empty((4, p.rows), dtype=torch.float32, device=x.device)
    p.x, p.y, p.a, p.saved = x.data_ptr(), _ptr(y), _ptr(a), saved.data_ptr()
    p.x_new = None if x_new is x else x_new.data_ptr()
    _launch(_lib.lib().dic_gated_norm_fwd, code, p, x.device, "gated_norm")
    return x_new, a, saved


def gated_norm_grad(dx_new, da, x_new, y, saved, *, post=None, gate=None, residual_scale=1.0, pre=None):
    """Gradients of gated_norm as a dict: "dx", "dy", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias", as far as there are such inputs.
    dx_new (None: zero) and da (None without pre) are the gradients of its outputs; x_new, y and saved as they went into and came out of that call."""
    _lib.require_gpu()
    _need(isinstance(x_new, torch.Tensor) and x_new.is_cuda, "x_new must be a tensor on the GPU")
    given = y if y is not None else da
    inner = given.dtype if isinstance(given, torch.Tensor) else x_new.dtype
    code = _norm_code(x_new.dtype, inner)
    _rows(x_new, x_new, "x_new", (x_new.dtype,), x_new.shape)
    _need((da is None) == (pre is None), "da is the gradient of pre's output: both or neither")
    if dx_new is not None:
        _rows(dx_new, x_new, "dx_new", (x_new.dtype,), x_new.shape)
    if da is not None:
        _rows(da, x_new, "da", (inner,), x_new.shape)
    if y is not None:
        _rows(y, x_new, "y", (inner,), x_new.shape)
    else:
        _need(post is None and gate is None and pre is not None, "without y there is a pre norm and nothing else")
    _need(dx_new is not None or da is not None, "neither output has a gradient")
    p = _norms(x_new, x_new, post, pre, gate, residual_scale)
    _rows(saved, x_new, "saved", (torch.float32,), (4, p.rows))
    new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
    got = {"dx": new(x_new)}
    if y is not None:
        got["dy"] = new(y)
    if gate is not None:
        got["gate"] = new(gate) if p.rows else torch.zeros_like(gate)
    for norm, side in ((post, "post"), (pre, "pre")):
        for name in ("weight", "bias"):
            t = getattr(norm, name) if norm is not None else None
            if t is not None:
                got[f"{side}_{name}"] = new(t)
    p.x_new, p.y, p.saved, p.dx_new, p.da = x_new.data_ptr(), _ptr(y), saved.data_ptr(), _ptr(dx_new), _ptr(da)
    p.dx, p.dy, p.dgate = _ptr(got["dx"]), _ptr(got.get("dy")), _ptr(got.get("gate"))
    p.dpost_w, p.dpost_b, p.dpre_w, p.dpre_b = (_ptr(got.get(k)) for k in ("post_weight", "post_bias", "pre_weight", "pre_bias"))
    L = _lib.lib()
    ws = _workspace(p, L.dic_gated_norm_ws_bytes(code, C.byref(p)), x_new.device)  # noqa: F841
    _launch(L.dic_gated_norm_bwd, code, p, x_new.device, "gated_norm_grad")
    return got
