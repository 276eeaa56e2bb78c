"""Operators of an encoder block over longer token rows than the reference's: attention in a sliding window whose first keys stay visible, and the norms
before and after a block with its gate and the residual scale (csrc/wattn.hip, csrc/gnorm.hip; include/dic_hip.h states the formulas).

As everywhere in this package there is no autograd: each forward call has a call that computes its gradients, and a tensor that asks for a gradient or
carries a forward-mode tangent is refused.
Calls run on the current stream of the tensors' device, allocate what they return and their workspaces from torch's allocator, never synchronise, and can
be captured into a graph.  Arguments that do not fit raise ValueError or TypeError before anything is launched."""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.DIC_F32, torch.bfloat16: _lib.DIC_BF16}
_RES_F32 = 0x200
_KINDS = {"layer": 1, "rms": 2}
_FAR = 2 ** 31 - 1
_FLT_MAX = 3.4028234663852886e38
# The parameter structs as bytes: packing one takes a fifth of the time of filling its ctypes mirror, and a call on one caption is all host time.
_WIN = struct.Struct("9P24q3P9if2P")
_NORM = struct.Struct("17Pif2Pif2qif2P")
_fns = {}


def _fn(name):
    """A C entry that takes its params as bytes."""
    f = _fns.get(name)
    if f is None:
        f = _lib.entry(name)
        f.argtypes = [C.c_int, C.c_int, C.c_char_p] if name == "dic_win_attn_ws_bytes" else [C.c_int, C.c_char_p] if name.endswith("ws_bytes") else [C.c_int, C.c_char_p, C.c_void_p]
        f.restype = C.c_size_t if name.endswith("ws_bytes") else C.c_int
        _fns[name] = f
    return f


def _launch(name, code, params, device):
    """One C call on the current stream of `device`."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)        # (torch.cuda.current_stream(device) without building the object)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = _fn(name)(code, params, stream)
    else:
        rc = _fn(name)(code, params, stream)
    if rc == 1001:
        raise ValueError(_lib.lib().dic_last_error().decode(errors="replace"))
    _lib.check(rc, name)


def _on(t, like, name, dtypes, shape=None):
    try:
        if t.dtype in dtypes and t.get_device() == like.get_device() and (shape is None or t.shape == shape) and not (t.requires_grad and torch.is_grad_enabled()):
            return
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {t.dtype} where {' or '.join(map(str, dtypes))} is needed")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    raise ValueError(f"{name} asks for a gradient: this package has no autograd, call the operator's _grad function on detached tensors")


def _unfit(e):
    """For what came up while the arguments were packed: sizes beyond 32 bits, and tensors that are sparse or inside a function transform."""
    return ValueError(f"a size that does not fit: {e}") if isinstance(e, struct.error) else TypeError(f"a tensor without memory of its own: {e}")


def _no_tangents(*tensors):
    """Inside forward-mode differentiation (forward_ad._current_level >= 0): a tangent would be dropped."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("a tensor carries a forward-mode tangent: this package has no autograd, call the operator on its primal")


def _ptr(t):
    try:
        return 0 if t is None else t.data_ptr()
    except RuntimeError as e:
        raise _unfit(e) from None


def _first(t, name):
    """What the other tensors are held against."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        _lib.require_gpu()
        raise ValueError(f"{name} must be on the GPU")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name}: {t.dtype} where torch.float32 or torch.bfloat16 is needed")


def _number(x, name):
    """x as a float that fp32 holds.  A tensor on the GPU would be waited for, and is refused."""
    if type(x) is not float:
        if isinstance(x, torch.Tensor) and (x.device.type != "cpu" or x.requires_grad or x.numel() != 1) or isinstance(x, (str, bytes)):
            raise TypeError(f"{name} must be a number")
        try:
            x = float(x)
        except OverflowError:
            raise ValueError(f"{name} must fit fp32") from None
        except (TypeError, ValueError, RuntimeError):
            raise TypeError(f"{name} must be a number") from None
    if not -_FLT_MAX <= x <= _FLT_MAX:
        raise ValueError(f"{name} must be finite and fit fp32")
    return x


# ------------------------------------------------------------------------------------------------ attention
def _bound(x, name):
    if x is None:
        return -1
    if type(x) is not int:
        value = _number(x, name)
        if value != int(value):
            raise ValueError(f"{name} must be a whole number")
        x = int(value)
    if x < 0:
        raise ValueError(f"{name} must be None (no bound) or at least 0")
    return min(x, _FAR)


def _check_rows(t, like, name, shape):
    _on(t, like, name, (like.dtype,), shape)
    if t.stride(3) != 1:
        raise ValueError(f"the rows of {name} must be contiguous")


def _complain(q, k, v):
    """What is wrong with them, as an exception."""
    _first(q, "q")
    if q.dim() != 4:
        raise ValueError(f"q has shape {tuple(q.shape)}, not [N, Tq, H, dh]")
    _check_rows(q, q, "q", q.shape)
    _on(k, q, "k", (q.dtype,))
    if k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"k has shape {tuple(k.shape)}, not [{q.shape[0]}, Tk, Hkv, {q.shape[3]}]")
    _check_rows(k, q, "k", k.shape)
    _check_rows(v, q, "v", k.shape)


def _attention(q, k, v, left, right, sinks, key_mask, kv_len, q_pos, scale):
    """The checked arguments: (strides of q, k and v, tail of the packed struct in front of the workspace, dtype code).  Alignment and what else the C entry
    checks are left to it."""
    try:
        t, at, (N, Tq, H, dh), (Nk, Tk, Hkv, dk) = q.dtype, q.get_device(), q.shape, k.shape
        sq, sk, sv = q.stride(), k.stride(), v.stride()
        code = _DTYPES[t]
        fine = (at >= 0 and k.dtype is t and v.dtype is t and k.get_device() == at and v.get_device() == at and N == Nk and dh == dk and v.shape == k.shape
                and sq[3] == sk[3] == sv[3] == 1 and not ((q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled()))
    except Exception:
        fine = False
    if not fine:
        _complain(q, k, v)
        raise ValueError("q, k and v do not fit together")
    if key_mask is not None:
        _on(key_mask, q, "key_mask", (torch.bool, torch.uint8), (N, Tk))
        if not key_mask.is_contiguous():
            raise ValueError("key_mask must be contiguous")
    for x, name in ((kv_len, "kv_len"), (q_pos, "q_pos")):
        if x is not None:
            _on(x, q, name, (torch.int32,), (N,))
            if not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    scale = (dh or 1) ** -0.5 if scale is None else _number(scale, "scale")
    if not scale > 0.0:
        raise ValueError("scale must be positive")
    return (*sq[:3], *sk[:3], *sv[:3]), (_ptr(key_mask), _ptr(kv_len), _ptr(q_pos), N, Tq, Tk, H, Hkv, dh, _bound(left, "left"), _bound(right, "right"), _bound(0 if sinks is None else sinks, "sinks"), scale), code


_NO_STRIDES = (0,) * 12


def window_attention(q, k, v, *, left=None, right=None, sinks=0, key_mask=None, kv_len=None, q_pos=None, scale=None, out=None):
    """softmax(scale q k^T) v over the keys each query row sees; returns (out like q, lse [N, H, Tq] fp32).

    q [N, Tq, H, dh]; k, v [N, Tk, Hkv, dh]: float32 or bfloat16, dh 64 or 128, any strides with contiguous 16-byte-aligned rows (views of a packed q|k|v
    tensor or of a longer cache); H a multiple of Hkv.  Row i of sequence n stands at position t = i + q_pos[n] (int32 [N]; 0 without).  It sees key j when
    j < kv_len[n] (int32 [N]; Tk without), key_mask[n, j] is true (bool or uint8 [N, Tk]), j <= t + right, and j >= t - left or j < sinks; left / right None:
    no bound.  A row that sees nothing gives zeros and lse = -inf.  `out`: write there instead of into a new tensor.

    One new token behind a cache: Tq = 1, kv_len = the cache's lengths with the new key in place, q_pos = kv_len - 1, right = 0."""
    if forward_ad._current_level >= 0:
        _no_tangents(q, k, v, out)
    strides, tail, code = _attention(q, k, v, left, right, sinks, key_mask, kv_len, q_pos, scale)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_rows(out, q, "out", q.shape)
    lse = q.new_empty((tail[3], tail[6], tail[4]), dtype=torch.float32)
    ws_bytes = _fn("dic_win_attn_ws_bytes")
    try:
        fields = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, *strides, *out.stride()[:3], *_NO_STRIDES, *tail)
        size = ws_bytes(code, 0, _WIN.pack(*fields, 0, 0))
    except (RuntimeError, struct.error) as e:
        raise _unfit(e) from None
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _launch("dic_win_attn_fwd", code, _WIN.pack(*fields, _ptr(ws), size), q.device)
    return out, lse


def window_attention_grad(dout, q, k, v, out, lse, *, left=None, right=None, sinks=0, key_mask=None, kv_len=None, q_pos=None, scale=None, grads=None):
    """(dq, dk, dv) of window_attention for the gradient `dout` of its output; the other arguments as they went into and came out of that call.
    `grads`: three tensors to write them into (views of a packed gradient, say).  dk and dv are summed over the query heads of each key head."""
    if forward_ad._current_level >= 0:
        _no_tangents(dout, q, k, v, out, lse)
    strides, tail, code = _attention(q, k, v, left, right, sinks, key_mask, kv_len, q_pos, scale)
    _on(dout, q, "dout", (q.dtype,), q.shape)
    _check_rows(out, q, "out", q.shape)
    _on(lse, q, "lse", (torch.float32,), (tail[3], tail[6], tail[4]))
    if not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    per = 16 // q.element_size()
    if not dout.is_contiguous() and (dout.stride(3) != 1 or any(s % per for s in dout.stride()[:3])) or _ptr(dout) % 16:
        if dout.layout is not torch.strided:
            raise TypeError("dout must be a dense tensor")
        dout = dout.clone(memory_format=torch.contiguous_format)                 # an expanded or transposed gradient
    if grads is None:
        dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    else:
        dq, dk, dv = grads
        if forward_ad._current_level >= 0:
            _no_tangents(dq, dk, dv)
        for t, like, name in ((dq, q, "dq"), (dk, k, "dk"), (dv, k, "dv")):
            _check_rows(t, q, name, like.shape)
    ws_bytes = _fn("dic_win_attn_ws_bytes")
    try:
        fields = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                  *strides, *out.stride()[:3], *dout.stride()[:3], *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3], *tail)
        size = ws_bytes(code, 1, _WIN.pack(*fields, 0, 0))
    except (RuntimeError, struct.error) as e:
        raise _unfit(e) from None
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _launch("dic_win_attn_bwd", code, _WIN.pack(*fields, _ptr(ws), size), q.device)
    return dq, dk, dv


# ------------------------------------------------------------------------------------------------ norms
class NormParams(NamedTuple):
    """A norm over the last dimension: kind "layer" or "rms", weight and bias [D] float32 (None: 1 and 0)."""
    kind: str = "layer"
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-12


_WEIGHT, _BIAS, _EPS = ({side: f"{side} {what}" for side in ("post", "pre")} for what in ("weight", "bias", "eps"))


def _inside(norm):
    return getattr(norm, "weight", None), getattr(norm, "bias", None), getattr(norm, "eps", None)


def _norm(norm, like, D, side):
    """The packed fields of one norm."""
    if norm is None:
        return 0, 0, 0, 0.0
    try:
        kind, weight, bias, eps = norm.kind, norm.weight, norm.bias, norm.eps
    except AttributeError:
        raise TypeError(f"{side} must be NormParams or None") from None
    if kind not in _KINDS:
        raise ValueError(f'{side}: a norm is "layer" or "rms"')
    for t, name in ((weight, _WEIGHT[side]), (bias, _BIAS[side])):
        if t is not None:
            _packed(t, like, name, torch.float32, (D,))
    return _ptr(weight), _ptr(bias), _KINDS[kind], _number(eps, _EPS[side])


def _shapes(x, gate):
    """(rows, D, rows that share a gate row) of x [..., D]."""
    if not (x.dim() >= 2 and 1 <= x.shape[-1] <= 8192):
        raise ValueError("rows of 1 to 8192 elements in at least two dimensions are needed")
    D = x.shape[-1]
    rows = x.numel() // D
    if gate is None:
        return rows, D, 1
    _on(gate, x, "gate", (torch.float32,))
    if not (gate.is_contiguous() and gate.dim() in (1, 2) and gate.shape[-1] == D):
        raise ValueError(f"gate must be contiguous, [{D}] or [sequences, {D}]")
    n = 1 if gate.dim() == 1 else gate.shape[0]
    if not (rows == 0 or (n > 0 and rows % n == 0)):
        raise ValueError(f"{rows} rows do not divide over {n} gates")
    return rows, D, max(rows // max(n, 1), 1)


def _packed(t, like, name, dtype, shape):
    try:                                                             # (the whole check in one expression: a call on one caption's rows is all host time)
        if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == like.get_device() and not (t.requires_grad and torch.is_grad_enabled()):
            return
    except (AttributeError, RuntimeError):
        pass
    _on(t, like, name, (dtype,), shape)
    raise ValueError(f"{name} must be contiguous")


def _norm_code(stream, inner):
    if inner not in _DTYPES or (stream, inner) == (torch.bfloat16, torch.float32):
        raise TypeError(f"a {stream} residual stream with {inner} blocks: float32 with float32 or bfloat16, or bfloat16 with bfloat16")
    return _DTYPES[inner] | (_RES_F32 if stream != inner else 0)


def gated_norm(x, y=None, *, post=None, gate=None, residual_scale=1.0, pre=None, dtype=None):
    """x_new = residual_scale x + gate * post(y) and a = pre(x_new), the next block's input, in one pass; returns (x_new, a, saved).

    y [..., D] is a block's output, x the residual stream in front of the block (x may be float32 beside a bfloat16 y).  post, pre: NormParams or None (no
    norm; without pre, a is None).  gate: float32 [D], [N, D] (one row for each of N equal runs of rows: the sequences of [N, T, D]), or None.  `saved`
    [4, rows] holds the rows' statistics for gated_norm_grad.  Without y it is a stack's first norm: a = pre(residual_scale x), of type `dtype` (x's); at
    scale 1 x_new is then x itself."""
    if forward_ad._current_level >= 0:
        _no_tangents(x, y, gate, residual_scale, *_inside(post), *_inside(pre))
    _first(x, "x")
    inner = y.dtype if isinstance(y, torch.Tensor) else (dtype or x.dtype)
    code = _norm_code(x.dtype, inner)
    _packed(x, x, "x", x.dtype, x.shape)
    if y is not None:
        _packed(y, x, "y", inner, x.shape)
        if not (dtype in (None, inner)):
            raise ValueError("dtype is the type of a without y")
    else:
        if not (post is None and gate is None and pre is not None):
            raise ValueError("without y there is a pre norm and nothing else")
    residual_scale = _number(residual_scale, "residual_scale")
    rows, D, per_gate = _shapes(x, gate)
    sides = *_norm(post, x, D, "post"), *_norm(pre, x, D, "pre")
    x_new = x if y is None and residual_scale == 1.0 else torch.empty_like(x)
    a = None if pre is None else torch.empty_like(x if y is None else y, dtype=inner)
    saved = x.new_empty((4, rows), dtype=torch.float32)
    try:
        params = _NORM.pack(x.data_ptr(), _ptr(y), 0 if x_new is x else x_new.data_ptr(), _ptr(a), _ptr(gate), saved.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0,
                            *sides, rows, per_gate, D, residual_scale, 0, 0)
    except (RuntimeError, struct.error) as e:
        raise _unfit(e) from None
    _launch("dic_gated_norm_fwd", code, params, x.device)
    return x_new, a, saved


def gated_norm_grad(dx_new, da, x_new, y, saved, *, post=None, gate=None, residual_scale=1.0, pre=None):
    """Gradients of gated_norm as a dict: "dx", "dy", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias", as far as there are such inputs.
    dx_new (None: zero) and da (None without pre) are the gradients of its outputs; x_new, y and saved as they went into and came out of that call."""
    if forward_ad._current_level >= 0:
        _no_tangents(dx_new, da, x_new, y, saved, gate, residual_scale, *_inside(post), *_inside(pre))
    _first(x_new, "x_new")
    given = y if y is not None else da
    inner = given.dtype if isinstance(given, torch.Tensor) else x_new.dtype
    code = _norm_code(x_new.dtype, inner)
    shape = x_new.shape
    _packed(x_new, x_new, "x_new", x_new.dtype, shape)
    if not ((da is None) == (pre is None)):
        raise ValueError("da is the gradient of pre's output: both or neither")
    if not (dx_new is not None or da is not None):
        raise ValueError("neither output has a gradient")
    if dx_new is not None:
        _packed(dx_new, x_new, "dx_new", x_new.dtype, shape)
    if da is not None:
        _packed(da, x_new, "da", inner, shape)
    if y is not None:
        _packed(y, x_new, "y", inner, shape)
    else:
        if not (post is None and gate is None and pre is not None):
            raise ValueError("without y there is a pre norm and nothing else")
    residual_scale = _number(residual_scale, "residual_scale")
    rows, D, per_gate = _shapes(x_new, gate)
    sides = *_norm(post, x_new, D, "post"), *_norm(pre, x_new, D, "pre")
    _packed(saved, x_new, "saved", torch.float32, (4, rows))
    got = {"dx": torch.empty_like(x_new)}
    if y is not None:
        got["dy"] = torch.empty_like(y)
    if gate is not None:
        got["gate"] = torch.empty_like(gate) if rows else torch.zeros_like(gate)
    names = [name for norm, side in ((post, "post"), (pre, "pre")) if norm is not None
             for name, t in ((side + "_weight", norm.weight), (side + "_bias", norm.bias)) if t is not None]
    if names:
        got.update(zip(names, x_new.new_empty((len(names), D), dtype=torch.float32).unbind(0)))      # (one allocation)
    fields = (0, _ptr(y), _ptr(x_new), 0, _ptr(gate), _ptr(saved), _ptr(dx_new), _ptr(da), got["dx"].data_ptr(), _ptr(got.get("dy")), _ptr(got.get("gate")),
              _ptr(got.get("post_weight")), _ptr(got.get("post_bias")), _ptr(got.get("pre_weight")), _ptr(got.get("pre_bias")), *sides, rows, per_gate, D, residual_scale)
    size = _fn("dic_gated_norm_ws_bytes")(code, _NORM.pack(*fields, 0, 0))
    ws = x_new.new_empty(size, dtype=torch.uint8) if size else None
    _launch("dic_gated_norm_bwd", code, _NORM.pack(*fields, _ptr(ws), size), x_new.device)
    return got
