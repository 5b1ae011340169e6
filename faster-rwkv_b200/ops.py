"""Operators of a recurrent layer over torch CUDA tensors: include/fr_b200.h's fr_b200_linear, fr_b200_conv_*, fr_b200_ssm_* and
fr_b200_slots_copy on the tensors' device and torch's current stream.

Tensors are [rows, width] with adjacent elements and any distance between rows, so that pieces of a wider projection go in as
they are; they are not copied or cast.  Results are new tensors unless `out` is given.  Sequences (`starts`) and slots are host
lists, numpy int32 arrays or CPU int32 tensors; a call that is captured into a CUDA graph holds them by value.
"""
from __future__ import annotations

import ctypes

import numpy as np

ACTIVATIONS = {"none": 0, "relu2": 1, "silu": 2, "sigmoid": 3, "gelu": 4, "softplus": 5}
_F16, _F32, _BF16 = 0, 1, 2
_ids = None        # torch dtype -> element type; torch is imported with the first call
_torch = None


def _setup():
    global _torch, _ids
    import torch
    _ids = {torch.float16: _F16, torch.float32: _F32, torch.bfloat16: _BF16}
    _torch = torch


def _call(name, args):
    from . import FrB200Error, lib
    L = lib()
    rc = getattr(L, name)(*args)
    if rc < 0:
        raise FrB200Error(rc, f"{name}: {L.fr_b200_strerror(rc).decode()}", L.fr_b200_op_last_error().decode())


def _rows(t, what, width=None, like=None):
    """A [rows, width] tensor on the GPU with adjacent elements -> address and distance of rows."""
    if t.dim() != 2:
        raise ValueError(f"{what} has {t.dim()} dimensions instead of 2")
    if width is not None and t.shape[1] != width:
        raise ValueError(f"{what} is {t.shape[1]} wide instead of {width}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[0] != like.shape[0]):
        raise ValueError(f"{what} differs from x in type, device or rows")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"the elements of a row of {what} are not adjacent")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    return t.data_ptr(), ld


def _param(t, what, shape, like):
    """An fp32 parameter, contiguous, or None."""
    if t is None:
        return None
    if t.dtype != _torch.float32 or t.device != like.device or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} is not a contiguous fp32 {list(shape)} tensor on the device of x")
    return t.data_ptr()


def _x(x):
    if _torch is None:
        _setup()
    if not x.is_cuda:
        raise ValueError("x is not on a GPU: there is no CPU path")
    if x.dtype not in _ids:
        raise ValueError(f"x has the type {x.dtype}: float16, bfloat16 and float32 are taken")
    return _ids[x.dtype]


def _place(x):
    index = x.device.index
    return index, _torch.cuda.current_stream(index).cuda_stream


def _ints(v, n, what):
    """A host list of n int32 -> (address, what keeps it), or None."""
    if v is None:
        return None, None
    if _torch is not None and isinstance(v, _torch.Tensor):
        if v.is_cuda:
            raise ValueError(f"{what} is on the GPU: the call holds it by value, from the host")
        v = v.numpy()
    elif isinstance(v, int):
        v = np.full(n, v, np.int32)
    a = np.asarray(v)
    if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
        raise ValueError(f"{what} is not a list of integers")
    if a.size != n:
        raise ValueError(f"{what} has {a.size} entries instead of {n}")
    if a.dtype != np.int32:
        if a.size and (a.min() < -2**31 or a.max() >= 2**31):
            raise ValueError(f"{what} has an entry that is no 32-bit integer")
        a = a.astype(np.int32)
    a = np.ascontiguousarray(a)
    return a.ctypes.data, a


def _sequences(starts, rows):
    if starts is None:
        return None, 1, None
    n = len(starts)
    if n < 1:
        raise ValueError("starts has the first row of every sequence and the end of the last")
    ptr, keep = _ints(starts, n, "starts")
    return ptr, n - 1, keep


def _pool(state, dtype, inner, like):
    """[slots, *inner] with whole slots -> address, distance of slots, slots."""
    if state is None:
        return None, 0, 0
    if state.dtype != dtype or state.device != like.device or state.dim() != 1 + len(inner) or tuple(state.shape[1:]) != inner:
        raise ValueError(f"state is not a {dtype} [slots, {', '.join(map(str, inner))}] tensor on the device of x")
    want = 1
    for size, stride in zip(reversed(inner), reversed(state.stride()[1:])):
        if size > 1 and stride != want:
            raise ValueError("a slot of state is not contiguous")
        want *= size
    slots = state.shape[0]
    return state.data_ptr(), state.stride(0) if slots > 1 else want, slots


def _out(out, x, rows, width, dtype):
    if out is None:
        return _torch.empty((rows, width), dtype=dtype, device=x.device)
    if out.dtype != dtype or out.device != x.device or tuple(out.shape) != (rows, width):
        raise ValueError(f"out is not a {dtype} [{rows}, {width}] tensor on the device of x")
    return out


def linear(x, w, bias=None, activation="none", residual=None, out=None, out_dtype=None):
    """residual + activation(x @ w.T + bias): x [rows, K], w [N, K] of one 16-bit type, bias [N] fp32; residual and the
    result [rows, N] in the type of x or out_dtype=torch.float32.  activation: none, relu2, silu, sigmoid, gelu, softplus.
    out may be the residual."""
    dt = _x(x)
    rows, k = x.shape if x.dim() == 2 else (None, None)
    xp, ldx = _rows(x, "x")
    n = w.shape[0]
    if w.dtype != x.dtype or w.device != x.device:
        raise ValueError("w differs from x in type or device")
    wp, ldw = _rows(w, "w", k)
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    out = _out(out, x, rows, n, out_dtype or (out.dtype if out is not None else x.dtype))
    op, ldo = _rows(out, "out")
    rp, ldr = None, 0
    if residual is not None:
        if residual.dtype != out.dtype or residual.device != x.device or residual.shape[0] != rows:
            raise ValueError("the residual differs from the result in type, device or rows")
        rp, ldr = _rows(residual, "residual", n)
    index, stream = _place(x)
    _call("fr_b200_linear", (xp, ldx, wp, ldw, dt, rows, k, n, _param(bias, "bias", (n,), x), ACTIVATIONS[activation], rp, ldr, op, ldo,
                             _ids.get(out.dtype, -1), index, stream))
    return out


def _conv(name, x, w, bias, activation, state, from_slots, to_slots, out, starts, seq):
    dt = _x(x)
    xp, ldx = _rows(x, "x")
    rows, d = x.shape
    taps = w.shape[1] if w.dim() == 2 else -1
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    wp, bp = _param(w, "w", (d, taps), x), _param(bias, "bias", (d,), x)
    out = _out(out, x, rows, d, x.dtype)
    op, ldo = _rows(out, "out")
    sp, stride, slots = _pool(state, x.dtype, (taps - 1, d), x)
    index, stream = _place(x)
    if seq:
        tp, n, k1 = _sequences(starts, rows)
    else:
        n = rows
    fp, k2 = _ints(from_slots, n, "from_slots")
    ip, k3 = _ints(to_slots, n, "to_slots")
    act = ACTIVATIONS[activation]
    if seq:
        _call(name, (xp, ldx, dt, rows, d, wp, taps, bp, act, tp, n, sp, stride, slots, fp, ip, op, ldo, index, stream))
    else:
        _call(name, (xp, ldx, dt, rows, d, wp, taps, bp, act, sp, stride, slots, fp, ip, op, ldo, index, stream))
    return out


def conv_seq(x, w, bias=None, activation="silu", starts=None, state=None, from_slots=None, to_slots=None, out=None):
    """Causal convolution of each channel over the last taps rows of its sequence: x [rows, D], w [D, taps] (2 to 4) and bias
    [D] fp32, activation none or silu.  starts: first rows of the sequences and the end of the last (None: one sequence).
    state: pool [slots, taps - 1, D] of the last rows; sequence i begins from slot from_slots[i] (-1: from zero; a single
    number stands for all) and leaves its state in to_slots[i] (-1: nowhere); None: slot i."""
    return _conv("fr_b200_conv_seq", x, w, bias, activation, state, from_slots, to_slots, out, starts, True)


def conv_step(x, w, bias=None, activation="silu", state=None, from_slots=None, to_slots=None, out=None):
    """conv_seq for one row of each stream: x [streams, D]."""
    return _conv("fr_b200_conv_step", x, w, bias, activation, state, from_slots, to_slots, out, None, False)


def _ssm(name, x, dt, A, B, C, D, z, dt_bias, dt_softplus, starts, state, from_slots, to_slots, out, seq):
    kind = _x(x)
    xp, ldx = _rows(x, "x")
    rows, d = x.shape
    if A.dim() != 2:
        raise ValueError("A is not [D, N]")
    n = A.shape[1]
    ap, skip, bias = _param(A, "A", (d, n), x), _param(D, "D", (d,), x), _param(dt_bias, "dt_bias", (d,), x)
    dtp, lddt = _rows(dt, "dt", d, x)
    bp, ldb = _rows(B, "B", None, x)
    cp, ldc = _rows(C, "C", B.shape[1], x)
    if n < 1 or B.shape[1] % n:
        raise ValueError("B is not [rows, groups * N]")
    groups = B.shape[1] // n
    zp, ldz = _rows(z, "z", d, x) if z is not None else (None, 0)
    out = _out(out, x, rows, d, x.dtype)
    op, ldo = _rows(out, "out")
    sp, stride, slots = _pool(state, _torch.float32, (d, n), x)
    index, stream = _place(x)
    if seq:
        tp, ns, k1 = _sequences(starts, rows)
    else:
        ns = rows
    fp, k2 = _ints(from_slots, ns, "from_slots")
    ip, k3 = _ints(to_slots, ns, "to_slots")
    head = (xp, ldx, dtp, lddt, ap, bp, ldb, cp, ldc, skip, zp, ldz, bias, 1 if dt_softplus else 0, kind, rows, d, n, groups)
    if not seq:
        _call(name, head + (sp, stride, slots, fp, ip, op, ldo, index, stream))
        return out
    from . import lib
    need = lib().fr_b200_ssm_seq_workspace(rows, ns, d, n)
    work = _torch.empty(need, dtype=_torch.uint8, device=x.device) if need else None
    _call(name, head + (tp, ns, sp, stride, slots, fp, ip, op, ldo, work.data_ptr() if need else None, need, index, stream))
    return out


def ssm_seq(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=True, starts=None, state=None, from_slots=None, to_slots=None, out=None):
    """Selective state space scan over the rows of each sequence: for channel d, state n,
        delta = softplus(dt + dt_bias);  h = exp(delta * A) * h + delta * x * B;  y = (sum_n C * h + D * x) * silu(z).
    x, dt, z [rows, channels] and B, C [rows, groups * N] of one type; A [channels, N], D and dt_bias [channels] fp32.
    state: pool [slots, channels, N] fp32; starts, from_slots and to_slots as in conv_seq."""
    return _ssm("fr_b200_ssm_seq", x, dt, A, B, C, D, z, dt_bias, dt_softplus, starts, state, from_slots, to_slots, out, True)


def ssm_step(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=True, state=None, from_slots=None, to_slots=None, out=None):
    """ssm_seq for one row of each stream."""
    return _ssm("fr_b200_ssm_step", x, dt, A, B, C, D, z, dt_bias, dt_softplus, None, state, from_slots, to_slots, out, False)


def copy_slots(pool, src, dst):
    """pool[dst[i]] takes what pool[src[i]] holds before the call (src -1: zeros): states of streams forked, moved, reordered
    and cleared.  pool: [slots, ...] of any type with contiguous slots; every slot appears in dst once at most."""
    if _torch is None:
        _setup()
    if not pool.is_cuda or pool.dim() < 1:
        raise ValueError("pool is not a GPU tensor of slots")
    per = 1
    for size, stride in zip(reversed(pool.shape[1:]), reversed(pool.stride()[1:])):
        if size > 1 and stride != per:
            raise ValueError("a slot of the pool is not contiguous")
        per *= size
    slots, es = pool.shape[0], pool.element_size()
    n = len(src)
    sp, k1 = _ints(src, n, "src")
    dp, k2 = _ints(dst, n, "dst")
    index, stream = _place(pool)
    _call("fr_b200_slots_copy", (pool.data_ptr(), per * es, (pool.stride(0) if slots > 1 else per) * es, slots, n, sp, dp, index, stream))
    return pool
