"""Operators of a recurrent layer over device tensors (linear, conv_seq / conv_step, ssm_seq / ssm_step, copy_slots,
Model.copy_states), each against its formula in 64 bits.

Tolerances are bounds of the rounding errors, derived here: a result of type t is off by half a step, eps(t) / 2 of its
value; what is computed in fp32 before that by the bounds that the helpers carry along."""
import itertools
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24          # half a step of fp32
EX2 = 2.0 ** -22          # the fast exponential: 2 ulp
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _half_step(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps    # the step of subnormal results


def _rand(*shape, dtype=F32, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(i * s for i, s in enumerate(shape, 1)))
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _check(got, want, err, what=""):
    """|got - want| <= err + the rounding of the result; same NaN and infinities."""
    t = got.dtype
    g, w = got.double(), want
    if not w.numel():
        return
    big = torch.isfinite(w)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    assert torch.equal(g[~big & ~torch.isnan(w)], w[~big & ~torch.isnan(w)]), what
    tol = (err + _half_step(t) * (w.abs() + err) + _tiny(t))[big]
    off = (g - w).abs()[big]
    assert bool((off <= tol).all()), (what, float((off / tol).max()), float(off.max()))


# ---- linear ------------------------------------------------------------------------------------------------------

ACTS = {
    "none": lambda v: v, "relu2": lambda v: torch.where(v < 0, torch.zeros_like(v), v * v), "silu": lambda v: v * torch.sigmoid(v),
    "sigmoid": torch.sigmoid, "gelu": lambda v: v * 0.5 * (1 + torch.erf(v / math.sqrt(2))), "softplus": lambda v: torch.logaddexp(v, torch.zeros_like(v)),
}


def _linear_want(x, w, bias, act, residual):
    """value and error bound: products of 16-bit numbers are exact in fp32; a sum of K of them, taken 16 at a time on the tensor cores
    (whose adders may truncate: a whole step), loses a step of at most the sum of magnitudes with each of K / 16 + 20 additions."""
    xd, wd = x.double(), w.double()
    v, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    err = (x.shape[1] / 16 + 20) * 2 * U32 * mag
    if bias is not None:
        v = v + bias.double()
        err = err + U32 * v.abs()
    r = ACTS[act](v)
    # slopes: relu2 2 |v|, the others at most 1.13; the functions themselves: a few steps of fp32, 8e-7 relative with fast exp and division,
    # erf's 2 ulp of 1, times |v| / 2
    err = err * (2 * v.abs() + err if act == "relu2" else 1.13) + (8e-7 * r.abs() + 4e-7 * v.abs() * (act in ("gelu",)) if act != "none" else 0)
    if residual is not None:
        r = r + residual.double()
        err = err + U32 * r.abs()
    return r, err


SIZES = [(1, 1, 1), (1, 64, 8), (1, 2048, 520), (2, 8, 24), (3, 33, 17), (7, 160, 100), (8, 4096, 128), (16, 72, 130), (17, 160, 96), (31, 40, 1000),
         (33, 512, 256), (64, 256, 136), (65, 72, 130), (100, 1000, 264), (128, 128, 128), (129, 520, 264), (200, 640, 328), (256, 64, 256),
         (257, 2048, 520), (300, 1031, 515), (1000, 512, 768), (2049, 136, 72)]


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear(pkg, rows, k, n, dtype):
    x, w = _rand(rows, k, dtype=dtype), _rand(n, k, dtype=dtype, scale=1 / math.sqrt(k), seed=1)
    b, r = _rand(n, seed=2), _rand(rows, n, dtype=dtype, scale=2.0, seed=3)
    for i, (bias, res, out_dtype) in enumerate(itertools.product((None, b), (None, r), (None, F32))):
        act = list(ACTS)[(i + rows) % len(ACTS)]
        resid = res if out_dtype is None or res is None else res.float()
        got = pkg.linear(x, w, bias, activation=act, residual=resid, out_dtype=out_dtype)
        assert got.dtype == (out_dtype or dtype) and got.shape == (rows, n)
        want, err = _linear_want(x, w, bias, act, resid)
        _check(got, want, err, (rows, k, n, act, bias is None, res is None, out_dtype))


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("rows,k,n", [(5, 96, 200), (140, 96, 200)])
def test_linear_activations(pkg, act, rows, k, n):
    x, w, b = _rand(rows, k, dtype=BF16, scale=3.0), _rand(n, k, dtype=BF16, scale=0.5, seed=1), _rand(n, scale=20.0, seed=2)
    for out_dtype in (BF16, F32):
        want, err = _linear_want(x, w, b, act, None)
        _check(pkg.linear(x, w, b, activation=act, out_dtype=out_dtype), want, err, act)


@pytest.mark.parametrize("rows,k,n", [(1, 256, 64), (12, 255, 65), (40, 256, 64), (300, 192, 136), (300, 191, 135), (520, 703, 650), (520, 704, 648)])
@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_linear_pieces_of_wider_rows(pkg, rows, k, n, shift):
    """x, w, residual and out as columns of wider tensors, at 16-byte boundaries and off them; what lies beside out stays."""
    X, W, R = _rand(rows, k + 24, dtype=F16), _rand(n, k + 40, dtype=F16, scale=0.1, seed=1), _rand(rows, n + 16, dtype=F16, seed=2)
    O = _rand(rows, n + 32, dtype=F16, seed=3)
    keep = O.clone()
    x, w, r, o = X[:, shift:shift + k], W[:, shift:shift + k], R[:, shift:shift + n], O[:, shift:shift + n]
    got = pkg.linear(x, w, None, activation="silu", residual=r, out=o)
    assert got is o
    want, err = _linear_want(x, w, None, "silu", r)
    _check(o, want, err)
    keep[:, shift:shift + n] = o
    assert torch.equal(O, keep)


@pytest.mark.parametrize("rows,k,n", [(5, 64, 70), (40, 640, 333), (100, 4096, 130), (260, 512, 77), (700, 256, 700)])
@pytest.mark.parametrize("out_dtype", [F16, F32])
def test_linear_with_ragged_results(pkg, rows, k, n, out_dtype):
    """operands at 16-byte boundaries, residual and out off them"""
    x, w, b = _rand(rows, k, dtype=F16), _rand(n, k, dtype=F16, scale=k ** -0.5, seed=1), _rand(n, seed=2)
    R, O = _rand(rows, n + 5, dtype=out_dtype, seed=3), torch.full((rows, n + 3), 9.0, dtype=out_dtype, device="cuda")
    for act, res in (("gelu", R[:, 2:2 + n]), ("none", None)):
        pkg.linear(x, w, b, activation=act, residual=res, out=O[:, 1:1 + n])
        want, err = _linear_want(x, w, b, act, res)
        _check(O[:, 1:1 + n], want, err, act)
        assert bool((O[:, 0] == 9).all()) and bool((O[:, n + 1:] == 9).all())


@pytest.mark.parametrize("rows", [1, 20, 200, 500])
def test_linear_onto_the_residual(pkg, rows):
    x, w = _rand(rows, 320, dtype=F16), _rand(264, 320, dtype=F16, scale=0.1, seed=1)
    for t in (F16, F32):
        r = _rand(rows, 264, dtype=t, seed=2)
        want, err = _linear_want(x, w, None, "none", r)
        got = pkg.linear(x, w, residual=r, out=r)
        assert got is r
        _check(r, want, err)


def test_linear_nan_and_infinities(pkg):
    for rows in (2, 80, 300):
        x, w = _rand(rows, 128, dtype=F16), _rand(72, 128, dtype=F16, seed=1)
        x[0, 5], x[1, 7] = float("nan"), float("inf")
        w[:, 7] = w[:, 7].abs() + 0.1
        got = pkg.linear(x, w, activation="relu2")
        assert torch.isnan(got[0]).all() and torch.isinf(got[1]).all()
        want, err = _linear_want(x[2:], w, None, "relu2", None)
        _check(got[2:], want, err)
        # a huge negative sum: silu and sigmoid go to zero, not to NaN
        b = torch.full((72,), -1e30, device="cuda")
        assert bool((pkg.linear(x[2:], w, b, activation="silu").abs() == 0).all())
        assert bool((pkg.linear(x[2:], w, b, activation="sigmoid").abs() == 0).all())
        assert bool((pkg.linear(x[2:], w, b, activation="softplus").abs() == 0).all())


def test_linear_is_the_same_every_time_and_on_any_stream(pkg):
    for rows in (1, 30, 129, 700):
        x, w, b = _rand(rows, 1024, dtype=BF16), _rand(520, 1024, dtype=BF16, scale=0.03, seed=1), _rand(520, seed=2)
        first = pkg.linear(x, w, b, activation="gelu")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [pkg.linear(x, w, b, activation="gelu") for _ in range(20)]
        torch.cuda.synchronize()
        assert all(torch.equal(first, a) for a in again)


def test_calls_on_several_streams_at_once(pkg):
    """products of every kind, scans and convolutions side by side: what each gives alone"""
    w, wide = _rand(2560, 2560, dtype=F16, scale=0.02, seed=1), _rand(640, 2560, dtype=F16, scale=0.02, seed=2)
    xs = [_rand(m, 2560, dtype=F16, seed=m) for m in (8, 40, 70, 150, 250, 700, 1500)]
    d, n = 320, 16
    sx, dt, A, B, C, D, z, bias = _ssm_inputs(300, d, n, 1, F16)
    cw = _rand(d, 4, seed=5)
    jobs = [lambda i=i: pkg.linear(xs[i], w, activation="silu") for i in range(len(xs))] + [lambda i=i: pkg.linear(xs[i], wide) for i in range(len(xs))]
    jobs += [lambda: pkg.ssm_seq(sx, dt, A, B, C, D=D, z=z, dt_bias=bias), lambda: pkg.conv_seq(sx, cw)]
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for r in range(12):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for i in range(s, len(jobs), len(streams)):
                    got.append((i + r) % len(jobs))
                    got.append(jobs[(i + r) % len(jobs)]())
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in zip(got[::2], got[1::2]))


def test_linear_rows_do_not_depend_on_their_neighbours(pkg):
    x, w = _rand(300, 512, dtype=F16), _rand(264, 512, dtype=F16, scale=0.05, seed=1)
    y = pkg.linear(x, w)
    x2 = x.clone()
    x2[150:] = float("nan")
    assert torch.equal(pkg.linear(x2, w)[:150], y[:150])


def test_linear_without_a_work_area(pkg):
    """a larger product off the 16-byte boundaries through the C entry, with scratch and without"""
    rows, k, n = 130, 1501, 900
    x, w = _rand(rows, k, dtype=BF16), _rand(n, k, dtype=BF16, scale=0.03, seed=1)
    want, err = _linear_want(x, w, None, "none", None)
    L = pkg.lib()
    need = L.fr_b200_linear_workspace(x.data_ptr(), k, w.data_ptr(), k, rows, k, n)
    assert need == (rows + n) * 188 * 16
    assert L.fr_b200_linear_workspace(x.data_ptr(), 1504, w.data_ptr(), 1504, rows, k, n) == 0 and L.fr_b200_linear_workspace(x.data_ptr(), k, w.data_ptr(), k, 32, k, n) == 0
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    for p, b in ((None, 0), (work.data_ptr(), need)):
        out = torch.empty((rows, n), dtype=BF16, device="cuda")
        rc = L.fr_b200_linear(x.data_ptr(), k, w.data_ptr(), k, 2, rows, k, n, None, 0, None, 0, out.data_ptr(), n, 2, p, b, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        _check(out, want, err)


def test_linear_without_rows(pkg):
    x, w = torch.empty((0, 64), dtype=F16, device="cuda"), _rand(32, 64, dtype=F16)
    assert pkg.linear(x, w).shape == (0, 32)


# ---- convolution -------------------------------------------------------------------------------------------------

def _conv_want(x, w, bias, act, starts, pool, fro, to):
    taps, d = w.shape[1], x.shape[1]
    y, err = torch.full_like(x, float("nan"), dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    new = pool.clone() if pool is not None else None
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        head = pool[fro[i]] if pool is not None and fro[i] >= 0 else torch.zeros((taps - 1, d), dtype=x.dtype, device="cuda")
        run = torch.cat([head, x[a:b]])
        v = sum(run[j:j + b - a].double() * w[:, j].double() for j in range(taps))
        mag = sum(run[j:j + b - a].double().abs() * w[:, j].double().abs() for j in range(taps))
        if bias is not None:
            v, mag = v + bias.double(), mag + bias.double().abs()
        e = (taps + 1) * U32 * mag
        r = ACTS[act](v)
        y[a:b], err[a:b] = r, 1.13 * e + (8e-7 * r.abs() if act == "silu" else 0)
        if new is not None and to[i] >= 0:
            new[to[i]] = run[b - a:]
    return y, err, new


LENGTHS = [[1], [2], [3], [16], [17], [1, 1, 1], [0, 5, 0, 0, 40, 2, 3, 16, 0], [33, 15, 1, 64, 2, 100], [500]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("taps,d,dtype", [(4, 512, F16), (4, 77, BF16), (3, 260, F32), (2, 1, F16), (2, 516, BF16), (4, 1030, F32)])
def test_conv_seq(pkg, lengths, taps, d, dtype):
    n = len(lengths)
    starts = np.cumsum([3] + lengths).tolist()           # rows in front of the first sequence and behind the last
    rows = starts[-1] + 5
    x, w = _rand(rows, d, dtype=dtype), _rand(d, taps, seed=1)
    pool = _rand(2 * n + 1, taps - 1, d, dtype=dtype, seed=2)
    fro = [(i * 5) % n if i % 3 else -1 for i in range(n)]
    fro = [f if f not in fro[:i] else -1 for i, f in enumerate(fro)]
    to = [2 * n - i if i % 4 != 1 else -1 for i in range(n)]
    for act, bias in (("silu", _rand(d, seed=3)), ("none", None)):
        p, out = pool.clone(), torch.full_like(x, 7.0)
        got = pkg.conv_seq(x, w, bias, activation=act, starts=starts, state=p, from_slots=fro, to_slots=to, out=out)
        assert got is out
        want, err, new = _conv_want(x, w, bias, act, starts, pool, fro, to)
        _check(out[3:starts[-1]], want[3:starts[-1]], err[3:starts[-1]])
        assert bool((out[:3] == 7).all()) and bool((out[starts[-1]:] == 7).all())
        assert torch.equal(p, new)


@pytest.mark.parametrize("d", [1, 5, 75])
def test_conv_looks_at_no_neighbours(pkg, d):
    """weights, bias and rows between NaN: a channel count that is no multiple of what a thread takes"""
    nan = torch.full((4, 4 * d + 64), float("nan"), device="cuda")
    x, w, b = _rand(20, d, dtype=F16), _rand(d, 4, seed=1), _rand(d, seed=2)
    nan[0, 16:16 + 4 * d], nan[1, 16:16 + d] = w.flatten(), b
    wide = torch.full((20, d + 9), float("nan"), dtype=F16, device="cuda")
    wide[:, 3:3 + d] = x
    wn, bn, xn = nan[0, 16:16 + 4 * d].view(d, 4), nan[1, 16:16 + d], wide[:, 3:3 + d]
    assert torch.equal(pkg.conv_seq(xn, wn, bn), pkg.conv_seq(x, w, b))
    assert torch.equal(pkg.conv_step(xn, wn, bn), pkg.conv_step(x, w, b))
    assert torch.isfinite(pkg.conv_seq(xn, wn, bn)).all()


def test_conv_seq_in_place_states_and_no_states(pkg):
    x, w, b = _rand(50, 64, dtype=F16), _rand(64, 4, seed=1), _rand(64, seed=2)
    starts, pool = [0, 1, 3, 50], _rand(3, 3, 64, dtype=F16, seed=3)
    p = pool.clone()
    got = pkg.conv_seq(x, w, b, starts=np.asarray(starts, np.int32), state=p)
    want, err, new = _conv_want(x, w, b, "silu", starts, pool, [0, 1, 2], [0, 1, 2])
    _check(got, want, err)
    assert torch.equal(p, new)
    want, err, _ = _conv_want(x, w, b, "silu", starts, None, None, None)
    _check(pkg.conv_seq(x, w, b, starts=torch.tensor(starts)), want, err)
    want, err, _ = _conv_want(x, w, b, "silu", [0, 50], None, None, None)
    _check(pkg.conv_seq(x, w, b), want, err)


@pytest.mark.parametrize("n,d,taps,dtype", [(1, 64, 4, F16), (5, 77, 4, BF16), (64, 512, 4, F16), (600, 12, 3, F32), (3, 1030, 2, BF16)])
def test_conv_step(pkg, n, d, taps, dtype):
    X, w, b = _rand(n, 2 * d, dtype=dtype), _rand(d, taps, seed=1), _rand(d, seed=2)
    x = X[:, d:]
    pool = _rand(2 * n, taps - 1, d, dtype=dtype, seed=3)
    fro, to = [n - 1 - i if i % 5 != 2 else -1 for i in range(n)], [n + i if i % 7 != 3 else -1 for i in range(n)]
    p = pool.clone()
    got = pkg.conv_step(x, w, b, state=p, from_slots=fro, to_slots=to)
    want, err, new = _conv_want(x, w, b, "silu", list(range(n + 1)), pool, fro, to)
    _check(got, want, err)
    assert torch.equal(p, new)
    # in place, slot i
    p = pool.clone()
    pkg.conv_step(x, w, b, state=p)
    _, _, new = _conv_want(x, w, b, "silu", list(range(n + 1)), pool, list(range(n)), list(range(n)))
    assert torch.equal(p, new)


def test_conv_tokens_follow_the_prompt(pkg):
    """a prompt in one piece, in pieces, and token by token: the same bits"""
    x, w, b = _rand(40, 96, dtype=F16), _rand(96, 4, seed=1), _rand(96, seed=2)
    whole = pkg.conv_seq(x, w, b)
    pool = torch.zeros((1, 3, 96), dtype=F16, device="cuda")
    parts = [pkg.conv_seq(x[:2], w, b, state=pool), pkg.conv_seq(x[2:25], w, b, state=pool)]
    parts += [pkg.conv_step(x[t:t + 1], w, b, state=pool) for t in range(25, 40)]
    assert torch.equal(torch.cat(parts), whole)
    assert torch.equal(pool[0], x[-3:])


# ---- selective scan ----------------------------------------------------------------------------------------------

def _ssm_inputs(rows, d, n, g, dtype, seed=0):
    wide = _rand(rows, 2 * d + 3 * g * n, dtype=dtype, seed=seed)
    x, z = wide[:, :d], wide[:, d:2 * d]
    B, C = wide[:, 2 * d:2 * d + g * n], wide[:, 2 * d + 2 * g * n:]
    dt = _rand(rows, d, dtype=dtype, scale=0.7, seed=seed + 1)
    A = -torch.arange(1, n + 1, device="cuda").float() * torch.exp(_rand(d, n, scale=0.3, seed=seed + 2))
    D, bias = _rand(d, seed=seed + 3), _rand(d, scale=1.0, seed=seed + 4) - 3
    return x, dt, A, B, C, D, z, bias


def _ssm_want(x, dt, A, B, C, D, z, bias, softplus, starts, pool, fro, to):
    """values and error bounds, carried along the recurrence: the decay exp(delta A) is off by EX2 + (the relative error of delta + three
    roundings) |delta A|, every product and sum by U32; delta by 1e-6 relative (fast exp, series and division) + what the rounding of its
    argument (of magnitude |dt| + |bias|) does to it, slope 1 at most times delta or less."""
    rows, d = x.shape
    n = A.shape[1]
    g = B.shape[1] // n
    xd, Ad = x.double(), A.double()
    raw = dt.double() + (bias.double() if bias is not None else 0)
    delta = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    mag = dt.double().abs() + (bias.double().abs() if bias is not None else 0)
    rd = 1.2e-6 + 4 * U32 * mag if softplus else 2 * U32 * mag / delta.abs().clamp(min=1e-300)       # relative error of delta
    y, ey = torch.zeros((rows, d), dtype=torch.float64, device="cuda"), torch.zeros((rows, d), dtype=torch.float64, device="cuda")
    new = pool.clone().double() if pool is not None else None
    enew = torch.zeros_like(new) if pool is not None else None
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        h = pool[fro[i]].double() if pool is not None and fro[i] >= 0 else torch.zeros((d, n), dtype=torch.float64, device="cuda")
        e = torch.zeros_like(h)
        for t in range(a, b):
            arg = delta[t][:, None] * Ad
            dec = torch.exp(arg)
            rel = EX2 + (rd[t][:, None] + 4 * U32) * arg.abs()
            Bt, Ct = (v[t].double().view(g, n).repeat_interleave(d // g, 0) for v in (B, C))
            add = (delta[t] * xd[t])[:, None] * Bt
            e = dec * (1 + rel) * e + dec * h.abs() * (rel + U32) + add.abs() * (rd[t][:, None] + 4 * U32)
            h = dec * h + add
            e = e + 2 * U32 * h.abs()
            v = (h * Ct).sum(1)
            ev = (e * Ct.abs()).sum(1) + (n + 4) * U32 * (h * Ct).abs().sum(1)
            if D is not None:
                v = v + D.double() * xd[t]
                ev = ev + 2 * U32 * (v.abs() + (D.double() * xd[t]).abs())
            if z is not None:
                zz = z[t].double()
                gate = zz * torch.sigmoid(zz)
                v, ev = v * gate, ev * gate.abs() + 1e-6 * (v * gate).abs()
            y[t], ey[t] = v, ev
        if new is not None and to[i] >= 0:
            new[to[i]], enew[to[i]] = h, e
    return y, ey, new, enew


SSM_SHAPES = [(8, 16, 1, F16), (64, 16, 1, BF16), (100, 16, 1, F32), (96, 16, 3, F16), (30, 5, 2, BF16), (33, 1, 1, F16), (64, 8, 2, F32),
              (48, 24, 1, F16), (40, 32, 2, BF16), (20, 64, 1, F32), (9, 100, 3, F16), (16, 128, 1, BF16), (264, 16, 1, F16)]


@pytest.mark.parametrize("lengths", [[1], [3], [32], [45], [0, 5, 0, 70, 1, 33], [200]], ids=str)
@pytest.mark.parametrize("d,n,g,dtype", SSM_SHAPES)
def test_ssm_seq(pkg, lengths, d, n, g, dtype):
    m = len(lengths)
    starts = np.cumsum([2] + lengths).tolist()
    rows = starts[-1] + 3
    x, dt, A, B, C, D, z, bias = _ssm_inputs(rows, d, n, g, dtype)
    pool = _rand(2 * m + 1, d, n, seed=9)
    fro, to = [i if i % 3 else -1 for i in range(m)], [2 * m - i if i % 4 != 1 else -1 for i in range(m)]
    for full in (True, False):
        p, out = pool.clone(), torch.full((rows, d), 7.0, dtype=dtype, device="cuda")
        kw = dict(D=D, z=z, dt_bias=bias) if full else dict(dt_softplus=False)
        dt_ = dt if full else dt.abs() * 0.1
        got = pkg.ssm_seq(x, dt_, A, B, C, starts=starts, state=p, from_slots=fro, to_slots=to, out=out, **kw)
        assert got is out
        y, ey, new, enew = _ssm_want(x, dt_, A, B, C, D if full else None, z if full else None, bias if full else None, full, starts, pool, fro, to)
        _check(out[2:starts[-1]], y[2:starts[-1]], ey[2:starts[-1]], "out")
        assert bool((out[:2] == 7).all()) and bool((out[starts[-1]:] == 7).all())
        _check(p, new, enew, "state")


@pytest.mark.parametrize("d,n,g,dtype", [(2056, 16, 1, F16), (2054, 16, 2, F32), (2560, 8, 1, BF16), (1600, 32, 2, F16), (1000, 64, 1, BF16), (160, 16, 1, F32), (1200, 16, 1, F16)])
def test_ssm_seq_of_wide_layers(pkg, d, n, g, dtype):
    """enough channels and sequences for every way of sharing the states among lanes"""
    lengths = [40, 7, 0, 64, 1, 12]
    starts = np.cumsum([0] + lengths).tolist()
    x, dt, A, B, C, D, z, bias = _ssm_inputs(starts[-1], d, n, g, dtype)
    for k in (6, 1):
        st = starts[:k + 1]
        pool = _rand(2 * k, d, n, seed=9)
        p = pool.clone()
        fro, to = [i if i % 3 else -1 for i in range(k)], [2 * k - 1 - i for i in range(k)]
        got = pkg.ssm_seq(x, dt, A, B, C, D=D, z=z, dt_bias=bias, starts=st, state=p, from_slots=fro, to_slots=to)
        y, ey, new, enew = _ssm_want(x, dt, A, B, C, D, z, bias, True, st, pool, fro, to)
        _check(got[:st[-1]], y[:st[-1]], ey[:st[-1]], "out")
        _check(p, new, enew, "state")


@pytest.mark.parametrize("streams", [1, 3, 40, 600])
@pytest.mark.parametrize("d,n,g,dtype", SSM_SHAPES)
def test_ssm_step(pkg, streams, d, n, g, dtype):
    x, dt, A, B, C, D, z, bias = _ssm_inputs(streams, d, n, g, dtype)
    pool = _rand(2 * streams, d, n, seed=9)
    fro, to = [streams - 1 - i if i % 5 != 2 else -1 for i in range(streams)], [streams + i if i % 7 != 3 else -1 for i in range(streams)]
    starts = list(range(streams + 1))
    p = pool.clone()
    got = pkg.ssm_step(x, dt, A, B, C, D=D, z=z, dt_bias=bias, state=p, from_slots=fro, to_slots=to)
    some = sorted({0, streams // 2, streams - 1, min(2, streams - 1), min(3, streams - 1)})
    want = [_ssm_want(v[0], v[1], A, v[2], v[3], D, v[4], bias, True, [0, 1], pool, [fro[i]], [to[i]])
            for i in some for v in [[t[i:i + 1] for t in (x, dt, B, C, z)]]]
    for i, (y, ey, new, enew) in zip(some, want):
        _check(got[i:i + 1], y, ey, i)
        if to[i] >= 0:
            _check(p[to[i]], new[to[i]], enew[to[i]], i)
    kept = sorted(set(range(2 * streams)) - {t for t in to if t >= 0})
    assert torch.equal(p[kept], pool[kept])
    # without a pool, and in place
    y, ey, _, _ = _ssm_want(x[:1], dt[:1], A, B[:1], C[:1], None, None, None, True, [0, 1], None, None, None)
    _check(pkg.ssm_step(x, dt, A, B, C)[:1], y, ey)
    p = pool.clone()
    again = pkg.ssm_step(x, dt, A, B, C, D=D, z=z, dt_bias=bias, state=p)
    y, ey, new, enew = _ssm_want(x[-1:], dt[-1:], A, B[-1:], C[-1:], D, z[-1:], bias, True, [0, 1], pool, [streams - 1], [streams - 1])
    _check(again[-1:], y, ey)
    _check(p[streams - 1], new[streams - 1], enew[streams - 1])


@pytest.mark.parametrize("rows,d,n", [(3000, 32, 16), (5000, 64, 4), (2500, 16, 40)])
def test_ssm_long_narrow_prompts(pkg, rows, d, n):
    """few channels and many rows: pieces of the sequence side by side, joined; the error bound of a scan that decays"""
    x, dt, A, B, C, D, z, bias = _ssm_inputs(rows, d, n, 1, F16)
    for starts, fro, to in (([0, rows], [1], [0]), ([0, 7, rows - 300, rows - 300, rows], [-1, 2, 1, 3], [4, 5, 6, 3])):
        pool = _rand(7, d, n, seed=9)
        p = pool.clone()
        got = pkg.ssm_seq(x, dt, A, B, C, D=D, z=z, dt_bias=bias, starts=starts, state=p, from_slots=fro, to_slots=to)
        y, ey, new, enew = _ssm_want(x, dt, A, B, C, D, z, bias, True, starts, pool, fro, to)
        # a piece's decay is the exponential of a sum of up to 1,024 time steps, off by as many roundings of it: |x| exp(-|x|) <= 0.37 of the state
        extra = 1024 * U32 * 0.37 * max(1.0, float(new.abs().max()))
        _check(got, y, ey + extra * C.double().abs().sum(1, keepdim=True) * (z.double().abs() + 1), "out")
        _check(p, new, enew + extra, "state")


def test_ssm_tokens_follow_the_prompt(pkg):
    d, n = 64, 16
    x, dt, A, B, C, D, z, bias = _ssm_inputs(60, d, n, 1, F32)
    kw = dict(D=D, dt_bias=bias)
    pool = torch.zeros((3, d, n), device="cuda")
    whole = pkg.ssm_seq(x, dt, A, B, C, z=z, state=pool, to_slots=[1], from_slots=-1, **kw)
    parts = [pkg.ssm_seq(x[:33], dt[:33], A, B[:33], C[:33], z=z[:33], state=pool, from_slots=-1, to_slots=[0], **kw)]
    parts += [pkg.ssm_step(x[t:t + 1], dt[t:t + 1], A, B[t:t + 1], C[t:t + 1], z=z[t:t + 1], state=pool, **kw) for t in range(33, 60)]
    y, ey, new, enew = _ssm_want(x, dt, A, B, C, D, z, bias, True, [0, 60], torch.zeros_like(pool), [0], [0])
    _check(torch.cat(parts), y, ey)
    _check(whole, y, ey)
    _check(pool[0], new[0], enew[0])
    _check(pool[1], new[0], enew[0])


def test_ssm_extremes(pkg):
    """time steps of 0 and far from it, decays of 0, NaN of one row or channel that stay where they belong"""
    d, n, rows = 40, 16, 70
    x, dt, A, B, C, D, z, bias = _ssm_inputs(rows, d, n, 1, F32)
    dt[:, 0], dt[:, 1] = -1e30, 1e4
    A[2] = -float("inf")
    y, ey, new, enew = _ssm_want(x, dt, A, B, C, D, z, bias, True, [0, rows], torch.zeros((1, d, n), device="cuda"), [-1], [0])
    p = torch.zeros((1, d, n), device="cuda")
    got = pkg.ssm_seq(x, dt, A, B, C, D=D, z=z, dt_bias=bias, state=p, from_slots=-1)
    fine = [c for c in range(d) if c not in (0, 2)]
    _check(got[:, fine], y[:, fine], ey[:, fine])
    _check(got[:, 0], (D[0].double() * x[:, 0].double() * z[:, 0].double() * torch.sigmoid(z[:, 0].double())), 1e-6 * torch.ones(rows, device="cuda", dtype=torch.float64))
    # the decay of channel 2 is 0: a row has what it adds itself, and the state stays finite behind the last row
    delta = torch.nn.functional.softplus(dt[:, 2].double() + bias[2].double())
    want = delta[-1] * x[-1, 2].double() * B[-1].double()
    _check(p[0, 2], want, 1e-5 * want.abs())
    x2 = x.clone()
    x2[30, 5] = float("nan")
    got2 = pkg.ssm_seq(x2, dt, A, B, C, D=D, z=z, dt_bias=bias)
    assert torch.isnan(got2[30:, 5]).all()
    rest = [c for c in range(d) if c != 5]
    assert torch.equal(got2[:, rest], got[:, rest]) and torch.equal(got2[:30], got[:30])


@pytest.mark.parametrize("d,n,dtype", [(24, 5, F16), (13, 5, F32), (16, 16, F16), (10, 3, BF16), (40, 70, F32)])
def test_ssm_infinite_inputs(pkg, d, n, dtype):
    """an infinite x makes its channel infinite, as the formula does: what fills up the lanes behind the last state adds no 0 x inf"""
    rows = 40
    x, dt, A, B, C, D, z, bias = _ssm_inputs(rows, d, n, 1, dtype)
    x, B, C = x.clone(), B.abs().contiguous(), C.abs().contiguous()
    x[7, 4], x[39, 6] = float("inf"), float("-inf")
    pool = torch.zeros((rows, d, n), device="cuda")
    y, ey, new, _ = _ssm_want(x, dt, A, B, C, None, z, bias, True, [0, rows], pool[:1], [-1], [0])
    assert torch.isinf(y[7:, 4]).all() and torch.isinf(y[39, 6])
    p = pool[:1].clone()
    _check(pkg.ssm_seq(x, dt, A, B, C, z=z, dt_bias=bias, state=p, from_slots=-1), y, ey)
    assert torch.equal(torch.isinf(p), torch.isinf(new)) and not torch.isnan(p).any()
    y, ey, new, _ = _ssm_want(x, dt, A, B, C, None, z, bias, True, list(range(rows + 1)), pool, list(range(rows)), list(range(rows)))
    p = pool.clone()
    _check(pkg.ssm_step(x, dt, A, B, C, z=z, dt_bias=bias, state=p), y, ey)
    assert torch.equal(torch.isinf(p), torch.isinf(new)) and not torch.isnan(p).any()


# ---- slots -------------------------------------------------------------------------------------------------------

def _moved(pool, src, dst):
    new = pool.clone()
    for a, b in zip(src, dst):
        new[b] = pool[a] if a >= 0 else 0
    return new


@pytest.mark.parametrize("dtype,row", [(F32, 1), (F32, 4), (F32, 1000), (F32, 40003), (F16, 1001), (F16, 8), (torch.uint8, 333), (torch.uint8, 4096), (BF16, 70002)])
def test_copy_slots(pkg, dtype, row):
    slots, rng = 37, np.random.default_rng(row)
    pool = torch.randint(0, 200, (slots, row), device="cuda").to(dtype)
    cases = {"fork": ([3] * 20, list(range(10, 30))), "swap": ([1, 0], [0, 1]), "ring": (list(range(slots)), [(i + 1) % slots for i in range(slots)]),
             "clear": ([-1, -1, 5], [4, 36, 0]), "same": ([7, 8], [7, 8]), "none": ([], []), "chain": ([5, 4, 3, 2], [6, 5, 4, 3]),
             "any": (rng.integers(-1, slots, slots).tolist(), rng.permutation(slots).tolist()), "one": ([36], [0])}
    for name, (src, dst) in cases.items():
        p = pool.clone()
        assert pkg.copy_slots(p, src, np.asarray(dst, np.int32)) is p
        assert torch.equal(p, _moved(pool, src, dst)), name


def test_copy_slots_of_a_wider_pool_and_many(pkg):
    wide = torch.randn((300, 5, 70), device="cuda")
    keep = wide.clone()
    view = wide[:, 1:3]                      # slots of 140 elements, 350 apart
    src, dst = list(range(299, -1, -1)), list(range(300))
    pkg.copy_slots(view, src, dst)
    assert torch.equal(wide[:, 1:3], keep[:, 1:3].flip(0)) and torch.equal(wide[:, 0], keep[:, 0]) and torch.equal(wide[:, 3:], keep[:, 3:])
    many = torch.randint(0, 1 << 30, (4096, 13), device="cuda", dtype=torch.int32)
    order = np.random.default_rng(1).permutation(4096)
    want = many[torch.from_numpy(order).cuda()]
    pkg.copy_slots(many, order.astype(np.int32), np.arange(4096, dtype=np.int32))
    assert torch.equal(many, want)


@pytest.mark.parametrize("shape_name,strategy", [("tiny4", "cuda fp16"), ("tiny4", "cuda int4"), ("tiny52", "cuda fp16")])
def test_model_copy_states(pkg, synth, shape_name, strategy):
    """streams forked after a prompt go on as the first; a cleared one begins anew; a chain of moves closes a gap"""
    shape = synth.SHAPES[shape_name]
    tensors = synth.to_file_dtypes(shape, synth.generate(shape, 3, ln_random=True), "fp16" if strategy.endswith("fp16") else "fp32")
    m = pkg.Model(tensors, strategy, shape=shape, max_batch=4)
    fresh = m.export_state(3)
    m.run([5, 9, 2])                                   # an odd number of tokens: the shift states lie in their other copy
    m.copy_states([0, 0], [1, 3])
    a = m.export_state(0)
    assert np.array_equal(a, m.export_state(1)) and np.array_equal(a, m.export_state(3))
    y = m.decode([7, 7, 1, 7])
    assert np.array_equal(y[0], y[1]) and np.array_equal(y[0], y[3])
    states = [m.export_state(i) for i in range(4)]
    m.copy_states([1, 2, -1], [0, 1, 2])               # stream 0 has finished
    assert np.array_equal(m.export_state(0), states[1]) and np.array_equal(m.export_state(1), states[2])
    assert np.array_equal(m.export_state(2), fresh) and np.array_equal(m.export_state(3), states[3])
    for bad in (([0], [4]), ([4], [0]), ([0, 1], [2, 2]), ([-2], [0])):
        with pytest.raises(pkg.FrB200Error):
            m.copy_states(*bad)
    before = [m.export_state(i) for i in range(4)]
    m.copy_states([0, 3], [0, 3])
    m.copy_states([], [])
    assert all(np.array_equal(m.export_state(i), b) for i, b in enumerate(before))
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    one = (np.array([0], np.int32), np.array([1], np.int32))
    with torch.cuda.graph(g, stream=s):
        rc = pkg.lib().fr_b200_state_copy(m.handle, 1, one[0].ctypes.data, one[1].ctypes.data, s.cuda_stream)
    assert rc == -4                                    # a capture is refused
    m.close()


# ---- what does not fit together ----------------------------------------------------------------------------------

def test_tensors_that_do_not_fit_are_refused(pkg):
    x, w, b = _rand(4, 64, dtype=F16), _rand(32, 64, dtype=F16), _rand(32)
    cw, pool = _rand(64, 4), _rand(6, 3, 64, dtype=F16)
    A, B, ssm = _rand(64, 8), _rand(4, 16, dtype=F16), _rand(6, 64, 8)
    no = [lambda: pkg.linear(x, w.bfloat16()), lambda: pkg.linear(x, w.cpu()), lambda: pkg.linear(x, w[:, :60]), lambda: pkg.linear(x.t(), w), lambda: pkg.linear(x[0], w),
          lambda: pkg.linear(x, w, b.half()), lambda: pkg.linear(x, w, b[:31]), lambda: pkg.linear(x, w, residual=_rand(4, 32)), lambda: pkg.linear(x, w, residual=_rand(5, 32, dtype=F16)),
          lambda: pkg.linear(x, w, out=_rand(4, 31, dtype=F16)), lambda: pkg.linear(x, w, out_dtype=torch.float64), lambda: pkg.linear(x, w, out_dtype="f32"),
          lambda: pkg.linear(x.double(), w.double()), lambda: pkg.conv_step(x, cw[:, 0]), lambda: pkg.conv_step(x, cw.t()), lambda: pkg.conv_step(x, cw, state=pool.float()),
          lambda: pkg.conv_step(x, cw, state=pool[:, :2]), lambda: pkg.conv_step(x, cw, state=pool.transpose(1, 2)), lambda: pkg.conv_step(x, cw, state=pool, from_slots=[0, 1, 2]),
          lambda: pkg.conv_step(x, cw, state=pool, from_slots=[0, 1, 2, 1.5]), lambda: pkg.conv_step(x, cw, state=pool, to_slots=[0, 1, 2, 1 << 40]),
          lambda: pkg.conv_step(x, cw, state=pool, to_slots=torch.arange(4, device="cuda")), lambda: pkg.conv_step(x, cw, state=pool, to_slots=np.zeros((4, 1), np.int32)),
          lambda: pkg.conv_seq(x, cw, starts=[]), lambda: pkg.conv_seq(x, cw, starts="12"), lambda: pkg.ssm_step(x, x, A, B, B[:, :8]), lambda: pkg.ssm_step(x, x, A, B[:, :12], B[:, :12]),
          lambda: pkg.ssm_step(x, x[:, :32], A, B, B), lambda: pkg.ssm_step(x, x.float(), A, B, B), lambda: pkg.ssm_step(x, x, A[:60], B, B), lambda: pkg.ssm_step(x, x, A, B[:3], B[:3]),
          lambda: pkg.ssm_step(x, x, A, B, B, z=x[:3]), lambda: pkg.ssm_step(x, x, A, B, B, state=ssm.half()), lambda: pkg.ssm_seq(x, x, A, B, B, D=_rand(63)),
          lambda: pkg.copy_slots(pool.transpose(1, 2), [0], [1]), lambda: pkg.copy_slots(pool, [0, 1], [1]), lambda: pkg.copy_slots(pool, None, [1]), lambda: pkg.copy_slots(pool, [0], 1)]
    for i, f in enumerate(no):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    lib = [lambda: pkg.linear(x.float(), w.float()), lambda: pkg.linear(x, w, out=x[:, :32]), lambda: pkg.conv_step(x, cw, activation="gelu"), lambda: pkg.conv_step(x, cw, out=x),
           lambda: pkg.conv_step(x, cw, state=pool, from_slots=[0, 1, 2, 6]), lambda: pkg.conv_step(x, cw, state=pool, to_slots=[0, 1, 2, 2]), lambda: pkg.conv_seq(x, cw, starts=[0, 5]),
           lambda: pkg.conv_seq(x, cw, starts=[3, 1]), lambda: pkg.conv_seq(x, cw, from_slots=[0]), lambda: pkg.ssm_seq(x, x.clone(), A, B, B, out=x),
           lambda: pkg.ssm_step(x, x, A, B, B, state=ssm[:3]), lambda: pkg.copy_slots(pool, [0, 1], [2, 2]), lambda: pkg.copy_slots(pool, [0], [6])]
    for i, f in enumerate(lib):
        with pytest.raises(pkg.FrB200Error):
            f()
            pytest.fail(f"call {i} was taken")


def test_lists_of_every_kind(pkg):
    x, w, pool = _rand(3, 8, dtype=F16), _rand(8, 4), _rand(5, 3, 8, dtype=F16)
    want = pkg.conv_step(x, w, state=pool.clone(), from_slots=[4, -1, 0], to_slots=[3, 1, 2])
    for f, t in (((4, -1, 0), (3, 1, 2)), (np.array([4, -1, 0], np.int32), np.array([3, 1, 2], np.int64)), (torch.tensor([4, -1, 0]), torch.tensor([3, 1, 2], dtype=torch.int32)),
                 (np.array([4, 9, -1, 9, 0, 9], np.int32)[::2], [np.int16(3), np.int64(1), 2])):
        p = pool.clone()
        assert torch.equal(pkg.conv_step(x, w, state=p, from_slots=f, to_slots=t), want)
        assert torch.equal(p[3, -1], x[0]) and torch.equal(p[1, -1], x[1]) and torch.equal(p[2, -1], x[2])
    assert torch.equal(pkg.conv_step(x, w, state=pool, from_slots=-1, to_slots=-1), pkg.conv_step(x, w))


# ---- together ----------------------------------------------------------------------------------------------------

class _Layer:
    """A selective state space layer: projection in, convolution, projections of the scan's inputs, scan, projection onto the residual."""

    def __init__(self, pkg, c=64, n=8, rank=16, dtype=F16):
        self.pkg, self.c, self.d, self.n, self.rank = pkg, c, 2 * c, n, rank
        d = self.d
        self.w_in, self.w_x = _rand(2 * d, c, dtype=dtype, scale=c ** -0.5), _rand(rank + 2 * n, d, dtype=dtype, scale=d ** -0.5, seed=1)
        self.w_dt, self.w_out = _rand(d, rank, dtype=dtype, scale=rank ** -0.5, seed=2), _rand(c, d, dtype=dtype, scale=d ** -0.5, seed=3)
        self.conv_w, self.conv_b = _rand(d, 4, scale=0.5, seed=4), _rand(d, seed=5)
        self.A, self.D, self.dt_b = -torch.exp(_rand(d, n, scale=0.5, seed=6)), _rand(d, seed=7), _rand(d, seed=8) - 2
        self.conv, self.ssm = torch.zeros((8, 3, d), dtype=dtype, device="cuda"), torch.zeros((8, d, n), device="cuda")

    def __call__(self, u, starts=None, **slots):
        p, d, n, r = self.pkg, self.d, self.n, self.rank
        xz = p.linear(u, self.w_in)
        if starts is None:
            x = p.conv_step(xz[:, :d], self.conv_w, self.conv_b, state=self.conv, **slots)
        else:
            x = p.conv_seq(xz[:, :d], self.conv_w, self.conv_b, starts=starts, state=self.conv, **slots)
        x_dbl = p.linear(x, self.w_x)
        dt = p.linear(x_dbl[:, :r], self.w_dt, self.dt_b, activation="softplus")
        a = (x, dt, self.A, x_dbl[:, r:r + n], x_dbl[:, r + n:])
        kw = dict(D=self.D, z=xz[:, d:], dt_softplus=False, state=self.ssm, **slots)
        y = p.ssm_step(*a, **kw) if starts is None else p.ssm_seq(*a, starts=starts, **kw)
        return p.linear(y, self.w_out, residual=u)

    def want(self, u):
        """one sequence from the start, in 64 bits, with the roundings of what is stored between the operators"""
        d, n, r, t = self.d, self.n, self.rank, u.dtype
        q = lambda v: v.to(t).double()  # noqa: E731
        xz = q(u.double() @ self.w_in.double().t())
        x, _, _ = _conv_want(xz[:, :d].to(t), self.conv_w, self.conv_b, "silu", [0, len(u)], None, None, None)
        x = q(x)
        dbl = q(x @ self.w_x.double().t())
        v = dbl[:, :r] @ self.w_dt.double().t() + self.dt_b.double()
        dt = q(torch.logaddexp(v, torch.zeros_like(v)))
        y, _, _, _ = _ssm_want(x, dt, self.A, dbl[:, r:r + n], dbl[:, r + n:], self.D, xz[:, d:], None, False, [0, len(u)], None, None, None)
        return q(q(y) @ self.w_out.double().t() + u.double())


def test_layer_prompts_then_tokens_then_a_fork(pkg):
    """Prompts of three streams back to back, tokens of all, one stream forked into two slots that go different ways: each stream as
    if it had run alone.  The stored values are rounded at the same places; an operand that falls on the other side of such a step moves
    it by eps, which the layer's gains (sums of unit variance) hand on: 32 half steps of values up to 8."""
    layer, c = _Layer(pkg), 64
    lengths = [5, 1, 37]
    prompts = [_rand(m, c, dtype=F16, seed=40 + m) for m in lengths]
    starts = np.cumsum([0] + lengths).astype(np.int32)
    out = layer(torch.cat(prompts), starts=starts, from_slots=-1, to_slots=[0, 1, 2])
    seen = [[p] for p in prompts] + [[prompts[2]]]
    got = [[out[a:b]] for a, b in zip(starts, starts[1:])] + [[out[starts[2]:]]]
    for step in range(3):
        u = _rand(3, c, dtype=F16, seed=60 + step)
        y = layer(u, from_slots=[0, 1, 2], to_slots=[0, 1, 2])
        for i in range(4):
            seen[i].append(u[min(i, 2):min(i, 2) + 1])
            got[i].append(y[min(i, 2):min(i, 2) + 1])
    for pool in (layer.conv, layer.ssm):
        pkg.copy_slots(pool, [2], [3])
    for step in range(3):
        u = _rand(4, c, dtype=F16, seed=80 + step)
        y = layer(u, from_slots=[0, 1, 2, 3], to_slots=[0, 1, 2, 3])
        for i in range(4):
            seen[i].append(u[i:i + 1])
            got[i].append(y[i:i + 1])
    for s, g in zip(seen, got):
        want = layer.want(torch.cat(s))
        off = (torch.cat(g).double() - want).abs().max()
        assert float(off) <= 32 * _half_step(F16) * 8, float(off)


def test_layer_captured_and_replayed(pkg):
    """Two captured graphs of the same layer at different sizes, replayed in turn with new inputs: the calls' own results."""
    layer, eager = _Layer(pkg), _Layer(pkg)
    u4, u9 = _rand(4, 64, dtype=F16, seed=1), _rand(90, 64, dtype=F16, seed=2)
    starts = [0, 30, 90]
    calls = {"step": (u4, lambda la, u: la(u, from_slots=[3, 2, 1, 0], to_slots=[4, 5, 6, 7])),
             "seq": (u9, lambda la, u: la(u, starts=starts, from_slots=[5, -1], to_slots=[0, 3]))}
    for u, f in calls.values():
        f(layer, u)
        f(eager, u)
    torch.cuda.synchronize()
    graphs = {}
    for name, (u, f) in calls.items():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f(layer, u)
        graphs[name] = (g, out)
    for pool in ("conv", "ssm"):
        getattr(layer, pool).copy_(getattr(eager, pool))
    for i in range(4):
        for name, (u, f) in calls.items():
            u.copy_(_rand(*u.shape, dtype=F16, seed=100 + i))
            graphs[name][0].replay()
            want = f(eager, u)
            torch.cuda.synchronize()
            assert torch.equal(graphs[name][1], want), (i, name)
    assert torch.equal(layer.conv, eager.conv) and torch.equal(layer.ssm, eager.ssm)


def test_offsets_past_32_bits(pkg):
    """rows and slots so far apart that elements and bytes between the first and the last pass 2^31 and 2^32: what they give side by side"""
    rows, d, n, far = 40, 64, 16, 2 ** 26 + 8
    space = torch.empty(rows * far, dtype=BF16, device="cuda")             # 5.4 GB, of which a few rows are touched
    assert (rows - 1) * far > 2 ** 31

    def spread(t, at):
        v = space.as_strided((rows, t.shape[1]), (far, 1), at)
        v.copy_(t)
        return v

    x, dt, A, B, C, D, z, bias = _ssm_inputs(rows, d, n, 1, BF16)
    fx, fdt, fB, fC, fz = (spread(t, at) for t, at in ((x, 0), (dt, 128), (B, 256), (C, 320), (z, 384)))
    fout = spread(torch.zeros_like(x), 512)
    w, b = _rand(96, d, dtype=BF16, scale=0.1, seed=3), _rand(d, 4, seed=4)
    for m in (8, rows):
        assert torch.equal(pkg.linear(fx[-m:], w), pkg.linear(x[-m:].contiguous(), w))
        y = spread(torch.zeros((rows, 96), dtype=BF16, device="cuda"), 640)[-m:]
        pkg.linear(fx[-m:], w, residual=y, out=y)
        assert torch.equal(y, pkg.linear(x[-m:].contiguous(), w))
    assert torch.equal(pkg.conv_seq(fx, b, out=fout), pkg.conv_seq(x, b))
    assert torch.equal(pkg.conv_step(fx, b, out=fout), pkg.conv_step(x, b))
    kw = dict(D=D, dt_bias=bias)
    assert torch.equal(pkg.ssm_seq(fx, fdt, A, fB, fC, z=fz, out=fout, **kw), pkg.ssm_seq(x, dt, A, B, C, z=z, **kw))
    assert torch.equal(pkg.ssm_step(fx, fdt, A, fB, fC, z=fz, out=fout, **kw), pkg.ssm_step(x, dt, A, B, C, z=z, **kw))
    del space, fx, fdt, fB, fC, fz, fout, y
    store = torch.empty(rows * far, dtype=F32, device="cuda")              # 10.7 GB
    pool, near = store.as_strided((rows, d, n), (far, n, 1)), _rand(rows, d, n, seed=5)
    pool.copy_(near)
    order, first = list(range(rows - 1, -1, -1)), [rows - 1 - i for i in range(rows)]
    pkg.copy_slots(pool, order, list(range(rows)))
    pkg.copy_slots(near, order, list(range(rows)))
    assert torch.equal(pool, near)
    assert torch.equal(pkg.ssm_step(x, dt, A, B, C, state=pool, from_slots=first, to_slots=first, **kw),
                       pkg.ssm_step(x, dt, A, B, C, state=near, from_slots=first, to_slots=first, **kw))
    assert torch.equal(pool, near)
    starts = [0, 7, 7, rows]
    assert torch.equal(pkg.ssm_seq(x, dt, A, B, C, state=pool, starts=starts, from_slots=[39, 0, 38], to_slots=[39, 37, 38], **kw),
                       pkg.ssm_seq(x, dt, A, B, C, state=near, starts=starts, from_slots=[39, 0, 38], to_slots=[39, 37, 38], **kw))
    assert torch.equal(pool, near)


def test_more_sequences_than_a_launch_holds(pkg):
    lengths = [(i * 7) % 5 for i in range(600)]
    starts = np.cumsum([0] + lengths).tolist()
    rows, d, n = starts[-1], 24, 8
    to = [(i * 77) % 601 for i in range(600)]
    fro = [t if i % 3 else -1 for i, t in enumerate(to)]
    x, w, b = _rand(rows, d, dtype=F16), _rand(d, 4, seed=1), _rand(d, seed=2)
    pool = _rand(601, 3, d, dtype=F16, seed=3)
    p = pool.clone()
    want, err, new = _conv_want(x, w, b, "silu", starts, pool, fro, to)
    _check(pkg.conv_seq(x, w, b, starts=starts, state=p, from_slots=fro, to_slots=to), want, err)
    assert torch.equal(p, new)
    x, dt, A, B, C, D, z, bias = _ssm_inputs(rows, d, n, 1, F16)
    pool = _rand(601, d, n, seed=4)
    p = pool.clone()
    y, ey, new, enew = _ssm_want(x, dt, A, B, C, D, z, bias, True, starts, pool, fro, to)
    _check(pkg.ssm_seq(x, dt, A, B, C, D=D, z=z, dt_bias=bias, starts=starts, state=p, from_slots=fro, to_slots=to), y, ey)
    _check(p, new, enew)


@pytest.mark.parametrize("k,n", [(72, 40), (71, 39), (8, 264)])
def test_linear_of_many_rows(pkg, k, n):
    x, w, b = _rand(100003, k, dtype=F16), _rand(n, k, dtype=F16, scale=0.2, seed=1), _rand(n, seed=2)
    want, err = _linear_want(x, w, b, "silu", None)
    _check(pkg.linear(x, w, b, activation="silu"), want, err)
