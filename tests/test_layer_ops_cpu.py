"""What the operators of a recurrent layer refuse, before anything is launched: shapes, types, alignment, overlaps, sequences
and slots.  Addresses here are numbers: no call gets as far as a device."""
import ctypes

import numpy as np
import pytest
import torch

F16, F32, BF16 = 0, 1, 2
X, W, O, R, S = (0x10000000 * i for i in range(1, 6))      # tensors far apart


def _i32(*v):
    return (ctypes.c_int32 * len(v))(*v)


def _refused(pkg, name, args, word):
    L = pkg.lib()
    assert getattr(L, name)(*args) == -1, name
    assert word in L.fr_b200_op_last_error().decode(), L.fr_b200_op_last_error()


def _linear(**kw):
    a = dict(x=X, ldx=64, w=W, ldw=64, dtype=F16, rows=4, K=64, N=32, bias=None, act=0, residual=None, ldr=0, out=O, ldo=32, out_dtype=F16, work=None, work_bytes=0,
             device=0, stream=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=F32), "f16 or bf16"), (dict(dtype=9), "f16 or bf16"), (dict(out_dtype=BF16), "out has the type"), (dict(act=6), "activation"),
    (dict(act=-1), "activation"), (dict(K=0), "shape"), (dict(N=0), "shape"), (dict(rows=-1), "shape"), (dict(rows=65535 * 64 + 1), "shape"), (dict(N=(1 << 24) + 1, ldo=1 << 25), "shape"), (dict(K=(1 << 24) + 1, ldx=1 << 25, ldw=1 << 25), "shape"),
    (dict(ldx=63), "closer"), (dict(ldw=0), "closer"), (dict(ldo=31), "closer"), (dict(residual=R, ldr=31), "closer"), (dict(x=None), "null"),
    (dict(w=None), "null"), (dict(out=None), "null"), (dict(x=X + 1), "misaligned"), (dict(bias=R + 2), "misaligned"),
    (dict(out_dtype=F32, out=O + 2), "misaligned"), (dict(out=X), "overlaps x"), (dict(out=W + 64), "overlaps x"), (dict(out=X + 2 * 64 * 3), "overlaps x"),
    (dict(rows=4000, K=1001, ldx=1001, ldw=1001, N=100, ldo=100, out=O, work=S, work_bytes=4100 * 126 * 16 - 1), "work area"), (dict(work=S + 8, work_bytes=99), "work area"),
    (dict(bias=O), "bias"), (dict(residual=O + 2, ldr=32), "residual"), (dict(residual=O, ldr=40), "residual"),
])
def test_linear_refuses(pkg, kw, word):
    _refused(pkg, "fr_b200_linear", _linear(**kw), word)


def _conv(**kw):
    a = dict(x=X, ldx=64, dtype=F16, rows=20, D=64, w=W, taps=4, bias=None, act=2, starts=None, n_seq=1, state=S, state_stride=192, n_slots=4, fro=None,
             to=None, out=O, ldo=64, device=0, stream=None)
    a.update(kw)
    return tuple(a.values())


SLOTS = [(dict(fro=_i32(4), to=_i32(0)), "read is out of range"), (dict(fro=_i32(-2)), "read is out of range"), (dict(to=_i32(4)), "write is out of range"),
         (dict(to=_i32(-2)), "write is out of range"), (dict(state=None, n_slots=0, fro=_i32(0)), "without a pool"), (dict(n_slots=0), "slots"),
         (dict(state_stride=191), "smaller"), (dict(state=S + 1), "misaligned")]


@pytest.mark.parametrize("kw,word", SLOTS + [
    (dict(dtype=3), "dtype"), (dict(taps=1), "taps"), (dict(taps=5), "taps"), (dict(act=1), "none or silu"), (dict(D=0), "shape"), (dict(D=(1 << 24) + 1), "shape"), (dict(rows=-1), "shape"),
    (dict(rows=1 << 31), "rows"), (dict(ldx=63), "shape"), (dict(ldo=63), "shape"), (dict(w=None), "null"), (dict(x=None), "null"), (dict(out=None), "null"),
    (dict(out=O + 1), "misaligned"), (dict(out=X + 128), "out overlaps"), (dict(out=S), "pool"), (dict(x=S + 128), "pool"),
    (dict(n_seq=2), "first rows"), (dict(n_seq=-1), "negative"), (dict(starts=_i32(-1, 5)), "outside"), (dict(starts=_i32(0, 21)), "outside"),
    (dict(starts=_i32(0, 9, 8), n_seq=2), "ends before"), (dict(starts=_i32(0, 9, 20), n_seq=2, to=_i32(1, 1)), "two streams"),
    (dict(starts=_i32(0, 9, 20), n_seq=2, fro=_i32(1, 2), to=_i32(2, 3)), "read by another"),
    (dict(starts=_i32(0, 1, 2, 3, 4, 5), n_seq=5), "more streams"),
])
def test_conv_seq_refuses(pkg, kw, word):
    _refused(pkg, "fr_b200_conv_seq", _conv(**kw), word)


@pytest.mark.parametrize("kw,word", SLOTS + [(dict(n_seq=9), "more streams")])
def test_conv_step_refuses(pkg, kw, word):
    a = dict(zip(("x", "ldx", "dtype", "rows", "D", "w", "taps", "bias", "act", "starts", "n_seq", "state", "state_stride", "n_slots", "fro", "to", "out",
                  "ldo", "device", "stream"), _conv(**kw)))
    a["rows"] = 5 if word == "more streams" else 1
    a.pop("starts"), a.pop("n_seq")
    _refused(pkg, "fr_b200_conv_step", tuple(a.values()), word)


def _ssm(seq=True, **kw):
    a = dict(x=X, ldx=64, dt=X + 0x1000000, lddt=64, A=W, B=X + 0x2000000, ldb=16, C=X + 0x3000000, ldc=16, D=None, z=None, ldz=0, bias=None, sp=1, dtype=F16,
             rows=20, d=64, n=16, groups=1, starts=None, n_seq=1, state=S, state_stride=1024, n_slots=4, fro=None, to=None, out=O, ldo=64, work=None, wb=0,
             device=0, stream=None)
    if not seq:
        a["rows"] = 1
    a.update(kw)
    if not seq:
        for k in ("starts", "n_seq", "work", "wb"):
            a.pop(k)
    return tuple(a.values())


SSM = [(dict(fro=_i32(4)), "read is out of range"), (dict(to=_i32(4)), "write is out of range"), (dict(state=None, n_slots=0, to=_i32(0)), "without a pool"),
       (dict(state_stride=1023), "smaller"), (dict(state=S + 2), "misaligned"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "shape"), (dict(d=0), "shape"), (dict(d=(1 << 23) + 1), "shape"),
       (dict(n=0), "states"), (dict(n=129), "states"), (dict(groups=0), "groups"), (dict(groups=3), "groups"), (dict(ldx=63), "closer"),
       (dict(lddt=1), "closer"), (dict(ldb=15), "closer"), (dict(ldc=31, groups=2), "closer"), (dict(z=R, ldz=63), "closer"), (dict(A=None), "null"),
       (dict(dt=None), "null"), (dict(B=None), "null"), (dict(out=None), "null"), (dict(out=O + 1), "misaligned"), (dict(A=W + 2), "misaligned"),
       (dict(out=X), "overlaps an input"), (dict(z=O, ldz=64), "overlaps an input"), (dict(C=S + 64), "overlaps an input"), (dict(out=S + 64), "overlaps the pool")]


@pytest.mark.parametrize("seq", [True, False])
@pytest.mark.parametrize("kw,word", SSM)
def test_ssm_refuses(pkg, kw, word, seq):
    _refused(pkg, "fr_b200_ssm_seq" if seq else "fr_b200_ssm_step", _ssm(seq, **kw), word)


def test_ssm_seq_refuses_sequences(pkg):
    for kw, word in ((dict(n_seq=2), "first rows"), (dict(starts=_i32(0, 21)), "outside"), (dict(starts=_i32(5, 4)), "ends before"),
                     (dict(starts=_i32(0, 4, 9), n_seq=2, to=_i32(3, 3)), "two streams")):
        _refused(pkg, "fr_b200_ssm_seq", _ssm(**kw), word)


def test_slots_copy_refuses(pkg):
    ok = (S, 64, 64, 8)
    for args, word in (((None, 64, 64, 8, 1, _i32(0), _i32(1)), "bad argument"), ((S, 0, 64, 8, 1, _i32(0), _i32(1)), "bad argument"),
                       ((S, 65, 64, 8, 1, _i32(0), _i32(1)), "bad argument"), ((S, 64, 64, 0, 1, _i32(0), _i32(1)), "slots"),
                       ((S, 64, 64, 65536, 1, _i32(0), _i32(1)), "slots"), (ok + (-1, _i32(0), _i32(1)), "moves"), (ok + (4097, _i32(0), _i32(1)), "moves"),
                       (ok + (1, None, _i32(1)), "null"), (ok + (1, _i32(0), None), "null"), (ok + (1, _i32(8), _i32(1)), "range"),
                       (ok + (1, _i32(-2), _i32(1)), "range"), (ok + (1, _i32(0), _i32(-1)), "range"), (ok + (1, _i32(0), _i32(8)), "range"),
                       (ok + (2, _i32(0, 1), _i32(3, 3)), "twice")):
        _refused(pkg, "fr_b200_slots_copy", args + (0, None), word)
    assert pkg.lib().fr_b200_state_copy(None, 0, None, None, None) == -1


def test_columns_of_the_same_rows_do_not_overlap(pkg):
    """x and out as halves of the same rows pass the check of overlaps (and stop at the missing device, without a GPU)"""
    if torch.cuda.is_available():
        pytest.skip("GPU present: the addresses are not memory")
    L = pkg.lib()
    rc = L.fr_b200_conv_seq(*_conv(ldx=128, ldo=128, out=X + 128))
    assert rc == -3
    _refused(pkg, "fr_b200_conv_seq", _conv(ldx=128, ldo=128, out=X + 126), "out overlaps")
    _refused(pkg, "fr_b200_conv_seq", _conv(ldx=128, ldo=128, out=X + 130), "out overlaps")
    assert L.fr_b200_linear(*_linear(rows=0, x=None, out=None)) == 0
    assert L.fr_b200_linear(*_linear()) == -3


def test_tensors_that_are_refused(pkg):
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="GPU"):
        pkg.linear(x, x)
    with pytest.raises(ValueError, match="GPU"):
        pkg.conv_step(x, x)
    with pytest.raises(ValueError, match="GPU"):
        pkg.ssm_seq(x, x, x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        pkg.copy_slots(x, [0], [1])
    for bad in ("tanh", None, 3):
        with pytest.raises(ValueError, match="activation"):
            pkg.linear(x, x, activation=bad)
    with pytest.raises(ValueError, match="not a tensor"):
        pkg.linear([1], x)


@pytest.mark.parametrize("seed", range(4))
def test_slots_are_checked_call_by_call(pkg, seed):
    """the record of who writes which slot is the call's own"""
    L, rng = pkg.lib(), np.random.default_rng(seed)
    for _ in range(50):
        n = int(rng.integers(1, 6))
        fro, to = rng.integers(-1, 6, n), rng.integers(-1, 6, n)
        writers = [t for t in to if t >= 0]
        good = len(set(writers)) == len(writers) and all(f < 0 or f not in writers or to[i] == f for i, f in enumerate(fro))
        a = _conv(rows=20, n_seq=n, starts=_i32(*range(n + 1)), n_slots=6, fro=_i32(*map(int, fro)), to=_i32(*map(int, to)), D=0)
        assert L.fr_b200_conv_seq(*a) == -1          # (D = 0 is refused first)
        a = _conv(rows=20, n_seq=n, starts=_i32(*range(n + 1)), n_slots=6, fro=_i32(*map(int, fro)), to=_i32(*map(int, to)))
        if torch.cuda.is_available():
            continue
        assert L.fr_b200_conv_seq(*a) == (-3 if good else -1)
