"""Edges of the operators of a recurrent layer: calls that their documentation allows and that lie beside the ordinary ones."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_batch import _capture
from test_gpu_layer_ops import BF16, EX2, F16, F32, U32, _check, _linear_want, _rand, _ssm_inputs, _ssm_want

pytestmark = pytest.mark.gpu


# ---- slots -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,row", [(F32, 25), (F32, 25001), (F32, 750001), (F16, 51), (F16, 50001), (F16, 1500001), (torch.uint8, 101), (torch.uint8, 100001),
                                       (torch.uint8, 3000001), (F32, 24), (F32, 25000)])
def test_copy_slots_that_only_clears(pkg, dtype, row):
    """no slot is read: slots of 4-, 2-, 1- and 16-byte granules, of one column of a CTA and of many"""
    pool = torch.randint(1, 200, (9, row), device="cuda").to(dtype)
    for dst in ([4], [0, 8], [7, 1, 2, 6, 3]):
        p = pool.clone()
        pkg.copy_slots(p, [-1] * len(dst), np.asarray(dst, np.int32))
        want = pool.clone()
        want[dst] = 0
        assert torch.equal(p, want)


def test_no_streams_and_no_rows(pkg):
    """a step of a server without streams, and sequences without a row in rows that are none: states are handed on"""
    e = lambda *s: torch.empty(s, dtype=F16, device="cuda")  # noqa: E731
    w, A = _rand(16, 4), -torch.ones((16, 8), device="cuda")
    conv, ssm = _rand(5, 3, 16, dtype=F16), _rand(5, 16, 8, seed=1)
    for f, t in (([], []), (np.zeros(0, np.int32), ()), (torch.zeros(0, dtype=torch.int32), []), (-1, -1), (None, None)):
        p, q = conv.clone(), ssm.clone()
        assert pkg.conv_step(e(0, 16), w, state=p, from_slots=f, to_slots=t).shape == (0, 16)
        assert pkg.ssm_step(e(0, 16), e(0, 16), A, e(0, 8), e(0, 8), state=q, from_slots=f, to_slots=t).shape == (0, 16)
        assert pkg.conv_seq(e(0, 16), w, state=p, starts=[0], from_slots=f, to_slots=t).shape == (0, 16)
        assert pkg.ssm_seq(e(0, 16), e(0, 16), A, e(0, 8), e(0, 8), state=q, starts=[0], from_slots=f, to_slots=t).shape == (0, 16)
        assert torch.equal(p, conv) and torch.equal(q, ssm)
    pkg.conv_seq(e(0, 16), w, state=p, starts=[0, 0, 0], from_slots=[1, -1], to_slots=[4, 2])
    pkg.ssm_seq(e(0, 16), e(0, 16), A, e(0, 8), e(0, 8), state=q, starts=[0, 0, 0], from_slots=[1, -1], to_slots=[4, 2])
    for new, old in ((p, conv), (q, ssm)):
        assert torch.equal(new[4], old[1]) and bool((new[2] == 0).all()) and torch.equal(new[[0, 1, 3]], old[[0, 1, 3]])
    for pool in (conv[:0], conv, conv[:, :0]):
        assert pkg.copy_slots(pool, [], []) is pool


@pytest.mark.parametrize("rows", [17, 40, 300, 2000])
@pytest.mark.parametrize("k,n", [(8, 1), (64, 1), (8, 8), (1, 3), (16, 2)])
def test_linear_of_the_smallest_matrices(pkg, rows, k, n):
    """one channel, and inputs of one word: boxes of a tile that reach past all of the matrix"""
    x, w = _rand(rows, k, dtype=F16), _rand(n, k, dtype=F16, seed=1)
    want, err = _linear_want(x, w, None, "none", None)
    _check(pkg.linear(x, w), want, err)


# ---- waits that give up ------------------------------------------------------------------------------------------

def test_a_wait_that_gave_up_is_told_once_and_refuses_nobody(pkg):
    """the status word is asked for; products that have nothing to do with it run, before and behind the question"""
    L = pkg.lib()
    pkg.check_operators()
    x, w = _rand(40, 64, dtype=F16), _rand(24, 64, dtype=F16, scale=0.1, seed=1)
    want, err = _linear_want(x, w, None, "none", None)
    assert L.fr_b200_op_wait_selftest(0, 1000, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    _check(pkg.linear(x, w), want, err)
    assert L.fr_b200_op_status(0) == -6 and b"gave up" in L.fr_b200_op_last_error()
    assert L.fr_b200_op_status(0) == 0
    _check(pkg.linear(x, w), want, err)
    assert L.fr_b200_op_wait_selftest(0, 1000, None) == 0
    torch.cuda.synchronize()
    with pytest.raises(pkg.FrB200Error):
        pkg.check_operators(0)
    pkg.check_operators(0)


# ---- long narrow prompts: pieces of a sequence side by side ------------------------------------------------------

def _cut(pkg, rows, d, n):
    assert pkg.lib().fr_b200_ssm_seq_workspace(rows, 1, d, n) > 0


@pytest.mark.parametrize("d,n,dtype,bias", [(24, 5, F16, -1.0), (13, 16, F32, -3.0), (10, 3, BF16, -1.0), (8, 70, F32, -4.0)])
def test_ssm_pieces_with_infinite_inputs(pkg, d, n, dtype, bias):
    """an infinite x, or an infinite state to begin with, makes its channel infinite to the end, however far the decay of a whole piece falls (that
    of a row stays in the range of fp32)"""
    rows = 1100
    _cut(pkg, rows, d, n)
    x, dt, A, B, C, D, z, _ = _ssm_inputs(rows, d, n, 1, dtype)
    bias = torch.full((d,), bias, device="cuda")
    step = torch.nn.functional.softplus(dt.double() + bias)
    assert float(step.max() * -A.min()) < 80 and float(step[:256].sum(0).max() * -A.min()) > 100
    x, B, C = x.clone(), B.abs().contiguous(), C.abs().contiguous()
    B[B == 0], C[C == 0] = 0.5, 0.5
    x[7, 4], x[300, 6] = float("inf"), float("-inf")
    start = torch.zeros((2, d, n), device="cuda")
    start[0, 5] = float("inf")
    y, ey, new, enew = _ssm_want(x, dt, A, B, C, None, z, bias, True, [0, rows], start, [0], [1])
    for c, t in ((4, 7), (5, 0), (6, 300)):
        assert torch.isinf(y[t:, c]).all()
    p = start.clone()
    got = pkg.ssm_seq(x, dt, A, B, C, z=z, dt_bias=bias, state=p, from_slots=[0], to_slots=[1])
    # a piece's decay is the exponential of a sum of up to 256 time steps, off by as many roundings of it: |x| exp(-|x|) <= 0.37 of the state
    extra = 256 * U32 * 0.37 * max(1.0, float(new[torch.isfinite(new)].abs().max()))
    _check(got, y, ey + extra * C.double().abs().sum(1, keepdim=True) * (z.double().abs() + 1), "out")
    _check(p, new, enew + extra, "state")


def test_ssm_pieces_whose_decays_leave_the_range(pkg):
    """products of a piece's decays beyond the range of fp32, where no row's are: states that are 0 stay so while decays grow, small ones grow
    to ordinary ones, large ones fall to
    them.  The decay of a piece is 2^arg with arg off by 44 roundings (a sum of 256 time steps in
    partial sums of 8 and 32, times A, log2 e and a third), cubed: 44 U32 |arg| + 3 EX2 + 4 U32 of the value."""
    rows, d, n = 1100, 4, 3
    _cut(pkg, rows, d, n)
    x, dt = torch.zeros((rows, d), device="cuda"), torch.zeros((rows, d), device="cuda")
    B, C = _rand(rows, n).abs() + 0.1, _rand(rows, n, seed=1).abs() + 0.1
    A = torch.tensor([0.5, 0.35, -0.4, -0.39], device="cuda")[:, None] * torch.ones(n, device="cuda")
    x[1050:, 0] = _rand(50, seed=2).abs()
    dt[:, 0] = 1.0                     # from zero: grows by 2^184 a piece, with nothing to grow before row 1050
    dt[:256, 1:] = 1.0                 # 1e-30 by 2^129, 1e30 by 2^-148, 1e36 by 2^-144; then unchanged
    x[1050:, 1:] = 1e-3
    start = torch.zeros((1, d, n), device="cuda")
    start[0, 1], start[0, 2], start[0, 3] = 1e-30, 1e30, 1e36
    y, ey, new, enew = _ssm_want(x, dt, A, B, C, None, None, None, False, [0, rows], start, [0], [0])
    assert torch.isfinite(y).all() and float(new[0, 1].min()) > 1e8 and 0 < float(new[0, 2].max()) < 1e-9
    extra = 44 * U32 * 150 + 3 * EX2 + 4 * U32
    p = start.clone()
    got = pkg.ssm_seq(x, dt, A, B, C, dt_softplus=False, state=p)
    _check(got, y, ey + extra * y.abs(), "out")
    _check(p, new, enew + extra * new.abs(), "state")


# ---- activations -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [3, 60, 300])
@pytest.mark.parametrize("out_dtype", [F16, F32])
def test_gelu_keeps_its_negative_tail(pkg, rows, out_dtype):
    """Values from the bias alone, exact in fp32: what the function itself is off by is relative, down to the smallest.  In half steps of fp32: the fit
    of the tail 2.2, the fast exponential 4, the fast division 4 and its argument 2 times a slope of at most 2.7, eight steps of a sum whose
    terms' magnitudes are at most twice the sum 16, three products 3; the exponent v^2 / 2 with its two products and constant 2.5 of itself: 42 + 1.3 v^2."""
    v = torch.linspace(-8.0, 3.0, 264, device="cuda")
    x, w = torch.zeros((rows, 64), dtype=F16, device="cuda"), _rand(264, 64, dtype=F16)
    got = pkg.linear(x, w, v, activation="gelu", out_dtype=out_dtype)
    want = (0.5 * v.double() * torch.special.erfc(-v.double() / 2 ** 0.5)).expand(rows, -1)
    assert float(want[0, 0].abs()) < 6e-15
    _check(got, want, (42 + 1.3 * v.double() ** 2) * U32 * want.abs())


@pytest.mark.parametrize("rows", [3, 60, 300])
def test_softplus_is_relative_far_below_zero(pkg, rows):
    """In half steps of fp32: the fast exponential 4, the fast division 4, the series and its sums 6; the exponential's argument v log2 e 1.25 of
    itself (a product and the constant)."""
    v = torch.cat([torch.linspace(-85.0, -10.0, 200), torch.linspace(-10.0, 4.0, 64), torch.tensor([-7.0, -20.0, -80.0, 0.0])]).cuda()
    x, w = torch.zeros((rows, 64), dtype=F16, device="cuda"), _rand(v.numel(), 64, dtype=F16)
    got = pkg.linear(x, w, v, activation="softplus", out_dtype=F32)
    want = torch.log1p(torch.exp(v.double())).expand(rows, -1)
    _check(got, want, (14 + 1.25 * v.double().clamp(max=0).abs()) * U32 * want)


# ---- states of a model -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("version,fmt", [("4", "cuda fp16"), ("4", "cuda int8"), ("5.2", "cuda fp16")])
def test_captured_steps_go_on_from_copied_states(pkg, synth, version, fmt):
    """Two tokens of two streams as a graph.  Between its replays their slots take states of streams that have seen one token more or less: a token reads
    one of two copies of the token-shift states, the graph always the same one."""
    shape = synth.Shape(version, 2, 128, 512, 96, n_head=2 if version != "4" else 0)
    tensors = synth.to_file_dtypes(shape, synth.generate(shape, seed=11, ln_random=True), "fp16" if fmt.endswith("fp16") else "fp32")
    m = pkg.Model(tensors, fmt, shape=shape, max_batch=6)
    ids = synth.token_ids(shape, 4, seed=9).reshape(2, 2).astype(np.int32)
    m.run([5])                                          # stream 0: one token, the others none
    m.copy_states([0], [4])
    m.run([9])
    m.copy_states([0, 0], [5, 3])                       # 4: one token, 5 and 3: two
    assert np.array_equal(m.export_state(5), m.export_state(0)) and np.array_equal(m.export_state(3), m.export_state(0))
    kept = {b: m.export_state(b) for b in (3, 4, 5)}
    m.copy_states([-1, -1], [0, 1])
    got = torch.zeros(2, 2, shape.vocab, device="cuda")
    graph = _capture(pkg, lambda st: [pkg.lib().fr_b200_decode(m.handle, ids[t].ctypes.data_as(ctypes.c_void_p), 2,
                                                               ctypes.c_void_p(got[t].data_ptr()), None, st) for t in (0, 1)])
    for pair in ((4, 5), (5, 4), (4, 4), (3, -1), (-1, 4)):
        for b in (0, 1):                                # what the same states give outside the graph, stream by stream
            m.import_state(kept[pair[b]] if pair[b] >= 0 else m.export_state(2), b)
        want = np.stack([m.decode(ids[t]) for t in (0, 1)])
        after = [m.export_state(b) for b in (0, 1)]
        m.copy_states(list(pair), [0, 1])
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(got.cpu().numpy(), want), pair
        assert all(np.array_equal(m.export_state(b), after[b]) for b in (0, 1)), pair
        assert all(np.array_equal(m.export_state(b), k) for b, k in kept.items())
    m.close()


@pytest.mark.parametrize("version", ["4", "5.2"])
def test_a_batch_forked_from_a_stream_out_of_step_is_captured(pkg, synth, version):
    """Streams of a batch take the state of one that has seen an odd number of tokens, beside others that have seen none; the batch is captured and replayed
    twice: four steps like those outside a graph.  (A stream out of step would be brought into it by copies that every replay makes again.)"""
    shape = synth.Shape(version, 2, 128, 512, 96, n_head=2 if version != "4" else 0)
    tensors = synth.to_file_dtypes(shape, synth.generate(shape, seed=11, ln_random=True), "fp16")
    m = pkg.Model(tensors, "cuda fp16", shape=shape, max_batch=5)
    ids = synth.token_ids(shape, 8, seed=9).reshape(2, 4).astype(np.int32)
    m.run([5, 9, 2])
    prompt = m.export_state(0)
    m.copy_states([0], [4])
    m.reset_states(0)
    m.copy_states([4, 4], [1, 3])
    assert all(np.array_equal(m.export_state(b), prompt) for b in (1, 3, 4))
    start = [m.export_state(b) for b in range(4)]
    got = torch.zeros(2, 4, shape.vocab, device="cuda")
    graph = _capture(pkg, lambda st: [pkg.lib().fr_b200_decode(m.handle, ids[t].ctypes.data_as(ctypes.c_void_p), 4, ctypes.c_void_p(got[t].data_ptr()), None, st)
                                      for t in (0, 1)])
    have = []
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        have.extend(got.cpu().numpy())
    end = [m.export_state(b) for b in range(4)]
    for b in range(4):
        m.import_state(start[b], b)
    assert np.array_equal(np.stack(have), np.stack([m.decode(ids[t]) for t in (0, 1, 0, 1)]))
    assert all(np.array_equal(m.export_state(b), end[b]) for b in range(4))
    m.close()


@pytest.mark.parametrize("version", ["4", "5.2"])
def test_captured_steps_go_on_from_cleared_states(pkg, synth, version):
    """a graph of two tokens, replayed behind streams that were cleared in the middle of a batch (the batch reads either copy), or reset as a whole behind
    an odd number of tokens (then it reads the first): what the same tokens give outside it, and the step behind them"""
    shape = synth.Shape(version, 2, 128, 512, 96, n_head=2 if version != "4" else 0)
    m = pkg.Model(synth.to_file_dtypes(shape, synth.generate(shape, seed=11, ln_random=True), "fp16"), "cuda fp16", shape=shape, max_batch=2)
    ids = synth.token_ids(shape, 6, seed=9).reshape(3, 2).astype(np.int32)
    want = np.stack([m.decode(ids[t]) for t in (0, 1, 2)])
    after = [m.export_state(b) for b in (0, 1)]
    got = torch.zeros(2, 2, shape.vocab, device="cuda")

    def graph():
        return _capture(pkg, lambda st: [pkg.lib().fr_b200_decode(m.handle, ids[t].ctypes.data_as(ctypes.c_void_p), 2, ctypes.c_void_p(got[t].data_ptr()), None, st)
                                         for t in (0, 1)])

    def replayed(g):
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(got.cpu().numpy(), want[:2])
        assert np.array_equal(m.decode(ids[2]), want[2])
        assert all(np.array_equal(m.export_state(b), after[b]) for b in (0, 1))

    g = graph()                                    # (an odd number of tokens: it reads the second copy)
    for _ in range(2):
        m.copy_states([-1, -1], [0, 1])
        replayed(g)
        m.decode(ids[2])                           # (an even number between the replays)
    m.reset_states()
    g = graph()
    for _ in range(2):
        replayed(g)                                # (three tokens in all)
        m.reset_states()
    m.close()


# ---- arguments ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("call", ["ssm_seq", "ssm_step"])
def test_dt_softplus_without_a_truth_value(pkg, call):
    """what cannot be asked for its truth raises what it raises, and nothing is launched"""
    x, dt, A, B, C, *_ = _ssm_inputs(4, 8, 2, 1, F16)
    out = torch.full((4, 8), 7.0, dtype=F16, device="cuda")
    with pytest.raises(ValueError, match="ambiguous"):
        getattr(pkg, call)(x, dt, A, B, C, dt_softplus=np.array([1, 2]), out=out)
    assert bool((out == 7).all())
    for yes in (True, 1, np.bool_(True), torch.tensor(True)):
        assert torch.equal(getattr(pkg, call)(x, dt, A, B, C, dt_softplus=yes), getattr(pkg, call)(x, dt, A, B, C))


def test_parameters_without_gradients(pkg):
    """weights that require a gradient: taken under no_grad, refused in every place outside it"""
    x, w, b = _rand(4, 64, dtype=F16), _rand(24, 64, dtype=F16, scale=0.1, seed=1), _rand(24, seed=2)
    want = pkg.linear(x, w, b)
    wp, bp = torch.nn.Parameter(w.clone()), torch.nn.Parameter(b.clone())
    with torch.no_grad():
        assert torch.equal(pkg.linear(x, wp, bp), want)
    assert torch.equal(pkg.linear(x, wp.detach(), bp.detach()), want)
    for args, kw in (((x, wp, b), {}), ((x, w, bp), {}), ((x, w, b), {"residual": want.clone().requires_grad_()}), ((x.clone().requires_grad_(), w, b), {})):
        with pytest.raises(ValueError, match="gradient"):
            pkg.linear(*args, **kw)
