"""Performance cases: the operators of a recurrent layer that a program calls on its own device tensors.

  linear     out = residual + act(x . w^T + bias): the projections of a layer with what follows them
  conv       the short causal convolution in front of a selective scan: prompts of any lengths back to back, or one
             token of each stream
  ssm        the selective state space scan, for the same prompts and tokens
  slots      states of streams forked, moved and freed: what a server does between two steps

The sizes are those of layers as wide as the models of `synth.SHAPES` (2048, 2560 and 5120 channels, 4 to a stream's
token-shift window, inner width twice the layer's).  States of streams are rows of a pool; a pass reads some slots and
writes others, so that it can be repeated.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ACTS = ("none", "relu2", "silu", "sigmoid", "gelu", "softplus")
TAPS = 4
MOST_FLOPS = 2.0 * 4096 * 2560 * 8960    # of a product
MOST_STATES = 4096 * 4096 * 16           # rows x channels x states of a scan
MOST_POOL = 1 << 28                      # elements of a pool


def listed():
    return [
        # one user's token through the projection into a layer of 2048 channels: a gate and a scan half side by side
        {"name": "linear_1_in", "kind": "linear", "rows": 1, "k": 2048, "n": 8192, "dtype": "fp16", "act": "none", "bias": False, "residual": False},
        # the time steps of a user's message: a narrow product out of a wider row, softplus behind it
        {"name": "linear_45_dt", "kind": "linear", "rows": 45, "k": 160, "n": 5120, "dtype": "fp16", "act": "softplus", "bias": True, "residual": False},
        # a busy server's projection back to the residual stream, as many streams as there happen to be
        {"name": "linear_200_out", "kind": "linear", "rows": 200, "k": 5120, "n": 2560, "dtype": "bf16", "act": "none", "bias": False, "residual": True},
        # the channel mix of the benchmark's longest prompt
        {"name": "linear_4096_ffn", "kind": "linear", "rows": 4096, "k": 2560, "n": 8960, "dtype": "fp16", "act": "relu2", "bias": True, "residual": False},
        # one token of each stream of a small server
        {"name": "conv_step_64", "kind": "conv_step", "streams": 64, "d": 4096, "dtype": "fp16", "act": "silu"},
        # prompts of a server, back to back, some of them later parts of one
        {"name": "conv_37_prompts", "kind": "conv_seq", "seqs": 37, "rows": 4001, "d": 5120, "dtype": "bf16", "act": "silu", "fresh": False},
        # one user's token
        {"name": "ssm_step_1", "kind": "ssm_step", "streams": 1, "d": 5120, "n": 16, "groups": 1, "dtype": "fp16"},
        # a full server's
        {"name": "ssm_step_256", "kind": "ssm_step", "streams": 256, "d": 4096, "n": 16, "groups": 1, "dtype": "bf16"},
        # a long prompt alone, from the start
        {"name": "ssm_prompt_4096", "kind": "ssm_seq", "seqs": 1, "rows": 4096, "d": 4096, "n": 16, "groups": 1, "dtype": "fp16", "fresh": True},
        # prompts of a server
        {"name": "ssm_11_prompts", "kind": "ssm_seq", "seqs": 11, "rows": 3001, "d": 5120, "n": 16, "groups": 1, "dtype": "bf16", "fresh": False},
        # a prompt answered in 31 ways
        {"name": "slots_fork_31", "kind": "slots", "what": "fork", "slots": 40, "moves": 31, "row": 5120 * 19, "dtype": "fp32"},
        # the survivors of a beam search over many streams, in place
        {"name": "slots_reorder_256", "kind": "slots", "what": "reorder", "slots": 256, "moves": 256, "row": 4096 * 16 * 8 + 24, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _channels(rng):
    if rng.random() < 0.4:
        return rng.choice((768, 1536, 2048, 2560, 4096, 5120))
    return _log_int(rng, 64, 5120)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "conv_step", "conv_seq", "ssm_step", "ssm_seq", "ssm_seq", "slots"))
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "linear":
        k, n = _channels(rng), _channels(rng)
        if rng.random() < 0.75:   # rows of whole 16 bytes, as most layers have them
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        rows = min(_log_int(rng, 1, 4096), int(MOST_FLOPS / (2.0 * k * n)))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "dtype": dtype, "act": rng.choice(ACTS), "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    if kind == "slots":
        row = _log_int(rng, 1000, 1 << 21)
        slots = max(4, min(_log_int(rng, 4, 512), MOST_POOL // row))
        what = rng.choice(("fork", "compact", "reorder", "free"))
        return {"kind": kind, "what": what, "slots": slots, "moves": rng.randint(1, slots if what == "reorder" else slots // 2), "row": row,
                "dtype": rng.choice(("fp16", "fp32"))}
    if rng.random() < 0.2:
        dtype = "fp32"
    d = _channels(rng)
    if kind.startswith("conv"):
        act = rng.choice(("none", "silu"))
        if kind == "conv_step":
            return {"kind": kind, "streams": _log_int(rng, 1, 512), "d": d, "dtype": dtype, "act": act}
        rows = _log_int(rng, 1, 4096)
        return {"kind": kind, "seqs": min(rows, _log_int(rng, 1, 64)), "rows": rows, "d": d, "dtype": dtype, "act": act, "fresh": rng.random() < 0.5}
    n = rng.choice((16, 16, 16, 8, 32, 64, rng.randint(1, 64)))
    groups = rng.choice((1, 1, 2, 4))
    d = (d + groups - 1) // groups * groups
    if kind == "ssm_step":
        streams = min(_log_int(rng, 1, 512), max(1, MOST_STATES // (8 * d * n)))
        return {"kind": kind, "streams": streams, "d": d, "n": n, "groups": groups, "dtype": dtype}
    rows = min(_log_int(rng, 1, 4096), max(1, MOST_STATES // (d * n)))
    return {"kind": kind, "seqs": min(rows, _log_int(rng, 1, 64)), "rows": rows, "d": d, "n": n, "groups": groups, "dtype": dtype, "fresh": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _normal(gen, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _starts(case):
    """First rows of the sequences, and the end of the last: lengths of at least one that differ by tens of times."""
    rng = random.Random(case["rows"] * 1000 + case["seqs"])
    weights = [rng.expovariate(1.0) for _ in range(case["seqs"])]
    left = case["rows"] - case["seqs"]
    lengths = [1 + int(left * w / sum(weights)) for w in weights]
    lengths[-1] += case["rows"] - sum(lengths)
    return np.cumsum([0] + lengths).astype(np.int32)


def _slots(case, gen, row, dtype, scale):
    """A pool of states of two slots a stream: streams read the first half (or begin from zero) and write the second, each in an order of its own."""
    n = case.get("seqs") or case["streams"]
    rng = random.Random(n)
    fro, to = list(range(n)), list(range(n, 2 * n))
    rng.shuffle(fro)
    rng.shuffle(to)
    pool = _normal(gen, (2 * n, *row), dtype, scale)
    fro = np.full(n, -1, np.int32) if case.get("fresh") else np.asarray(fro, np.int32)
    return {"pool": pool, "from": fro, "to": np.asarray(to, np.int32),
            "from_gpu": torch.from_numpy(fro).long().cuda(), "to_gpu": torch.tensor(to, device="cuda")}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        wide = k if k % 8 else k + 32 if k < 256 else k   # a narrow operand is a piece of a wider row
        s["x"] = _normal(gen, (rows, wide), dt)[:, :k]
        s["w"] = _normal(gen, (n, k), dt, 1.0 / math.sqrt(k))
        s["bias"] = _normal(gen, (n,), scale=0.5) if case["bias"] else None
        s["residual"] = _normal(gen, (rows, n), dt, 2.0) if case["residual"] else None
        return s
    if kind == "slots":
        rng = random.Random(case["slots"] * 1000 + case["moves"])
        slots, moves, what = case["slots"], case["moves"], case["what"]
        order = list(range(slots))
        rng.shuffle(order)
        if what == "fork":          # one state into free slots
            src, dst = [order[0]] * moves, order[1:1 + moves]
        elif what == "compact":     # the highest live slots into the lowest free ones
            src, dst = sorted(range(slots - moves, slots)), sorted(range(moves))
        elif what == "free":
            src, dst = [-1] * moves, order[:moves]
        else:                       # every slot takes the state of some slot, several of the same one
            src, dst = [rng.choice(order[:moves]) for _ in range(moves)], order[:moves]
        s["pool"] = _normal(gen, (slots, case["row"]), dt)
        s["src"], s["dst"] = np.asarray(src, np.int32), np.asarray(dst, np.int32)
        s["src_gpu"], s["dst_gpu"] = torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda")
        return s
    d = case["d"]
    rows = case["rows"] if "rows" in case else case["streams"]
    xz = _normal(gen, (rows, 2 * d), dt)   # the projection into the layer: the scan's half, and the gate's
    if "seqs" in case:
        s["starts"] = _starts(case)
        s["starts_gpu"] = torch.from_numpy(s["starts"]).long().cuda()
        s["longest"] = int(np.diff(s["starts"]).max())
    if kind.startswith("conv"):
        s["x"] = xz[:, :d]
        s["w"], s["bias"] = _normal(gen, (d, TAPS), scale=0.5), _normal(gen, (d,), scale=0.2)
        s.update(_slots(case, gen, (TAPS - 1, d), dt, 1.0))
        return s
    n, g = case["n"], case["groups"]
    s["x"] = torch.nn.functional.silu(_normal(gen, (rows, d))).to(dt)
    s["z"] = xz[:, d:]
    s["dt"] = _normal(gen, (rows, d), dt, 0.5)
    bc = _normal(gen, (rows, 160 + 2 * g * n), dt)   # B and C come out of one projection, behind the time steps' low rank
    s["B"], s["C"] = bc[:, 160:160 + g * n], bc[:, 160 + g * n:]
    s["A"] = -torch.arange(1, n + 1, device="cuda").float() * torch.exp(_normal(gen, (d, n), scale=0.2))
    step = torch.exp(torch.rand(d, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))   # 0.001 to 0.1
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["D"] = 1.0 + _normal(gen, (d,), scale=0.1)
    s.update(_slots(case, gen, (d, n), torch.float32, 0.5))
    return s


# ---- the operators in their plain form ---------------------------------------------------------------------------

def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _act(v, name):
    if name == "relu2":
        return torch.clamp(v, min=0) ** 2
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return _softplus(v) if name == "softplus" else v


def _linear(s):
    v = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        v = v + s["bias"]
    v = _act(v, s["case"]["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["x"].dtype)


def _read_slots(s):
    fro = s["from_gpu"]
    live = (fro >= 0).float().view(-1, *[1] * (s["pool"].dim() - 1))
    return s["pool"][fro.clamp(min=0)].float() * live


def _conv_step(s):
    window = torch.cat([_read_slots(s), s["x"].float()[:, None]], 1)          # [streams, taps, channels]
    y = _act((window * s["w"].t()).sum(1) + s["bias"], s["case"]["act"])
    s["pool"][s["to_gpu"]] = window[:, 1:].to(s["pool"].dtype)
    return y.to(s["x"].dtype), s["pool"]


def _conv_seq(s):
    x, starts, back = s["x"], s["starts_gpu"], TAPS - 1
    rows, seqs = x.shape[0], starts.numel() - 1
    # what came before every sequence, then the rows: tap j of a row is one row of these
    before = _read_slots(s).reshape(seqs * back, -1)
    rows_all = torch.cat([before, x.float()], 0)
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    at = row[:, None] - back + torch.arange(TAPS, device="cuda")              # [rows, taps]
    first = starts[seq][:, None]
    at = torch.where(at >= first, seqs * back + at, seq[:, None] * back + back + at - first)
    y = _act((rows_all[at] * s["w"].t()).sum(1) + s["bias"], s["case"]["act"])
    last = starts[1:, None] - back + torch.arange(back, device="cuda")
    first = starts[:-1, None]
    i = torch.arange(seqs, device="cuda")[:, None]
    last = torch.where(last >= first, seqs * back + last, i * back + back + last - first)
    s["pool"][s["to_gpu"]] = rows_all[last].to(s["pool"].dtype)
    return y.to(x.dtype), s["pool"]


def _per_channel(v, d, groups):
    """[rows, groups * n] -> [rows, channels, n], a view"""
    rows = v.shape[0]
    return v.float().view(rows, groups, 1, -1).expand(rows, groups, d // groups, -1).reshape(rows, d, -1)


def _ssm_inputs(s):
    d, groups = s["case"]["d"], s["case"]["groups"]
    x = s["x"].float()
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    decay = torch.exp(delta[:, :, None] * s["A"])
    adds = (delta * x)[:, :, None] * _per_channel(s["B"], d, groups)
    return x, decay, adds, _per_channel(s["C"], d, groups)


def _ssm_out(s, x, h, c):
    y = (h * c).sum(2) + s["D"] * x
    return (y * _act(s["z"].float(), "silu")).to(s["x"].dtype)


def _ssm_step(s):
    x, decay, adds, c = _ssm_inputs(s)
    h = decay * _read_slots(s) + adds
    s["pool"][s["to_gpu"]] = h
    return _ssm_out(s, x, h, c), s["pool"]


def _ssm_seq(s):
    x, decay, h, c = _ssm_inputs(s)
    first = s["starts_gpu"][:-1]
    h[first] += decay[first] * _read_slots(s)
    decay[first] = 0
    reach = 1
    while reach < s["longest"]:     # after each pass h holds the sum over twice as many rows
        h[reach:] += decay[reach:] * h[:-reach]
        decay[reach:] = decay[reach:] * decay[:-reach]
        reach *= 2
    s["pool"][s["to_gpu"]] = h[s["starts_gpu"][1:] - 1]
    return _ssm_out(s, x, h, c), s["pool"]


def _slots_copy(s):
    src, pool = s["src_gpu"], s["pool"]
    pool[s["dst_gpu"]] = pool[src.clamp(min=0)] * (src >= 0).to(pool.dtype)[:, None]
    return pool


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if own:
        frb = importlib.import_module("faster-rwkv_b200")
        if kind == "linear":
            return frb.linear(s["x"], s["w"], s["bias"], activation=case["act"], residual=s["residual"])
        if kind == "slots":
            frb.copy_slots(s["pool"], s["src"], s["dst"])
            return s["pool"]
        slots = {"state": s["pool"], "from_slots": s["from"], "to_slots": s["to"]}
        if kind == "conv_step":
            return frb.conv_step(s["x"], s["w"], s["bias"], activation=case["act"], **slots), s["pool"]
        if kind == "conv_seq":
            return frb.conv_seq(s["x"], s["w"], s["bias"], activation=case["act"], starts=s["starts"], **slots), s["pool"]
        params = {"D": s["D"], "z": s["z"], "dt_bias": s["dt_bias"], "dt_softplus": True}
        if kind == "ssm_step":
            return frb.ssm_step(s["x"], s["dt"], s["A"], s["B"], s["C"], **params, **slots), s["pool"]
        return frb.ssm_seq(s["x"], s["dt"], s["A"], s["B"], s["C"], starts=s["starts"], **params, **slots), s["pool"]
    return {"linear": _linear, "slots": _slots_copy, "conv_step": _conv_step, "conv_seq": _conv_seq, "ssm_step": _ssm_step, "ssm_seq": _ssm_seq}[kind](s)


def work(case):
    kind, es = case["kind"], torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": es * (rows * k + n * k + rows * n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0), "flops": 2.0 * rows * k * n}
    if kind == "slots":
        row, moves = es * case["row"], case["moves"]
        read = {"fork": 1, "free": 0, "compact": moves, "reorder": moves}[case["what"]]
        if case["what"] == "reorder":   # the states that some slot takes, and those that change
            rng = random.Random(case["slots"] * 1000 + moves)
            order = list(range(case["slots"]))
            rng.shuffle(order)
            src = [rng.choice(order[:moves]) for _ in range(moves)]
            read = len({a for a, b in zip(src, order) if a != b})
            moves = sum(a != b for a, b in zip(src, order))
        return {"bytes": row * (read + moves), "flops": 0}
    d, streams = case["d"], case.get("seqs") or case.get("streams")
    rows = case.get("rows") or streams
    states = (1 if case.get("fresh") else 2) * streams
    if kind.startswith("conv"):
        return {"bytes": es * (2 * rows * d + states * (TAPS - 1) * d) + 4 * d * (TAPS + 1), "flops": rows * d * (2.0 * TAPS + 4)}
    n, g = case["n"], case["groups"]
    return {"bytes": es * (4 * rows * d + 2 * rows * g * n) + 4 * states * d * n + 4 * d * (n + 2), "flops": rows * d * (7.0 * n + 16)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    kind = case["kind"]
    if kind == "slots" and case["what"] == "reorder":
        return None     # each pass moves on from the one before
    s = prepare(case, seed)
    if kind == "slots":
        moved = s["pool"].double()
        source = moved.clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            moved[b] = source[a] if a >= 0 else 0.0
        return moved
    f = torch.nn.functional
    acts = {"none": lambda v: v, "relu2": lambda v: f.relu(v).square(), "silu": lambda v: v * torch.sigmoid(v), "sigmoid": torch.sigmoid,
            "gelu": lambda v: v * torch.special.ndtr(v), "softplus": lambda v: torch.logaddexp(v, torch.zeros_like(v))}
    if kind == "linear":
        v = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        v = acts[case["act"]](v + s["bias"].double() if case["bias"] else v)
        return v + s["residual"].double() if case["residual"] else v
    pool, x = s["pool"].double(), s["x"].double()
    fro, to = s["from"].tolist(), s["to"].tolist()
    starts = s["starts"].tolist() if "starts" in s else list(range(len(to) + 1))
    y = torch.empty_like(x)
    if kind.startswith("conv"):
        old = pool.clone()
        for i, (a, b) in enumerate(zip(starts, starts[1:])):
            head = old[fro[i]] if fro[i] >= 0 else torch.zeros_like(old[0])
            run_of = torch.cat([head, x[a:b]])
            acc = sum(run_of[j:j + b - a] * s["w"][:, j].double() for j in range(TAPS))
            y[a:b] = acts[case["act"]](acc + s["bias"].double())
            pool[to[i]] = run_of[b - a:]
        return y, pool
    # all sequences side by side, one row of each at a time
    d, g = case["d"], case["groups"]
    begin = torch.tensor(starts[:-1], device="cuda")
    length = torch.tensor(np.diff(starts), device="cuda")
    h = torch.stack([pool[i] if i >= 0 else torch.zeros_like(pool[0]) for i in fro])
    delta = acts["softplus"](s["dt"].double() + s["dt_bias"].double())
    a64, gate, skip = s["A"].double(), acts["silu"](s["z"].double()), s["D"].double() * x
    for t in range(int(max(np.diff(starts)))):
        at = torch.nonzero(length > t)[:, 0] if len(to) > 1 else torch.zeros(1, dtype=torch.long, device="cuda")
        r = begin[at] + t
        b = s["B"][r].double().view(len(r), g, -1).repeat_interleave(d // g, 1)
        c = s["C"][r].double().view(len(r), g, -1).repeat_interleave(d // g, 1)
        now = h[at] * torch.exp(delta[r][:, :, None] * a64) + (delta[r] * x[r])[:, :, None] * b
        h[at] = now
        y[r] = ((now * c).sum(2) + skip[r]) * gate[r]
    pool[torch.tensor(to, device="cuda")] = h
    return y, pool
