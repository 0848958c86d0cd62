"""What the sequence and gradient operators are measured on.

Three operators:

* ``scan``: the gated linear recurrence over a whole sequence, forward alone or
  forward and backward (``ptamd.scan.gated_scan``);
* ``step``: the same recurrence for one new token or frame of every row, the
  state updated in place (``ptamd.scan.gated_scan_step``);
* ``clip``: the global norm of many gradient tensors and their scaling to a
  largest norm (``ptamd.clip.clip_grads``).

The recurrence has two forms, by the gates that the input holds (pre-activation,
stacked along one dimension):

  leaky  z, n        h_t = (1 - s(z_t)) h_{t-1} + s(z_t) n_t            y_t = h_t
  lstm   i, f, n, o  c_t = s(f_t) c_{t-1} + s(i_t) tanh(n_t)            y_t = s(o_t) tanh(c_t)

with s the logistic function.  Rows of a batch may be shorter than the batch
(``lengths``): what stands behind a row's end is not read, y is 0 there and so
are the gradients.

``run`` takes the plain form (elementary torch operations in 32 bits) where
``own`` is false, the framework's operators where it is true; ``exact`` is the
definition in 64 bits, frame by frame, with gradients from autograd.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GATES = {"leaky": 2, "lstm": 4}
LOOP_STEPS = 512          # the plain form walks up to this many steps, and doubles above


# ---------------------------------------------------------------- the cases

def _scan_case(name, form, dtype, layout, batch, steps, train, h0=False, ragged=False, seq=True,
               **size):
    return dict(name=name, op="scan", form=form, dtype=dtype, layout=layout, batch=batch,
                steps=steps, train=train, h0=h0, ragged=ragged, seq=seq, **size)


def listed():
    return [
        # one token of one sequence while it is generated: the call's latency
        dict(name="step_leaky_bf16_1x2048", op="step", form="leaky", dtype="bf16", batch=1, width=2048),
        # 64 clips streamed frame by frame through 25 channels of 32x32 (the ConvLSTM's state)
        dict(name="step_lstm_f32_64x25600", op="step", form="lstm", dtype="f32", batch=64, width=25600),
        # a short odd sequence, carried on from an earlier one: latency of the forward alone
        _scan_case("fwd_leaky_f32_2x37x200", "leaky", "f32", "btd", 2, 37, False, h0=True, width=200),
        # one long prompt: no rows to spread over, the time axis has to be split
        _scan_case("fwd_leaky_bf16_1x16384x2048", "leaky", "bf16", "btd", 1, 16384, False, width=2048),
        # a training batch of token sequences of different lengths
        _scan_case("train_leaky_bf16_8x2048x2048", "leaky", "bf16", "btd", 8, 2048, True, ragged=True,
                   width=2048),
        # a clip batch, channels before time as a Conv3d leaves it: InT's 32 channels, 64 frames
        _scan_case("train_leaky_f32_clips32", "leaky", "f32", "clip_c", 32, 64, True, channels=32, side=32),
        # nothing divides anything
        _scan_case("train_leaky_f16_3x1013x777", "leaky", "f16", "btd", 3, 1013, True, h0=True, ragged=True,
                   width=777),
        # the clip ConvLSTM's sizes (25 channels, 64 frames of 32x32), read out at the last frame alone
        _scan_case("train_lstm_bf16_clips64_last", "lstm", "bf16", "clip_t", 64, 64, True, seq=False,
                   channels=25, side=32),
        # few long rows in training, every step read out
        _scan_case("train_lstm_bf16_2x8192x512", "lstm", "bf16", "btd", 2, 8192, True, h0=True, width=512),
        # the InT trainer's own 30 gradients, 107,158 numbers: launches are all there is
        dict(name="clip_int_f32", op="clip", kind="int", dtype="f32", count=30, total=107158, shapes=0,
             out="f32", above=True, norm="2"),
        # the gradients of a 24-layer model of width 1024, clipped into the optimizer's f32 buffers
        dict(name="clip_layers_bf16", op="clip", kind="layers", dtype="bf16", count=194, total=334808064,
             shapes=0, out="f32", above=True, norm="2"),
        # ragged tensors of all types, empty ones among them, below the threshold: in place
        dict(name="clip_ragged_mixed", op="clip", kind="ragged", dtype="mixed", count=257,
             total=20000003, shapes=11, out="place", above=False, norm="2"),
    ]


def draw(rng):
    """One more case of the same ranges: never more bytes than the largest listed one."""
    top = max(work(c)["bytes"] for c in listed())
    while True:
        case = _draw(rng)
        if work(case)["bytes"] <= top:
            return case


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["scan", "scan", "scan", "step", "clip"])
    if op == "clip":
        count = _logint(rng, 1, 400)
        place = rng.random() < 0.4
        return dict(op="clip", kind="ragged", dtype=rng.choice(["f32", "bf16", "f16", "mixed"]), count=count,
                    total=_logint(rng, count, 200_000_000), shapes=rng.randrange(1 << 20),
                    out="place" if place else "f32", above=not place and rng.random() < 0.7,
                    norm=rng.choice(["2", "2", "2", "1", "inf"]))
    form = rng.choice(["leaky", "lstm"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "step":
        return dict(op="step", form=form, dtype=dtype, batch=_logint(rng, 1, 256),
                    width=_logint(rng, 1, 30000))
    case = dict(op="scan", form=form, dtype=dtype, train=rng.random() < 0.6, h0=rng.random() < 0.5,
                ragged=rng.random() < 0.5)
    case["seq"] = case["ragged"] or not case["train"] or rng.random() < 0.7
    case["layout"] = rng.choice(["btd", "btd", "clip_c", "clip_t"])
    if case["layout"] == "btd":
        case.update(batch=_logint(rng, 1, 64), steps=_logint(rng, 1, 16384), width=_logint(rng, 1, 4096))
    else:
        case.update(batch=_logint(rng, 1, 64), steps=_logint(rng, 1, 128), channels=rng.randint(1, 32),
                    side=rng.choice([7, 16, 20, 32, 32, 33, 64]))
    return case


def _features(case):
    return case["width"] if "width" in case else case["channels"] * case["side"] ** 2


def _tensor_sizes(case):
    """The gradients' element counts, in order."""
    if case["kind"] == "int":
        c = 32
        sizes = [3 * c, c, 49 * c * c, 49 * c * c] + 4 * [c] + 6 * [c * c, c] + 4 * [c]
        return sizes + [c, 1, 50, 1, 1, 1]
    if case["kind"] == "layers":
        d = 1024
        sizes = [32000 * d]
        for _ in range(24):
            sizes += [d, d, d * d, d * d, d * d, d * d, 4 * d * d, 4 * d * d]
        return sizes + [d]
    rng = np.random.default_rng(case["shapes"])
    part = rng.exponential(size=case["count"]) ** 2
    part[rng.random(case["count"]) < 0.05] = 0.0
    if part.sum() == 0:
        part[0] = 1.0
    return [int(s) for s in np.floor(part / part.sum() * case["total"])]


def _tensor_types(case):
    if case["dtype"] != "mixed":
        return [DTYPES[case["dtype"]]] * case["count"]
    rng = np.random.default_rng(case["shapes"] + 1)
    return [list(DTYPES.values())[k] for k in rng.integers(0, 3, case["count"])]


def work(case):
    if case["op"] == "clip":
        read = sum(n * t.itemsize for n, t in zip(_tensor_sizes(case), _tensor_types(case)))
        write = 4 * sum(_tensor_sizes(case)) if case["out"] == "f32" else 0
        if case["out"] == "place" and case["above"]:
            write = read
        return {"bytes": read + write + 4, "flops": 3 * sum(_tensor_sizes(case))}
    size, gates = DTYPES[case["dtype"]].itemsize, GATES[case["form"]]
    row = _features(case)
    if case["op"] == "step":
        n = case["batch"] * row
        return {"bytes": n * ((gates + 1) * size + 8), "flops": 12 * gates * n}
    # every input once, every output once: the gates, y, the states; in training
    # the gradients of y and of the gates too
    n = case["batch"] * case["steps"] * row
    ends = case["batch"] * row * 4 * (gates // 2 + (1 if case["h0"] else 0))
    total = n * (gates + (1 if case["seq"] else 0)) * size
    if case["train"]:
        total, ends = 2 * total, 2 * ends
    return {"bytes": total + ends, "flops": 12 * gates * n * (3 if case["train"] else 1)}


# ---------------------------------------------------------------- the inputs

def _lengths(case, gen):
    """Row ends of a batch padded to its longest row; one row is full, one may be short."""
    t = case["steps"]
    u = torch.rand(case["batch"], generator=gen)
    n = (t * (0.35 + 0.65 * u)).long().clamp(1, t)
    n[0] = t
    return n


def _shape(case, n):
    """Shape of a tensor of n gates, the gates' dimension, the time dimension."""
    if case["layout"] == "btd":
        return (case["batch"], case["steps"], n * case["width"]), 2, 1
    s = case["side"]
    if case["layout"] == "clip_c":
        return (case["batch"], n * case["channels"], case["steps"], s, s), 1, 2
    return (case["batch"], case["steps"], n * case["channels"], s, s), 2, 1


def _gates(shape, gate_dim, form, dtype, gen):
    """Pre-activations as a trained cell has them: slow leaks, forget gates mostly open."""
    x = torch.randn(shape, generator=gen, device="cuda")
    parts = x.chunk(GATES[form], gate_dim)
    if form == "leaky":
        parts[0].mul_(1.5).sub_(2.0)
    else:
        parts[1].add_(2.0)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    st = {"case": case}
    if case["op"] == "clip":
        sizes, types = _tensor_sizes(case), _tensor_types(case)
        if case["out"] == "f32":         # a tensor each, clipped into views of the optimizer's flat buffer
            st["grads"] = [(0.02 * torch.randn(n, generator=gen, device="cuda")).to(t)
                           for n, t in zip(sizes, types)]
            st["flat"] = [torch.empty(sum(sizes), device="cuda")]
            st["out"] = list(st["flat"][0].split(sizes))
        else:                            # views of one bucket for each type, clipped in place
            st["flat"], st["grads"], st["out"] = [], [None] * len(sizes), None
            for t in DTYPES.values():
                mine = [k for k in range(len(sizes)) if types[k] is t]
                if mine:
                    own_sizes = [sizes[k] for k in mine]
                    st["flat"].append((0.02 * torch.randn(sum(own_sizes), generator=gen, device="cuda")).to(t))
                    for k, v in zip(mine, st["flat"][-1].split(own_sizes)):
                        st["grads"][k] = v
        n = max(1, sum(_tensor_sizes(case)))
        like = {"2": 0.02 * math.sqrt(n), "1": 0.016 * n, "inf": 0.04}[case["norm"]]
        st["max_norm"] = like * (0.25 if case["above"] else 100.0)
        st["norm_type"] = float(case["norm"])
    elif case["op"] == "step":
        shape = (case["batch"], GATES[case["form"]] * case["width"])
        st["x"] = _gates(shape, 1, case["form"], DTYPES[case["dtype"]], gen)
        st["state"] = torch.randn(case["batch"], case["width"], generator=gen, device="cuda")
    else:
        dtype = DTYPES[case["dtype"]]
        shape, gate_dim, dim = _shape(case, GATES[case["form"]])
        x = _gates(shape, gate_dim, case["form"], dtype, gen)
        y_shape = _shape(case, 1)[0]
        end = y_shape[:dim] + y_shape[dim + 1:]
        h0 = torch.randn(end, generator=gen, device="cuda") if case["h0"] else None
        st.update(gate_dim=gate_dim, dim=dim, h0=h0,
                  lengths=_lengths(case, host).cuda() if case["ragged"] else None)
        if case["train"]:
            x.requires_grad_()
            if h0 is not None:
                h0.requires_grad_()
            st["dy"] = torch.randn(y_shape, generator=gen, device="cuda").to(dtype) if case["seq"] else None
            st["dh"] = torch.randn(end, generator=gen, device="cuda")
        st["x"] = x
    if own:
        st["clip"], st["scan"] = _package()
    return st


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pathtracker-models_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ptamd import clip, scan
    return clip, scan


# ---------------------------------------------------------------- one pass

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    case = st["case"]
    if case["op"] == "clip":
        norm = st["clip"].clip_grads(st["grads"], st["max_norm"], norm_type=st["norm_type"], out=st["out"])
        return [norm] + st["flat"]
    if case["op"] == "step":
        return [st["scan"].gated_scan_step(st["x"], st["state"], form=case["form"]), st["state"]]
    with torch.set_grad_enabled(case["train"]):
        res = st["scan"].gated_scan(st["x"], st["h0"], form=case["form"], dim=st["dim"],
                                    gate_dim=st["gate_dim"], lengths=st["lengths"], want_seq=case["seq"])
    out = [r.detach() for r in res if r is not None]
    if not case["train"]:
        return out
    heads, ds = ([res[0], res[1]], [st["dy"], st["dh"]]) if case["seq"] else ([res[1]], [st["dh"]])
    leaves = [st["x"]] + ([st["h0"]] if case["h0"] else [])
    return out + list(torch.autograd.grad(heads, leaves, ds))


def _logistic(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _linear(a, b, dim, reverse=False):
    """h_t = a_t h_{t-1} + b_t along ``dim`` (from the far end when ``reverse``)."""
    n = a.shape[dim]
    if n <= LOOP_STEPS:
        out = torch.empty_like(b)
        h = torch.zeros_like(b.select(dim, 0))
        for t in (reversed(range(n)) if reverse else range(n)):
            h = a.select(dim, t) * h + b.select(dim, t)
            out.select(dim, t).copy_(h)
        return out
    a, b = a.clone(), b.clone()
    k = 1
    while k < n:
        late, early = (0, k) if reverse else (k, 0)
        at = a.narrow(dim, late, n - k)
        b.narrow(dim, late, n - k).add_(at * b.narrow(dim, early, n - k))
        at.copy_(at * a.narrow(dim, early, n - k))
        k *= 2
    return b


def _run_plain(st):
    case = st["case"]
    if case["op"] == "clip":
        return _plain_clip(st)
    if case["op"] == "step":
        return _plain_step(st)
    with torch.no_grad():
        return _plain_scan(st)


def _plain_clip(st):
    p = st["norm_type"]
    parts = [g.float() for g in st["grads"] if g.numel()]
    if p == math.inf:
        norm = torch.stack([g.abs().max() for g in parts]).max()
    elif p == 1.0:
        norm = torch.stack([g.abs().sum(dtype=torch.float64) for g in parts]).sum()
    else:
        norm = torch.stack([(g * g).sum(dtype=torch.float64) for g in parts]).sum().sqrt()
    coef = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0).float()
    for g, o in zip(st["grads"], st["out"] or st["grads"]):
        o.copy_(g.float() * coef)
    return [norm.float()] + st["flat"]


def _plain_step(st):
    parts = [p.float() for p in st["x"].chunk(GATES[st["case"]["form"]], 1)]
    if st["case"]["form"] == "leaky":
        z, n = parts
        h = _logistic(-z) * st["state"] + _logistic(z) * n
        y = h
    else:
        i, f, n, o = parts
        h = _logistic(f) * st["state"] + _logistic(i) * torch.tanh(n)
        y = _logistic(o) * torch.tanh(h)
    st["state"].copy_(h)
    return [y.to(st["x"].dtype), st["state"]]


def _plain_scan(st):
    case, dim, gate_dim = st["case"], st["dim"], st["gate_dim"]
    x = st["x"].detach()
    steps = case["steps"]
    parts = [p.float() for p in x.chunk(GATES[case["form"]], gate_dim)]
    one = torch.ones((), device=x.device)
    zero = torch.zeros((), device=x.device)
    live = last = None
    if st["lengths"] is not None:
        view = [1] * parts[0].dim()
        view[0], view[dim] = -1, 1
        ends = st["lengths"].view(view)
        view[0], view[dim] = 1, steps
        t = torch.arange(steps, device=x.device).view(view)
        live, last = t < ends, t == ends - 1

    def valid(v, other):
        return v if live is None else torch.where(live, v, other)

    if case["form"] == "leaky":
        z, n = parts
        keep, take = _logistic(-z), _logistic(z)
        put = take * n
    else:
        i, f, n, o = parts
        keep, take, cand, show = _logistic(f), _logistic(i), torch.tanh(n), _logistic(o)
        put = take * cand
    keep, put = valid(keep, one), valid(put, zero)
    first = put.clone()
    if st["h0"] is not None:
        h0 = st["h0"].detach()
        first.select(dim, 0).add_(keep.select(dim, 0) * h0)
    state = _linear(keep, first, dim)
    if case["form"] == "leaky":
        y, end_y = state, state.select(dim, steps - 1)
    else:
        tc = torch.tanh(state)
        y = show * tc
        end_y = y.select(dim, steps - 1) if last is None else torch.where(last, y, zero).sum(dim)
    end = state.select(dim, steps - 1)
    out = [valid(y, zero).to(x.dtype)] if case["seq"] else []
    out += [end_y] if case["form"] == "leaky" else [end_y, end]
    if not case["train"]:
        return out

    dy = st["dy"].float() if st["dy"] is not None else torch.zeros_like(y)
    dy = valid(dy, zero)
    if case["form"] == "lstm":
        if last is None:
            dy = dy.clone()
            dy.select(dim, steps - 1).add_(st["dh"])
        else:
            dy = dy + torch.where(last, st["dh"].unsqueeze(dim), zero)
        local = dy * show * (1.0 - tc * tc)
    else:
        local = dy.clone()
        local.select(dim, steps - 1).add_(st["dh"])       # behind a row's end the state is carried along
    ahead = torch.zeros_like(keep)
    ahead.narrow(dim, 0, steps - 1).copy_(keep.narrow(dim, 1, steps - 1))
    grad = _linear(ahead, local, dim, reverse=True)
    before = torch.zeros_like(state)
    before.narrow(dim, 1, steps - 1).copy_(state.narrow(dim, 0, steps - 1))
    if st["h0"] is not None:
        before.select(dim, 0).copy_(h0)
    if case["form"] == "leaky":
        ds = [grad * (n - before) * take * keep, grad * take]
    else:
        ds = [grad * cand * take * _logistic(-i), grad * before * keep * _logistic(-f),
              grad * take * (1.0 - cand * cand), dy * tc * show * _logistic(-o)]
    out.append(torch.cat([valid(d, zero) for d in ds], gate_dim).to(x.dtype))
    if st["h0"] is not None:
        out.append(keep.select(dim, 0) * grad.select(dim, 0))
    return out


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "clip":
        return _exact_clip(st)
    if case["op"] == "step":
        s = torch.sigmoid
        h = st["state"].double()
        w = case["width"]
        g = [st["x"][:, k * w:(k + 1) * w].double() for k in range(GATES[case["form"]])]
        if case["form"] == "leaky":
            h = h + s(g[0]) * (g[1] - h)
            return [h, h]
        h = s(g[1]) * h + s(g[0]) * torch.tanh(g[2])
        return [s(g[3]) * torch.tanh(h), h]
    rows = max(1, int(1.5e8 // (case["steps"] * _features(case))))
    got = [_exact_rows(st, r, min(r + rows, case["batch"])) for r in range(0, case["batch"], rows)]
    return [torch.cat(parts) for parts in zip(*got)]


def _exact_clip(st):
    p = st["norm_type"]
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in st["grads"]:
        if g.numel() == 0:
            continue
        v = torch.linalg.vector_norm(g.double(), p)
        total = torch.maximum(total, v) if p == math.inf else total + v ** p
    norm = total if p == math.inf else total ** (1.0 / p)
    coef = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
    if st["out"] is not None:
        return [norm, torch.cat([g.double() * coef for g in st["grads"]])]
    return [norm] + [f.double() * coef for f in st["flat"]]


def _exact_rows(st, r0, r1):
    """Rows r0 <= b < r1: one frame after the other, gradients from autograd."""
    case, dim = st["case"], st["dim"]
    x = st["x"].detach()[r0:r1].double()
    h0 = st["h0"].detach()[r0:r1].double() if st["h0"] is not None else None
    train = case["train"]
    if train:
        x.requires_grad_()
        if h0 is not None:
            h0.requires_grad_()
    n = st["lengths"][r0:r1] if st["lengths"] is not None else None
    with torch.set_grad_enabled(train):
        w = x.shape[st["gate_dim"]] // GATES[case["form"]]
        gate = [x.narrow(st["gate_dim"], k * w, w) for k in range(GATES[case["form"]])]
        if case["form"] == "leaky":
            leak = torch.sigmoid(gate[0])
            seq = [v.unbind(dim) for v in (leak, gate[1])]
        else:
            seq = [v.unbind(dim) for v in (torch.sigmoid(gate[0]), torch.sigmoid(gate[1]),
                                           torch.tanh(gate[2]), torch.sigmoid(gate[3]))]
        h = h0 if h0 is not None else torch.zeros_like(seq[0][0])
        end_y = h if case["form"] == "leaky" else torch.zeros_like(h)
        ys = []
        for t in range(case["steps"]):
            if case["form"] == "leaky":
                new = h + seq[0][t] * (seq[1][t] - h)
                y = new
            else:
                new = seq[1][t] * h + seq[0][t] * seq[2][t]
                y = seq[3][t] * torch.tanh(new)
            if n is not None:
                on = (t < n).view(-1, *([1] * (h.dim() - 1)))
                new, end_y = torch.where(on, new, h), torch.where(on, y, end_y)
                y = torch.where(on, y, torch.zeros_like(y))
            else:
                end_y = y
            h = new
            if case["seq"]:
                ys.append(y)
        out = [torch.stack(ys, dim)] if case["seq"] else []
        out += [end_y] if case["form"] == "leaky" else [end_y, h]
        if not train:
            return out
        heads, ds = [end_y], [st["dh"][r0:r1].double()]
        if case["seq"]:
            heads.append(out[0])
            ds.append(st["dy"][r0:r1].double())
        grads = torch.autograd.grad(heads, [x] + ([h0] if h0 is not None else []), ds)
    return [v.detach() for v in out] + list(grads)
