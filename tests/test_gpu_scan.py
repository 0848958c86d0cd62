"""The gated scan on the GPU (ptamd/scan.py) against the 64-bit oracle, inside
bounds that follow the recurrence (oracle/scan_ref.py) plus half a step of the
output's type: forms, types, layouts, row ends, states, strides, streams,
graphs, and a prompt continued step by step."""
import math

import pytest
import torch

from oracle import scan_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GATES = {"leaky": 2, "lstm": 4}


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def _gates(form, shape, dtype, seed, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    out = [scale * torch.randn(shape, generator=g) for _ in range(GATES[form])]
    out[0 if form == "leaky" else 1].add_(-2.0 if form == "leaky" else 2.0)
    return [v.to(dtype) for v in out], g


def _close(got, want, bound, what):
    """|got - want| within the bound and half a step of got's type, everywhere."""
    got_d, want = got.detach().cpu().double(), want.reshape(got.shape)
    bound = bound.reshape(got.shape)
    tol = bound + scan_ref.rounding(want.abs() + bound, got.dtype)
    bad = ~((got_d - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got_d - want).abs() / tol.clamp(min=1e-300)).max()))


def _btf(t, dim):
    """[.., T, ..] to [B, T, F] with the batch in front (dimension 0, or all of it where time is first)."""
    if dim == 0:
        return t.reshape(1, t.shape[0], -1)
    return t.movedim(dim, 1).reshape(t.shape[0], t.shape[dim], -1)


def _check(form, gates, dim, *, stack=None, h0=None, lengths=None, dy=None, dh=None, dc=None, want_seq=True,
           device=None):
    """One forward and backward through ``gated_scan`` against the oracle.  ``stack``: the
    dimension to stack the gates along (None: one tensor per gate)."""
    from ptamd import scan
    dev = device or _dev()
    flat = [_btf(v, dim) for v in gates]
    b, t, f = flat[0].shape
    val, bnd = scan_ref.walk(form, flat, None if h0 is None else h0.reshape(b, f), lengths,
                             None if dy is None else _btf(dy, dim), None if dh is None else dh.reshape(b, f),
                             None if dc is None else dc.reshape(b, f))
    if stack is None:
        xs = [v.to(dev).requires_grad_() for v in gates]
        arg, kw = xs, {}
    else:
        xs = [torch.cat(gates, stack).to(dev).requires_grad_()]
        arg, kw = xs[0], dict(gate_dim=stack)
    h0d = None if h0 is None else h0.to(dev).requires_grad_()
    res = scan.gated_scan(arg, h0d, form=form, dim=dim, lengths=None if lengths is None else lengths.to(dev),
                          want_seq=want_seq, **kw)
    y, h = res[0], res[1]
    if want_seq:
        assert y.shape == gates[0].shape and y.dtype == gates[0].dtype
        _close(_btf(y.cpu(), dim), val["y"], bnd["y"], "y")
    else:
        assert y is None
    _close(h, val["h"], bnd["h"], "h_last")
    if form == "lstm":
        _close(res[2], val["c"], bnd["c"], "c_last")
    heads, ds = [], []
    for out, d in ((y, dy), (h, dh), (res[2] if form == "lstm" else None, dc)):
        if d is not None:
            heads.append(out)
            ds.append(d.to(dev))
    leaves = xs + ([h0d] if h0d is not None else [])
    grads = torch.autograd.grad(heads, leaves, ds)
    dx = grads[:len(xs)]
    if stack is not None:
        dx = dx[0].chunk(len(gates), stack)
    for k, g in enumerate(dx):
        _close(_btf(g.cpu(), dim), val["dgates"][k], bnd["dgates"][k], f"gate {k}")
    if h0d is not None:
        _close(grads[-1], val["dh0"], bnd["dh0"], "h0")


def _run(form, dtype, b, t, f, seed, h0=True, lengths=None, stack=2, want_seq=True):
    gates, g = _gates(form, (b, t, f), TYPES[dtype], seed)
    h = torch.randn(b, f, generator=g) if h0 else None
    dy = torch.randn(b, t, f, generator=g).to(TYPES[dtype]) if want_seq else None
    dh = torch.randn(b, f, generator=g)
    dc = torch.randn(b, f, generator=g) if form == "lstm" else None
    _check(form, gates, 1, stack=stack, h0=h, lengths=lengths, dy=dy, dh=dh, dc=dc, want_seq=want_seq)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form", list(GATES))
@pytest.mark.parametrize("b,t,f", [
    (1, 1, 1), (2, 3, 5), (3, 8, 64), (2, 9, 130),     # one wave; one chunk
    (2, 37, 200), (1, 33, 127), (3, 129, 66),          # several waves, ragged chunks
    (1, 129, 3), (1, 700, 65), (2, 1025, 34),          # the chain: chunks of a row in workgroups of their own
    (1, 9001, 3), (70, 400, 40),                       # more chunks than a group; more than the card holds
    (520, 41, 256),                                    # many columns: the four-wave groups
    (1000, 9, 3), (300, 140, 7), (9000, 3, 1),         # rows of few columns, side by side
])
def test_sizes(form, dtype, b, t, f):
    _run(form, dtype, b, t, f, seed=b * 1000 + t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", list(GATES))
@pytest.mark.parametrize("t,f", [(5, 70), (70, 6), (600, 130), (2049, 2), (8200, 3)])
def test_row_ends(form, dtype, t, f):
    """Ends of 0, 1, around a chunk's, the whole row, and outside [0, T]."""
    ends = torch.tensor([0, 1, min(t, 31), min(t, 129), t - 1, t, t + 7, -3, min(t, 4096), min(t, 4097)])
    _run(form, dtype, len(ends), t, f, seed=t, lengths=ends)
    _run(form, dtype, len(ends), t, f, seed=t + 1, lengths=ends.to(torch.int32), h0=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", list(GATES))
def test_last_state_only(form, dtype):
    _run(form, dtype, 2, 75, 96, seed=3, want_seq=False)
    _run(form, dtype, 3, 900, 31, seed=4, want_seq=False, lengths=torch.tensor([0, 900, 333]), h0=False)


@pytest.mark.parametrize("form", list(GATES))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape,dim,stack", [
    ((2, 3, 20, 4, 32), 2, 1),        # a clip batch, channels before time; inner = whole tiles
    ((2, 5, 20, 3, 7), 2, 1),         # the same, odd
    ((2, 20, 5, 4, 8), 1, 2),         # frames before channels
    ((20, 3, 10), 0, 2),              # time first
    ((20, 3, 10), 0, 1),
    ((2, 11, 45), 2, 1),              # time last
    ((2, 3, 11, 40, 2), 3, 1),
    ((4, 12), 1, None),               # one column per row
    ((300, 2), 0, None),
])
def test_layouts(form, dtype, shape, dim, stack):
    gates, g = _gates(form, shape, TYPES[dtype], 17)
    end = shape[:dim] + shape[dim + 1:]
    kw = dict(h0=torch.randn(end, generator=g), dy=torch.randn(shape, generator=g).to(TYPES[dtype]),
              dh=torch.randn(end, generator=g))
    _check(form, gates, dim, stack=None, **kw)
    if stack is not None:
        _check(form, gates, dim, stack=stack, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_alignment(dtype):
    """Views that begin off a pair of elements, step over elements, differ from
    gate to gate, or hold their axes in another order."""
    from ptamd import scan
    dev = _dev()
    gates, g = _gates("leaky", (2, 50, 64), TYPES[dtype], 23)
    dy = torch.randn(2, 50, 64, generator=g).to(TYPES[dtype])
    val, bnd = scan_ref.walk("leaky", gates, dy=dy)

    def wide(v, how):
        if how == "off":
            out = torch.full((2, 50, 67), math.nan, dtype=v.dtype, device=dev)[..., 1:65]
        elif how == "step":
            out = torch.full((2, 100, 64), math.nan, dtype=v.dtype, device=dev)[:, ::2]
        elif how == "skip":
            out = torch.full((2, 50, 128), math.nan, dtype=v.dtype, device=dev)[..., ::2]
        elif how == "order":
            out = torch.full((50, 2, 64), math.nan, dtype=v.dtype, device=dev).transpose(0, 1)
        else:
            out = torch.full((2, 64, 50), math.nan, dtype=v.dtype, device=dev).transpose(1, 2)
        return out.copy_(v).detach().requires_grad_()

    for hows in (("off", "off"), ("step", "order"), ("skip", "off"), ("order", "order"), ("last", "step")):
        xs = [wide(v, h) for v, h in zip(gates, hows)]
        y, _ = scan.gated_scan(xs)
        _close(y, val["y"], bnd["y"], hows)
        for k, d in enumerate(torch.autograd.grad(y, xs, dy.to(dev))):
            _close(d, val["dgates"][k], bnd["dgates"][k], (hows, k))
    # an expanded gradient (of a sum) and one in another order
    xs = [v.to(dev).requires_grad_() for v in gates]
    y, _ = scan.gated_scan(xs)
    v1, b1 = scan_ref.walk("leaky", gates, dy=torch.ones(2, 50, 64))
    for k, d in enumerate(torch.autograd.grad(y.float().sum(), xs, retain_graph=True)):
        _close(d, v1["dgates"][k], b1["dgates"][k], ("sum", k))
    turned = dy.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    for k, d in enumerate(torch.autograd.grad(y, xs, turned)):
        _close(d, val["dgates"][k], bnd["dgates"][k], ("turned", k))


@pytest.mark.parametrize("form", list(GATES))
def test_layouts_that_lie_like_a_larger_batch(form):
    """Batch and a further axis one behind the other in memory, the rest padded: row
    ends stay those of the batch, and a backward whose dy lies differently finds the
    forward's states."""
    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, (4, 30, 6, 5, 8), torch.float32, 71)
    ends = torch.tensor([30, 0, 17, 1])
    val, bnd = scan_ref.walk(form, [_btf(v, 1) for v in gates], lengths=ends)
    padded = []
    for v in gates:
        p = torch.full((30, 4, 6, 6, 9), math.nan, device=dev)[:, :, :, :5, :8].transpose(0, 1)
        padded.append(p.copy_(v))
    res = scan.gated_scan(padded, form=form, lengths=ends.to(dev), want_seq=False)
    _close(res[1], val["h"], bnd["h"], "h_last")

    for shape, dim in (((300, 130, 2, 5), 0), ((130, 300, 2, 5), 1), ((130, 2, 300, 5), 2)):
        gates, g = _gates(form, shape, torch.float32, 73)
        dy = torch.randn(shape, generator=g)
        val, bnd = scan_ref.walk(form, [_btf(v, dim) for v in gates], dy=_btf(dy, dim))
        xs = [v.to(dev).requires_grad_() for v in gates]
        y = scan.gated_scan(xs, form=form, dim=dim)[0]
        _close(_btf(y, dim), val["y"], bnd["y"], (dim, "y"))
        wide = torch.full([n + 1 for n in shape], math.nan, device=dev)
        apart = wide[tuple(slice(0, n) for n in shape)].copy_(dy)
        for k, d in enumerate(torch.autograd.grad(y, xs, apart)):
            _close(_btf(d.cpu(), dim), val["dgates"][k], bnd["dgates"][k], (dim, k))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form", list(GATES))
def test_what_stands_behind_a_row_is_never_used(form, dtype):
    """NaN, infinities and the type's lowest value behind the rows' ends change nothing."""
    from ptamd import scan
    dev = _dev()
    ends = torch.tensor([0, 1, 40, 130, 300])
    gates, g = _gates(form, (5, 300, 48), TYPES[dtype], 31)
    dy = torch.randn(5, 300, 48, generator=g).to(TYPES[dtype])
    behind = (torch.arange(300)[None] >= ends[:, None])[:, :, None].expand(5, 300, 48)
    outs = []
    for fill in (0.0, math.nan, math.inf, -math.inf, torch.finfo(TYPES[dtype]).min):
        x = torch.cat([torch.where(behind, torch.full_like(v, fill), v) for v in gates], 2).to(dev).requires_grad_()
        d = torch.where(behind, torch.full_like(dy, fill), dy).to(dev)
        res = scan.gated_scan(x, form=form, lengths=ends.to(dev))
        outs.append([r.detach() for r in res] + list(torch.autograd.grad(res[0], x, d)))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))
    assert not outs[0][0][behind.to(dev)].any()
    assert not outs[0][-1][behind.repeat(1, 1, GATES[form]).to(dev)].any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_saturated_gates(dtype):
    """Gates at the ends of their type: the state is kept, or replaced, exactly."""
    from ptamd import scan
    dev = _dev()
    t = TYPES[dtype]
    n = torch.randn(1, 40, 8).to(t)
    h0 = torch.randn(1, 8)
    for z, keep in ((-math.inf, True), (torch.finfo(t).min, True), (math.inf, False), (torch.finfo(t).max, False)):
        x = torch.cat([torch.full_like(n, z), n], 2).to(dev).requires_grad_()
        h = h0.to(dev).requires_grad_()
        y, last = scan.gated_scan(x, h)
        want = h0[:, None].expand(1, 40, 8).to(t) if keep else n
        assert torch.equal(y.cpu(), want) and torch.equal(last.cpu(), h0 if keep else n[:, -1].float())
        dx, dh0 = torch.autograd.grad(y.float().sum(), [x, h])
        assert not dx[..., :8].any()                       # s' = 0
        assert torch.equal(dx[..., 8:].cpu(), torch.zeros_like(n) if keep else torch.ones_like(n))
        assert torch.equal(dh0.cpu(), torch.full((1, 8), 40.0 if keep else 0.0))
    big = torch.finfo(t).max
    x = torch.full((1, 30, 32), big, dtype=t)             # all lstm gates open, candidate 1
    y, h, c = scan.gated_scan(x.to(dev), form="lstm")
    assert torch.equal(c.cpu(), torch.full((1, 8), 30.0)) and torch.equal(h.cpu(), torch.ones(1, 8))
    x = torch.randn(1, 30, 16).to(t)
    x[0, 7, 3] = math.nan                                  # a NaN stays in its column, from its step on
    y, _ = scan.gated_scan(x.to(dev))
    bad = torch.isnan(y.cpu())
    assert bool(bad[0, 7:, 3].all()) and int(bad.sum()) == 23


@pytest.mark.parametrize("form", list(GATES))
def test_gradient_against_differences(form):
    """The f32 kernels' own difference quotient: the loss is summed in 64 bits, so
    the quotient of step s is off by s^2 |f'''| / 6 + bound(f) / s."""
    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, (2, 60, 16), torch.float32, 41, scale=1.0)
    x = torch.cat(gates, 2).to(dev)
    h0 = torch.randn(2, 16, generator=g).to(dev)
    dy = torch.randn(2, 60, 16, generator=g).to(dev).double()
    v = torch.randn(x.shape, generator=g).to(dev)
    v = v / v.norm()

    def f(xx):
        return float((scan.gated_scan(xx, h0, form=form)[0].double() * dy).sum())

    xr = x.clone().requires_grad_()
    y = scan.gated_scan(xr, h0, form=form)[0]
    slope = float((torch.autograd.grad(y, xr, dy.float())[0].double() * v).sum())
    s = 2.0 ** -4
    quot = (f(x + s * v) - f(x - s * v)) / (2 * s)
    # along a unit direction of 1920+ gates a third derivative of a sum of 1920
    # outputs of size 1 is below 1; the f32 evaluations are off by their bound
    _, bnd = scan_ref.walk(form, gates, h0.cpu(), backward=False)
    noise = float((bnd["y"] ** 2).sum().sqrt()) * float((dy ** 2).sum().sqrt())
    assert abs(quot - slope) <= s * s / 6 + noise / s, (quot, slope)


def test_two_runs_agree_bit_for_bit_and_other_streams_do():
    from ptamd import scan
    dev = _dev()
    gates, g = _gates("lstm", (2, 1500, 96), torch.bfloat16, 53)
    x = torch.cat(gates, 2).to(dev).requires_grad_()
    dy = torch.randn(2, 1500, 96, generator=g).bfloat16().to(dev)

    def once():
        res = scan.gated_scan(x, form="lstm")
        return [r.detach() for r in res] + list(torch.autograd.grad(res[0], x, dy))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_two_chains_at_once():
    """Long rows on two streams at the same time: each call has a chain of its own."""
    from ptamd import scan
    dev = _dev()
    xs, want = [], []
    for k in range(2):
        gates, _ = _gates("leaky", (1, 6000 + 500 * k, 256), torch.bfloat16, 90 + k)
        xs.append(torch.cat(gates, 2).to(dev).requires_grad_())
    one = torch.ones((), device=dev)

    def once(k):
        y, h = scan.gated_scan(xs[k])
        return [y.detach(), h.detach(), torch.autograd.grad(h.sum(), xs[k], one)[0]]

    want = [once(k) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(once(k))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k])), k


@pytest.mark.parametrize("t,f", [(40, 64), (1500, 33)])
def test_captured_forward_and_backward(t, f):
    """Two graphs with workspaces of their own, replayed in turn with eager work between."""
    from ptamd import scan
    dev = _dev()
    xs, dys, graphs, outs = [], [], [], []
    for k in range(2):
        gates, g = _gates("leaky", (2, t, f), torch.float32, 60 + k)
        xs.append(torch.cat(gates, 2).to(dev).requires_grad_())
        dys.append(torch.randn(2, t, f, generator=g).to(dev))

    def once(k):
        y, h = scan.gated_scan(xs[k])
        return [y.detach(), h.detach(), torch.autograd.grad([y, h], xs[k], [dys[k], h.detach()])[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k in range(2):
            once(k)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(once(k))
        graphs.append(graph)
    for rep in range(3):
        with torch.no_grad():
            for x in xs:
                x.add_(0.125)
        for k in (0, 1, 0):
            graphs[k].replay()
        want = [once(k) for k in range(2)]
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[k])), (rep, k)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form", list(GATES))
@pytest.mark.parametrize("b,f", [(1, 1), (1, 2048), (3, 77), (64, 512), (5, 8)])
def test_step(form, dtype, b, f):
    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, (b, 1, f), TYPES[dtype], b * 100 + f)
    h0 = torch.randn(b, f, generator=g)
    val, bnd = scan_ref.walk(form, gates, h0, backward=False)
    x = torch.cat(gates, 2)[:, 0].to(dev)
    for state in (h0.to(dev), torch.zeros(b, 2 * f + 1, device=dev)[:, 1:f + 1].copy_(h0),
                  torch.zeros(f, b, device=dev).t().copy_(h0)):
        keep = state.data_ptr()
        y = scan.gated_scan_step(x, state, form=form)
        assert state.data_ptr() == keep
        _close(y, val["y"][:, 0], bnd["y"][:, 0], "y")
        _close(state, val["c"], bnd["c"], "state")
    state = h0.to(dev)
    y = scan.gated_scan_step([v[:, 0].to(dev) for v in gates], state, form=form)
    _close(y, val["y"][:, 0], bnd["y"][:, 0], "y, one tensor per gate")


@pytest.mark.parametrize("form", list(GATES))
def test_step_on_frames(form):
    """[B, G C, H, W] frames against states [B, C, H, W], channels-last ones too."""
    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, (3, 5, 6, 7), torch.float32, 9)
    h0 = torch.randn(3, 5, 6, 7, generator=g)
    val, bnd = scan_ref.walk(form, [v.reshape(3, 1, -1) for v in gates], h0.reshape(3, -1), backward=False)
    for fmt in (torch.contiguous_format, torch.channels_last):
        x = torch.cat(gates, 1).to(dev).contiguous(memory_format=fmt)
        state = h0.to(dev).contiguous(memory_format=fmt)
        y = scan.gated_scan_step(x, state, form=form)
        _close(y.reshape(3, -1), val["y"][:, 0], bnd["y"][:, 0], fmt)
        _close(state.reshape(3, -1), val["c"], bnd["c"], fmt)


@pytest.mark.parametrize("form", list(GATES))
def test_a_prompt_continued_step_by_step(form):
    """A scan over a prefix, then single steps from its last state: the whole scan's outputs."""
    from ptamd import scan
    dev = _dev()
    t, cut = 300, 273
    gates, _ = _gates(form, (2, t, 64), torch.float32, 77)
    val, bnd = scan_ref.walk(form, gates, backward=False)
    x = torch.cat(gates, 2).to(dev)
    res = scan.gated_scan(x[:, :cut], form=form)
    state = res[-1].clone()
    ys = [res[0]] + [scan.gated_scan_step(x[:, k], state, form=form)[:, None] for k in range(cut, t)]
    _close(torch.cat(ys, 1), val["y"], bnd["y"], "continued")
    _close(state, val["c"], bnd["c"], "state")


@pytest.mark.parametrize("form", list(GATES))
def test_step_with_the_state_inside_the_gates(form):
    """Overlapping memory: every gate is read before the state is written."""
    from ptamd import scan
    dev = _dev()
    n = GATES[form]
    buf = torch.randn(3, (n + 1) * 700, generator=torch.Generator().manual_seed(5)).to(dev)
    x, state = buf[:, :n * 700], buf[:, 350:1050]
    want_state = state.clone()
    want = scan.gated_scan_step(x.clone(), want_state, form=form)
    y = scan.gated_scan_step(x, state, form=form)
    assert torch.equal(y, want) and torch.equal(state, want_state)


def test_a_step_tells_autograd_that_it_wrote():
    from ptamd import scan
    dev = _dev()
    w = torch.ones(2, 4, device=dev, requires_grad=True)
    for state in (torch.ones(2, 4, device=dev), torch.ones(2, 8, device=dev)[:, ::2]):
        out = (w * state).sum()
        scan.gated_scan_step(torch.zeros(2, 8, device=dev), state)
        with pytest.raises(RuntimeError, match="inplace"):
            out.backward()
    with torch.inference_mode():
        state = torch.ones(2, 4, device=dev)
        assert float(scan.gated_scan_step(torch.zeros(2, 8, device=dev), state).sum()) == 4.0
        assert float(state.sum()) == 4.0


@pytest.mark.parametrize("t", [40, 900])
@pytest.mark.parametrize("form,which", [("leaky", "y"), ("leaky", "h"), ("lstm", "y"), ("lstm", "h"), ("lstm", "c")])
def test_one_output_alone_has_a_gradient(form, which, t):
    """The others' gradients are absent, not zero tensors."""
    gates, g = _gates(form, (2, t, 70), torch.bfloat16, t + len(which))
    d = torch.randn((2, t, 70) if which == "y" else (2, 70), generator=g)
    ends = torch.tensor([t, t // 3])
    _check(form, gates, 1, stack=2, h0=torch.randn(2, 70, generator=g), lengths=ends,
           **{"d" + which: d.to(torch.bfloat16) if which == "y" else d})


def test_graphs_of_the_gradients():
    """create_graph leaves the first gradients as they are and refuses the second."""
    from ptamd import scan
    dev = _dev()
    x = torch.randn(2, 30, 16, device=dev, requires_grad=True)
    want, = torch.autograd.grad(scan.gated_scan(x)[0].sum(), x)
    got, = torch.autograd.grad(scan.gated_scan(x)[0].sum(), x, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="differentiable once"):
        got.sum().backward()


@pytest.mark.parametrize("t,f", [(600_000, 2048), (60_000, 20_480)])
def test_offsets_past_32_bits(t, f):
    """4.9 GB of gates in one row (chunks of a row in workgroups of their own, and a
    workgroup walking it): both ends as scans of their own give them.

    A state is a mean of n's under weights that fall off fast: at most some 64
    roundings of 2^-24 of max |n| < 7 count, 3e-5; the gradients' factors are G < 30
    and |n - c| < 14, with s(z) s(-z) <= 1/4: 64 2^-24 30 14 / 4 < 5e-4.  bf16
    outputs are off by half a step, 2^-8, on either side."""
    from ptamd import scan
    g = torch.Generator(device=_dev()).manual_seed(t)
    x = torch.randn(1, t, 2 * f, generator=g, device=_dev(), dtype=torch.bfloat16)
    dy = torch.randn(1, t, f, generator=g, device=_dev(), dtype=torch.bfloat16)
    x.requires_grad_()
    y, h = scan.gated_scan(x)
    dx, = torch.autograd.grad(y, x, dy)
    y, h, x = y.detach(), h.detach(), x.detach()
    k = 1000

    def same(got, want, tol):
        assert bool(((got.float() - want.float()).abs() <= 2 ** -7 * want.float().abs() + tol).all())

    def part(sl, h0):
        xs = x[:, sl].clone().requires_grad_()
        ys, hs = scan.gated_scan(xs, h0)
        return ys.detach(), hs.detach(), torch.autograd.grad(ys, xs, dy[:, sl].clone())[0]

    ys, _, dxs = part(slice(0, k), None)
    same(y[:, :k], ys, 3e-5)
    same(dx[:, :k // 2], dxs[:, :k // 2], 5e-4)
    with torch.no_grad():
        before = scan.gated_scan(x[:, :t - k], want_seq=False)[1]
    ys, hs, dxs = part(slice(t - k, t), before)
    same(y[:, t - k:], ys, 3e-5)
    same(h, hs, 3e-5)
    same(dx[:, t - k:], dxs, 5e-4)


def test_empty_and_refused_calls():
    from ptamd import scan
    dev = _dev()
    h0 = torch.randn(2, 4, device=dev, requires_grad=True)
    x = torch.zeros(2, 0, 8, device=dev, requires_grad=True)
    y, h = scan.gated_scan(x, h0)
    assert y.shape == (2, 0, 4) and torch.equal(h, h0)
    (y.sum() + h.sum()).backward()
    assert x.grad.shape == x.shape and torch.equal(h0.grad, torch.ones_like(h0))
    y, h, c = scan.gated_scan(torch.zeros(0, 5, 16, device=dev), form="lstm")
    assert y.shape == (0, 5, 4) and h.shape == c.shape == (0, 4)
    assert scan.gated_scan_step(torch.zeros(0, 8, device=dev), torch.zeros(0, 4, device=dev)).shape == (0, 4)
    x = torch.zeros(2, 5, 8, device=dev)
    for kw, err, word in ((dict(dim=5), ValueError, "dim"), (dict(dim=2), ValueError, "time"),
                          (dict(dim=0, lengths=torch.ones(5, dtype=torch.int64, device=dev)), ValueError, "batch"),
                          (dict(lengths=torch.ones(3, dtype=torch.int64, device=dev)), ValueError, "lengths"),
                          (dict(lengths=torch.ones(2, device=dev)), TypeError, "integer"),
                          (dict(lengths=torch.ones(2, dtype=torch.int64)), TypeError, "device")):
        with pytest.raises(err, match=word):
            scan.gated_scan(x, **kw)
    with pytest.raises(ValueError, match="h0"):
        scan.gated_scan(x, torch.zeros(2, 5, device=dev))
    with pytest.raises(TypeError, match="h0"):
        scan.gated_scan(x, torch.zeros(2, 4))
    s = torch.zeros(2, 4, device=dev)
    with pytest.raises(TypeError, match="float32"):
        scan.gated_scan_step(x[:, 0], s.bfloat16())
    with pytest.raises(ValueError, match="shape"):
        scan.gated_scan_step(x[:, 0], s[:1])
    with pytest.raises(ValueError, match="share memory"):
        scan.gated_scan_step(x[:, 0], s[:1].expand(2, 4))
    with pytest.raises(scan.PtScanError, match="backward"):
        scan.gated_scan_step(x[:, 0].requires_grad_(), s)
