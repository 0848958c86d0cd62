"""Calls of the gated scan and of clipping that a program makes around them: graphs
whose inputs and row ends change between replays, graphs that share memory, a
captured step, hooks and checkpoints, inference mode, several threads, broadcast
and repeated inputs, negative dimensions."""
import threading

import pytest
import torch

from oracle import scan_ref
from test_gpu_scan import GATES, TYPES, _btf, _check, _close, _dev, _gates

pytestmark = pytest.mark.gpu


def _warm(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()


def _capture(fn, pool=None):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=pool):
        out = fn()
    return graph, out


@pytest.mark.parametrize("t,f", [(40, 130), (1500, 33), (300, 9000)])        # several waves, the chain, 16 waves
@pytest.mark.parametrize("form", list(GATES))
def test_row_ends_change_between_replays(form, t, f):
    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, (2, t, f), torch.bfloat16, t)
    x = torch.cat(gates, 2).to(dev).requires_grad_()
    h0 = torch.randn(2, f, generator=g).to(dev).requires_grad_()
    dy, dh = torch.randn(2, t, f, generator=g).bfloat16().to(dev), torch.randn(2, f, generator=g).to(dev)
    ends = torch.tensor([t, t // 2], device=dev)

    def once():
        res = scan.gated_scan(x, h0, form=form, lengths=ends)
        return [r.detach() for r in res] + list(torch.autograd.grad(res[:2], [x, h0], [dy, dh]))

    _warm(once)
    graph, out = _capture(once)
    for new in ([0, t], [1, t - 1], [t + 9, -4], [t // 3, t // 3 + 1]):
        ends.copy_(torch.tensor(new))
        with torch.no_grad():
            x.add_(0.0625)
        graph.replay()
        want = once()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), new


def test_graphs_that_share_a_pool():
    """One graph's scratch lies where the other's did: replayed in any order, one at a time."""
    from ptamd import scan
    dev = _dev()
    xs = [torch.cat(_gates("leaky", (1, 3000 + 700 * k, 192), torch.float32, k)[0], 2).to(dev).requires_grad_()
          for k in range(2)]

    def once(k):
        y, h = scan.gated_scan(xs[k])
        return y.detach(), torch.autograd.grad(h.sum(), xs[k])[0]

    _warm(lambda: [once(0), once(1)])
    first = _capture(lambda: once(0))
    second = _capture(lambda: once(1), first[0].pool())
    want = [[v.clone() for v in once(k)] for k in range(2)]
    for k in (0, 1, 1, 0, 1):
        graph, out = (first, second)[k]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k])), k


@pytest.mark.parametrize("form", list(GATES))
@pytest.mark.parametrize("strided", [False, True])
def test_captured_steps(form, strided):
    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, (6, 5, 200), torch.bfloat16, 3)
    xs = torch.cat(gates, 2).to(dev)
    x = xs[:, 0].clone()
    start = torch.randn(5, 6, 40, 5, generator=g).to(dev)
    make = (lambda: start[0].clone().view(6, 200)) if not strided else \
        (lambda: torch.empty(200, 6, device=dev).t().copy_(start[0].view(6, 200)))
    state = make()
    _warm(lambda: scan.gated_scan_step(x, state.clone(), form=form))
    graph, y = _capture(lambda: scan.gated_scan_step(x, state, form=form))
    state.copy_(make())
    eager = make()
    for k in range(5):
        x.copy_(xs[:, k])
        graph.replay()
        want = scan.gated_scan_step(xs[:, k], eager, form=form)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(state, eager), k


def test_captured_clipping_in_place_of_many_and_of_strided_gradients():
    from ptamd import clip
    dev = _dev()
    g = torch.Generator().manual_seed(9)
    base = [torch.randn(32 * k + 1, generator=g).to(list(TYPES.values())[k % 3]).to(dev) for k in range(400)]
    wide = torch.randn(50, 60, generator=g).to(dev)
    grads = [v.clone() for v in base] + [wide.clone()[:, ::2]]
    own = grads[-1]._base
    _warm(lambda: clip.clip_grads([v.clone() for v in grads], 1.0))
    graph, norm = _capture(lambda: clip.clip_grads(grads, 1.0))
    for scale in (1.0, 4.0, 1e-4, 0.25):                  # (above the threshold, below it, above)
        for v, b in zip(grads, base):
            v.copy_(b * scale)
        own.copy_(wide * scale)
        want = [v.clone() for v in grads]
        graph.replay()
        n = clip.clip_grads(want, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(grads, want)), scale
        assert torch.equal(own[:, 1::2], (wide * scale)[:, 1::2])


@pytest.mark.parametrize("form", list(GATES))
def test_saved_tensors_pass_through_hooks_and_checkpoints(form):
    from torch.utils.checkpoint import checkpoint

    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, (2, 900, 65), torch.bfloat16, 21)
    x = torch.cat(gates, 2).to(dev).requires_grad_()
    h0 = torch.randn(2, 65, generator=g).to(dev).requires_grad_()
    ends = torch.tensor([900, 411], device=dev)

    def loss(v, h):
        res = scan.gated_scan(v, h, form=form, lengths=ends)
        return res[0].float().square().sum() + res[-1].sum()

    want = torch.autograd.grad(loss(x, h0), [x, h0])
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        kept = loss(x, h0)
    out = kept, checkpoint(loss, x, h0, use_reentrant=False)
    for v in out:
        for _ in range(2 if v is kept else 1):           # twice over the same saved states
            got = torch.autograd.grad(v, [x, h0], retain_graph=v is kept)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        y = loss(x, h0)
    with torch.inference_mode():
        assert torch.equal(loss(x.detach().clone(), h0.detach().clone()), y)


def test_an_input_changed_before_the_backward_is_noticed():
    from ptamd import scan
    x = torch.randn(2, 30, 16, device=_dev(), requires_grad=True)
    for spoil in (0, 1):
        v, ends = x * 1.0, torch.tensor([30, 9], device=_dev())
        y = scan.gated_scan(v, lengths=ends)[0]
        (v if spoil == 0 else ends).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()


def test_threads_call_at_once():
    """A stream each; a thread's result is the one it gets alone."""
    from ptamd import clip, scan
    dev = _dev()
    xs = [torch.cat(_gates("lstm", (2, 1200 + 100 * k, 48), torch.float32, k)[0], 2).to(dev) for k in range(4)]
    grads = [[v[:, :, :50].clone() for v in xs[k:k + 1]] for k in range(4)]

    def once(k):
        x = xs[k].clone().requires_grad_()
        res = scan.gated_scan(x, form="lstm")
        out = [r.detach() for r in res] + list(torch.autograd.grad(res[1].sum(), x))
        buf = [torch.empty_like(v) for v in grads[k]]
        return out + [clip.clip_grads(grads[k], 1.0, out=buf)] + buf

    want = [once(k) for k in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[k] = once(k)
                torch.cuda.current_stream().synchronize()
        except Exception as e:            # noqa: BLE001  (the main thread raises it)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not errors, errors
    torch.cuda.synchronize()
    for k in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k])), k


@pytest.mark.parametrize("form", list(GATES))
def test_broadcast_and_repeated_inputs(form):
    """Gates shared by the rows, one tensor for every gate, a state for all rows: the
    gradients are the sums over the uses."""
    from ptamd import scan
    dev = _dev()
    n = GATES[form]
    gates, g = _gates(form, (1, 50, 70), torch.float32, 33)
    dy = torch.randn(3, 50, 70, generator=g)
    h0 = torch.randn(1, 70, generator=g)
    val, bnd = scan_ref.walk(form, [v.expand(3, 50, 70) for v in gates], h0.expand(3, 70), None, dy)
    xs = [v.to(dev).requires_grad_() for v in gates]
    hd = h0.to(dev).requires_grad_()
    for stacked in (False, True):
        x = torch.cat(xs, 2).expand(3, 50, n * 70) if stacked else [v.expand(3, 50, 70) for v in xs]
        y = scan.gated_scan(x, hd.expand(3, 70), form=form)[0]
        _close(y, val["y"], bnd["y"], "y")
        grads = torch.autograd.grad(y, xs + [hd], dy.to(dev))
        for k, d in enumerate(grads):
            want, tol = (val["dgates"][k], bnd["dgates"][k]) if k < n else (val["dh0"], bnd["dh0"])
            # three f32 values are added: each rounded once, and two sums
            tol = tol + 2 * scan_ref.rounding(want, torch.float32)
            _close(d, want.sum(0, keepdim=True), tol.sum(0, keepdim=True) +
                   2 * scan_ref.rounding(want.abs().sum(0, keepdim=True), torch.float32), (stacked, k))
    one = gates[0].to(dev).requires_grad_()
    val, bnd = scan_ref.walk(form, [gates[0]] * n, dy=dy[:1])
    y = scan.gated_scan([one] * n, form=form)[0]
    _close(y, val["y"], bnd["y"], "one tensor")
    d, = torch.autograd.grad(y, one, dy[:1].to(dev))
    parts = torch.stack(val["dgates"])
    _close(d, parts.sum(0), sum(bnd["dgates"]) + 5 * scan_ref.rounding(parts.abs().sum(0), torch.float32), "summed")


@pytest.mark.parametrize("form", list(GATES))
@pytest.mark.parametrize("shape,dim,stack", [((3, 40, 24), -2, -1), ((3, 24, 40), -1, -2), ((40, 3, 24), -3, -1),
                                             ((6, 40, 5), 1, 0), ((6, 5, 40), 2, 0), ((2, 3, 4, 40), -1, 1)])
def test_negative_dimensions_and_gates_in_front(form, shape, dim, stack):
    from ptamd import scan
    dev = _dev()
    gates, g = _gates(form, shape, torch.float32, 5)
    at = dim % len(shape)
    ends = torch.randint(0, 41, (shape[0],), generator=g) if at else None
    flat = [_btf(v, at) for v in gates]
    val, bnd = scan_ref.walk(form, flat, lengths=ends, backward=False)
    y, h = scan.gated_scan(torch.cat(gates, stack).to(dev), form=form, dim=dim, gate_dim=stack,
                           lengths=None if ends is None else ends.to(dev))[:2]
    _close(_btf(y, at), val["y"], bnd["y"], "y")
    _close(h, val["h"], bnd["h"], "h")
    _check(form, gates, at, stack=stack % len(shape), lengths=ends, dh=torch.randn(h.shape, generator=g))


def test_odd_strides_of_single_elements_and_types_of_row_ends():
    """Axes of one element may have any stride; ends in any integer type, strided."""
    from ptamd import scan
    dev = _dev()
    gates, g = _gates("leaky", (1, 60, 33), torch.bfloat16, 8)
    val, bnd = scan_ref.walk("leaky", gates, lengths=torch.tensor([41]), dy=torch.ones(1, 60, 33))
    mem = [v.to(dev).view(60, 33) for v in gates]
    for stride in (0, 1, 7, 10 ** 9):
        xs = [m.as_strided((1, 60, 33), (stride + k, 33, 1)).requires_grad_() for k, m in enumerate(mem)]
        for ends in (torch.tensor([41], dtype=torch.uint8, device=dev), torch.tensor([41, 0, 3], device=dev)[::3],
                     torch.tensor([41], dtype=torch.int16, device=dev)):
            y = scan.gated_scan(xs, lengths=ends)[0]
            _close(y, val["y"], bnd["y"], stride)
            for k, d in enumerate(torch.autograd.grad(y, xs, torch.ones_like(y))):
                _close(d, val["dgates"][k], bnd["dgates"][k], (stride, k))
