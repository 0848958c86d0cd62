"""Backwards captured into a graph while another autograd graph of the same leaves
lives: one from the default stream is refused (before anything of the backward is
launched), any other goes on."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _leaf():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.randn(2, 40, 64, device="cuda", requires_grad=True)


def _on(stream, fn):
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = fn()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    return out


def test_which_graphs_go_on_to_the_default_stream():
    """Without any capture: what the refusal looks at."""
    from ptamd import scan
    seen, side = scan.native().waits_on_default_stream, torch.cuda.Stream()
    x, w = _leaf(), torch.randn(64, 64, device="cuda", requires_grad=True)

    def pair():
        return scan.gated_scan(x)[0], scan.gated_scan(x @ w)[0]

    direct, behind = pair()
    assert seen(direct) and seen(behind)                     # built on the default stream
    direct = behind = None
    direct, behind = _on(side, pair)
    assert not seen(direct) and not seen(behind)
    direct = behind = None
    eager = (w * 2).sum()                                    # keeps w's accumulator, made here
    direct, behind = _on(side, pair)
    assert not seen(direct) and seen(behind)
    direct = behind = None
    eager = None
    direct, behind = _on(side, pair)
    assert not seen(direct) and not seen(behind)


def test_what_a_running_backward_does_not_reach_does_not_count():
    """As the refusal asks: from within a backward, for the leaves that it was asked for."""
    from ptamd import scan
    x, w = _leaf(), torch.randn(64, 64, device="cuda", requires_grad=True)
    eager = (w * 2).sum()
    asked = []

    def once(*leaves):
        y = scan.gated_scan(x @ w)[0]
        y.register_hook(lambda g: asked.append(scan.native().waits_on_default_stream(y)))
        torch.autograd.grad(y.sum(), leaves)

    side = torch.cuda.Stream()
    for leaves, want in (((x,), False), ((w,), True), ((x, w), True)):
        _on(side, lambda: once(*leaves))
        assert asked.pop() is want, leaves
    assert eager.requires_grad


@pytest.mark.parametrize("through", [False, True])
def test_a_capture_that_cannot_end_is_refused(through):
    from ptamd import scan
    x = _leaf()
    w = torch.randn(64, 64, device="cuda", requires_grad=True)
    leaf = w if through else x
    dy = torch.randn(2, 40, 32, device="cuda")

    def forward():
        return scan.gated_scan(x.detach() @ w if through else x)[0]

    want, = _on(torch.cuda.Stream(), lambda: torch.autograd.grad(forward(), leaf, dy))     # warm: libraries, buffers
    eager = (leaf * 2).sum()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forward()
        with pytest.raises(RuntimeError, match="default stream"):
            torch.autograd.grad(y, leaf, dy)
    y = graph = None
    # the forward alone may be captured, and the backward once the other graph is gone
    eager = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(forward(), leaf, dy)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        torch.testing.assert_close(got, want)


def test_a_graph_of_other_leaves_may_live():
    from ptamd import scan
    x, other = _leaf(), _leaf()
    dy = torch.randn(2, 40, 32, device="cuda")
    want, = _on(torch.cuda.Stream(), lambda: torch.autograd.grad(scan.gated_scan(x)[0], x, dy))
    eager = scan.gated_scan(other)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(scan.gated_scan(x)[0], x, dy)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert eager.requires_grad
