"""Sequences of no steps and batches of no rows, in training."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form,count", [("leaky", 2), ("lstm", 4)])
@pytest.mark.parametrize("shape", [(2, 0, 5), (0, 3, 5), (2, 3, 0)])
@pytest.mark.parametrize("state", [None, False, True])
def test_every_output_has_a_gradient_of_the_gates(form, count, shape, state):
    from ptamd import scan
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    b, t, f = shape
    h0 = None if state is None else torch.randn(b, f, device="cuda", requires_grad=state)
    for want_seq in (True, False):
        for stacked in (True, False):
            x = torch.randn(b, t, count * f, device="cuda", requires_grad=True)
            xs = x if stacked else list(x.chunk(count, 2))
            res = [r for r in scan.gated_scan(xs, h0, form=form, want_seq=want_seq) if r is not None]
            assert len(res) == (2 if form == "lstm" else 1) + want_seq
            for r in res:
                assert r.requires_grad
                grads = torch.autograd.grad(r.sum(), [x] + ([h0] if state else []), retain_graph=True,
                                            allow_unused=True)
                assert grads[0].shape == x.shape and not grads[0].any()
            end = res[-1]                       # the state after no steps is the one before
            assert torch.equal(end, torch.zeros(b, f, device="cuda") if h0 is None else h0)
            if state:
                assert torch.equal(torch.autograd.grad(end.sum(), h0)[0], torch.ones_like(h0))
