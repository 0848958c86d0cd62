"""What ptamd.scan and ptamd.clip refuse because the kernels would answer it
wrongly; all before any look at the device, so without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from ptamd import clip, scan


def _dual(*shape, **kw):
    return fwAD.make_dual(torch.zeros(*shape, **kw), torch.ones(*shape, **kw))


@pytest.mark.parametrize("grad", [False, True])
def test_inputs_with_a_tangent_are_refused(grad):
    plain = torch.zeros(2, 5, 8, requires_grad=grad)
    with fwAD.dual_level():
        calls = [
            (scan.PtScanError, lambda: scan.gated_scan(_dual(2, 5, 8))),
            (scan.PtScanError, lambda: scan.gated_scan([plain, _dual(2, 5, 8)])),
            (scan.PtScanError, lambda: scan.gated_scan(plain, _dual(2, 4))),
            (scan.PtScanError, lambda: scan.gated_scan_step(_dual(2, 8), torch.zeros(2, 4))),
            (scan.PtScanError, lambda: scan.gated_scan_step(torch.zeros(2, 8), _dual(2, 4))),
            (clip.PtClipError, lambda: clip.grad_norm([torch.zeros(3), _dual(3)])),
            (clip.PtClipError, lambda: clip.clip_grads([_dual(3)], 1.0)),
            (clip.PtClipError, lambda: clip.clip_grads([torch.zeros(3)], 1.0, out=[_dual(3)])),
        ]
        for error, call in calls:
            with pytest.raises(error, match="forward-mode"):
                call()
    with pytest.raises(scan.PtScanError, match="ROCm device"):      # without one the call goes on
        scan.gated_scan(plain)


def _calls(x, state):
    """(error, call) of every entry on gates x [B, T, 2 D] and a state [B, D]."""
    return [(scan.PtScanError, lambda: scan.gated_scan(x)[0]),
            (scan.PtScanError, lambda: scan.gated_scan_step(x[:, 0], state)),
            (clip.PtClipError, lambda: clip.grad_norm([state])),
            (clip.PtClipError, lambda: clip.clip_grads([state], 1.0)),
            (clip.PtClipError, lambda: clip.clip_grads([state], 1.0, out=[state]))]


@pytest.mark.parametrize("k", range(5))
def test_tracing_is_refused(k):
    def f(x, state):
        return _calls(x, state)[k][1]()

    x, state = torch.zeros(2, 5, 8), torch.zeros(2, 4)
    error = _calls(x, state)[k][0]
    with pytest.raises(error, match="traced"):
        torch.jit.trace(f, (x, state))
    for mode in ("real", "fake"):
        with pytest.raises(error, match="traced"):
            make_fx(f, tracing_mode=mode)(x, state)
    with FakeTensorMode() as fake:
        with pytest.raises(error, match="traced"):
            f(fake.from_tensor(x), fake.from_tensor(state))
    with pytest.raises(error, match="ROCm device"):
        f(x, state)


def test_tensors_without_memory_of_their_own_are_refused():
    with FakeTensorMode() as fake:
        x, state = (fake.from_tensor(torch.zeros(s)) for s in ((2, 5, 8), (2, 4)))
    for error, call in _calls(x, state):
        with pytest.raises(error, match="plain tensors"):
            call()
    with pytest.raises(scan.PtScanError, match="plain tensors"):
        scan.gated_scan(torch.zeros(2, 5, 8), state)


def test_writing_into_a_negated_view_is_refused():
    """x.conj().imag holds the values' negatives: a kernel's store would land with the other sign."""
    state = torch.zeros(2, 4, dtype=torch.complex64).conj().imag
    assert state.is_neg() and state.dtype == torch.float32
    with pytest.raises(scan.PtScanError, match="negated view"):
        scan.gated_scan_step(torch.zeros(2, 8), state)
    with pytest.raises(clip.PtClipError, match="negated view"):
        clip.clip_grads([torch.zeros(2, 4)], 1.0, out=[state])
