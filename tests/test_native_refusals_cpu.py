"""What ptamd.scan and ptamd.clip refuse because the kernels would answer it
wrongly; all before any look at the device, so without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

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
