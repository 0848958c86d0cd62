"""The lstm form of the gated scan where candidates and states are small: tanh keeps
its relative accuracy there, whatever the gates' type (bounds: oracle/scan_ref.py)."""
import pytest
import torch

from oracle import scan_ref
from test_gpu_scan import TYPES, _check, _close, _dev

pytestmark = pytest.mark.gpu


def _small(b, t, f, dtype, scale, seed):
    """Gates of size 1.5 and candidates and states of size ``scale``."""
    g = torch.Generator().manual_seed(seed)
    i, fg, n, o = (1.5 * torch.randn(b, t, f, generator=g) for _ in range(4))
    gates = [v.to(TYPES[dtype]) for v in (i, fg + 2.0, scale * n, o)]
    return gates, scale * torch.randn(b, f, generator=g), g


@pytest.mark.parametrize("scale", [1e-1, 1e-3, 1e-5, 1e-7])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("b,t,f", [(2, 3, 130), (2, 40, 70), (1, 700, 65)])   # one wave, several, the chain
def test_scan_of_small_candidates_and_states(b, t, f, dtype, scale):
    gates, h0, g = _small(b, t, f, dtype, scale, 7 * t)
    dy = torch.randn(b, t, f, generator=g).to(TYPES[dtype])
    _check("lstm", gates, 1, stack=2, h0=h0, dy=dy, dh=torch.randn(b, f, generator=g),
           dc=torch.randn(b, f, generator=g))
    _check("lstm", gates, 1, stack=2, h0=h0, dh=torch.randn(b, f, generator=g), want_seq=False)


@pytest.mark.parametrize("scale", [1e-1, 1e-3, 1e-5, 1e-7])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("f", [77, 512])
def test_step_of_small_candidates_and_states(f, dtype, scale):
    from ptamd import scan
    gates, h0, _ = _small(3, 1, f, dtype, scale, f)
    val, bnd = scan_ref.walk("lstm", gates, h0, backward=False)
    state = h0.to(_dev())
    y = scan.gated_scan_step(torch.cat(gates, 2)[:, 0].to(_dev()), state, form="lstm")
    _close(y, val["y"][:, 0], bnd["y"][:, 0], "y")
    _close(state, val["c"], bnd["c"], "state")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_tanh_over_its_whole_range(dtype):
    """One step from c = 0 with open gates is tanh(tanh(n)), n from 2^-24 to 2^4 and
    both signs, around the borders of its branches too."""
    from ptamd import scan
    n = torch.cat([2.0 ** torch.linspace(-24, 4, 3001, dtype=torch.float64),
                   torch.linspace(0.02, 0.08, 601, dtype=torch.float64),
                   torch.linspace(0.30, 0.40, 601, dtype=torch.float64)]).to(TYPES[dtype])
    n = torch.cat([n, -n])[None]
    gates = [torch.full_like(n, 40.0), torch.zeros_like(n), n, torch.full_like(n, 40.0)]
    val, bnd = scan_ref.walk("lstm", [v[:, None] for v in gates], backward=False)
    x = torch.cat(gates, 1).to(_dev())
    y, h, c = scan.gated_scan(x[:, None], form="lstm")
    _close(c, val["c"], bnd["c"], "c")
    _close(h, val["h"], bnd["h"], "h")
    _close(y, val["y"], bnd["y"], "y")
    state = torch.zeros(n.shape, device=_dev())
    y = scan.gated_scan_step(x, state, form="lstm")
    _close(state, val["c"], bnd["c"], "step's c")
    _close(y, val["y"][:, 0], bnd["y"][:, 0], "step's y")
