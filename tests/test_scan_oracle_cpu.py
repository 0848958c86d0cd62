"""The 64-bit oracle of the gated scan (oracle/scan_ref.py) against autograd
through the definition and against central differences."""
import pytest
import torch

from oracle import scan_ref


def _definition(form, gates, h0, lengths):
    b, t_len, _ = gates[0].shape
    h = h0
    end = h if form == "leaky" else torch.zeros_like(h)
    ys = []
    for t in range(t_len):
        on = (t < lengths)[:, None]
        g = [v[:, t] for v in gates]
        if form == "leaky":
            new = (1 - torch.sigmoid(g[0])) * h + torch.sigmoid(g[0]) * g[1]
            y = new
        else:
            new = torch.sigmoid(g[1]) * h + torch.sigmoid(g[0]) * torch.tanh(g[2])
            y = torch.sigmoid(g[3]) * torch.tanh(new)
        h = torch.where(on, new, h)
        end = torch.where(on, y, end)
        ys.append(torch.where(on, y, torch.zeros_like(y)))
    return torch.stack(ys, 1), end, h


@pytest.mark.parametrize("form,count", [("leaky", 2), ("lstm", 4)])
def test_oracle_against_autograd_and_differences(form, count):
    g = torch.Generator().manual_seed(5)
    b, t, f = 4, 6, 3
    gates = [torch.randn(b, t, f, generator=g, dtype=torch.float64).requires_grad_() for _ in range(count)]
    h0 = torch.randn(b, f, generator=g, dtype=torch.float64).requires_grad_()
    lengths = torch.tensor([6, 0, 1, 4])
    dy, dh, dc = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((b, t, f), (b, f), (b, f)))
    y, end, c = _definition(form, gates, h0, lengths)
    loss = (y * dy).sum() + (end * dh).sum() + (c * dc).sum()
    want = torch.autograd.grad(loss, [*gates, h0])
    val, bnd = scan_ref.walk(form, [v.detach() for v in gates], h0.detach(), lengths, dy, dh, dc)
    for got, ref in zip((val["y"], val["h"], val["c"], *val["dgates"], val["dh0"]), (y, end, c, *want)):
        torch.testing.assert_close(got, ref.detach(), rtol=1e-12, atol=1e-14)
    assert all(bool((v >= 0).all()) for v in (bnd["y"], bnd["h"], bnd["c"], *bnd["dgates"], bnd["dh0"]))

    def scalar(gs):
        yy, e, cc = _definition(form, gs, h0.detach(), lengths)
        return ((yy * dy).sum() + (e * dh).sum() + (cc * dc).sum()).item()

    step = 1e-5                                  # error of the difference: step^2 |f'''| + 2^-52 / step ~ 1e-10
    for k in range(count):
        v = torch.randn(gates[k].shape, generator=g, dtype=torch.float64)
        up = [w.detach() + (step * v if j == k else 0) for j, w in enumerate(gates)]
        down = [w.detach() - (step * v if j == k else 0) for j, w in enumerate(gates)]
        assert abs((scalar(up) - scalar(down)) / (2 * step) - (val["dgates"][k] * v).sum().item()) < 1e-8


@pytest.mark.parametrize("form,count", [("leaky", 2), ("lstm", 4)])
def test_bounds_hold_for_the_definition_in_f32(form, count):
    """An f32 walk of the same formulas stays inside the bounds that the GPU tests use."""
    g = torch.Generator().manual_seed(6)
    gates = [2 * torch.randn(3, 200, 5, generator=g) for _ in range(count)]
    h0 = torch.randn(3, 5, generator=g)
    lengths = torch.tensor([200, 57, 1])
    val, bnd = scan_ref.walk(form, gates, h0, lengths, backward=False)
    y, end, c = _definition(form, gates, h0, lengths)
    for got, k in ((y, "y"), (end, "h"), (c, "c")):
        assert bool(((got.double() - val[k]).abs() <= bnd[k] + scan_ref.rounding(val[k], torch.float32)).all()), k
