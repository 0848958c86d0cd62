"""The scanned recurrence and the clipping as a trainer uses them: the ConvLSTM
without hidden convolutions (models/convlstm.py), a training step with clipped
gradients, and mainclean.py --clip-grad."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def _model(t, k=5):
    from models.convlstm import ConvLSTMVideo
    torch.manual_seed(3)
    m = ConvLSTMVideo(dimensions=6, timesteps=t, kernel_size=k, lesion_hidden=True)
    with torch.no_grad():
        m.readout_dense.weight.fill_(1.5)
    return m


def _reference(m, x):
    """(logits, h_1..T) in float64 on the CPU, frame by frame: the cell's own step with h = 0."""
    cell = m.unit1
    frames = F.softplus(m.preproc(x))
    h = c = torch.zeros_like(frames[:, :, 0])
    hs = []
    for t in range(frames.shape[2]):
        xt = frames[:, :, t]
        i, f, n, o = (getattr(cell, f"Wx{g}")(xt) for g in "ifco")
        c = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(n)
        h = torch.sigmoid(o) * torch.tanh(c)
        hs.append(h)
    out = torch.cat([m.readout_conv(h), x[:, 2, 0][:, None]], 1)
    out = F.avg_pool2d(m.target_conv(out), kernel_size=h.shape[2:])
    return m.readout_dense(out.reshape(x.shape[0], -1)), torch.stack(hs, 1)


def test_convlstm_without_hidden_convolutions_matches_the_cell_step():
    dev = _dev()
    t = 9
    m = _model(t)
    x = torch.rand(3, 3, t, 32, 32, generator=torch.Generator().manual_seed(1))
    ref = _model(t).double()
    lo_ref, hs_ref = _reference(ref, x.double())
    w = torch.randn(3, 1, generator=torch.Generator().manual_seed(2))
    lo_ref.backward(w.double())
    m = m.to(dev).train()
    out, jv = m(x.to(dev))
    out.backward(w.to(dev))
    # f32 convolutions of at most 6 x 25 products, 9 steps: 1e-5 of the values' size
    torch.testing.assert_close(out.detach().cpu().double(), lo_ref.detach(), rtol=1e-5, atol=1e-5)
    assert torch.equal(jv.cpu(), torch.ones(1))
    for (n, p), q in zip(m.named_parameters(), ref.parameters()):
        if ".Wh" in n:
            assert p.grad is None
            continue
        scale = float(q.grad.abs().max())
        assert float((p.grad.cpu().double() - q.grad).abs().max()) <= 1e-4 * scale + 1e-9, n
    m.eval()
    with torch.no_grad():
        out2, states, hidden = m(x.to(dev), testmode=True)
    assert torch.equal(out2, out.detach()) and states.shape == (3, t, 1, 32, 32)
    torch.testing.assert_close(hidden.cpu().double(), hs_ref.detach(), rtol=1e-5, atol=1e-5)


def test_bf16_gates_stay_near_f32():
    dev = _dev()
    m = _model(16).to(dev)
    u8 = torch.randint(0, 256, (2, 16, 32, 32, 3), dtype=torch.uint8, device=dev)
    a = m(u8)[0].detach()
    m.cell_dtype = "bf16"
    b, _ = m(u8)
    b.sum().backward()
    # a gate is off by a few 2^-9 of its size (about 1); the pooled logit averages 1024 pixels
    assert float((a - b.detach()).abs().max()) <= 0.02
    assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)


def test_a_training_step_with_clipped_gradients():
    """Scan -> loss -> backward -> clip -> Adam, against the same step with the
    gradients scaled by hand."""
    from ptamd import clip, scan
    dev = _dev()
    torch.manual_seed(0)
    lin = torch.nn.Linear(24, 2 * 48).to(dev)
    x = torch.randn(4, 70, 24, device=dev)
    lengths = torch.tensor([70, 1, 33, 64], device=dev)
    state = {k: v.clone() for k, v in lin.state_dict().items()}

    def grads():
        lin.zero_grad(set_to_none=True)
        y, h = scan.gated_scan(lin(x), lengths=lengths)
        (y.square().sum() + h.sum()).backward()
        return [p.grad for p in lin.parameters()]

    runs = []
    for by_hand in (False, True):
        lin.load_state_dict(state)
        opt = torch.optim.Adam(lin.parameters(), lr=0.1)
        g = grads()
        if by_hand:
            total = torch.sqrt(sum((v.double() ** 2).sum() for v in g))
            k = torch.clamp(0.25 / (total + 1e-6), max=1.0)
            for v in g:
                v.copy_((v.double() * k).float())
            norm = total.float()
        else:
            norm = clip.clip_grad_norm_(lin.parameters(), 0.25)
        opt.step()
        runs.append([norm] + [p.detach().clone() for p in lin.parameters()] + [v.clone() for v in g])
    assert float(runs[0][0]) > 0.25
    for a, b in zip(*runs):      # the factor and the product are rounded once each
        torch.testing.assert_close(a, b, rtol=4 * 2.0 ** -24, atol=1e-9)


@pytest.mark.parametrize("model", ["InT", "convlstm_no_hidden"])
def test_mainclean_with_clipping(tmp_path, model):
    _dev()
    import mainclean
    out = mainclean.main(["--model", model, "--name", "clip", "--dist", "14", "--speed", "1",
                          "--length", "8", "-b", "4", "--epochs", "1", "--print-freq", "1",
                          "--data-root", str(tmp_path / "data"), "--synthetic", "16",
                          "--results-root", str(tmp_path / "res"), "--max-iters", "3",
                          "--clip-grad", "1e-3"])
    tr = out["train"]
    assert len(tr["loss"]) == len(tr["gradnorm"]) == 3
    assert all(np.isfinite(tr["loss"])) and all(np.isfinite(tr["gradnorm"])) and min(tr["gradnorm"]) > 0
