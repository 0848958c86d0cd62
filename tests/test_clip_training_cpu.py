"""The training harness's clipping option and the scanned ConvLSTM's registry
entry, host logic only."""
import types

import pytest
import torch

from ptamd import clip
from utils import engine, misc_functions
from utils.opts import parser


def test_clip_flag_is_off_by_default_and_reaches_the_reference_name():
    base = "--model InT --length 64 --speed 1 --dist 14".split()
    assert parser.parse_args(base).clip_grad == 0.0
    assert parser.parse_args(base + ["--clip-grad", "0.5"]).clip_grad == 0.5
    assert misc_functions.clip_grad_norm_ is clip.clip_grad_norm_


def test_convlstm_without_hidden_convolutions_keeps_the_parameters():
    args = types.SimpleNamespace(model="convlstm", algo="bptt", penalty=False)
    torch.manual_seed(0)
    whole = engine.model_selector(args, timesteps=8, device="cpu")
    args.model = "convlstm_no_hidden"
    torch.manual_seed(0)
    cut = engine.model_selector(args, timesteps=8, device="cpu")
    assert list(whole.state_dict()) == list(cut.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(whole.state_dict().values(), cut.state_dict().values()))
    assert whole.lesion_hidden is False and all(p.requires_grad for p in whole.parameters())
    frozen = {n for n, p in cut.named_parameters() if not p.requires_grad}
    assert frozen == {f"unit1.Wh{g}.weight" for g in "ifco"}
    with pytest.raises(RuntimeError, match="ROCm device"):
        cut(torch.zeros(1, 3, 8, 32, 32))


class _Tiny(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.lin = torch.nn.Linear(3, 1)

    def forward(self, x):
        return self.lin(x.mean(dim=(2, 3, 4))), torch.ones(1)


def _harness(tmp_path, monkeypatch, *flags):
    """mainclean.py over synthetic clips with a CPU model and a CPU stand-in for the clipping."""
    import mainclean
    log = []

    class Norm:
        def item(self):
            log.append("read")
            return 1.5

    def fake_clip(params, max_norm):
        log.append(("clip", max_norm))
        return Norm()

    class Adam(torch.optim.SGD):
        def __init__(self, params, lr, fused):
            super().__init__(params, lr=lr)

        def step(self):
            log.append("step")
            return super().step()

    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    monkeypatch.setattr(mainclean.engine, "model_selector", lambda **kw: _Tiny())
    monkeypatch.setattr(mainclean, "clip_grad_norm_", fake_clip)
    monkeypatch.setattr(torch.optim, "Adam", Adam)
    out = mainclean.main(["--model", "InT", "--name", "t", "--dist", "14", "--speed", "1", "--length", "4", "-b", "4",
                          "--epochs", "1", "--data-root", str(tmp_path / "data"), "--synthetic", "16",
                          "--results-root", str(tmp_path / "res"), "--max-iters", "2", *flags])
    return log, out


def test_the_norm_is_read_behind_the_step(tmp_path, monkeypatch):
    """Its read waits for the whole backward: the step's launches go first."""
    log, out = _harness(tmp_path, monkeypatch, "--clip-grad", "0.5")
    assert log == [("clip", 0.5), "step", "read"] * 2
    assert out["train"]["gradnorm"] == [1.5, 1.5]


@pytest.mark.parametrize("bad", ["-1", "nan", "-0.5", "x"])
def test_a_norm_that_cannot_be_clipped_to_is_refused(bad, capsys):
    """(-1 and nan would have trained without clipping, and said nothing)"""
    with pytest.raises(SystemExit):
        parser.parse_args(["--model", "InT", f"--clip-grad={bad}"])
    assert "--clip-grad" in capsys.readouterr().err
    assert parser.parse_args(["--model", "InT", "--clip-grad", "inf"]).clip_grad == float("inf")   # the norm alone
