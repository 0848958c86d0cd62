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
