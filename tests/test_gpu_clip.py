"""The gradient norm and clipping on the GPU (ptamd/clip.py) against 64 bits.

Tolerances: squares and sums are held in 64 bits, so the norm is off by its
rounding to f32, 2^-24 relative, and the sums' n 2^-53, below 2^-29 here.  The
factor is rounded to f32 once, the product once: 2 x 2^-24, and half a step of
the output's type.
"""
import math

import numpy as np
import pytest
import torch

from oracle.scan_ref import rounding

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def _norm(grads, p):
    v = np.concatenate([g.cpu().double().reshape(-1).numpy() for g in grads] + [np.zeros(0)])
    if p == math.inf:
        return float(np.abs(v).max()) if v.size else 0.0
    return float((np.abs(v) ** p).sum()) ** (1.0 / p)


def _check(outs, befores, norm, max_norm, p, exact_below=True):
    want = _norm(befores, p)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= want * (U + 2 ** -29) + 2.0 ** -149
    k = min(1.0, max_norm / (want + 1e-6))
    for o, b in zip(outs, befores):
        ref = b.cpu().double() * k
        got = o.cpu().double()
        if k == 1.0 and exact_below:
            assert torch.equal(got, ref)
        else:
            # the kernel's factor is within one more 2^-52 of k before its rounding
            assert bool(((got - ref).abs() <= ref.abs() * 2.01 * U + rounding(ref, o.dtype) + 2.0 ** -149).all())


def _tensors(sizes, dtype, seed, scale=0.02):
    g = torch.Generator().manual_seed(seed)
    kinds = list(TYPES.values())
    return [(scale * torch.randn(n, generator=g)).to(kinds[k % 3] if dtype == "mixed" else TYPES[dtype]).to(_dev())
            for k, n in enumerate(sizes)]


SIZES = [
    [1], [7], [0, 3, 0], [8191, 8192, 8193], [1, 255, 256, 257, 2047, 2049, 65536, 40000],
    [32 * k + 1 for k in range(200)],                # three tables of pointers
    [9_000_001, 5, 3_000_000],
]


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip(sizes, dtype, p):
    from ptamd import clip
    grads = _tensors(sizes, dtype, len(sizes) + sum(sizes))
    before = [g.clone() for g in grads]
    want = _norm(before, p)
    assert abs(float(clip.grad_norm(grads, p)) - want) <= want * (U + 2 ** -29)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    # below the threshold: untouched; above it: into f32 buffers, then in place
    norm = clip.clip_grads(grads, 4 * want + 1.0, norm_type=p)
    _check(grads, before, norm, 4 * want + 1.0, p)
    out = [torch.full(g.shape, math.nan, device=g.device) for g in grads]
    norm = clip.clip_grads(grads, 0.3 * want, norm_type=p, out=out)
    _check(out, before, norm, 0.3 * want, p)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    norm = clip.clip_grads(grads, 4 * want + 1.0, norm_type=p, out=out)     # k = 1, another place: a copy
    _check(out, before, norm, 4 * want + 1.0, p)
    norm = clip.clip_grads(grads, 0.3 * want, norm_type=p)
    _check(grads, before, norm, 0.3 * want, p)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_odd_starts_leave_their_neighbours_alone(dtype):
    """Tensors packed without a gap in one buffer, some of them clipped."""
    from ptamd import clip
    sizes = [3, 1, 8192, 5, 20000, 7, 8200, 1, 0, 4097]
    flat = _tensors([sum(sizes)], dtype, 4)[0]
    before = flat.clone()
    parts, old = list(flat.split(sizes)), list(before.split(sizes))
    some = [k for k in range(len(sizes)) if k % 3 != 1]
    want = _norm([old[k] for k in some], 2.0)
    norm = clip.clip_grads([parts[k] for k in some], 0.5 * want)
    _check([parts[k] for k in some], [old[k] for k in some], norm, 0.5 * want, 2.0)
    assert all(torch.equal(parts[k], old[k]) for k in range(len(sizes)) if k not in some)


def test_large_and_tiny_values():
    """f32 squares would overflow above 1.8e19 and vanish below 1e-23; the sums do not."""
    from ptamd import clip
    dev = _dev()
    for scale in (1e30, 1e-30, 3e38, 1e-40):
        grads = [torch.full((1000,), scale, device=dev), torch.full((77,), -scale, device=dev)]
        before = [g.clone() for g in grads]
        want = _norm(before, 2.0)
        norm = clip.grad_norm(grads)
        if want < 3.4e38:
            assert abs(float(norm) - want) <= want * 2 * U + 2.0 ** -149
        else:
            assert math.isinf(float(norm))               # beyond f32; the factor is still right
        clip.clip_grads(grads, 1.0)
        for g, b in zip(grads, before):
            ref = b.cpu().double() * min(1.0, 1.0 / (want + 1e-6))
            assert bool(((g.cpu().double() - ref).abs() <= ref.abs() * 2.01 * U + 2.0 ** -149).all())


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_nan_and_inf_follow_the_formula(p):
    from ptamd import clip
    dev = _dev()
    for bad, where in ((math.nan, 0), (math.nan, 9999), (math.inf, 5000), (-math.inf, 123)):
        g = torch.ones(10000, device=dev)
        g[where] = bad
        h = torch.ones(3, device=dev, dtype=torch.bfloat16)
        norm = clip.clip_grads([g, h], 1.0, norm_type=p)
        if math.isnan(bad):
            assert math.isnan(float(norm)) and bool(torch.isnan(g).all()) and bool(torch.isnan(h).all())
        else:                                            # k = 0; 0 x inf is NaN
            assert float(norm) == math.inf and not h.any() and bool(torch.isnan(g[where]))
            assert int(torch.isnan(g).sum()) == 1 and int((g == 0).sum()) == 9999
    q = torch.nn.Parameter(torch.zeros(4, device=dev))
    q.grad = torch.tensor([1.0, math.inf, 2.0, 3.0], device=dev)
    kept = q.grad.clone()
    with pytest.raises(RuntimeError, match="norm is inf"):
        clip.clip_grad_norm_([q], 1.0, error_if_nonfinite=True)
    assert torch.equal(q.grad, kept)
    assert float(clip.clip_grads([torch.zeros(5, device=dev)], 0.0)) == 0.0     # 0 / (0 + 1e-6) = 0: no NaN


def test_orders_and_strides():
    from ptamd import clip
    dev = _dev()
    base = [torch.randn(6, 5, 4, 3, device=dev), torch.randn(40, 30, device=dev)]
    grads = [base[0].contiguous(memory_format=torch.channels_last), base[1].t(),
             torch.randn(20, 20, device=dev)[:, ::2], torch.randn(9, device=dev)]
    hole = grads[2]
    around = hole._base.clone()
    before = [g.clone() for g in grads]
    want = _norm(before, 2.0)
    out = [torch.empty_like(grads[0]), torch.empty(30, 40, device=dev), torch.empty(10, 20, device=dev).t(),
           torch.empty(18, device=dev)[::2]]
    norm = clip.clip_grads(grads, 0.5 * want, out=out)
    _check(out, before, norm, 0.5 * want, 2.0)
    norm = clip.clip_grads(grads, 0.5 * want)
    _check(grads, before, norm, 0.5 * want, 2.0)
    assert torch.equal(hole._base[:, 1::2], around[:, 1::2])
    with pytest.raises(clip.PtClipError, match="share memory"):
        clip.clip_grads([torch.ones(3, device=dev).expand(4, 3)], 1.0)
    with pytest.raises(clip.PtClipError, match="shares memory"):
        clip.clip_grads([grads[3], grads[3]], 1.0)
    with pytest.raises(clip.PtClipError, match="shares memory"):
        clip.clip_grads([base[0], base[0].view(-1)[:10]], 1.0)
    with pytest.raises(ValueError, match="shape"):
        clip.clip_grads([grads[3]], 1.0, out=[torch.empty(8, device=dev)])
    with pytest.raises(TypeError, match="output"):
        clip.clip_grads([grads[3]], 1.0, out=[torch.empty(9, device=dev, dtype=torch.bfloat16)])


def test_two_runs_agree_bit_for_bit_on_any_stream():
    from ptamd import clip
    grads = _tensors([100_003, 7, 5_000_000], "mixed", 8)
    out1, out2 = ([torch.empty(g.shape, device=g.device) for g in grads] for _ in range(2))
    n1 = clip.clip_grads(grads, 0.5, out=out1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n2 = clip.clip_grads(grads, 0.5, out=out2)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(n1, n2) and all(torch.equal(a, b) for a, b in zip(out1, out2))


def test_captured_clipping():
    """Replayed with other gradients in the same buffers, with eager work between."""
    from ptamd import clip
    grads = _tensors([30_000, 3, 100_000], "mixed", 12, scale=1.0)
    out = [torch.empty(g.shape, device=g.device) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip.clip_grads(grads, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip.clip_grads(grads, 1.0, out=out)
    for rep in range(3):
        for g in grads:
            g.mul_(0.25)
        graph.replay()
        got = [norm.clone()] + [o.clone() for o in out]
        want = [torch.empty_like(o) for o in out]
        n = clip.clip_grads(grads, 1.0, out=want)
        torch.cuda.synchronize()
        assert torch.equal(got[0], n) and all(torch.equal(a, b) for a, b in zip(got[1:], want)), rep


def test_parameters_of_a_model_as_the_reference_clips_them():
    """clip_grad_norm_ against the reference's formula (utils/misc_functions.py:48-69)."""
    from ptamd import clip
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Linear(65, 7), torch.nn.Linear(7, 1)).to(_dev())
    m(torch.randn(5, 33, device=_dev())).sum().backward()
    m[2].bias.grad = None
    params = [p for p in m.parameters()]
    before = [p.grad.clone() for p in params if p.grad is not None]
    want = _norm(before, 2.0)
    norm = clip.clip_grad_norm_(m.parameters(), 0.1)
    assert want > 0.1
    _check([p.grad for p in params if p.grad is not None], before, norm, 0.1, 2.0)
    assert m[2].bias.grad is None
    one = clip.clip_grad_norm_(params[0], 100.0)
    assert abs(float(one) - _norm([params[0].grad], 2.0)) <= float(one) * 2 * U


def test_clipping_tells_autograd_that_it_wrote():
    from ptamd import clip
    dev = _dev()
    w = torch.ones(8, device=dev, requires_grad=True)
    for grads, out in (([torch.ones(8, device=dev)], None), ([torch.ones(16, device=dev)[::2]], None),
                       ([torch.ones(8, device=dev)], [torch.ones(8, device=dev)])):
        loss = (w * (out or grads)[0]).sum()
        clip.grad_norm(grads)
        clip.clip_grads(grads, 0.5, out=out)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()


def test_a_parameter_listed_twice_is_refused():
    from ptamd import clip
    p = torch.nn.Parameter(torch.ones(8, device=_dev()))
    p.grad = torch.ones_like(p)
    with pytest.raises(clip.PtClipError, match="shares memory"):
        clip.clip_grad_norm_([p, p], 1.0)
    assert torch.equal(p.grad, torch.ones_like(p))
    assert abs(float(clip.clip_grad_norm_([p], 100.0, norm_type="inf")) - 1.0) <= U


def test_a_tensor_of_more_than_2_31_elements():
    """It takes several entries of the pointer table; values around their seams."""
    from ptamd import clip
    n = 2 ** 31 + 12_345
    g = torch.zeros(n, dtype=torch.bfloat16, device=_dev())
    at = [0, 2 ** 28 - 1, 2 ** 28, 2 ** 31 - 1, 2 ** 31, n - 1]
    for i in at:
        g[i] = 2.0
    norm = clip.clip_grads([g], 6.0 ** 0.5)
    assert abs(float(norm) - 24.0 ** 0.5) <= 24.0 ** 0.5 * U
    # k = sqrt(6) / (sqrt(24) + 1e-6): 2 k is below 1 by less than half a step of bf16
    assert [float(g[i]) for i in at] == [1.0] * len(at)
    g.abs_()
    assert float(g.max()) == 1.0 and int(torch.count_nonzero(g)) == len(at)


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_so_many_partial_sums_that_they_are_added_in_a_launch_of_their_own(p):
    from ptamd import clip
    flat = torch.randn(1300, 32_768, generator=torch.Generator(device=_dev()).manual_seed(3), device=_dev())
    before = flat.double()
    want = float(torch.linalg.vector_norm(before, p))
    norm = clip.clip_grads(list(flat), want / 8, norm_type=p)
    assert abs(float(norm) - want) <= want * (U + 2 ** -29)
    # k in 64 bits from a norm within 2^-29, the product rounded once
    k = (want / 8) / (want + 1e-6)
    assert bool(((flat.double() - before * k).abs() <= before.abs() * k * (U + 2 ** -28)).all())
