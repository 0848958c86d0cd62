"""When strided tensors share memory, against a walk over every element."""
import random

import pytest
import torch

from ptamd import clip, scan


def _places(t):
    at = torch.zeros((), dtype=torch.int64)
    for n, st in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * st
    return (at.reshape(-1) * t.element_size() + t.data_ptr()).tolist()


def _bytes(t):
    return [p + k for p in _places(t) for k in range(t.element_size())]


def _view(rng, base):
    flat = base.view(torch.float32) if rng.random() < 0.7 else base.view(torch.bfloat16)
    sizes = [rng.randint(1, 5) for _ in range(rng.randint(0, 4))]
    strides = [rng.choice([0, 1, 1, 2, 3, 5, 6, 10, 15, 30]) for _ in sizes]
    reach = sum((n - 1) * s for n, s in zip(sizes, strides))
    return flat.as_strided(sizes, strides, rng.randint(0, max(0, min(40, flat.numel() - reach - 1))))


@pytest.mark.parametrize("seed", range(4))
def test_intersections_are_exact(seed):
    rng, base = random.Random(seed), torch.zeros(4096, dtype=torch.uint8)
    apart = together = 0
    for _ in range(1500):
        a, b = _view(rng, base), _view(rng, base)
        want = bool(set(_bytes(a)) & set(_bytes(b)))
        assert scan.native().intersect(a, b) == scan.native().intersect(b, a) == want, (a.shape, a.stride(), b.shape,
                                                                                   b.stride())
        places = _places(a)
        assert scan.native().meets_itself(a) == (len(set(places)) < len(places)), (a.shape, a.stride())
        spans = min(_bytes(a)) <= max(_bytes(b)) and min(_bytes(b)) <= max(_bytes(a))
        apart, together = apart + (spans and not want), together + want
    assert apart > 50 and together > 50             # (interleaved ones are among them)


def test_large_views_are_told_apart_quickly():
    base = torch.empty(1, dtype=torch.float32).expand(1)
    wide = torch.empty(0).set_(base.untyped_storage(), 0, (0,))
    assert not scan.native().intersect(wide, base)
    flat = torch.empty(4_000_000)
    x = flat.view(1000, 4000)
    assert not scan.native().intersect(x[:, ::2], x[:, 1::2])
    assert scan.native().intersect(x[:, ::2], x[500:, 2:3])
    assert not scan.native().intersect(x[:, :2000].t(), x[:, 2000:])
    assert scan.native().intersect(x.t(), x[999:, 3999:])
    assert not scan.native().meets_itself(x[::3, ::7].t())
    assert clip.native() is scan.native()
