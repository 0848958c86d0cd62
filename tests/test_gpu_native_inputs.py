"""ptamd.scan and ptamd.clip on tensors whose memory does not hold their values as
they are: views with the negative bit (x.conj().imag)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def _negated(v):
    """The values of ``v`` in a view that holds their negatives."""
    out = torch.complex(torch.zeros_like(v), -v).conj().imag
    assert out.is_neg() and torch.equal(out, v)
    return out


@pytest.mark.parametrize("form,count", [("leaky", 2), ("lstm", 4)])
def test_scan_of_negated_views(form, count):
    from ptamd import scan
    dev = _dev()
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 40, count * 24, generator=g).to(dev)
    h0 = torch.randn(3, 24, generator=g).to(dev)
    dy, dh = torch.randn(3, 40, 24, generator=g).to(dev), torch.randn(3, 24, generator=g).to(dev)
    ends = torch.tensor([40, 0, 17], device=dev)
    outs = []
    for neg in (lambda v: v, _negated):
        for stacked in (True, False):
            leaves = [v.clone().requires_grad_() for v in ([x] if stacked else x.chunk(count, 2))] + \
                [h0.clone().requires_grad_()]
            xs = [neg(v) for v in leaves[:-1]]
            lengths = ends if neg is not _negated else torch._neg_view(-ends)
            res = scan.gated_scan(xs[0] if stacked else xs, neg(leaves[-1]), form=form, lengths=lengths)
            grads = torch.autograd.grad(res[:2], leaves, [neg(dy), neg(dh)])
            with torch.no_grad():
                again = scan.gated_scan(xs[0] if stacked else xs, neg(leaves[-1]), form=form, lengths=lengths)
            outs.append([*(r.detach() for r in res), torch.cat(grads[:-1], 2), grads[-1], *again])
            state = h0.clone()
            one = [v[:, 3].detach() for v in xs]
            outs[-1] += [scan.gated_scan_step(one[0] if stacked else one, state, form=form), state]
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_clipping_of_negated_views():
    from ptamd import clip
    dev = _dev()
    v = torch.randn(500, generator=torch.Generator().manual_seed(3)).to(dev)
    for g in (_negated(v), _negated(torch.stack([v, v], 1))[:, 0]):
        want = [torch.empty_like(v)]
        norm = clip.clip_grads([v], 0.5, out=want)
        got = [torch.empty_like(v)]
        assert torch.equal(clip.clip_grads([g], 0.5, out=got), norm) and torch.equal(got[0], want[0])
        assert torch.equal(clip.grad_norm([g]), norm)
        assert torch.equal(clip.clip_grads([g], 0.5), norm) and torch.equal(g, want[0])     # in place
    base = torch.complex(torch.zeros_like(v), -v)                     # its own memory as the output
    g, o = base.conj().imag, base.imag
    clip.clip_grads([g], 0.5, out=[o])
    assert torch.equal(o, want[0])


def test_strided_tensors_that_share_memory_are_refused():
    from ptamd import clip
    dev = _dev()
    base = torch.randn(40, 60, generator=torch.Generator().manual_seed(4)).to(dev)
    kept = base.clone()
    p = torch.nn.Parameter(torch.zeros(40, 30, device=dev))
    p.grad = base[:, ::2]
    free = torch.ones(40, 30, device=dev)
    wide = torch.zeros(80, 60, device=dev)

    def refused(*args, **kw):
        with pytest.raises(clip.PtClipError, match="share"):
            clip.clip_grads(*args, 1.0, **kw)
        assert torch.equal(base, kept) and not wide.any()

    with pytest.raises(clip.PtClipError, match="shares memory"):
        clip.clip_grad_norm_([p, p], 1.0)
    refused([base[:, ::2], base[:, ::2]])                                   # the same twice
    refused([base[:, ::2], base[:, 2:4]])                                   # a column in both
    refused([base[:, ::2], base.view(-1)[:70]])                             # a dense one over it
    strided = [base[:, ::2], free]
    refused(strided, out=[wide[::2, ::2], base[:, 2:32]])                   # an output on another gradient
    refused(strided, out=[wide[::2, ::2], base.view(-1)[:1200].view(40, 30)])
    refused(strided, out=[wide[::2, ::2], wide[::2, ::2]])                  # on another output
    refused(strided, out=[wide[::2, ::2], wide[::2, :30]])
    refused([free, kept[:, ::2]], out=[wide[::2, ::2], wide.view(-1)[:1200].view(40, 30)])
    refused([base.as_strided((30, 4), (2, 1))])                             # elements of one gradient
    # what interleaves, or is only read twice, goes on
    norm = clip.clip_grads([base[:, ::2], base[:, 1::2]], 1.0)
    want = kept.double().norm()
    assert abs(float(norm) - float(want)) <= float(want) * 2.0 ** -23
    torch.testing.assert_close(base, (kept.double() / (want + 1e-6)).float(), rtol=2.0 ** -22, atol=0)
    out = [wide[::2, ::2], wide[1::2, 1::2]]
    clip.clip_grads([kept[:, ::2], kept[:, ::2]], 1e9, out=out)
    assert torch.equal(out[0], kept[:, ::2]) and torch.equal(out[1], kept[:, ::2])


def test_one_overlap_among_many_strided_gradients():
    """Wherever it stands in the list and in memory."""
    from ptamd import clip
    dev = _dev()
    flat = torch.ones(300, 40, 10, device=dev)
    grads = [flat[k, :, ::2] for k in range(300)]
    assert abs(float(clip.clip_grads(grads, 1e9)) - 60_000 ** 0.5) < 1e-4
    for k in (0, 123, 299):
        other = flat[k, 5:9, 4:7]
        for at in (0, 77, 300):
            with pytest.raises(clip.PtClipError, match="share"):
                clip.clip_grads(grads[:at] + [other] + grads[at:], 1.0)
    wide = flat[:, 0].t()                                    # over all of them
    with pytest.raises(clip.PtClipError, match="share"):
        clip.clip_grads(grads[7:9] + [wide], 1.0)
    assert bool((flat == 1).all())


def test_an_output_on_a_negated_gradient_is_refused():
    from ptamd import clip
    v, w = torch.ones(60, device=_dev()), torch.ones(60, device=_dev())
    with pytest.raises(clip.PtClipError, match="share"):
        clip.clip_grads([torch._neg_view(v), w], 1.0, out=[torch.empty_like(v), v])
    assert bool((v == 1).all())


class _Wrapped(torch.Tensor):
    """A tensor that holds another and has no memory of its own."""

    @staticmethod
    def __new__(cls, inner):
        out = torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(), dtype=inner.dtype,
                                                  device=inner.device)
        out.inner = inner
        return out

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        def plain(v):
            return v.inner if isinstance(v, cls) else v
        return func(*torch.utils._pytree.tree_map(plain, args), **torch.utils._pytree.tree_map(plain, kwargs or {}))


def test_gradients_that_are_no_plain_tensors_are_refused():
    from ptamd import scan
    import torch.autograd.forward_ad as fwAD
    dev = _dev()
    x = torch.randn(2, 30, 16, device=dev, requires_grad=True)
    d = torch.randn(2, 30, 8, device=dev)
    y, h = scan.gated_scan(x)
    with pytest.raises(RuntimeError, match="plain tensors"):
        torch.autograd.grad(y, x, _Wrapped(d), retain_graph=True)
    with pytest.raises(RuntimeError, match="plain tensors"):
        torch.autograd.grad([y, h], x, [d, _Wrapped(d[:, 0].contiguous())], retain_graph=True)
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(y, x, fwAD.make_dual(d, torch.ones_like(d)), retain_graph=True)
    with pytest.raises(scan.PtScanError, match="plain tensors"):
        scan.gated_scan(_Wrapped(x.detach()))
    want, = torch.autograd.grad(y, x, d, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, x, d)[0], want) and bool(want.any())
