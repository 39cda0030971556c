"""dp/optim8.py: a parameter whose memory order changes in place, gradients of other strides."""
import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def _bytes(opt):
    return {k: v.view(torch.uint8).clone() for k, v in opt.state_buffers().items()}


def _same(opt, held):
    now = _bytes(opt)
    return now.keys() == held.keys() and all(torch.equal(now[k], held[k]) for k in held)


def _transpose(p):
    p.data = p.data.t()                                       # the same address and size


def _other_strides(p):
    n, c, h, w = p.shape
    p.data = p.data.as_strided((n, c, h, w), (c * h * w, 1, w * c, c))


def _cut_rows(p):
    p.data = p.data[:p.shape[0] // 2]


@pytest.mark.parametrize("shape,change", [((64, 80), _transpose), ((72, 72), _transpose), ((16, 32, 3, 3), _other_strides), ((40, 30), _transpose), ((64, 80), _cut_rows)])
@pytest.mark.parametrize("stale", [False, True])
def test_a_parameter_permuted_in_place_is_refused(mmt_lib, shape, change, stale):
    """Same address, same number of elements, another memory order (or fewer rows), under a contiguous gradient of the new shape or the gradient
    that was there: elements would be paired in the wrong order.  Nothing is touched, and the old layout goes on."""
    from mm_training_amd.dp.optim8 import ClipAdamW8
    g = torch.Generator().manual_seed(1)
    p = P(torch.randn(shape, generator=g).cuda())
    other = P(torch.randn(300, generator=g).cuda())
    opt = ClipAdamW8([other, p], max_norm=1.0)
    grad = torch.randn(shape, generator=g).cuda()
    p.grad, other.grad = grad, torch.ones_like(other)
    opt.step()
    before = p.data
    change(p)
    if not stale:
        p.grad = None
        p.grad = torch.randn(p.shape, generator=g).cuda()
    values, state = [q.detach().clone() for q in (p, other)], _bytes(opt)
    for _ in range(2):
        with pytest.raises((RuntimeError, TypeError), match="ClipAdamW8"):
            opt.step()
    assert torch.equal(p, values[0]) and torch.equal(other, values[1]) and _same(opt, state)
    p.data = before
    p.grad = None
    p.grad = grad
    opt.step()
    assert not torch.equal(other, values[1])


def test_gradients_whose_strides_alternate(mmt_lib):
    """Contiguous and channels_last gradients of one channels_last weight in turn, 1 x 1 weights whose strides say nothing, a reshaped vector: each step as if
    its gradient came in the parameter's own layout."""
    from mm_training_amd.dp.optim8 import ClipAdamW8
    g = torch.Generator().manual_seed(2)
    make = lambda: [P(torch.randn(s, generator=torch.Generator().manual_seed(7)).cuda().contiguous(memory_format=torch.channels_last))  # noqa: E731
                    for s in ((32, 16, 3, 3), (128, 64, 1, 1))]
    a, b = make(), make()
    one, two = ClipAdamW8(a, seed=1), ClipAdamW8(b, seed=1)
    for step in range(6):
        for p, q in zip(a, b):
            d = torch.randn(p.shape, generator=g).cuda()
            p.grad = d.contiguous(memory_format=torch.channels_last)
            q.grad = d.clone() if step % 3 else d.contiguous(memory_format=torch.channels_last)
        one.step()
        two.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), step
