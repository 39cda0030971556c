"""dp/optim8.py: state that a program clears, groups and states that it edits directly."""
import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter
SIZES = (5000, 300, 6000)


def _go(n_steps, cls_kw=None):
    from mm_training_amd.dp.optim8 import ClipAdamW8
    ps = [P(torch.linspace(-1, 1, n).cuda()) for n in SIZES]
    opt = ClipAdamW8(ps, lr=0.05, seed=4, **(cls_kw or {}))
    for i in range(n_steps):
        for p in ps:
            p.grad = torch.full_like(p, 1.0 + i)
        opt.step()
    return ps, opt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [None, 0, 1, 2])
def test_cleared_state_begins_anew(mmt_lib, which, dtype):
    """``state.clear()`` (or one parameter's entry taken out): the next step is a first step -- of zero moments and step count 1 -- for those
    parameters, and the next one for the rest; under rounding bits that have not been drawn yet."""
    from mm_training_amd import _lib
    from mm_training_amd.dp.optim8 import ClipAdamW8
    ps = [P(torch.linspace(-1, 1, n).to(dtype).cuda()) for n in SIZES]
    opt = ClipAdamW8(ps, lr=0.05, seed=4)
    keys, plain = [], _lib.timed_call
    _lib.timed_call = lambda kind, name, *a: (keys.append(a[6]), plain(kind, name, *a))[1]
    try:
        for i in range(3):
            for p in ps:
                p.grad = torch.full_like(p, 1.0 + i)
            opt.step()
        if which is None:
            opt.state.clear()
        else:
            del opt.state[ps[which]]
        before = [p.detach().clone() for p in ps]
        for p in ps:
            p.grad = torch.full_like(p, -2.0)
        opt.step()
    finally:
        _lib.timed_call = plain
    assert len(set(keys)) == 4
    for k, p in enumerate(ps):
        fresh = which is None or k == which
        assert int(opt.state[p]["step"]) == (1 if fresh else 4)
        if fresh:           # a first step moves against the gradient by lr (and decay): m / sqrt(v) = -1 to roundings, bf16 to a step of 2^-7
            want = before[k].double() * (1 - 0.05 * 1e-2) + 0.05
            assert float((p.detach().double() - want).abs().max()) <= (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -7)
        else:               # three steps the other way: the first moment is still above zero, the parameter goes down
            assert float((p.detach().double() - before[k].double()).max()) < 0.0


def test_groups_edited_directly_are_refused(mmt_lib):
    def pop(opt, ps):
        opt.param_groups[0]["params"].pop()

    def replace(opt, ps):
        opt.param_groups[0]["params"][0] = P(ps[0].detach().clone())

    def add(opt, ps):
        opt.param_groups[0]["params"].append(P(torch.ones(10, device="cuda")))

    def swap(opt, ps):
        q = opt.param_groups[0]["params"]
        q[0], q[1] = q[1], q[0]

    def pop_group(opt, ps):
        opt.param_groups.append(dict(opt.param_groups[0], params=[opt.param_groups[0]["params"].pop()]))

    for change in (pop, replace, add, swap, pop_group):
        ps, opt = _go(2)
        change(opt, ps)
        for g in opt.param_groups:
            for p in g["params"]:
                p.grad = torch.ones_like(p)
        values = [p.detach().clone() for p in ps]
        for _ in range(2):
            with pytest.raises(RuntimeError, match="ClipAdamW8"):
                opt.step()
        assert all(torch.equal(p, v) for p, v in zip(ps, values)), change.__name__


def test_states_replaced_directly_are_refused(mmt_lib):
    """A state of other tensors than the optimizer's own would never be read: load_state_dict is the way in."""
    ps, opt = _go(2)
    opt.state[ps[2]] = {k: v.clone() for k, v in opt.state[ps[2]].items()}
    values = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="ClipAdamW8"):
        opt.step()
    assert all(torch.equal(p, v) for p, v in zip(ps, values))


def test_a_sparse_gradient_is_refused(mmt_lib):
    ps, opt = _go(1)
    ps[1].grad = None
    ps[1].grad = torch.ones_like(ps[1]).to_sparse()
    values = [p.detach().clone() for p in ps]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="sparse"):
            opt.step()
    assert all(torch.equal(p, v) for p, v in zip(ps, values))
    ps[1].grad = None
    opt.step()
    assert [int(opt.state[p]["step"]) for p in ps] == [2, 1, 2]


def test_groups_edited_directly_then_laid_out_anew(mmt_lib):
    """After a parameter was taken out of its group (or given a state directly) a further group is refused and does not stay; a loaded state lays everything out for
    the parameters that are there."""
    ps, opt = _go(2)
    late = P(torch.ones(5000, device="cuda"))
    gone = opt.param_groups[0]["params"].pop()
    with pytest.raises(RuntimeError, match="ClipAdamW8"):
        opt.add_param_group(dict(params=[late]))
    assert len(opt.param_groups) == 1
    del opt.state[gone]
    given = {k: v.clone() for k, v in opt.state[ps[0]].items() if k != "draw"}
    opt.state[late] = given
    with pytest.raises(RuntimeError, match="ClipAdamW8"):
        opt.add_param_group(dict(params=[late]))
    assert len(opt.param_groups) == 1
    del opt.state[late]
    opt.load_state_dict(opt.state_dict())
    for p in ps:
        p.grad = torch.ones_like(p)
    before = gone.detach().clone()
    opt.step()
    assert torch.equal(gone, before) and [int(opt.state[p]["step"]) for p in ps[:2]] == [3, 3] and gone not in opt.state
    twin_ps, twin = _go(2)
    for p in twin_ps:
        p.grad = torch.ones_like(p)
    twin.step()
    assert all(torch.equal(a, b) for a, b in zip(ps[:2], twin_ps[:2]))
