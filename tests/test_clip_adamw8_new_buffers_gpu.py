"""dp/optim8.py: the moments laid out anew (an added group, a loaded state) after a parameter changed."""
import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def _bytes(opt):
    return {k: v.view(torch.uint8).clone() for k, v in opt.state_buffers().items()}


def _same(opt, held):
    now = _bytes(opt)
    return now.keys() == held.keys() and all(torch.equal(now[k], held[k]) for k in held)


def _channels_last(p):
    p.data = p.data.contiguous(memory_format=torch.channels_last)


def _turn(p):
    p.data = p.data.transpose(0, 1).contiguous()


def _halve(p):
    p.data = p.data[:p.shape[0] // 2].clone()


def _shrink(p):
    p.data = p.data[:2].clone()                               # below min_8bit_size: another form of state


@pytest.mark.parametrize("change", [_channels_last, _turn, _halve, _shrink])
def test_a_group_added_after_a_parameter_changed(mmt_lib, change):
    """add_param_group lays the moments out anew: a parameter that no longer fits its moments is refused, groups and moments stay; with the
    parameter put back, the group joins and steps go on as if nothing had happened."""
    from mm_training_amd.dp.optim8 import ClipAdamW8
    g = torch.Generator().manual_seed(3)
    start, grads = torch.randn(32, 16, 3, 3, generator=g).cuda(), [torch.randn(32, 16, 3, 3, generator=g).cuda() for _ in range(3)]
    runs = []
    for disturbed in (False, True):
        p, late = P(start.clone()), P(torch.ones(5000, device="cuda"))
        opt = ClipAdamW8([p], seed=5)
        p.grad = grads[0].clone()
        opt.step()
        if disturbed:
            held, state = p.data, _bytes(opt)
            change(p)
            with pytest.raises(RuntimeError, match="ClipAdamW8"):
                opt.add_param_group(dict(params=[late]))
            assert len(opt.param_groups) == 1 and _same(opt, state)
            p.data = held
        opt.add_param_group(dict(params=[late]))
        for d in grads[1:]:
            p.grad = None
            p.grad, late.grad = d.clone(), torch.ones_like(late)
            opt.step()
        runs.append((p.detach().clone(), late.detach().clone(), _bytes(opt)))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert all(torch.equal(runs[0][2][k], runs[1][2][k]) for k in runs[0][2])


def test_a_state_loaded_after_the_form_changed(mmt_lib):
    """A parameter that grew over (or fell under) min_8bit_size before its state is loaded: the loaded moments take the form of its present size."""
    from mm_training_amd.dp.optim8 import ClipAdamW8, pack_moment
    for sizes in ((1000, 9000), (9000, 1000)):
        p = P(torch.ones(sizes[0], device="cuda"))
        opt = ClipAdamW8([p])
        p.data = torch.ones(sizes[1], device="cuda")
        m, v = torch.randn(sizes[1], device="cuda"), torch.rand(sizes[1], device="cuda")
        opt.load_state_dict({"state": {0: dict(step=torch.tensor(3.0), exp_avg=m, exp_avg_sq=v)}, "param_groups": opt.state_dict()["param_groups"]})
        for key, x in (("exp_avg", m), ("exp_avg_sq", v)):
            if sizes[1] >= 4096:
                codes, scales = pack_moment(x, key == "exp_avg_sq")
                assert torch.equal(opt.state[p][key].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(opt.state[p][key + "_scale"], scales)
            else:
                assert torch.equal(opt.state[p][key], x)
        p.grad = torch.ones_like(p)
        opt.step()
        assert int(opt.state[p]["step"]) == 4
