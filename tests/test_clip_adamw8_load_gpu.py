"""dp/optim8.py: checkpoints through hooks, and ones that fail."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def _bytes(opt):
    return {k: v.view(torch.uint8).clone() for k, v in opt.state_buffers().items()}


def _same(opt, held):
    now = _bytes(opt)
    return now.keys() == held.keys() and all(torch.equal(now[k], held[k]) for k in held)


def _stepped(n=5000, seed=1, steps=2):
    from mm_training_amd.dp.optim8 import ClipAdamW8
    ps = [P(torch.linspace(-1, 1, k).cuda()) for k in (n, 200)]
    opt = ClipAdamW8(ps, lr=0.25, seed=seed)
    for i in range(steps):
        for p in ps:
            p.grad = torch.full_like(p, 0.5 + i)
        opt.step()
    return ps, opt


def test_load_hooks(mmt_lib):
    """A pre-hook's result is what is loaded (state and groups), in the order the hooks were registered; post-hooks find the loaded moments, and what they put into the
    state stays."""
    from mm_training_amd.dp.optim8 import ClipAdamW8
    ps, opt = _stepped()
    saved = copy.deepcopy(opt.state_dict())
    renamed = {"state": {k: {("renamed_" + n): t for n, t in st.items()} for k, st in saved["state"].items()}, "param_groups": saved["param_groups"]}
    seen = []

    def rename(o, sd):
        seen.append(("pre", sorted(sd["state"][0])))
        return {"state": {k: {n.replace("renamed_", ""): t for n, t in st.items()} for k, st in sd["state"].items()}, "param_groups": sd["param_groups"]}

    def slower(o, sd):
        seen.append(("pre", sorted(sd["state"][0])))
        sd["param_groups"] = [dict(g, lr=0.125) for g in sd["param_groups"]]

    def after(o):
        p = o.param_groups[0]["params"][0]
        seen.append(("post", int(o.state[p]["step"]), bool(o.state[p]["exp_avg"].view(torch.uint8).any()), o.param_groups[0]["lr"]))
        o.state[p]["mine"] = 7

    fresh = [P(p.detach().clone()) for p in ps]
    other = ClipAdamW8(fresh, lr=1.0, seed=1)
    other.register_load_state_dict_pre_hook(rename)
    other.register_load_state_dict_pre_hook(slower)
    other.register_load_state_dict_post_hook(after)
    other.load_state_dict(renamed)
    assert [s[0] for s in seen] == ["pre", "pre", "post"]
    assert "renamed_exp_avg" in seen[0][1] and "exp_avg" in seen[1][1]
    assert seen[2][1:] == (2, True, 0.125) and other.state[fresh[0]]["mine"] == 7
    assert _same(other, _bytes(opt)) and sorted(renamed["state"][0])[0].startswith("renamed_")
    other.load_state_dict(renamed)                            # the hooks are as they were
    assert len(seen) == 6


@pytest.mark.parametrize("spoil", ["scale", "missing", "step", "shape", "group", "hyper", "split"])
def test_a_failing_load_leaves_everything(mmt_lib, spoil):
    ps, opt = _stepped()
    sd = copy.deepcopy(opt.state_dict())
    sd["param_groups"][0]["lr"] = 0.5
    st = sd["state"]
    if spoil == "scale":
        st[0]["exp_avg_sq_scale"] = st[0]["exp_avg_sq_scale"][:-1]
    elif spoil == "missing":
        del st[1]["exp_avg_sq"]
    elif spoil == "step":
        del st[1]["step"]
    elif spoil == "shape":
        st[1]["exp_avg"] = st[1]["exp_avg"][:-1]
    elif spoil == "group":
        sd["param_groups"][0]["params"] = [0]
    elif spoil == "hyper":
        sd["param_groups"][0]["betas"] = (0.9, 1.0)
    else:
        g = sd["param_groups"][0]
        sd["param_groups"] = [dict(g, params=[0]), dict(g, params=[1])]
    state = _bytes(opt)
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] == 0.25 and len(opt.param_groups) == 1 and _same(opt, state)
    assert all(int(opt.state[p]["step"]) == 2 for p in ps)
    twin_ps, twin = _stepped()
    for a, b in zip(ps, twin_ps):
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    twin.step()
    assert all(torch.equal(a, b) for a, b in zip(ps, twin_ps)) and _same(opt, _bytes(twin))
