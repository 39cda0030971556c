"""dp/optim8.py: the key of the rounding bits where parameters come and go."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def test_no_parameter_meets_the_same_rounding_bits_twice(mmt_lib, monkeypatch):
    """The key of every launch, by who takes part: parameters that join late, outlive the older ones, take turns, go through a checkpoint, are joined by a group."""
    from mm_training_amd import _lib
    from mm_training_amd.dp import optim8
    keys = []
    plain = _lib.timed_call
    monkeypatch.setattr(_lib, "timed_call", lambda kind, name, *a: (keys.append(a[6]), plain(kind, name, *a))[1])
    ps = [P(torch.ones(n, device="cuda")) for n in (5000, 6000, 100)]
    opt = optim8.ClipAdamW8(ps, seed=9)
    met = {k: [] for k in range(4)}

    def step(*who):
        for k, p in enumerate(ps):
            p.grad = torch.ones_like(p) if k in who else None
        opt.step()
        for k in who:
            assert keys[-1] not in met[k], (k, len(met[k]))
            met[k].append(keys[-1])

    for _ in range(6):
        step(0)
    for _ in range(3):
        step(0, 1)
    for _ in range(8):
        step(1)
    step(0, 1, 2)
    for _ in range(3):
        step(2)
        step(0)
    held = copy.deepcopy(opt.state_dict())
    opt = optim8.ClipAdamW8(ps, seed=9)
    opt.load_state_dict(held)
    for _ in range(12):
        step(1)
        step(2)
    ps.append(P(torch.ones(7000, device="cuda")))
    opt.add_param_group(dict(params=[ps[3]]))
    for _ in range(4):
        step(3)
        step(0, 3)
    step(0, 1, 2, 3)
    # a state that does not say which bits were drawn: none of the counts' can have been
    held = copy.deepcopy(opt.state_dict())
    for st in held["state"].values():
        for name in [n for n in st if n not in ("step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")]:
            del st[name]
    counts = {k: int(st["step"]) for k, st in held["state"].items()}
    older = optim8.ClipAdamW8(ps[:3], seed=9)
    older.add_param_group(dict(params=[ps[3]]))
    older.load_state_dict(held)
    opt, met = older, {k: [older._key(c) for c in range(1, max(counts.values()) + 1)] for k in range(4)}
    for k in range(4):
        for _ in range(max(counts.values())):
            step(k)


def test_the_state_for_adamw_names_nothing_else(mmt_lib):
    from mm_training_amd.dp.optim8 import ClipAdamW8
    p = P(torch.linspace(-1, 1, 5000).cuda())
    opt = ClipAdamW8([p])
    p.grad = torch.ones_like(p)
    opt.step()
    for st in opt.state_dict_32bit()["state"].values():
        assert sorted(st) == ["exp_avg", "exp_avg_sq", "step"]
