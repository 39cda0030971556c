"""dp/optim8.py: streams and lifetimes of the state."""
import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def _busy(n):
    x = torch.randn(4096, 4096, device="cuda")
    for _ in range(n):
        x = x @ x * 1e-4
    return x


def test_an_optimizer_made_behind_queued_work_and_dropped_before_its_step_has_run(mmt_lib):
    """Made on a busy stream, stepped on another that does not wait for it, dropped while that step is still queued, its memory asked for again at once."""
    from mm_training_amd.dp.optim8 import ClipAdamW8

    def go(hurried):
        ps = [P(torch.ones(n, device="cuda")) for n in (300000, 500)]
        for p in ps:
            p.grad = torch.full_like(p, 0.5)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        if hurried:
            _busy(30)
        opt = ClipAdamW8(ps, lr=0.1, seed=3)
        with torch.cuda.stream(side):
            if hurried:
                _busy(30)
            opt.step()
            opt.step()
        norm = opt.last_norm
        sizes = [v.view(torch.uint8).numel() for v in opt.state_buffers().values()]
        if hurried:
            del opt
            again = [torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") for n in sizes * 3]
            again += [torch.full((k,), 0x7F, dtype=torch.uint8, device="cuda") for k in (8, 512, 1024, 2048) for _ in range(20)]
        torch.cuda.synchronize()
        return [p.detach().clone() for p in ps], norm
    (a, _), (b, _) = go(False), go(True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
