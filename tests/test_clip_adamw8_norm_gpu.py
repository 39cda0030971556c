"""dp/optim8.py: norms that a caller keeps."""
import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def test_norms_that_are_kept(mmt_lib):
    from mm_training_amd.dp.optim8 import ClipAdamW8
    p = P(torch.zeros(4096, device="cuda"))
    opt = ClipAdamW8([p], max_norm=1.0)
    kept = []
    for i in range(10):
        p.grad = torch.full_like(p, float(i + 1))
        opt.step()
        kept.append(opt.last_norm)
    for i, norm in enumerate(kept):                           # (whole numbers: exact)
        assert float(norm[0]) == 64.0 * (i + 1), i
        assert abs(float(norm[1]) - 1 / (64.0 * (i + 1) + 1e-6)) <= 2.0 ** -22
