"""dp/optim8.py: bf16 copies of parameters that change."""
import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def _channels_last(p):
    p.data = p.data.contiguous(memory_format=torch.channels_last)


def test_a_bf16_copy_that_no_longer_fits_is_refused(mmt_lib):
    """Copies are made in the parameter's memory order and type: one that changed before the first step would be written in another order, or not at all."""
    from mm_training_amd.dp.optim8 import ClipAdamW8

    def retype(p):
        p.data = p.data.bfloat16()

    for change in (_channels_last, retype):
        p = P(torch.randn(32, 16, 3, 3, generator=torch.Generator().manual_seed(1)).cuda())
        opt = ClipAdamW8([p])
        opt.make_bf16_shadows([p])
        change(p)
        p.grad = torch.ones_like(p)
        value, shadow = p.detach().clone(), opt.shadows[p].clone()
        with pytest.raises(RuntimeError, match="copy"):
            opt.step()
        assert torch.equal(p, value) and torch.equal(opt.shadows[p], shadow)
        opt.make_bf16_shadows([p]) if p.dtype == torch.float32 else opt.shadows.clear()
        opt.step()
        assert p.dtype != torch.float32 or torch.equal(opt.shadows[p], p.detach().bfloat16())
