"""dp/optim8.py: NaN of any payload, in gradients, moments and codes."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

P = torch.nn.Parameter


def _bits(values, dtype=torch.int32):
    """fp32 values of the given bit patterns"""
    return torch.tensor([v - (1 << 32) if v >= 1 << 31 else v for v in values], dtype=dtype).view(torch.float32)


@pytest.mark.parametrize("bits", [0x7FFFFFFF, 0xFFFFFFFF, 0x7FC0FFFF, 0x7F800001])
def test_a_nan_of_any_payload_stays_one_in_bf16(mmt_lib, bits):
    """16 random bits added to a NaN's lowest ones must not carry it past the largest pattern, into zero."""
    from mm_training_amd.dp.optim8 import ClipAdamW8
    nan = _bits([bits]).cuda()
    source = P(torch.ones(64, device="cuda"))
    packed, small = P(torch.ones(5003, device="cuda", dtype=torch.bfloat16)), P(torch.ones(99, device="cuda", dtype=torch.bfloat16))
    opt = ClipAdamW8([source, packed, small], max_norm=1.0, seed=2)
    for p in (source, packed, small):
        p.grad = torch.ones_like(p)
    source.grad[3:4] = nan                                    # through the norm
    opt.step()
    assert torch.isnan(opt.last_norm).all() and torch.isnan(packed).all() and torch.isnan(small).all()
    small = P(torch.ones(99, device="cuda", dtype=torch.bfloat16))
    opt = ClipAdamW8([small], seed=2)
    m = torch.zeros(99, device="cuda")                        # through a loaded fp32 moment
    m[5:6] = nan
    opt.load_state_dict({"state": {0: dict(step=1.0, exp_avg=m, exp_avg_sq=torch.ones(99, device="cuda"))}, "param_groups": opt.state_dict()["param_groups"]})
    small.grad = torch.ones_like(small)
    opt.step()
    assert torch.isnan(small).nonzero().flatten().tolist() == [5]


def test_codes_that_are_nan(mmt_lib):
    """NaN codes of a loaded state, of either format and sign, under fp32 and bf16 parameters."""
    from mm_training_amd.dp.optim8 import ClipAdamW8
    for dtype in (torch.float32, torch.bfloat16):
        for key, codes in (("exp_avg", (0x7F, 0xFF)), ("exp_avg_sq", (0x7D, 0x7E, 0x7F, 0xFF))):
            for code in codes:
                p = P(torch.ones(4096, device="cuda", dtype=dtype))
                p.grad = torch.ones_like(p)
                opt = ClipAdamW8([p], seed=4)
                opt.step()
                sd = copy.deepcopy(opt.state_dict())
                sd["state"][0][key].view(torch.uint8)[37] = code
                opt.load_state_dict(sd)
                opt.step()
                assert torch.isnan(p).nonzero().flatten().tolist() == [37], (dtype, key, code)
