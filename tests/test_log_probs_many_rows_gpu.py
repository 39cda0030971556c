"""ops/log_probs.py: more rows than the grid has waves, so that every wave's list of candidates in LDS is written again for its next rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D,top", [(600_011, 300, 8), (530_007, 257, 40), (1_050_001, 40, 5)])
def test_alternatives_of_more_rows_than_waves(mmt_lib, rows, D, top, dtype):
    """Every row's alternatives against a stable sort; their log probabilities against 64 bits.  |logits| <= 16, so an exponent's argument is off by at most
    8 (32 + log 300) roundings of 2^-24 and the sum by D / 16 + 64."""
    from mm_training_amd.ops.log_probs import log_probs
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, D, device="cuda", generator=g) * 2).clamp(-16, 16).to(dtype)          # (bf16: ties in every row)
    r = log_probs(x, top=top)
    tol = 2.0 ** -24 * (8 * (32 + 6) + D / 16 + 64)
    for at in range(0, rows, 150_000):
        part = x[at:at + 150_000]
        order = torch.sort(part.float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids[at:at + 150_000], order)
        want = part.double().log_softmax(1).gather(1, order)
        assert float((r.top_log_prob[at:at + 150_000].double() - want).abs().max()) <= tol
