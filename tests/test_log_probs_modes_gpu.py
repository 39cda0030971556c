"""ops/log_probs.py under forward-mode differentiation: refused like the framework's other operators, never a tangent dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,dim", [((4, 10), -1), ((2, 112, 3, 5), 1), ((3, 5000), 1)])
def test_dual_tensors_are_refused(mmt_lib, shape, dim):
    from mm_training_amd.ops.log_probs import log_probs
    g = torch.Generator().manual_seed(0)
    x, way = (torch.randn(shape, generator=g).cuda() for _ in range(2))
    want = log_probs(x, dim=dim)
    with fwd.dual_level():
        for leaf in (x, x.clone().requires_grad_(True)):
            dual = fwd.make_dual(leaf, way)
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                    log_probs(dual, dim=dim)
        plain = log_probs(x, dim=dim)                          # no tangent: as ever
    assert torch.equal(plain.lse, want.lse) and torch.equal(plain.entropy, want.entropy)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda q: log_probs(q, dim=dim).lse, (x,), (way,))
