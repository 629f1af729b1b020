"""A network one of whose layer norms has a weight of zero, through the policies that keep least."""
import pytest
import torch

from tests.test_norm_dropout_cpu import Net
from tests.test_norm_dropout_runner_gpu import reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("policy", ["low_memory", "budget_10gb"])
@pytest.mark.parametrize("fuse", [False, True])
def test_gradients_with_zero_weights(cuda, policy, fuse):
    from monet_b200 import runner
    torch.manual_seed(0)
    model = Net().to(cuda).train()
    with torch.no_grad():
        model.blocks[1].norm.weight[::3] = 0.0
        model.blocks[2].norm.weight[4] = 0.0
    x, gout = torch.randn(200, 24, device=cuda), torch.randn(200, 10, device=cuda)
    run = runner.Runner(model, getattr(runner, policy), fuse=fuse, counter_dropout=True)
    out = run.forward(x)
    ref, grads = reference(model, run, x, gout)
    run.backward(gout.clone())
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())     # noqa: E731
    # the bounds of the network without zeros: operands of eight linear layers truncated to 2^-10 each, and a
    # share of 4.7e-3 of the ReLU gates that may flip, each moving its element by its own size
    assert rel(out, ref) < 2e-2
    for k, p in model.named_parameters():
        assert bool(p.grad.isfinite().all()), k
        assert rel(p.grad, grads[k]) < 6.9e-2, (k, rel(p.grad, grads[k]))
