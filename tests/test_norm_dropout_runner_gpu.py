"""Networks of linear layers, dropout and layer norm through the executor, against 64-bit autograd
with the masks that the operators drew."""
import copy

import pytest
import torch

from oracle import lm_ops_oracle as oracle
from tests.test_norm_dropout_cpu import Net

pytestmark = pytest.mark.gpu


def reference(model, run, x, gout, width=32):
    """(output, {name: gradient}) in 64 bits; each dropout takes the mask of the runner's operator."""
    m = copy.deepcopy(model).double().cpu()
    masks = {}
    drops = [n for n in run.nodes if n.op in ("monet::dropout", "monet::dropout_add_layer_norm")]
    for n in drops:
        params = run._ops[n.id].params
        p, seed = (params[0], params[1]) if n.op == "monet::dropout" else (params[1], params[2])
        if p:
            keep = oracle.dropout_keep(int(seed), 0, x.shape[0] * width, p).view(-1, width)
            masks.setdefault(p, keep.double() / (1 - p))

    class Given(torch.nn.Module):
        def __init__(self, mask):
            super().__init__()
            self.mask = mask

        def forward(self, v):
            return v * self.mask

    m.inner = Given(masks[0.25])
    for b in m.blocks:
        if b.has_drop:
            b.drop = Given(masks[b.drop.p])
    out = m(x.cpu().double())
    out.backward(gout.cpu().double())
    return out.detach(), {k: p.grad for k, p in m.named_parameters()}


@pytest.mark.parametrize("policy", ["store_all", "low_memory"])
@pytest.mark.parametrize("fuse", [False, True])
def test_network(cuda, policy, fuse):
    from monet_b200 import runner
    torch.manual_seed(0)
    model = Net().to(cuda).train()
    x, gout = torch.randn(200, 24, device=cuda), torch.randn(200, 10, device=cuda)
    run = runner.Runner(model, getattr(runner, policy), fuse=fuse, counter_dropout=True)
    out = run.forward(x)
    ref, grads = reference(model, run, x, gout)
    run.backward(gout.clone())
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())     # noqa: E731
    # TF32 truncates the operands of eight linear layers: 2^-10 each, the bound of the layer's own tests
    assert rel(out, ref) < 2e-2
    # A gradient also feels the ReLU gates.  Truncated operands move a pre-activation by up to 2^-10 of
    # its deviation per layer, d = 6 * 2^-10 behind the six layers before the last gate; the density of
    # a normal value at zero is 0.4 per deviation, so a share 2 * 0.4 * d = 4.7e-3 of the gates may
    # flip, each moving its element by its own size: sqrt(4.7e-3) = 6.9e-2 in the norm.
    for k, p in model.named_parameters():
        assert rel(p.grad, grads[k]) < 6.9e-2, (k, rel(p.grad, grads[k]))


def test_low_memory_keeps_less(cuda):
    """From the output and with regenerated masks, the post-norm blocks keep one tensor less each."""
    from monet_b200 import runner
    model = Net(width=1024).to(cuda).train()
    x = torch.randn(4096, 24, device=cuda)
    peak = {}
    for name, policy, fuse, counter in (("all", runner.store_all, False, False), ("low", runner.low_memory, True, True)):
        run = runner.Runner(model, policy, fuse=fuse, counter_dropout=counter)
        run.forward(x)
        del run
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        run = runner.Runner(model, policy, fuse=fuse, counter_dropout=counter)
        base = torch.cuda.memory_allocated()
        run.forward(x)
        peak[name] = torch.cuda.memory_allocated() - base
        del run
    act = 4096 * 1024 * 4
    # kept by `all`: beyond `low`, at least the input of each of the three block norms
    assert peak["low"] <= peak["all"] - 3 * act, peak


def test_captured_step(cuda):
    """A whole training step as one CUDA graph: the loss of each replay is that of the eager step where
    nothing is dropped, and with dropout each replay has masks of its own."""
    from monet_b200 import runner
    from monet_b200.lm_ops.softmax import SoftmaxCrossEntropy
    torch.manual_seed(1)
    for p in (0.0, 0.4):
        model = Net().to(cuda).train()
        for m in model.modules():
            if isinstance(m, torch.nn.Dropout):
                m.p = p
        x, y = torch.randn(64, 24, device=cuda), torch.randint(0, 10, (64,), device=cuda)
        run = runner.Runner(model, runner.low_memory, fuse=True, counter_dropout=True)
        step = runner.GraphedStep(run, SoftmaxCrossEntropy(), torch.optim.SGD(model.parameters(), lr=0.0), x, y)
        losses = [float(step(x, y)) for _ in range(4)]
        assert all(v == v and v < 100 for v in losses)
        if p:
            assert len(set(losses)) > 1
        else:
            loss = torch.nn.functional.cross_entropy(copy.deepcopy(model).double()(x.double()), y)
            assert len(set(losses)) == 1 and abs(losses[0] - float(loss.detach())) < 2e-2


def test_three_dimensional_operators(cuda):
    """The operator classes on [batch, tokens, width] activations, both storage forms, by protocol."""
    import monet_b200.lm_ops as L
    from monet_b200.lm_ops import fused  # noqa: F401
    m = "multiway_newnode"
    x, r, dy = (torch.randn(3, 17, 48, device=cuda) for _ in range(3))
    w, b = torch.rand(48, device=cuda) + 0.5, torch.randn(48, device=cuda)
    grads = []
    for cls in L.list_ops(m, "aten::layer_norm"):
        op = cls()
        y = op.forward(x, [48], w, b, 1e-5, True)
        stored = [x, w, b] if cls.__name__.startswith("Input") else [w, b, y]
        grads.append(op.backward(dy, stored))
        assert stored == [] and len(grads[-1]) == 3
    for cls in L.list_ops(m, "monet::dropout_add_layer_norm"):
        torch.manual_seed(3)
        op = cls()
        out = op.forward(x, r, [48], w, b, 1e-5, 0.25, True)
        stored = [w, b, out[1]] if isinstance(out, tuple) else [w, b, out]
        grads.append(op.backward(dy, stored, nodel=True))
        assert len(stored) == 3 and len(grads[-1]) == 4
        again = cls()
        again.params = op.params
        second = again.forward(x, r, [48], w, b, 1e-5, 0.25, True)
        assert torch.equal(second[0], out[0]) if isinstance(out, tuple) else torch.equal(second, out)
    for a, c in ((0, 1), (2, 3)):
        for p, q in zip(grads[a], grads[c]):
            assert p.shape == q.shape and torch.allclose(p, q, rtol=1e-4, atol=1e-4)
    plain = L.list_ops(m, "aten::layer_norm")[0]()
    plain.forward(x, [48], None, None, 1e-5, True)
    assert len(plain.backward(dy, [x, None, None])) == 1
