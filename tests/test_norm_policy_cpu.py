"""Which form of layer norm the executor picks where a weight is zero: backward from the output divides by it."""
import pytest
import torch

from tests.test_norm_dropout_cpu import Net


@pytest.mark.parametrize("policy", ["low_memory", "budget_10gb"])
@pytest.mark.parametrize("fuse", [False, True])
def test_a_zero_weight_keeps_the_input(policy, fuse):
    from monet_b200 import runner
    torch.manual_seed(0)
    model = Net()
    with torch.no_grad():
        model.blocks[0].norm.weight.zero_()
        model.blocks[1].norm.weight[5] = -0.0
    run = runner.Runner(model, getattr(runner, policy), fuse=fuse, counter_dropout=True)
    norms = {n.module: run.choices[n.id] for n in run.nodes if n.op in ("aten::layer_norm", "monet::dropout_add_layer_norm")}
    assert set(norms) == {"first", "blocks.0.norm", "blocks.1.norm", "blocks.2.norm"}
    for name in ("blocks.0.norm", "blocks.1.norm"):
        assert norms[name].impl == 0 and not norms[name].inplace
    for name in ("first", "blocks.2.norm"):      # no weight, and none that is zero
        assert norms[name].impl == 1


def test_other_policies_are_taken_as_they_are():
    from monet_b200 import runner
    model = Net()
    with torch.no_grad():
        model.blocks[0].norm.weight.zero_()
    run = runner.Runner(model, runner.store_all)
    assert all(run.choices[n.id] == runner.store_all(run.nodes, n) for n in run.nodes)
