"""Layer norm and dropout without a GPU: the generator's published vectors, the definitions against
autograd, registry slots, graph extraction and fusion, and refusals that precede any launch."""
import ctypes as C

import pytest
import torch
import torch.nn as nn

from oracle import lm_ops_oracle as oracle


def test_generator_against_published_vectors():
    """Known answers of Philox-4x32-10 (Salmon et al., SC 2011)."""
    assert [hex(v) for v in oracle.philox_words([0] * 4, 0)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    assert [hex(v) for v in oracle.philox_words([0xFFFFFFFF] * 4, (1 << 64) - 1)[0]] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


def test_kept_share_is_one_minus_p():
    n = 1 << 18
    for p in (0.1, 0.5, 0.9):
        share = float(oracle.dropout_keep(12345, 6, n, p).double().mean())
        assert abs(share - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5


def test_definitions_against_autograd():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 12, generator=g, dtype=torch.float64, requires_grad=True)
    w = (torch.rand(12, generator=g, dtype=torch.float64) + 0.5).requires_grad_(True)
    b = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(5, 12, generator=g, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(x, (12,), w, b, 1e-5)
    y.backward(dy)
    oy, mean, rstd = oracle.layer_norm_forward(x.detach(), w.detach(), b.detach(), 1e-5)
    assert torch.allclose(oy, y.detach(), atol=1e-12)
    dx, dw, db = oracle.layer_norm_backward(dy, (oy - b.detach()) / w.detach(), w.detach(), rstd)
    assert torch.allclose(dx, x.grad, atol=1e-12) and torch.allclose(dw, w.grad, atol=1e-12) and torch.allclose(db, b.grad, atol=1e-12)


def test_registry():
    import monet_b200.lm_ops as L
    from monet_b200.lm_ops import fused  # noqa: F401
    names = lambda mode, op: [c.__name__ for c in L.list_ops(mode, op)]   # noqa: E731
    m = "conv_multiway_newnode"
    assert names(m, "aten::layer_norm") == ["InputActLayerNorm", "OutputActLayerNorm"]
    assert names("normal", "aten::layer_norm") == ["InputActLayerNorm"]
    assert names(m, "monet::dropout_add_layer_norm") == ["SumActDropoutAddLayerNorm", "OutputActDropoutAddLayerNorm"]
    assert names(m, "monet::dropout") == ["CounterDropout"] and names(m, "aten::dropout") == ["Dropout"]
    size = L.list_ops(m, "monet::dropout_add_layer_norm")[0].backward_storage[1].size
    assert size((7, 33)) == 7 * 33 * 4


class Block(nn.Module):
    """A post-norm block: layer_norm(x + dropout(f(x))), and a plain x + f(x) norm when p is None."""

    def __init__(self, width, p, swap=False):
        super().__init__()
        self.up, self.act, self.down = nn.Linear(width, 2 * width), nn.ReLU(), nn.Linear(2 * width, width)
        self.drop = nn.Dropout(p) if p is not None else nn.Identity()
        self.has_drop, self.swap = p is not None, swap
        self.norm = nn.LayerNorm(width)

    def forward(self, x):
        h = self.down(self.act(self.up(x)))
        if self.has_drop:
            h = self.drop(h)
        return self.norm(h + x if self.swap else x + h)


class Net(nn.Module):
    def __init__(self, width=32, classes=10):
        super().__init__()
        self.stem, self.first = nn.Linear(24, width), nn.LayerNorm(width, elementwise_affine=False)
        self.inner = nn.Dropout(0.25)
        self.blocks = nn.Sequential(Block(width, 0.1), Block(width, None), Block(width, 0.5, swap=True))
        self.head = nn.Linear(width, classes)

    def forward(self, x):
        return self.head(self.blocks(self.inner(self.first(self.stem(x)))))


def test_extraction_and_fusion():
    from monet_b200 import runner
    nodes, out = runner.extract_graph(Net())
    ops = [n.op for n in nodes]
    assert ops.count("aten::layer_norm") == 4 and ops.count("aten::dropout") == 3
    first = next(n for n in nodes if n.op == "aten::layer_norm")
    assert [a.value for a in first.args[1:5]] == [[32], None, None, 1e-5]
    fused, fout = runner.fuse_graph(nodes, out)
    ops = [n.op for n in fused]
    assert ops.count("monet::dropout_add_layer_norm") == 3 and ops.count("aten::layer_norm") == 1
    assert ops.count("aten::dropout") == 1 and "aten::add" not in ops and fused[fout].op == "aten::addmm"
    ends = [n for n in fused if n.op == "monet::dropout_add_layer_norm"]
    assert [n.args[6].value for n in ends] == [0.1, 0.0, 0.5]
    for n in ends:                                  # x comes from the block's last linear layer when it is dropped
        if n.args[6].value:
            assert fused[n.args[0].value].op == "aten::addmm"
    for n in fused:
        for a in n.args:
            if a.kind == "node":
                assert a.value < n.id and n.id in fused[a.value].users


def test_sums_with_another_reader_stay_separate():
    """Pre-norm: the sum goes on beside the norm, so no single-output node can replace the pair; a dropout
    with a second reader stays a node of its own."""
    from monet_b200 import runner

    class PreNorm(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b, self.d, self.n = nn.Linear(8, 8), nn.Linear(8, 8), nn.Dropout(0.2), nn.LayerNorm(8)

        def forward(self, x):
            x = self.a(x)
            z = x + self.d(self.b(x))
            return self.n(z) + z

    class SharedDropout(PreNorm):
        def forward(self, x):
            x = self.a(x)
            h = self.d(self.b(x))
            return self.n(x + h) + h

    nodes, out = runner.fuse_graph(*runner.extract_graph(PreNorm()))
    assert "monet::dropout_add_layer_norm" not in [n.op for n in nodes]
    nodes, out = runner.fuse_graph(*runner.extract_graph(SharedDropout()))
    n = next(n for n in nodes if n.op == "monet::dropout_add_layer_norm")
    assert n.args[6].value == 0.0 and "aten::dropout" in [n.op for n in nodes]


def test_policies():
    from monet_b200 import runner
    r = runner.Runner(Net(), runner.low_memory, fuse=True, counter_dropout=True)
    pick = {n.op: r.choices[n.id] for n in r.nodes}
    assert pick["monet::dropout"].recompute and pick["monet::dropout_add_layer_norm"].impl == 1
    assert pick["aten::layer_norm"].impl == 1 and pick["aten::layer_norm"].inplace
    r = runner.Runner(Net(), runner.store_all)
    assert all(r.choices[n.id].impl == 0 and not r.choices[n.id].inplace for n in r.nodes if n.op == "aten::layer_norm")
    assert "aten::dropout" in [n.op for n in r.nodes]


def test_refused_before_any_launch(built_lib):
    """Descriptors are checked first: no device is touched."""
    from monet_b200 import _lib
    api = _lib.lib()
    one = C.c_void_p(64)          # non-null and aligned: never dereferenced

    def fwd(d, drop=None, x=one, residual=None, y=one, ws=None, nbytes=0):
        return api.mb_layer_norm_fwd(x, residual, None, None, y, None, one, one, C.byref(d) if d else None,
                                     C.byref(drop) if drop else None, ws, nbytes, None)

    def bwd(d, drop=None, ws=one, nbytes=0, dx=None, mean=one, out=0):
        return api.mb_layer_norm_bwd(one, one, out, None, None, None, mean, one, one, dx, one, one, C.byref(d),
                                     C.byref(drop) if drop else None, ws, nbytes, None)

    ok = lambda **k: _lib.LnDesc(*[{**dict(rows=4, cols=16, a=16, b=16, c=16, dtype=0, pdtype=0, eps=1e-5), **k}[n]   # noqa: E731
                                   for n in ("rows", "cols", "a", "b", "c", "dtype", "pdtype", "eps")])
    cases = [(fwd(None), 1, "descriptor"), (fwd(ok(dtype=9)), 1, "dtype"), (fwd(ok(cols=0)), 2, "cols"), (fwd(ok(cols=1 << 31)), 2, "cols"),
             (fwd(ok(pdtype=1)), 1, "parameters"), (fwd(ok(eps=-1.0)), 1, "eps")]
    for rc, code, _ in cases:
        assert rc == code
    for call, code, word in [
            (lambda: fwd(ok(), x=None), 1, "null"), (lambda: fwd(ok(), y=C.c_void_p(66)), 1, "misaligned"),
            (lambda: fwd(ok(), _lib.DropoutDesc(0.5, 64, 0)), 1, "residual"),
            (lambda: fwd(ok(), _lib.DropoutDesc(1.5, 64, 0), residual=one), 1, "probability"),
            (lambda: fwd(ok(), _lib.DropoutDesc(0.5, None, 0), residual=one), 1, "seed"),
            (lambda: fwd(ok(), _lib.DropoutDesc(0.5, 68, 0), residual=one), 1, "seed"),
            (lambda: fwd(ok(a=32), y=one, x=one), 1, "dense"), (lambda: fwd(ok(b=0), x=C.c_void_p(128), residual=one), 1, "dense"),
            (lambda: bwd(ok(), dx=one, nbytes=1 << 20), 1, "same buffer"), (lambda: bwd(ok(a=32), nbytes=1 << 20), 1, "dense"),
            (lambda: bwd(ok()), 3, "workspace"), (lambda: bwd(ok(), ws=None, nbytes=1 << 20), 3, "workspace"),
            (lambda: bwd(ok(), mean=None, nbytes=1 << 20), 1, "null"),
            (lambda: bwd(ok(), _lib.DropoutDesc(0.5, 64, 0), nbytes=1 << 20), 1, "dx"),
            (lambda: api.mb_dropout(one, one, 8, 7, C.byref(_lib.DropoutDesc(0.5, 64, 0)), None), 1, "dtype"),
            (lambda: api.mb_dropout(None, one, 8, 0, C.byref(_lib.DropoutDesc(0.5, 64, 0)), None), 1, "null"),
            (lambda: api.mb_dropout(one, one, 8, 0, None, None), 1, "descriptor"),
            (lambda: api.mb_dropout(one, one, 8, 0, C.byref(_lib.DropoutDesc(float("nan"), 64, 0)), None), 1, "probability")]:
        rc = call()
        assert rc == code and word in _lib.last_error(), (rc, code, word, _lib.last_error())
    assert api.mb_layer_norm_bwd_workspace_bytes(C.byref(ok())) >= 2 * 16 * 4
    assert api.mb_layer_norm_bwd_workspace_bytes(C.byref(ok(rows=0))) == 0 and api.mb_layer_norm_bwd_workspace_bytes(None) == 0
    assert api.mb_layer_norm_fwd_workspace_bytes(C.byref(ok())) == 0
    long = ok(cols=1 << 20, a=1 << 20, b=1 << 20)       # rows walked twice need room for their sums
    need = api.mb_layer_norm_fwd_workspace_bytes(C.byref(long))
    assert need > 0
    for ws, nbytes in ((None, need), (one, need - 4), (C.c_void_p(66), need)):
        assert fwd(long, ws=ws, nbytes=nbytes) == 3 and "workspace" in _lib.last_error()


def test_cpu_tensors_are_refused(built_lib):
    from monet_b200 import functional as F
    x = torch.randn(4, 8)
    for call in (lambda: F.layer_norm(x, (8,)), lambda: F.dropout(x, 0.5, torch.tensor([1])),
                 lambda: F.dropout_add_layer_norm(x, x, (8,)), lambda: F.layer_norm_bwd_from_input(x, x, (8,), None, x[:, 0], x[:, 0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
