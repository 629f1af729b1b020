"""Counter-based dropout: the mask is the oracle's element for element, kept values are scaled and
rounded once, and the operator regenerates its mask in backward and recomputation."""
import numpy as np
import pytest
import torch

from oracle import lm_ops_oracle as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 4096, 70001, 1 << 20])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.3000077, 0.999])
def test_mask_and_values(cuda, t, n, p):
    from monet_b200 import functional as F
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g).to(t)
    seed, offset = 0x123456789ABCDEF - n, 3_000_000_000
    y = F.dropout(x.to(cuda), p, torch.tensor([seed], device=cuda), offset).cpu()
    keep = oracle.dropout_keep(seed, offset, n, p)
    scale = torch.tensor(1.0 / (1.0 - p), dtype=torch.float32)
    assert y.dtype == t and torch.equal(y, torch.where(keep, x.float() * scale, torch.zeros(n)).to(t))
    dx = F.dropout_bwd(x.to(cuda), p, torch.tensor([seed], device=cuda), offset).cpu()
    assert torch.equal(dx, y)


def test_ties_of_the_upper_half_go_by_the_lower_half(cuda):
    """p set so that its threshold lies between the numbers of elements with the same upper half."""
    from monet_b200 import functional as F
    n, seed = 1 << 20, 17
    u = oracle.dropout_numbers(seed, 0, n).astype(np.int64)
    s = torch.tensor([seed], device=cuda)
    ones = torch.ones(n, device=cuda)
    order = np.sort(u)
    near = np.nonzero(np.diff(order) == np.diff(order)[np.diff(order) > 0].min())[0][:1]
    for at in list(near) + [0, 5, n // 3, n - 2]:
        for t in (int(order[at]), int(order[at]) + 1, (int(order[at]) >> 16 << 16), (int(order[at]) >> 16 << 16) + 1):
            p = t / 2.0 ** 32
            got = F.dropout(ones, p, s).cpu() == 0
            assert torch.equal(got, torch.from_numpy(u < t)), (at, t)


def test_edges(cuda):
    from monet_b200 import functional as F
    s = torch.tensor([3], device=cuda)
    x = torch.randn(1000, device=cuda)
    assert torch.equal(F.dropout(x, 0.0, None), x) and torch.equal(F.dropout(x, 1e-12, None), x)
    bad = torch.full((1000,), float("nan"), device=cuda)
    assert not bool(F.dropout(bad, 1.0, s).any())                      # all dropped: zero, not NaN
    keep = oracle.dropout_keep(3, 0, 1000, 0.5)
    half = F.dropout(bad, 0.5, s).cpu()
    assert bool(half[keep].isnan().all()) and not bool(half[~keep].any())
    assert F.dropout(x[:0], 0.5, s).numel() == 0
    z = x.clone()
    y = F.dropout(z, 0.5, s, inplace=True)
    assert y.data_ptr() == z.data_ptr() and torch.equal(y, F.dropout(x, 0.5, s))
    assert not torch.equal(F.dropout(x, 0.5, s, 1), F.dropout(x, 0.5, s, 2))
    # a start off the vector boundary, a strided tensor, channels_last
    base = torch.randn(4003, device=cuda)
    for t in TYPES:
        b = base.to(t)
        for v in (b[1:2002], b[2:], b[4:1000], b[::3]):
            keep = oracle.dropout_keep(3, 0, v.numel(), 0.5).to(cuda)
            assert torch.equal(F.dropout(v, 0.5, s), torch.where(keep, v.float() * 2, torch.zeros_like(v.float())).to(t))
    c = torch.randn(2, 3, 4, 5, device=cuda).contiguous(memory_format=torch.channels_last)
    d = F.dropout(c, 0.5, s)
    assert d.stride() == c.stride()
    keep = oracle.dropout_keep(3, 0, c.numel(), 0.5).to(cuda)
    assert torch.equal(d.permute(0, 2, 3, 1).flatten() != 0, keep)


def test_many_elements(cuda):
    from monet_b200 import functional as F
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device=cuda)
    F.dropout(x, 0.5, torch.tensor([29], device=cuda), inplace=True)
    tail = x[-4096:].cpu()
    first = (n - 4096) // 8
    words = oracle.philox_words([(np.arange(514, dtype=np.uint64) + np.uint64(first)) & np.uint64(0xFFFFFFFF),
                                 (np.arange(514, dtype=np.uint64) + np.uint64(first)) >> np.uint64(32), 0, 0], 29)
    skip = (n - 4096) % 8
    halves = words.view("<u2").reshape(-1)[skip:skip + 4096]
    assert torch.equal(tail, torch.from_numpy(np.where(halves >= 0x8000, 2.0, 0.0)).to(torch.bfloat16))


def test_operator_recomputes_its_mask(cuda):
    """Later instances of a node get ``params``; a recomputed forward, a backward and a gradient in
    another layout all see the first forward's mask."""
    import monet_b200.lm_ops as L
    make = L.list_ops("normal", "monet::dropout")[0]
    x = torch.randn(4, 6, 10, 10, device=cuda).contiguous(memory_format=torch.channels_last)
    torch.manual_seed(5)
    op = make()
    y = op.forward(x, 0.4, True)
    again = make()
    again.params = op.params
    assert torch.equal(again.forward(x, 0.4, True), y)
    ones = torch.ones(4, 6, 10, 10, device=cuda)
    back = make()
    back.params = op.params
    dx = back.backward(ones, [])
    assert torch.equal(dx != 0, y != 0) and bool(((dx == 0) | (dx == torch.tensor(1 / 0.6, device=cuda))).all())
    assert not torch.equal(make().forward(x, 0.4, True), y)
    torch.manual_seed(5)
    assert torch.equal(make().forward(x, 0.4, True), y)
    still = make()
    assert torch.equal(still.forward(x, 0.4, False), x) and torch.equal(still.backward(ones, []), ones)


def test_replay_draws_anew(cuda):
    """The seed comes from PyTorch's generator, so each replay of a captured step has its own mask, and
    its forward and backward share it."""
    import monet_b200.lm_ops as L
    make = L.list_ops("normal", "monet::dropout")[0]
    x = torch.randn(5000, device=cuda).abs() + 0.1

    def step():
        op = make()
        y = op.forward(x, 0.5, True)
        return y, op.backward(torch.ones_like(x), [])

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, dx = step()
    seen = []
    for _ in range(3):
        g.replay()
        assert torch.equal(y != 0, dx != 0)
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_refusals(cuda):
    from monet_b200 import functional as F
    x, s = torch.randn(16, device=cuda), torch.tensor([1], device=cuda)
    for call in (lambda: F.dropout(x.double(), 0.5, s), lambda: F.dropout(x, -0.1, s), lambda: F.dropout(x, 1.1, s),
                 lambda: F.dropout(x, float("nan"), s), lambda: F.dropout(x, 0.5, None), lambda: F.dropout(x, 0.5, 7),
                 lambda: F.dropout(x, 0.5, s.cpu()), lambda: F.dropout(x, 0.5, torch.cat([s, s])),
                 lambda: F.dropout(x, 0.5, s.float()), lambda: F.dropout(x, 0.5, s, 1 << 32), lambda: F.dropout(x.cpu(), 0.5, s)):
        with pytest.raises(RuntimeError):
            call()
