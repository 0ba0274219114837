"""Dropout from a counter-based generator (HIP) against its formula: masks exactly, values to the one rounding."""
import pytest
import torch

from tests import row_truth

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 4096, 65537, 3 * 1024 * 1024 + 5])
@pytest.mark.parametrize("p,residual", [(0.1, False), (0.5, True), (0.999, True), (1.0, True)])
def test_values_and_gradients(n, dtype, p, residual):
    from graspbalance_amd import fused_rows
    g = torch.Generator().manual_seed(n)
    x, dy = torch.randn(n, generator=g).to(dtype), torch.randn(n, generator=g).to(dtype)
    res = torch.randn(n, generator=g).to(dtype) if residual else None
    pair = (-5 - n, (1 << 40) + 3)
    xd = x.to("cuda:0").requires_grad_()
    rd = res.to("cuda:0").requires_grad_() if residual else None
    y = fused_rows.dropout(xd, p, pair, residual=rd)
    keep, scale = row_truth.keep_mask(n, p, *pair)
    factor = keep.double() * scale
    want = x.double() * factor + (res.double() if residual else 0)
    # x * scale (scale itself rounded): 2 U of the product, the sum: U, and the rounding to the type
    bound = 4 * 2.0 ** -24 * (x.double() * factor).abs() + (2.0 ** -24 + HALF[dtype]) * want.abs() + TINY[dtype]
    assert bool(((y.detach().double().cpu() - want).abs() <= bound).all())
    if not residual:
        assert torch.equal(y.detach().cpu() != 0, keep & (x != 0))
    y.backward(dy.to("cuda:0"))
    want = dy.double() * factor
    bound = (4 * 2.0 ** -24 + HALF[dtype]) * want.abs() + TINY[dtype]
    assert bool(((xd.grad.double().cpu() - want).abs() <= bound).all())
    if residual:
        assert torch.equal(rd.grad.cpu(), dy)


def test_numbers_past_32_bits_of_elements():
    """Elements behind 2^32: the counter's second word."""
    from graspbalance_amd import fused_rows
    n = (1 << 32) + 4096
    x = torch.ones(n, device="cuda:0", dtype=torch.float16)
    y = fused_rows.dropout(x, 0.5, (123, 9))
    del x
    tail = (y[-4096:] != 0).cpu()
    blocks = torch.arange((n - 4096) >> 3, n >> 3)
    import numpy as np
    c = np.zeros((blocks.numel(), 4), np.uint64)
    c[:, 0], c[:, 1], c[:, 2] = blocks.numpy() & 0xFFFFFFFF, blocks.numpy() >> 32, 9
    w = row_truth.philox(c, (123, 0))
    h = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(-1)
    assert torch.equal(tail, torch.from_numpy(h >= 32768))


def test_fp32_past_the_caches():
    """Over 96 MB of fp32: the streamed form keeps the places and values of the others."""
    from graspbalance_amd import fused_rows
    n = (96 << 18) + 4099
    x, res = torch.randn(n, device="cuda:0"), torch.randn(n, device="cuda:0")
    for r in (None, res):
        y = fused_rows.dropout(x, 0.4, (3, 7), residual=r)
        cut = 1 << 20
        head = fused_rows.dropout(x[:cut], 0.4, (3, 7), residual=None if r is None else r[:cut])
        assert torch.equal(y[:cut], head)
        keep, scale = row_truth.keep_mask(n, 0.4, 3, 7)
        want = torch.where(keep.to("cuda:0"), x * scale, 0.0) + (0 if r is None else r)
        assert bool(((y - want).abs() <= 4 * 2.0 ** -24 * (x.abs() * scale + want.abs())).all())


def test_rates_and_independence():
    """The share of kept elements and of places kept by two calls: within 6 sigma of p and p^2."""
    from graspbalance_amd import fused_rows
    n = 1 << 22
    x = torch.ones(n, device="cuda:0")
    for p in (0.1, 0.5, 0.9):
        a, b = (fused_rows.dropout(x, p, (42, call)) != 0 for call in (0, 1))
        for share, want in ((a, 1 - p), (b, 1 - p), (a & b, (1 - p) ** 2)):
            sigma = (want * (1 - want) / n) ** 0.5
            assert abs(share.double().mean().item() - want) < 6 * sigma + 2.0 ** -16
    assert torch.equal(fused_rows.dropout(x, 0.5, (1, 2)), fused_rows.dropout(x, 0.5, (1, 2)))
    assert not torch.equal(fused_rows.dropout(x, 0.5, (1, 2)), fused_rows.dropout(x, 0.5, (2, 1)))


def test_dropped_places_hide_what_they_hold():
    from graspbalance_amd import fused_rows
    x = torch.randn(4096, device="cuda:0")
    keep = fused_rows.dropout(torch.ones_like(x), 0.5, (8, 8)) != 0
    bad = torch.where(keep, x, torch.tensor(float("nan"), device="cuda:0"))
    assert torch.equal(fused_rows.dropout(bad, 0.5, (8, 8)), fused_rows.dropout(torch.where(keep, x, 0.0), 0.5, (8, 8)))


def test_layer_moves_on_and_evaluates_to_the_input():
    from graspbalance_amd import fused_rows
    layer = fused_rows.Dropout(0.5, seed=6).to("cuda:0")
    x = torch.randn(2, 3, 128, device="cuda:0", requires_grad=True)
    a = layer(x)
    b = layer(x, residual=x.detach())
    assert layer.rng.tolist() == [6, 2]
    assert torch.equal(a, fused_rows.dropout(x, 0.5, (6, 0)))
    assert torch.equal(b, fused_rows.dropout(x, 0.5, (6, 1), residual=x.detach()))
    # the backward pass of the first call uses the first call's numbers although the layer has moved on
    ga, = torch.autograd.grad(a, x, torch.ones_like(a))
    assert torch.equal(ga != 0, fused_rows.dropout(torch.ones_like(x), 0.5, (6, 0)) != 0)
    assert layer.state_dict()["rng"].tolist() == [6, 2] and list(layer.state_dict()) == ["rng"]
    layer.eval()
    assert layer(x) is x and torch.equal(layer(x, residual=x), x + x)
    assert layer.rng.tolist() == [6, 2]


def test_captured_layer_draws_new_numbers_at_every_replay():
    from graspbalance_amd import fused_rows
    layer = fused_rows.Dropout(0.5, seed=1).to("cuda:0")
    x = torch.randn(5000, device="cuda:0", requires_grad=True)
    dy = torch.randn(5000, device="cuda:0")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = layer(x)
        torch.autograd.grad(y, x, dy)
        del y
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
        gx, = torch.autograd.grad(y, x, dy)
    for call in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        want = fused_rows.dropout(x.detach(), 0.5, (1, call))
        assert torch.equal(y.detach(), want), call
        assert torch.equal(gx, fused_rows.dropout(dy, 0.5, (1, call)))


def test_misaligned_and_strided_inputs():
    from graspbalance_amd import fused_rows
    flat = torch.randn(5001, device="cuda:0").to(torch.bfloat16)
    assert torch.equal(fused_rows.dropout(flat[1:], 0.5, (3, 3)), fused_rows.dropout(flat[1:].clone(), 0.5, (3, 3)))
    m = torch.randn(64, 33, device="cuda:0")
    assert torch.equal(fused_rows.dropout(m.t(), 0.5, (3, 3)), fused_rows.dropout(m.t().contiguous(), 0.5, (3, 3)))
    e = torch.empty(0, 4, device="cuda:0", requires_grad=True)
    y = fused_rows.dropout(e, 0.5, (3, 3))
    assert y.shape == (0, 4) and torch.autograd.grad(y.sum(), e)[0].shape == (0, 4)


def test_refusals():
    from graspbalance_amd import fused_rows
    x = torch.randn(8, device="cuda:0")
    for call in (lambda: fused_rows.dropout(x, -0.1, (1, 2)), lambda: fused_rows.dropout(x, 1.1, (1, 2)),
                 lambda: fused_rows.dropout(x.double(), 0.5, (1, 2)), lambda: fused_rows.dropout(x, 0.5, None),
                 lambda: fused_rows.dropout(x, 0.5, (1,)), lambda: fused_rows.dropout(x, 0.5, torch.tensor([1, 2])),
                 lambda: fused_rows.dropout(x, 0.5, torch.tensor([1, 2], dtype=torch.int32, device="cuda:0")),
                 lambda: fused_rows.dropout(x, 0.5, (1, 2), residual=x[:4])):
        with pytest.raises(RuntimeError):
            call()
