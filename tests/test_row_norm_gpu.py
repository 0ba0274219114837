"""Group norm with an activation on channel-last rows (HIP) against the formulas in 64 bits."""
import math

import pytest
import torch

from tests import row_truth

pytestmark = pytest.mark.gpu
U = 2.0 ** -24           # half a step of fp32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _inputs(R, C, dtype, residual, seed=0, shift=2.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    x = (r(R, C) * (0.5 + torch.rand(C, generator=g)) + shift * r(C)).to(dtype)
    return dict(x=x, weight=1 + 0.3 * r(C), bias=0.3 * r(C), residual=r(R, C).to(dtype) if residual else None,
                dy=r(R, C).to(dtype))


def _check(case, groups, dtype, act, cuts=None, shape=None, p=0.0, eps=1e-5, slope=0.01, train=True, rng=(77, 3)):
    """One call against the truth.  Bounds, element by element, from the arithmetic of the operator (U = 2^-24):
    z comes out of about 16 roundings, each at most U of the largest term |xh w| + |b| + |residual|, and of the mean, which is
    held in 32 bits: |mean| rstd |w| U, again under 16 (statistics: four rows at a time, joined in 64 bits).  The activations
    are 1.13-Lipschitz, their own evaluation adds a few U of (1 + |z|): 32 U in all.  The slopes act' are 1.13-Lipschitz too
    (away from the corners of relu: inputs of those cases are kept off them by the test), so g carries |dy| times that.
    Sums over a lane's rows are fp32 over at most 64 of them before they are joined in fp32 trees of depth < 10 and in 64
    bits: 128 U of the sum of magnitudes.  The result is rounded once: half a step of its type."""
    from graspbalance_amd import fused_rows
    dev = "cuda:0"
    x, w, b, res, dy = (case[k] for k in ("x", "weight", "bias", "residual", "dy"))
    R, C = x.shape
    shape = shape or (R, C)
    if cuts is None:
        n = shape[0]
        borders, offs = [i * (R // n) for i in range(n + 1)], None
    else:
        borders, offs = cuts, torch.tensor(cuts, device=dev)
    leaves = {k: (None if t is None else t.to(dev).reshape(shape if t.dim() == 2 else t.shape).requires_grad_(train))
              for k, t in (("x", x), ("weight", w), ("bias", b), ("residual", res))}
    y = fused_rows.group_norm_act(leaves["x"], groups, leaves["weight"], leaves["bias"], eps=eps, act=act, negative_slope=slope,
                                  residual=leaves["residual"], offsets=offs, dropout_p=p, rng=rng if p else None)
    assert y.dtype == dtype and y.shape == shape
    keep, scale = row_truth.keep_mask(R * C, p, *rng) if p else (None, 1.0)
    factor = keep.view(R, C).double() * scale if p else None
    dbl = lambda t: None if t is None else t.double()   # noqa: E731
    want = row_truth.group_norm(dbl(x), groups, dbl(w), dbl(b), eps, act, slope, dbl(res), borders, factor,
                                dbl(dy) if train else None)
    aw = torch.ones(C, dtype=torch.float64) if w is None else dbl(w).abs()
    zero = torch.zeros(1, dtype=torch.float64)
    ez = 32 * U * (1 + want["z"].abs() + want["xh"].abs() * aw + want["offset"] * aw + (zero if b is None else dbl(b).abs())
                   + (zero if res is None else dbl(res).abs()))
    half, tiny = HALF[dtype], TINY[dtype]

    def close(name, got, truth, bound):
        got = got.detach().double().cpu().reshape(truth.shape)
        off = (got - truth).abs()
        worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
        assert torch.isfinite(got).all() and worst <= 1, (name, worst)

    f = scale if p else 1.0
    close("y", y, want["y"], half * want["y"].abs() + f * ez + tiny)
    if p:
        flat = y.detach().reshape(R, C).cpu()
        inside = torch.zeros(R, dtype=torch.bool)
        inside[borders[0]:borders[-1]] = True
        assert bool((flat[~keep.view(R, C) & inside[:, None]] == 0).all())
    if not train:
        return y
    grads = torch.autograd.grad(y, [t for t in leaves.values() if t is not None], dy.to(dev).reshape(shape))
    got = dict(zip([k for k, t in leaves.items() if t is not None], grads))
    eg = f * dbl(dy).abs() * (1.2 * ez + 8 * U)
    mean_eg = eg.max() if eg.numel() else zero
    ex = want["rstd"] * (aw * eg + (1 + want["xh"].abs()) * mean_eg * aw.max()
                         + 128 * U * ((aw * want["dres"].abs()) + want["spread1"] + want["xh"].abs() * want["spread2"])
                         + ez * want["spread2"])
    inside = torch.zeros(R, 1, dtype=torch.float64)
    inside[borders[0]:borders[-1]] = 1
    close("dx", got["x"], want["dx"], half * want["dx"].abs() + ex + tiny)
    if res is not None:
        close("dresidual", got["residual"], want["dres"], half * want["dres"].abs() + eg * inside + tiny)
    if w is not None:
        close("dweight", got["weight"], want["dw"], 128 * U * want["aw"] + (eg * (1 + want["xh"].abs()) + ez * want["dres"].abs()).sum(0) + 1e-30)
        close("dbias", got["bias"], want["db"], 128 * U * want["ab"] + eg.sum(0) + 1e-30)
    outside = inside[:, 0] == 0
    assert bool((y.detach().reshape(R, C).cpu()[outside] == 0).all())
    assert bool((got["x"].reshape(R, C).cpu()[outside] == 0).all())
    return y


def _off_the_corner(case, groups, samples, eps=1e-5):
    """Moves the residual so that no z is within 1e-3 of zero (relu's slope jumps there)."""
    x, R, C = case["x"].double(), *case["x"].shape
    want = row_truth.group_norm(x, groups, case["weight"].double(), case["bias"].double(), eps, "none", 0.0,
                                case["residual"].double(), [i * (R // samples) for i in range(samples + 1)], None, None)
    z = want["z"]
    move = torch.where(z.abs() < 0.02, torch.where(z >= 0, 0.1, -0.1).double(), 0.0)
    case["residual"] = (case["residual"].double() + move).to(case["residual"].dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,groups", [
    ((1, 1, 8), 1), ((1, 1, 4), 4), ((2, 1, 1), 1), ((1, 256, 256), 8), ((3, 37, 90), 6), ((2, 129, 12), 4), ((2, 64, 67), 67),
    ((1, 5, 1021), 1), ((2, 3, 4096), 1), ((2, 3, 4096), 4096), ((1, 700, 1000), 8), ((4, 1024, 256), 32), ((1, 9000, 48), 3),
    ((2, 5000, 65), 5), ((3, 2049, 128), 8), ((70, 33, 24), 2)])
def test_norm_shapes(shape, groups, dtype):
    R, C = math.prod(shape[:-1]), shape[-1]
    _check(_inputs(R, C, dtype, False, seed=R + C), groups, dtype, "silu", shape=shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((1, 400, 4096), 1), ((1, 400, 4096), 4096), ((1, 90, 4096), 512), ((300, 40, 16), 2),
                                          ((2, 20000, 1023), 33)])
def test_norm_wide_and_many(shape, groups, dtype):
    """The widest rows read twice, groups of one channel, many samples, odd rows of a thousand channels."""
    R, C = math.prod(shape[:-1]), shape[-1]
    _check(_inputs(R, C, dtype, True, seed=R + C), groups, dtype, "gelu", shape=shape, p=0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tensors_past_the_caches(dtype):
    """Over 96 MB: the streamed loads and stores.  The truth in 64 bits on the GPU; bounds as in _check for terms of size one
    to ten (|x|, |dy| < 8, rstd < 2, |w| < 3): 32 U * 40 on y, 256 U * 40 on dx."""
    from graspbalance_amd import fused_rows
    rows, C, G = (110000, 128, 8) if dtype == torch.float32 else (110000, 264, 8)
    g = torch.Generator(device="cuda:0").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda:0")   # noqa: E731
    x, dy = r(2, rows, C).to(dtype).requires_grad_(), r(2, rows, C).to(dtype)
    w, b = (1 + 0.2 * r(C)).requires_grad_(), (0.2 * r(C)).requires_grad_()
    assert x.numel() * x.element_size() > 96 << 20
    y = fused_rows.group_norm_act(x, G, w, b, act="silu")
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    half = HALF[dtype]
    tw, tb = torch.zeros(C, dtype=torch.float64, device="cuda:0"), torch.zeros(C, dtype=torch.float64, device="cuda:0")
    with torch.no_grad():
        for s in range(2):
            p = x[s].double().view(rows, G, C // G)
            mean = p.mean((0, 2), keepdim=True)
            rstd = 1 / torch.sqrt(((p - mean) ** 2).mean((0, 2), keepdim=True) + 1e-5)
            xh = ((p - mean) * rstd).view(rows, C)
            z = xh * w.double() + b.double()
            sig = torch.sigmoid(z)
            want = z * sig
            assert bool(((y[s].double() - want).abs() <= half * want.abs() + 32 * 40 * U).all())
            gr = dy[s].double() * (sig + z * sig * (1 - sig))
            h, v = (gr * w.double()).view(rows, G, C // G), xh.view(rows, G, C // G)
            want = ((h - h.mean((0, 2), keepdim=True) - v * (h * v).mean((0, 2), keepdim=True)) * rstd).view(rows, C)
            assert bool(((dx[s].double() - want).abs() <= half * want.abs() + 256 * 40 * U).all())
            tw += (gr * xh).sum(0)
            tb += gr.sum(0)
    # sums of 220000 terms of size ~1: fp32 over at most 64 of them, then 64 bits
    assert bool(((dw.double() - tw).abs() <= 128 * U * 220000).all()) and bool(((db.double() - tb).abs() <= 128 * U * 220000).all())
    assert float((dw.double() - tw).norm() / tw.norm()) < 1e-5


def test_many_packed_samples():
    """A thousand clouds of 0 to 40 rows, some of one row, against the same clouds one by one."""
    from graspbalance_amd import fused_rows
    g = torch.Generator().manual_seed(8)
    sizes = torch.randint(0, 40, (1000,), generator=g)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)])
    R = int(off[-1])
    case = _inputs(R, 48, torch.float32, False, seed=8)
    _check(case, 6, torch.float32, "silu", cuts=off.tolist())
    x = case["x"].to("cuda:0")
    y = fused_rows.group_norm_act(x, 6, offsets=off.to("cuda:0"))
    for s in (0, 17, 500, 999):
        lo, hi = int(off[s]), int(off[s + 1])
        if hi > lo:
            one = fused_rows.group_norm_act(x[lo:hi].unsqueeze(0), 6)[0]
            assert float((one - y[lo:hi]).abs().max()) <= 64 * U * (1 + float(one.abs().max()) * 40)


def test_two_streams_at_once():
    """Two calls in flight on two streams, with workspaces of their own."""
    from graspbalance_amd import fused_rows
    x = [torch.randn(4, 20000, 64, device="cuda:0") for _ in range(2)]
    want = [fused_rows.group_norm_act(t, 8, act="gelu") for t in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fused_rows.group_norm_act(x[i], 8, act="gelu"))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i]) for i in range(2) for a in got[i])


@pytest.mark.parametrize("act", ["none", "relu", "leaky_relu", "silu", "gelu"])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("shape,groups,dtype", [((2, 100, 40), 5, torch.float32), ((2, 4000, 72), 4, torch.bfloat16),
                                                ((1, 3000, 45), 9, torch.float16), ((1, 3000, 45), 9, torch.float32)])
def test_activations_residual_dropout(shape, groups, dtype, act, p):
    R, C = math.prod(shape[:-1]), shape[-1]
    case = _inputs(R, C, dtype, True, seed=5)
    if act in ("relu", "leaky_relu"):
        _off_the_corner(case, groups, shape[0])
    _check(case, groups, dtype, act, shape=shape, p=p, slope=0.2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C,groups,cuts,R", [
    (90, 6, [0, 0, 1, 1, 700, 3001, 3001], 3001), (64, 8, [3, 3, 50, 51, 4000], 4100), (67, 1, [0, 2, 2, 9], 20),
    (128, 8, [0, 20000, 20001, 30000], 30007), (24, 3, [5, 5], 5), (24, 3, [2, 2], 5), (1021, 1, [1, 40, 90], 95)])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_packed_samples(C, groups, cuts, R, dtype, p):
    """Empty samples, single rows, rows before the first and behind the last sample (zeros), odd starts."""
    _check(_inputs(R, C, dtype, True, seed=R), groups, dtype, "gelu", cuts=cuts, p=p)


def test_offsets_outside_the_tensor_stay_inside_it():
    from graspbalance_amd import fused_rows
    x = torch.randn(100, 16, device="cuda:0")
    off = torch.tensor([-7, 40, 2 ** 40], device="cuda:0")
    y = fused_rows.group_norm_act(x, 4, offsets=off)
    want = fused_rows.group_norm_act(x, 4, offsets=torch.tensor([0, 40, 100], device="cuda:0"))
    assert torch.equal(y, want)


@pytest.mark.parametrize("shape", [(1, 512, 32), (1, 70000, 32)])
def test_a_large_offset_costs_no_bits(shape):
    """mean 1000 times the width: the bound holds |mean| rstd U and nothing that grows with its square."""
    _check(_inputs(shape[1], shape[2], torch.float32, False, seed=9, shift=1000.0), 4, torch.float32, "none", shape=shape)


def test_no_weight_no_bias_and_constant_input():
    case = _inputs(300, 48, torch.float32, False)
    case["weight"] = case["bias"] = None
    _check(case, 4, torch.float32, "silu", shape=(2, 150, 48))
    case["x"] = torch.full((300, 48), 3.25)
    _check(case, 4, torch.float32, "none", shape=(2, 150, 48))


def test_non_finite_values_stay_in_their_group():
    from graspbalance_amd import fused_rows
    x = torch.randn(2, 300, 32, device="cuda:0")
    clean = fused_rows.group_norm_act(x, 4, act="relu")
    for bad in (float("inf"), float("nan"), -float("inf")):
        y = x.clone()
        y[1, 7, 9] = bad                   # group 1 of sample 1
        y = fused_rows.group_norm_act(y, 4, act="relu")
        assert bool(torch.isnan(y[1, :, 8:16]).all())
        y[1, :, 8:16] = clean[1, :, 8:16]
        assert torch.equal(y, clean)


def test_views_of_other_tensors_and_strides():
    """A base address that is a multiple of the element only, transposed rows, an expanded gradient."""
    from graspbalance_amd import fused_rows
    flat = torch.randn(2 * 301 * 40 + 3, device="cuda:0").to(torch.bfloat16)
    x = flat[3:].view(2, 301, 40)
    y = fused_rows.group_norm_act(x, 5, act="silu")
    assert torch.equal(y, fused_rows.group_norm_act(x.clone(), 5, act="silu"))
    t = torch.randn(40, 301, device="cuda:0").t().unsqueeze(0).requires_grad_()
    z = fused_rows.group_norm_act(t, 5, act="silu")
    z.sum().backward()
    u = t.detach().contiguous().requires_grad_()
    fused_rows.group_norm_act(u, 5, act="silu").backward(torch.ones_like(u))
    assert torch.equal(t.grad, u.grad)


def test_gradients_against_differences():
    """Central differences of the 64-bit formula at fp32 inputs: the gradient as a whole, not the formula alone."""
    from graspbalance_amd import fused_rows
    case = _inputs(33, 12, torch.float32, True, seed=4)
    args = [case[k] for k in ("x", "weight", "bias", "residual")]
    leaves = [t.to("cuda:0").requires_grad_() for t in args]
    y = fused_rows.group_norm_act(leaves[0].view(1, 33, 12), 3, leaves[1], leaves[2], act="gelu",
                                  residual=leaves[3].view(1, 33, 12), dropout_p=0.25, rng=(4, 4))
    grads = torch.autograd.grad(y, leaves, case["dy"].to("cuda:0").view(1, 33, 12))
    keep, scale = row_truth.keep_mask(33 * 12, 0.25, 4, 4)
    factor = keep.view(33, 12).double() * scale

    def value(ts):
        out = row_truth.group_norm(ts[0], 3, ts[1], ts[2], 1e-5, "gelu", 0, ts[3], [0, 33], factor, None)
        return (out["y"] * case["dy"].double()).sum()

    g = torch.Generator().manual_seed(1)
    dbl = [t.double() for t in args]
    for i, grad in enumerate(grads):
        d = torch.randn(dbl[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = list(dbl), list(dbl)
        up[i], down[i] = dbl[i] + h * d, dbl[i] - h * d
        slope = ((value(up) - value(down)) / (2 * h)).item()
        # differences: h^2 of third derivatives (~1e-8 here); the gradient: 2^-24 times some 400 terms of size ~10
        assert abs((grad.double().cpu().reshape(d.shape) * d).sum().item() - slope) < 1e-3


def test_repeats_bit_for_bit_and_on_a_side_stream():
    from graspbalance_amd import fused_rows
    x = torch.randn(3, 5000, 96, device="cuda:0", requires_grad=True)
    w = torch.randn(96, device="cuda:0", requires_grad=True)
    b = torch.randn(96, device="cuda:0", requires_grad=True)
    dy = torch.randn(3, 5000, 96, device="cuda:0")

    def once():
        y = fused_rows.group_norm_act(x, 8, w, b, act="gelu")
        return [y.detach()] + list(torch.autograd.grad(y, [x, w, b], dy))
    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(first, second))


def test_captured_step_replays_with_new_numbers():
    """Forward and backward in a graph, dropout included: every replay equals the eager call with the pair it found."""
    from graspbalance_amd import fused_rows
    dev = "cuda:0"
    x = torch.randn(2, 900, 64, device=dev, requires_grad=True)
    w = torch.randn(64, device=dev, requires_grad=True)
    b = torch.randn(64, device=dev, requires_grad=True)
    dy = torch.randn(2, 900, 64, device=dev)
    rng = torch.tensor([11, 0], device=dev)
    step = torch.tensor([0, 1], device=dev)

    def once(pair):
        y = fused_rows.group_norm_act(x, 4, w, b, act="silu", dropout_p=0.4, rng=pair)
        return [y] + list(torch.autograd.grad(y, [x, w, b], dy))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            del once(rng)[:]
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(rng)
        rng.add_(step)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(2, 900, 64, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        want = [t.detach() for t in once((11, i))]
        assert all(torch.equal(a, c) for a, c in zip(got, want)), i
        assert rng.tolist() == [11, i + 1]


def test_refusals():
    from graspbalance_amd import fused_rows
    x = torch.randn(2, 10, 16, device="cuda:0")
    off = torch.tensor([0, 20], device="cuda:0")
    for call in (lambda: fused_rows.group_norm_act(x, 3), lambda: fused_rows.group_norm_act(x, 0),
                 lambda: fused_rows.group_norm_act(x, 4, act="tanh"), lambda: fused_rows.group_norm_act(x.double(), 4),
                 lambda: fused_rows.group_norm_act(x[0, 0], 4), lambda: fused_rows.group_norm_act(x, 4, eps=-1.0),
                 lambda: fused_rows.group_norm_act(x, 4, weight=torch.ones(8, device="cuda:0")),
                 lambda: fused_rows.group_norm_act(x, 4, weight=torch.ones(16)),
                 lambda: fused_rows.group_norm_act(x, 4, residual=x[:1]),
                 lambda: fused_rows.group_norm_act(x, 4, residual=x.half()),
                 lambda: fused_rows.group_norm_act(x, 4, offsets=off),
                 lambda: fused_rows.group_norm_act(x.view(20, 16), 4, offsets=off.int()),
                 lambda: fused_rows.group_norm_act(x.view(20, 16), 4, offsets=off.cpu()),
                 lambda: fused_rows.group_norm_act(x.view(20, 16), 4, offsets=off[:1]),
                 lambda: fused_rows.group_norm_act(x, 4, dropout_p=0.5),
                 lambda: fused_rows.group_norm_act(x, 4, dropout_p=2.0, rng=(1, 2)),
                 lambda: fused_rows.group_norm_act(x, 4, dropout_p=0.5, rng=torch.tensor([1, 2])),
                 lambda: fused_rows.group_norm_act(torch.randn(1, 2, 1025, device="cuda:0"), 1)):
        with pytest.raises(RuntimeError):
            call()
    y = fused_rows.group_norm_act(x.requires_grad_(), 4)
    g = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_empty_tensors():
    from graspbalance_amd import fused_rows
    for shape in ((0, 5, 16), (3, 0, 16)):
        x = torch.empty(shape, device="cuda:0", requires_grad=True)
        w = torch.ones(16, device="cuda:0", requires_grad=True)
        y = fused_rows.group_norm_act(x, 4, w, None, act="relu")
        gx, gw = torch.autograd.grad(y.sum(), [x, w])
        assert y.shape == shape and gx.shape == shape and bool((gw == 0).all())


def test_long_runs_keep_their_bits():
    """512 samples of 8000 x 128: a lane adds 1000 terms.  Equal terms 1 + 0.99 * 2^-15 lose their tail at every addition to a
    sum of 512 or more, all in one direction: 250 U in plain fp32.  The bound: 64 additions in fp32 (and the two that end a
    range) before they join a sum of 64 bits, trees of depth under 10, the workgroups' sums and the result rounded once."""
    from graspbalance_amd import fused_rows
    S, rows, C = 512, 8000, 128
    x = torch.randn(S, rows, C, device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(0))
    w, b = (torch.ones(C, device="cuda:0").requires_grad_() for _ in range(2))
    y = fused_rows.group_norm_act(x, 8, w, b)
    c = torch.tensor(1 + 0.99 * 2.0 ** -15, device="cuda:0")
    dw, db = torch.autograd.grad(y, [w, b], c.expand_as(y))
    total = float(c) * S * rows
    assert bool(((db.double() - total).abs() <= 80 * U * total).all()), float((db.double() / total - 1).abs().max() / U)
    # z = xh + 1, so xh is y - 1 to a few U
    xh = sum((y[s].double() - 1).sum(0) for s in range(S)) * float(c)
    mag = sum((y[s].double() - 1).abs().sum(0) for s in range(S)) * float(c)
    assert bool(((dw.double() - xh).abs() <= 90 * U * mag).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((9, 16, 1024), 8), ((64, 3, 40), 4), ((129, 3, 65), 5), ((3000, 2, 33), 3), ((17000, 1, 24), 2),
                                          ((40, 700, 1021), 1)])
def test_many_samples(shape, groups, dtype):
    """The samples' sums added by the applying kernel's last row, by one workgroup a column block, by several."""
    R, C = math.prod(shape[:-1]), shape[-1]
    _check(_inputs(R, C, dtype, False, seed=R), groups, dtype, "silu", shape=shape)


@pytest.mark.parametrize("S,before,behind", [(64, 5, 0), (700, 0, 9000), (2500, 30, 70)])
def test_many_packed_samples_and_rows_outside(S, before, behind):
    """Rows in front of the first and behind the last of many samples, some of them empty, some long."""
    g = torch.Generator().manual_seed(S)
    sizes = torch.randint(0, 7, (S,), generator=g)
    sizes[S // 3] = 3000
    cuts = (torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]) + before).tolist()
    _check(_inputs(cuts[-1] + behind, 40, torch.float32, True, seed=S), 4, torch.float32, "gelu", cuts=cuts, p=0.25)


def test_many_samples_take_no_longer_than_few():
    """The same rows as 4096 samples and as 64, dense and packed with as many rows again behind the last, the best of seven
    passes: about the same time; 7.5 times as long where one workgroup adds the samples' sums (1.58 ms against 0.21), and longer
    still where one clears the rows behind them."""
    from graspbalance_amd import fused_rows

    def best(S, rows, pad):
        x = torch.randn(S * rows + pad, 128, device="cuda:0") if pad else torch.randn(S, rows, 128, device="cuda:0")
        off = torch.arange(S + 1, device="cuda:0") * rows if pad else None
        leaves = [x.requires_grad_()] + [torch.ones(128, device="cuda:0").requires_grad_() for _ in range(2)]
        dy, times = torch.randn_like(x), []
        for _ in range(7):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            y = fused_rows.group_norm_act(leaves[0], 8, *leaves[1:], act="silu", offsets=off)
            torch.autograd.grad(y, leaves, dy)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    for pad in (0, 1 << 18):
        few, many = best(64, 4096, pad), best(4096, 64, pad)
        assert many <= 4 * few, (pad, many, few)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu", "leaky_relu", "silu", "gelu"])
@pytest.mark.parametrize("shape", [(2, 60, 48), (1, 9000, 45)])
def test_dropped_places_hide_the_residual(shape, act, dtype):
    """Infinities and NaN of the residual and of dy in dropped places reach no output and no gradient: the same bits as zeros."""
    from graspbalance_amd import fused_rows
    n, C = math.prod(shape), shape[-1]
    keep, _ = row_truth.keep_mask(n, 0.5, 4, 7)
    keep = keep.view(shape).to("cuda:0")
    case = _inputs(n // C, C, dtype, True, seed=n)
    x, w, b, res, dy = (case[k].to("cuda:0") for k in ("x", "weight", "bias", "residual", "dy"))
    x, res, dy = x.view(shape), res.view(shape), dy.view(shape)

    def run(fill):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, torch.where(keep, res, fill))]
        y = fused_rows.group_norm_act(leaves[0], 3, *leaves[1:3], act=act, residual=leaves[3], dropout_p=0.5, rng=(4, 7))
        return [y.detach()] + list(torch.autograd.grad(y, leaves, torch.where(keep, dy, fill)))
    clean = run(torch.zeros((), dtype=dtype, device="cuda:0"))
    assert all(bool(torch.isfinite(t).all()) for t in clean)
    for bad in (float("inf"), -float("inf"), float("nan")):
        assert all(torch.equal(a, c) for a, c in zip(run(torch.tensor(bad, dtype=dtype, device="cuda:0")), clean)), bad


def test_tensors_past_32_bits_of_elements():
    """Two samples of 2^31 elements and more: the ends of both against the formulas (statistics in 64 bits, on the GPU), dweight
    and dbias; bounds as in test_tensors_past_the_caches."""
    from graspbalance_amd import fused_rows
    rows, C, G = (1 << 24) + 3, 128, 4
    g = torch.Generator(device="cuda:0").manual_seed(5)
    x, dy = (torch.randn(2, rows, C, generator=g, device="cuda:0", dtype=torch.bfloat16) for _ in range(2))
    x[1] += 0.5
    w, b = (1 + 0.2 * torch.randn(C, generator=g, device="cuda:0")).requires_grad_(), torch.zeros(C, device="cuda:0").requires_grad_()
    x.requires_grad_()
    y = fused_rows.group_norm_act(x, G, w, b, act="relu")
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    tw, tb, mw, mb = (torch.zeros(C, dtype=torch.float64, device="cuda:0") for _ in range(4))
    step = 1 << 20
    with torch.no_grad():
        for s in range(2):
            part = lambda t, i: t[s, i:i + step].double().view(-1, G, C // G)   # noqa: E731
            n, sums = rows * (C // G), torch.zeros(4, G, 1, dtype=torch.float64, device="cuda:0")
            for i in range(0, rows, step):
                sums[0] += part(x, i).sum((0, 2)).view(G, 1)
            mean = sums[0] / n
            for i in range(0, rows, step):
                sums[1] += ((part(x, i) - mean) ** 2).sum((0, 2)).view(G, 1)
            rstd = 1 / torch.sqrt(sums[1] / n + 1e-5)
            wd = w.double().view(G, -1)
            for i in range(0, rows, step):
                xh = (part(x, i) - mean) * rstd
                gr = part(dy, i) * (xh * wd > 0)
                sums[2] += (gr * wd).sum((0, 2)).view(G, 1)
                sums[3] += (gr * wd * xh).sum((0, 2)).view(G, 1)
                tw += (gr * xh).sum(0).view(C)
                tb += gr.sum(0).view(C)
                mw += (gr * xh).abs().sum(0).view(C)
                mb += gr.abs().sum(0).view(C)
            for at in (slice(0, 1000), slice(rows - 1000, rows)):
                xh = (x[s, at].double().view(-1, G, C // G) - mean) * rstd
                z = xh * wd
                want = z.clamp(min=0).view(-1, C)
                assert bool(((y[s, at].double() - want).abs() <= HALF[torch.bfloat16] * want + 32 * 40 * U).all()), s
                gr = dy[s, at].double().view(-1, G, C // G) * (z > 0)
                want = ((gr * wd - sums[2] / n - xh * sums[3] / n) * rstd).view(-1, C)
                clear = (z.abs() > 1e-4).view(-1, C)     # (relu's slope jumps at zero)
                off = (dx[s, at].double() - want).abs()
                assert bool((off <= HALF[torch.bfloat16] * want.abs() + 256 * 40 * U)[clear].all()), s
    # (elements within rounding of relu's corner, 1e-6 of them, may fall on the other side)
    assert bool(((dw.double() - tw).abs() <= 128 * U * mw).all()) and bool(((db.double() - tb).abs() <= 128 * U * mb + 1e-5 * mb).all())


def test_gelu_over_its_range():
    """gelu and its slope by themselves (weight 0: z is the bias), relative to the true values: the polynomial's 1.1e-7, the
    roundings of the exponent (two of z^2 / 2, which exp multiplies by) and twelve more - down to z = -9, where the value is 1e-18."""
    from graspbalance_amd import fused_rows
    C = 4096
    z = torch.linspace(-9, 9, C)
    z[C // 2] = 0.0
    b = z.to("cuda:0").requires_grad_()
    x = torch.ones(1, 1, C, device="cuda:0")
    y = fused_rows.group_norm_act(x, C, torch.zeros(C, device="cuda:0"), b, act="gelu")
    slope, = torch.autograd.grad(y, b, torch.ones_like(y))
    zd = z.double()
    cdf = 0.5 * torch.special.erfc(-zd / math.sqrt(2.0))
    pdf = torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)
    part = 1.1e-7 + (zd * zd + 12) * U
    off = (y.detach().double().cpu().view(C) - zd * cdf).abs()
    assert bool((off <= part * (zd * cdf).abs()).all()), (off / (zd * cdf).abs()).max()
    off = (slope.double().cpu() - (cdf + zd * pdf)).abs()
    assert bool((off <= part * (cdf + zd.abs() * pdf)).all())
