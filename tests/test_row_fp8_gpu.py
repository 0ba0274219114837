"""Products in 8-bit floats with a scale for each block of 128 (HIP) against the definition in 64 bits."""
import pytest
import torch

from tests import row_truth

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _maxima(a):
    """Largest magnitude of every block of 128 along the rows of a: (R, blocks)."""
    pad = torch.nn.functional.pad(a.abs(), (0, -a.shape[1] % 128))
    return pad.view(a.shape[0], -1, 128).amax(2)


def _check(got, a, b, bias, dtype, name, length=None):
    """got against a @ b^T + bias in double.  fp32 results: exact products of bf16 operands and fp32 additions - the
    instruction adds in groups, so at most length / 8 roundings of 2^-24 follow a term, and 64 where ranges are joined.
    16-bit results: in a step of at most 128 products none loses more than 2^-14 of the largest, which is no larger than the
    product of the two blocks' largest; the steps are added in fp32.  Then one rounding to the type."""
    truth = a @ b.t()
    terms = a.abs() @ b.abs().t()
    if bias is not None:
        truth, terms = truth + bias, terms + bias.abs()
    bound = 2.0 ** -24 * ((length or a.shape[1]) / 8 + 64) * terms + HALF[dtype] * truth.abs() + TINY[dtype]
    if dtype != torch.float32:
        bound = bound + 128 * 2.0 ** -14 * (_maxima(a) @ _maxima(b).t())
    off = (got.detach().double().cpu() - truth).abs()
    assert got.dtype == dtype and got.shape == truth.shape and torch.isfinite(got).all()
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1, (name, worst)


def _data(P, K, N, dtype, wtype=torch.float32, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed + P + 3 * K + 7 * N)
    x = (torch.randn(P, K, generator=g) * torch.exp(torch.randn(P, 1, generator=g))).to(dtype)
    w = (torch.randn(N, K, generator=g) * (2.0 / K) ** 0.5).to(wtype)
    return x, w, torch.randn(N, generator=g) if bias else None, torch.randn(P, N, generator=g).to(dtype)


SHAPES = [(1, 1, 1), (1, 1024, 1024), (2, 130, 17), (5, 128, 128), (16, 1000, 33), (16, 1025, 40), (17, 64, 300), (33, 259, 65),
          (64, 512, 129), (65, 127, 127), (100, 384, 130), (300, 129, 302), (1000, 640, 96), (4096, 259, 302), (700, 2048, 515),
          (2500, 136, 4104), (70, 5000, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,K,N", SHAPES)
def test_forward_and_gradients(P, K, N, dtype):
    from graspbalance_amd import fused_rows
    x, w, b, dy = _data(P, K, N, dtype)
    leaves = [t.to("cuda:0").requires_grad_() for t in (x, w, b)]
    y = fused_rows.fp8_linear(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to("cuda:0"))
    xq, wq, dq = row_truth.in_8_bits(x.double(), 1), row_truth.in_8_bits(w.double(), 128), row_truth.in_8_bits(dy.double(), 1)
    _check(y, xq, wq, b.double(), dtype, "y")
    _check(dx, dq, wq.t().contiguous(), None, dtype, "dx")
    _check(dw, dq.t().contiguous(), xq.t().contiguous(), None, torch.float32, "dw", length=P)
    sums = dy.double().sum(0)
    assert bool(((db.double().cpu() - sums).abs() <= 2.0 ** -24 * (64 * dy.double().abs().sum(0) + sums.abs())).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("P,K,N", [(1, 1024, 1024), (3, 300, 500), (16, 1024, 64), (16, 1152, 64), (40, 130, 77), (900, 200, 300),
                                   (20000, 128, 192)])
def test_kept_weight_gives_what_the_float_one_does(P, K, N, dtype):
    """A weight quantised once, its codes given back as tensors, and one quantised in the call: the same bits."""
    from graspbalance_amd import fused_rows
    x, w, b, dy = (t.to("cuda:0") for t in _data(P, K, N, dtype))
    held = fused_rows.Fp8Weight.quantize(w, input_gradients=True)
    codes = held.codes.float().cpu().double()
    scale = torch.exp2(held.scales.cpu().double() - 127).repeat_interleave(128, 0).repeat_interleave(128, 1)[:N]
    assert torch.equal((codes * scale)[:, :K], row_truth.in_8_bits(w.cpu().double(), 128))
    assert bool((codes[:, K:] == 0).all())
    assert torch.equal(held.codes_t.float().cpu()[:, :N].t().double(), codes[:, :K])
    y = fused_rows.fp8_linear(x, held, b)
    again = fused_rows.Fp8Weight(held.codes.view(torch.uint8), held.scales, K)
    assert torch.equal(y, fused_rows.fp8_linear(x, again, b))
    _check(y, row_truth.in_8_bits(x.cpu().double(), 1), row_truth.in_8_bits(w.cpu().double(), 128), b.cpu().double(), dtype, "y")
    xg = x.clone().requires_grad_()
    wg = w.clone().requires_grad_()
    gx, = torch.autograd.grad(fused_rows.fp8_linear(xg, held, b), xg, dy)
    want, _ = torch.autograd.grad(fused_rows.fp8_linear(xg, wg, b), [xg, wg], dy)
    assert torch.equal(gx, want)
    with pytest.raises(RuntimeError, match="input_gradients"):
        fused_rows.fp8_linear(xg, again, b)


def test_many_rows():
    """More rows than a range of the weight gradient, tiles of 256, an odd tail; the truth on the GPU in 64 bits."""
    from graspbalance_amd import fused_rows
    P, K, N = 70001, 200, 264
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, dy = (t.to("cuda:0") for t in _data(P, K, N, dtype))
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = fused_rows.fp8_linear(*leaves)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        xq, wq, dq = (row_truth.in_8_bits(t.detach().cpu().double(), n) for t, n in ((x, 1), (w, 128), (dy, 1)))
        _check(y, xq, wq, b.detach().cpu().double(), dtype, "y")
        _check(dx, dq, wq.t().contiguous(), None, dtype, "dx")
        _check(dw, dq.t().contiguous(), xq.t().contiguous(), None, torch.float32, "dw", length=P)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,K,N", [(32768, 128, 128), (33001, 131, 100), (40003, 100, 255), (35000, 127, 470), (32770, 512, 90),
                                   (120007, 256, 130)])
def test_streamed_rows(P, K, N, dtype):
    """Many rows and a weight that LDS holds: every column variant, one and several steps, odd widths, kept codes, sums."""
    from graspbalance_amd import fused_rows
    x, w, b, dy = (t.to("cuda:0") for t in _data(P, K, N, dtype))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = fused_rows.fp8_linear(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    xq, wq, dq = (row_truth.in_8_bits(t.detach().cpu().double(), n) for t, n in ((x, 1), (w, 128), (dy, 1)))
    _check(y, xq, wq, b.detach().cpu().double(), dtype, "y")
    _check(dx, dq, wq.t().contiguous(), None, dtype, "dx")
    _check(dw, dq.t().contiguous(), xq.t().contiguous(), None, torch.float32, "dw", length=P)
    sums = dy.cpu().double().sum(0)
    assert bool(((db.double().cpu() - sums).abs() <= 2.0 ** -24 * (256 * dy.cpu().double().abs().sum(0) + sums.abs())).all())
    with torch.no_grad():      # nothing kept
        assert torch.equal(fused_rows.fp8_linear(x, fused_rows.Fp8Weight.quantize(w), b), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,K,N", [(33, 4096, 70), (64, 4300, 130), (65, 1030, 64), (200, 1153, 321), (1000, 2100, 100),
                                   (1100, 1100, 1100), (2100, 1664, 515)])
def test_long_reductions_of_few_tiles(P, K, N, dtype):
    """The steps split over groups of waves: two and four of them, ranges that are short or empty, tiles that end inside."""
    from graspbalance_amd import fused_rows
    x, w, b, _ = _data(P, K, N, dtype)
    held = fused_rows.Fp8Weight.quantize(w.to("cuda:0"))
    y = fused_rows.fp8_linear(x.to("cuda:0"), held, b.to("cuda:0"))
    _check(y, row_truth.in_8_bits(x.double(), 1), row_truth.in_8_bits(w.double(), 128), b.double(), dtype, "y")
    assert torch.equal(y, fused_rows.fp8_linear(x.to("cuda:0"), held, b.to("cuda:0")))
    bad = x.clone()
    bad[P // 2, K - 1] = float("nan")
    again = fused_rows.fp8_linear(bad.to("cuda:0"), held, b.to("cuda:0"))
    rest = torch.arange(P, device="cuda:0") != P // 2
    assert bool(torch.isnan(again[P // 2]).all()) and torch.equal(again[rest], y[rest])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("P,K,N", [(420000, 128, 128), (13000, 640, 4100)])
def test_results_past_the_caches(P, K, N, dtype):
    """Over 96 MB of x or y: streamed loads and stores, in both ways through the kernels; 300 rows against the truth, all of
    them against the same rows in parts.  A part of many rows is added in the same order; the one row that is left over
    goes through another kernel, whose sums are off by what _check allows fp32 sums, as the others are: twice that."""
    from graspbalance_amd import fused_rows
    x, w, b, _ = (t.to("cuda:0") for t in _data(P, K, N, dtype))
    held = fused_rows.Fp8Weight.quantize(w)
    y = fused_rows.fp8_linear(x, held, b)
    pick = torch.randperm(P, generator=torch.Generator().manual_seed(0))[:300]
    _check(y[pick.to("cuda:0")], row_truth.in_8_bits(x[pick.to("cuda:0")].cpu().double(), 1),
           row_truth.in_8_bits(w.cpu().double(), 128), b.cpu().double(), dtype, "y")
    part = P // 3
    for lo in range(0, P, part):
        mine, whole = fused_rows.fp8_linear(x[lo:lo + part], held, b), y[lo:lo + part]
        if mine.shape[0] > 64:
            assert torch.equal(mine, whole)
        else:
            xq, wq = row_truth.in_8_bits(x[lo:].cpu().double(), 1), row_truth.in_8_bits(w.cpu().double(), 128)
            bound = 2.0 ** -24 * (K / 8 + 64) * (xq.abs() @ wq.abs().t() + b.cpu().double().abs()) + HALF[dtype] * whole.abs().cpu().double()
            if dtype != torch.float32:
                bound = bound + 128 * 2.0 ** -14 * (_maxima(xq) @ _maxima(wq).t())
            assert bool(((mine - whole).abs().cpu().double() <= 2 * bound).all())


def _codes(x):
    from graspbalance_amd import fused_rows
    codes, scales = fused_rows._quantise_rows(x)
    return codes.view(torch.float8_e4m3fn).float().cpu().double(), scales.cpu().int()


def test_quantiser_at_its_borders():
    """The largest value at 448 * 2^e and one step beyond, ties between codes, the smallest codes, blocks of zeros, the
    smallest and largest magnitudes."""
    up = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9)).item()
    rows = []
    for top in (448.0, up, 447.0, 1.0, 0.875, 0.8750001, 3.4028234e38, 1e-38, 2.0 ** -126, 2.0 ** -149, 7 * 2.0 ** -149):
        r = torch.zeros(130)
        r[0] = top
        r[1:9] = top * torch.tensor([1 / 3, 0.03125, 0.0013, 2.0 ** -15, 2.0 ** -18.5, 17 / 32, 19 / 32, -1.0])
        r[129] = -top
        rows.append(r)
    rows.append(torch.zeros(130))
    x = torch.stack(rows)
    codes, scales = _codes(x.to("cuda:0"))
    want = row_truth.in_8_bits(x.double(), 1)
    got = codes * torch.exp2(scales[:, :2].double() - 127).repeat_interleave(128, 1)
    assert torch.equal(got[:, :130], want) and bool((codes[:, 130:] == 0).all())
    assert scales[0, 0] == 127 and scales[1, 0] == 128 and scales[-1, 0] == 127 and int(scales[:, :2].min()) >= 1
    assert codes.abs().max() == 448


def test_ties_go_to_even_codes():
    x = torch.zeros(1, 128)
    x[0, 0] = 448.0
    x[0, 1:7] = torch.tensor([17.0, 19.0, 21.0, 2.0 ** -10, 3 * 2.0 ** -10, -17.0])
    codes, _ = _codes(x.to("cuda:0"))
    assert codes[0, 1:7].tolist() == [16.0, 20.0, 20.0, 0.0, 2 * 2.0 ** -9, -16.0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("P", [1, 40, 300])
def test_non_finite_values(P, dtype):
    """An infinity or NaN spoils its row of y (of x) or its column (of weight) and nothing else."""
    from graspbalance_amd import fused_rows
    x, w, _, _ = (None if t is None else t.to("cuda:0") for t in _data(P, 260, 50, dtype, bias=False))
    clean = fused_rows.fp8_linear(x, w)
    for bad in (float("inf"), float("nan")):
        y = x.clone()
        y[P // 2, 131] = bad
        y = fused_rows.fp8_linear(y, w)
        assert bool(torch.isnan(y[P // 2]).all())
        rest = torch.arange(P, device="cuda:0") != P // 2
        assert torch.equal(y[rest], clean[rest])
        v = w.clone()
        v[7, 259] = bad
        y = fused_rows.fp8_linear(x, v)
        assert bool(torch.isnan(y[:, 7]).all()) and bool(torch.isfinite(y[:, 8:]).all())


def test_gradients_against_differences():
    """On inputs that 8 bits hold exactly, steps that stay on the codes leave the quantisers the identity, so differences of
    the operator itself are exact: y is linear in x and in weight."""
    from graspbalance_amd import fused_rows
    g = torch.Generator().manual_seed(3)
    P, K, N = 40, 256, 48
    x = torch.randint(-6, 7, (P, K), generator=g).float()
    w = torch.randint(-6, 7, (N, K), generator=g).float()
    dy = torch.randint(-3, 4, (P, N), generator=g).float()
    x[:, 0::128], w[:, 0::128], dy[:, 0] = 448.0, 448.0, 448.0     # every block's scale is 1 whatever the rest does
    leaves = [t.to("cuda:0").requires_grad_() for t in (x, w)]
    y = fused_rows.fp8_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy.to("cuda:0"))
    for i in range(2):
        d = torch.randint(-1, 2, leaves[i].shape, generator=g).float()
        d[:, 0::128] = 0
        moved = [t.detach().cpu() for t in leaves]
        moved[i] = moved[i] + d
        diff = (fused_rows.fp8_linear(*(t.to("cuda:0") for t in moved)).double().cpu() - y.detach().double().cpu())
        want = (diff * dy.double()).sum().item()
        got = (grads[i].double().cpu() * d.double()).sum().item()
        assert abs(got - want) <= 1e-6 * (diff * dy.double()).abs().sum().item() + 1e-3


def test_views_batches_streams_and_repeats():
    from graspbalance_amd import fused_rows
    x = torch.randn(3, 50, 96, device="cuda:0")
    w = torch.randn(40, 96, 1, 1, device="cuda:0")
    y = fused_rows.fp8_linear(x, w)
    assert y.shape == (3, 50, 40)
    assert torch.equal(y.view(150, 40), fused_rows.fp8_linear(x.view(150, 96), w.view(40, 96)))
    wide = torch.randn(150, 101, device="cuda:0")
    wide[:, 3:99] = x.view(150, 96)
    assert torch.equal(fused_rows.fp8_linear(wide[:, 3:99], w), y.view(150, 40))
    flat = torch.cat([torch.zeros(1, device="cuda:0"), x.flatten()])[1:].view(150, 96)     # a base 4 bytes off a line
    assert torch.equal(fused_rows.fp8_linear(flat, w), y.view(150, 40))
    t = torch.randn(96, 40, device="cuda:0").t()
    assert torch.equal(fused_rows.fp8_linear(x, t), fused_rows.fp8_linear(x, t.contiguous()))
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()

    def once():
        out = fused_rows.fp8_linear(xs, ws)
        return [out.detach()] + list(torch.autograd.grad(out, [xs, ws], torch.ones_like(out)))
    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_step():
    from graspbalance_amd import fused_rows
    dev = "cuda:0"
    x, w, b, dy = (t.to(dev) for t in _data(900, 130, 70, torch.float32))
    x, w, b = (t.requires_grad_() for t in (x, w, b))

    def once():
        y = fused_rows.fp8_linear(x, w, b)
        return [y] + list(torch.autograd.grad(y, [x, w, b], dy))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        del once()[:]
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(900, 130, device=dev))
            w.copy_(torch.randn(70, 130, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        assert all(torch.equal(a, c.detach()) for a, c in zip(got, once())), i


def test_other_weight_types_partial_gradients_and_empty_rows():
    from graspbalance_amd import fused_rows
    x = torch.randn(60, 100, device="cuda:0")
    w = torch.randn(30, 100, device="cuda:0").to(torch.bfloat16).requires_grad_()
    y = fused_rows.fp8_linear(x, w)
    gw, = torch.autograd.grad(y.sum(), w)
    assert gw.dtype == torch.bfloat16
    b = torch.randn(30, device="cuda:0").half().requires_grad_()
    gb, = torch.autograd.grad(fused_rows.fp8_linear(x, w.detach(), b).sum(), b)
    assert gb.dtype == torch.float16 and bool((gb == 60).all())
    e = torch.empty(0, 100, device="cuda:0", requires_grad=True)
    y = fused_rows.fp8_linear(e, w, b)
    ge, gw, gb = torch.autograd.grad(y.sum(), [e, w, b])
    assert y.shape == (0, 30) and ge.shape == (0, 100) and bool((gw == 0).all()) and bool((gb == 0).all())


def test_refusals():
    from graspbalance_amd import fused_rows
    x, w = torch.randn(4, 64, device="cuda:0"), torch.randn(8, 64, device="cuda:0")
    held = fused_rows.Fp8Weight.quantize(w)
    for call in (lambda: fused_rows.fp8_linear(x.double(), w), lambda: fused_rows.fp8_linear(x, w.double()),
                 lambda: fused_rows.fp8_linear(x[:, :63], w), lambda: fused_rows.fp8_linear(x, w.cpu()),
                 lambda: fused_rows.fp8_linear(x.cpu(), w), lambda: fused_rows.fp8_linear(x, w, torch.ones(9, device="cuda:0")),
                 lambda: fused_rows.fp8_linear(x, w.view(8, 32, 2)), lambda: fused_rows.fp8_linear(x, w[:0]),
                 lambda: fused_rows.fp8_linear(x[:, :32], held),
                 lambda: fused_rows.Fp8Weight(held.codes, held.scales, 200),
                 lambda: fused_rows.Fp8Weight(held.codes, held.scales.int(), 64),
                 lambda: fused_rows.Fp8Weight(held.codes[:, :64], held.scales, 64),
                 lambda: fused_rows.Fp8Weight(held.codes.cpu(), held.scales, 64),
                 lambda: fused_rows.Fp8Weight(held.codes.float(), held.scales, 64)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,K,N", [(1, 1024, 1024), (40, 1300, 70), (200, 1153, 321), (1100, 1100, 1100), (16500, 256, 200),
                                   (20000, 128, 128), (2500, 136, 4104)])
def test_sums_of_16_bit_products_are_fp32(P, K, N, dtype):
    """The bound of fp32 results (see _check: K / 8 roundings of 2^-24 and 64 where ranges are joined) and the one rounding to
    the type, on every route: values and the input's gradient.  Outputs whose terms cancel show sums of fewer bits."""
    from graspbalance_amd import fused_rows
    x, w, b, dy = _data(P, K, N, dtype)
    xg = x.to("cuda:0").requires_grad_()
    y = fused_rows.fp8_linear(xg, fused_rows.Fp8Weight.quantize(w.to("cuda:0"), input_gradients=True), b.to("cuda:0"))
    dx, = torch.autograd.grad(y, xg, dy.to("cuda:0"))
    xq, wq, dq = row_truth.in_8_bits(x.double(), 1), row_truth.in_8_bits(w.double(), 128), row_truth.in_8_bits(dy.double(), 1)
    for got, left, right, bias in ((y, xq, wq, b.double()), (dx, dq, wq.t().contiguous(), None)):
        truth, terms = left @ right.t(), left.abs() @ right.abs().t()
        if bias is not None:
            truth, terms = truth + bias, terms + bias.abs()
        bound = 2.0 ** -24 * (left.shape[1] / 8 + 64) * terms + HALF[dtype] * truth.abs() + TINY[dtype]
        off = (got.detach().double().cpu() - truth).abs()
        assert bool((off <= bound).all()), (off / bound).max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,K,N", SHAPES + [(20000, 128, 192), (33001, 131, 100), (35000, 127, 470), (1100, 1100, 1100)])
def test_short_sums_on_request(P, K, N, dtype):
    """The 8-bit matrix instructions where they are asked for, within _check's bound for them; fp32 rows take no notice."""
    from graspbalance_amd import fused_rows
    x, w, b, dy = _data(P, K, N, dtype)
    leaves = [t.to("cuda:0").requires_grad_() for t in (x, w, b)]
    y = fused_rows.fp8_linear(*leaves, short_sums=True)
    grads = torch.autograd.grad(y, leaves, dy.to("cuda:0"))
    xq, wq, dq = row_truth.in_8_bits(x.double(), 1), row_truth.in_8_bits(w.double(), 128), row_truth.in_8_bits(dy.double(), 1)
    _check(y, xq, wq, b.double(), dtype, "y")
    _check(grads[0], dq, wq.t().contiguous(), None, dtype, "dx")
    _check(grads[1], dq.t().contiguous(), xq.t().contiguous(), None, torch.float32, "dw", length=P)
    if dtype == torch.float32:
        plain = fused_rows.fp8_linear(*leaves)
        assert torch.equal(y, plain)
        assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(plain, leaves, dy.to("cuda:0"))))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,K,N", [(420000, 128, 128), (13000, 640, 4100)])
def test_short_sums_past_the_caches(P, K, N, dtype):
    """The streamed loads and stores of that form: 300 rows against the truth."""
    from graspbalance_amd import fused_rows
    x, w, b, _ = (t.to("cuda:0") for t in _data(P, K, N, dtype))
    y = fused_rows.fp8_linear(x, w, b, short_sums=True)
    pick = torch.randperm(P, generator=torch.Generator().manual_seed(0))[:300].to("cuda:0")
    xq, wq = row_truth.in_8_bits(x[pick].cpu().double(), 1), row_truth.in_8_bits(w.cpu().double(), 128)
    _check(y[pick], xq, wq, b.cpu().double(), dtype, "y")


def test_kept_codes_are_autograds_to_watch():
    """Codes or exponents of a kept weight rewritten between the passes raise; saved-tensor hooks see what is kept."""
    from graspbalance_amd import fused_rows
    x, w, b, dy = (t.to("cuda:0") for t in _data(40, 130, 70, torch.float32))
    x.requires_grad_()
    for change in (lambda h: h.codes_t.view(torch.uint8).zero_(), lambda h: h.scales.add_(1)):
        held = fused_rows.Fp8Weight.quantize(w, input_gradients=True)
        parts = [t.clone() for t in (held.codes, held.scales, held.codes_t)]
        for h in (held, fused_rows.Fp8Weight(parts[0], parts[1], 130, parts[2])):
            y = fused_rows.fp8_linear(x, h, b)
            change(h)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, x, dy)
    held = fused_rows.Fp8Weight.quantize(w, input_gradients=True)
    for weight in (held, w):
        want, = torch.autograd.grad(fused_rows.fp8_linear(x, weight, b), x, dy)
        seen = []

        def unpack(t):
            seen.append(t)
            return t.to("cuda:0")
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
            y = fused_rows.fp8_linear(x, weight, b)
        got, = torch.autograd.grad(y, x, dy)
        assert torch.equal(got, want) and sum(t.numel() for t in seen) >= held.codes_t.numel() + held.scales.numel()


@pytest.mark.parametrize("rows,excess,needs_x", [(1 << 23, 0.99 * 2.0 ** -15, False), (1 << 25, 0.99 * 2.0 ** -17, True)])
def test_bias_gradient_of_many_rows(rows, excess, needs_x):
    """Equal terms 1 + excess lose their tail at every addition to a sum of 512 or more (there a lane's four rows are added
    first, hence the smaller excess), all in one direction: over 100 U of 2^-24 where a lane adds a thousand rows in fp32.
    The bound: at most 64 such additions, the workgroups' sums and the result rounded once.  Both ways through the kernels."""
    from graspbalance_amd import fused_rows
    x = torch.ones(rows, 1, device="cuda:0").requires_grad_(needs_x)
    bias = torch.zeros(128, device="cuda:0").requires_grad_()
    y = fused_rows.fp8_linear(x, fused_rows.Fp8Weight.quantize(torch.ones(128, 1, device="cuda:0"), input_gradients=True), bias)
    c = torch.tensor(1 + excess, device="cuda:0")
    db = torch.autograd.grad(y, [bias] + [x] * needs_x, c.expand_as(y))[0]
    total = float(c) * rows
    assert bool(((db.double() - total).abs() <= 68 * 2.0 ** -24 * total).all()), float((db.double() / total - 1).abs().max()) * 2 ** 24


@pytest.mark.parametrize("P,K,N", [((1 << 20) + 77, 4104, 8), ((1 << 25) + 5, 128, 130)])
def test_products_past_32_bits_of_elements(P, K, N):
    """Codes, rows and outputs behind 2^32 elements, in tiles and streamed: the first and last rows of y and dx; in tiles the last columns of dw too."""
    from graspbalance_amd import fused_rows
    g = torch.Generator(device="cuda:0").manual_seed(1)
    x, dy = (torch.randn(P, n, generator=g, device="cuda:0", dtype=torch.bfloat16) for n in (K, N))
    w = (torch.randn(N, K, generator=g, device="cuda:0") * (2.0 / K) ** 0.5).requires_grad_()
    y = fused_rows.fp8_linear(x.requires_grad_(), w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    wq = row_truth.in_8_bits(w.detach().cpu().double(), 128)
    for at in (slice(0, 150), slice(P - 150, P)):
        _check(y[at], row_truth.in_8_bits(x[at].detach().cpu().double(), 1), wq, None, torch.bfloat16, "y")
        _check(dx[at], row_truth.in_8_bits(dy[at].cpu().double(), 1), wq.t().contiguous(), None, torch.bfloat16, "dx")
    if K > 128:      # (the truth of every row of the last block of columns: a minute of the CPU for 2^25 of them)
        xq = row_truth.in_8_bits(x[:, (K - 1) // 128 * 128:].detach().cpu().double(), 1)
        _check(dw[:, -xq.shape[1]:], row_truth.in_8_bits(dy.cpu().double(), 1).t().contiguous(), xq.t().contiguous(), None,
               torch.float32, "dw", length=P)
