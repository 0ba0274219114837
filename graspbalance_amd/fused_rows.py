"""Channel-last row operators beside the BatchNorm stacks of fused_mlp (no reference counterpart): group norm with an
activation, dropout from a counter-based generator, products in 8-bit floats with a scale for each block of 128.

Rows are (..., C) tensors in fp32, bf16 or fp16 with the channels last, as everywhere on the fused path.  Kernels run on the
current stream of the tensors' device; workspaces come from torch's allocator inside the call, so that every captured graph
has its own.  CPU tensors raise, like every operator of this package.  Gradients are exact to rounding and repeat bit for
bit (no atomics); differentiating them again is refused, and so are operands of forward-mode differentiation.
"""
import ctypes
import functools

import torch
import torch.nn as nn
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .fused_mlp import _call, linear_bias

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # GB_T_*


def _s(t):
    return _lib.raw_stream(t.device)


def _refuse(what, why):
    raise RuntimeError("%s: %s" % (what, why))


def supports(t):
    """Whether the operators of this module take tensor t."""
    return t.is_cuda and t.dtype in _TYPES


def _rows_tensor(what, name, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(what, "CPU not supported (%s)" % name)
    if t.dtype not in _TYPES:
        _refuse(what, "%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))


def _like(what, name, t, x):
    """A tensor that goes with x element by element."""
    if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        _refuse(what, "%s must have the input's shape, type and device" % name)


def _channel_vector(what, name, t, n, x):
    """A per-channel parameter as contiguous fp32 (None stays None); its gradient comes back in its own type."""
    if t is None:
        return None
    if t.shape != (n,) or t.device != x.device or not t.is_floating_point():
        _refuse(what, "%s must be a float tensor of %d elements on the input's device" % (name, n))
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _rate(what, p, rng, x):
    """(q, rng) of a dropout rate: q / 65536 is the rate, rng an int64 pair on the device or a pair of ints."""
    if not 0.0 <= p <= 1.0:
        _refuse(what, "a dropout rate of %r is not in [0, 1]" % (p,))
    q = int(p * 65536 + 0.5)
    if q == 0:
        return 0, (0, 0)
    if isinstance(rng, torch.Tensor):
        if rng.shape != (2,) or rng.dtype != torch.int64 or rng.device != x.device or not rng.is_contiguous():
            _refuse(what, "rng must be an int64 tensor [seed, call] on the input's device, or a pair of ints")
        return q, rng
    try:
        seed, call = (int(v) for v in rng)
    except (TypeError, ValueError):
        _refuse(what, "rng must be an int64 tensor [seed, call] on the input's device, or a pair of ints")
    wrap = lambda v: (v + (1 << 63)) % (1 << 64) - (1 << 63)   # noqa: E731  (64 bits as C's signed type holds them)
    return q, (wrap(seed), wrap(call))


def _rng_args(rng):
    """(device pointer | None, seed, call) of a launch."""
    return (_lib.ptr(rng), 0, 0) if isinstance(rng, torch.Tensor) else (None, rng[0], rng[1])


def _grads(*tensors):
    """Whether a call goes through autograd: to be recorded for a backward pass, or because an operand carries a tangent of
    forward-mode differentiation, which the autograd functions refuse (a tangent must not vanish)."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _once(backward):
    """once_differentiable without its 3 - 5 us where no graph of the backward pass is being recorded."""
    guarded = once_differentiable(backward)

    def run(ctx, dy):
        return guarded(ctx, dy) if torch.is_grad_enabled() else backward(ctx, dy)
    return run


def _dropout(x, residual, q, rng, keep):
    """(y, the pair that was used | None)"""
    y = torch.empty_like(x)
    at, seed, call = _rng_args(rng)
    # the numbers' key is kept as it was used: the owner may write the next call's into rng before the backward pass
    used = torch.empty_like(rng) if keep and at is not None else None
    _call("gb_dropout", x.device, x.data_ptr(), _lib.ptr(residual), y.data_ptr(), x.numel(), _TYPES[x.dtype], q, at, seed, call,
          _lib.ptr(used), _s(x))
    return y, used


class _Dropout(Function):
    @staticmethod
    def forward(ctx, x, residual, q, rng):
        y, used = _dropout(x, residual, q, rng, True)
        ctx.q, ctx.rng, ctx.has_residual = q, None if used is not None else rng, residual is not None
        ctx.save_for_backward(*(() if used is None else (used,)))
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            dx, _ = _dropout(dy.contiguous(), None, ctx.q, ctx.saved_tensors[0] if ctx.rng is None else ctx.rng, False)
        return dx, dy if ctx.has_residual and ctx.needs_input_grad[1] else None, None, None


def dropout(x, p, rng, residual=None):
    """x with every element dropped (zero, whatever it held) with probability p and the others divided by 1 - p, plus
    `residual`.  p is taken to the nearest 65536th.  rng: [seed, call] - an int64 tensor on the device, which a captured
    graph reads at every replay, or two ints.  Element i (in the order of the contiguous tensor) is kept by number i of
    that pair alone (Philox4x32-10, include/graspbal.h gb_dropout): equal pairs drop equal places, pairs that differ in
    either number are independent.  Nothing of the mask is stored; the backward pass computes it again."""
    _rows_tensor("dropout", "x", x)
    q, rng = _rate("dropout", p, rng, x)
    if residual is not None:
        _like("dropout", "residual", residual, x)
    if q == 0:
        return x if residual is None else x + residual
    x, residual = x.contiguous(), None if residual is None else residual.contiguous()
    if not _grads(x, residual):
        return _dropout(x, residual, q, rng, False)[0]
    return _Dropout.apply(x, residual, q, rng)


class Dropout(nn.Module):
    """dropout() as a layer: owns its [seed, call] pair on the device as the buffer ``rng`` (saved with the module) and moves
    to the next call at every training forward - also at every replay of a captured one, and at a recomputed one: under
    activation checkpointing call dropout() with a pair of your own.  Without a seed, one is drawn from torch's CPU generator;
    ranks that draw the same one (or share their buffers) drop the same places of their own rows."""

    def __init__(self, p=0.5, seed=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            _refuse("Dropout", "a dropout rate of %r is not in [0, 1]" % (p,))
        self.p = p
        if seed is None:
            seed = int(torch.randint(0, 1 << 62, (1,)))
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))
        self.register_buffer("_next", torch.tensor([0, 1], dtype=torch.int64), persistent=False)

    def extra_repr(self):
        return "p=%g" % self.p

    def take(self):
        """The pair for one call; the next call gets another.  (A copy: what the caller's kernels read later is not
        moved.)"""
        used = self.rng.clone()
        self.rng.add_(self._next)
        return used

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else x + residual
        return dropout(x, self.p, self.take(), residual)


def _norm_struct(x, weight, bias, residual, offsets, stats, at, used, seed, call, cfg):
    """GbGroupNorm of one call, in the order of its fields."""
    samples, groups, eps, act, slope, q = cfg
    C, at_stats = x.shape[-1], stats.data_ptr()
    return _lib.GroupNorm(x.data_ptr(), _lib.ptr(residual), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(offsets), at_stats,
                          at_stats + 4 * samples * groups, at, used, x.numel() // C, seed, call, samples, C, groups,
                          _TYPES[x.dtype], act, q, eps, slope)


def _norm(x, weight, bias, residual, offsets, cfg, rng, keep):
    """(y, statistics, the pair that was used | None)"""
    dev = x.device
    samples, groups = cfg[:2]
    y = torch.empty_like(x)
    stats = torch.empty((2, samples, groups), dtype=torch.float32, device=dev)
    at, seed, call = _rng_args(rng)
    used = torch.empty_like(rng) if keep and at is not None else None
    n = _norm_struct(x, weight, bias, residual, offsets, stats, at, _lib.ptr(used), seed, call, cfg)
    size = _norm_workspace_bytes(n.rows, samples, n.channels, groups, n.dtype, n.act, n.q, offsets is not None, 0)
    ws = _bytes(size, dev)
    _call("gb_group_norm_fwd", dev, ctypes.byref(n), y.data_ptr(), _lib.ptr(ws), size, _s(x))
    return y, stats, used


class _GroupNormAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, offsets, cfg, rng):
        y, stats, used = _norm(x, weight, bias, residual, offsets, cfg, rng, True)
        # (without an activation the gradient does not depend on the residual)
        ctx.save_for_backward(x, weight, bias, residual if cfg[3] else None, offsets, stats, used)
        ctx.cfg, ctx.rng = cfg, None if used is not None else rng
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, bias, residual, offsets, stats, used = ctx.saved_tensors
        samples, groups, _, act, _, q = cfg = ctx.cfg
        dev, C = x.device, x.shape[-1]
        dy = dy.contiguous()
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = torch.empty_like(x)
        # (the residual's gradient is dy itself where nothing stands between it and y)
        plain = act == 0 and q == 0 and offsets is None
        dres = torch.empty_like(x) if need_r and not plain else None
        make = torch.empty if x.numel() else torch.zeros
        dw = make(C, dtype=torch.float32, device=dev) if need_w else None
        db = make(C, dtype=torch.float32, device=dev) if need_b else None
        at, seed, call = _rng_args(used if ctx.rng is None else ctx.rng)
        n = _norm_struct(x, weight, bias, residual, offsets, stats, at, None, seed, call, cfg)
        size = _norm_workspace_bytes(n.rows, samples, C, groups, n.dtype, act, q, offsets is not None, 1)
        ws = _bytes(size, dev)
        _call("gb_group_norm_bwd", dev, ctypes.byref(n), dy.data_ptr(), dx.data_ptr(), _lib.ptr(dres), _lib.ptr(dw),
              _lib.ptr(db), _lib.ptr(ws), size, _s(x))
        return dx if need_x else None, dw, db, (dy if plain else dres) if need_r else None, None, None, None


@functools.lru_cache(maxsize=1024)
def _norm_workspace_bytes(rows, samples, channels, groups, dtype, act, q, packed, backward):
    n = _lib.GroupNorm(rows=rows, samples=samples, channels=channels, groups=groups, dtype=dtype, act=act, q=q,
                       offsets=8 if packed else None)
    size = ctypes.c_longlong()
    _lib.check(_lib.lib().gb_group_norm_workspace(ctypes.byref(n), backward, ctypes.byref(size)), "group_norm_act")
    return size.value


def _bytes(size, dev):
    return torch.empty(size, dtype=torch.uint8, device=dev) if size else None


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", negative_slope=0.01, residual=None,
                   offsets=None, dropout_p=0.0, rng=None):
    """act(group_norm(x) * weight + bias + residual) on channel-last rows, then dropout when dropout_p > 0, in one pass.

    x: (B, ..., C), every x[b] a sample of its own; or with `offsets` (S + 1 ascending row numbers, int64 on the device)
    packed rows (R, C), sample s being rows offsets[s] up to offsets[s + 1] - none, where they are equal.  Rows outside
    every sample give zeros and get zero gradients.  Statistics are taken over all rows of a sample and the C / num_groups
    channels of a group, biased, as nn.GroupNorm does; a single element per group is legal and gives act(bias).
    act: "none", "relu", "leaky_relu" (negative_slope), "silu", "gelu" (the erf form).  weight, bias: (C,) or None.
    dropout_p, rng: as in dropout().  -> like x."""
    what = "group_norm_act"
    _rows_tensor(what, "x", x)
    if x.dim() < 2:
        _refuse(what, "x must be (samples, ..., channels)")
    C, groups = x.shape[-1], int(num_groups)
    if groups <= 0 or C <= 0 or C % groups:
        _refuse(what, "%d channels do not make %d groups" % (C, groups))
    if act not in _lib.ACTIVATIONS:
        _refuse(what, "act must be one of %s" % ", ".join(_lib.ACTIVATIONS))
    if not eps >= 0:
        _refuse(what, "eps must not be negative")
    if offsets is not None:
        if x.dim() != 2:
            _refuse(what, "packed rows must be (rows, channels)")
        if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.numel() < 2 \
                or offsets.dtype != torch.int64 or offsets.device != x.device:
            _refuse(what, "offsets must be an int64 tensor of samples + 1 row numbers on the input's device")
        offsets = offsets.contiguous()
        samples = offsets.numel() - 1
    else:
        samples = max(1, x.shape[0])
    if residual is not None:
        _like(what, "residual", residual, x)
        residual = residual.contiguous()
    q, rng = _rate(what, dropout_p, rng, x)
    x = x.contiguous()
    weight, bias = _channel_vector(what, "weight", weight, C, x), _channel_vector(what, "bias", bias, C, x)
    cfg = (samples, groups, float(eps), _lib.ACTIVATIONS[act], float(negative_slope), q)
    if not _grads(x, weight, bias, residual):
        return _norm(x, weight, bias, residual, offsets, cfg, rng, False)[0]
    return _GroupNormAct.apply(x, weight, bias, residual, offsets, cfg, rng)


# ---- products in 8-bit floats -----------------------------------------------------------------------------------------

_WS_COLSUM, _WS_WGRAD, _WS_LINEAR, _KEEP, _SUM = 0, 1, 4, 1, 2     # GB_FP8_*
_TRANSPOSED, _SHORT_SUMS = 1, 2


def _up(n, m):
    return (n + m - 1) // m * m


def _row_bytes(P, K):
    """(bytes of the codes of rows (P, K), bytes of their exponents): kept one behind the other in one allocation."""
    Kp = _up(K, 128)
    return P * Kp, P * _up(Kp // 128, 4)


def _quantise_rows(x2):
    """(codes, scales) of rows (P, K)."""
    P, K = x2.shape
    n, m = _row_bytes(P, K)
    both = torch.empty(n + m, dtype=torch.uint8, device=x2.device)
    _quantise_rows_to(x2, both.data_ptr(), None, None, 0)
    return both[:n].view(P, -1), both[n:].view(P, -1)


def _quantise_rows_to(x2, at, sums, ws, size):
    P, K = x2.shape
    _call("gb_fp8_quant_rows", x2.device, x2.data_ptr(), _TYPES[x2.dtype], P, K, at, at + _row_bytes(P, K)[0], _lib.ptr(sums), ws,
          size, _s(x2))


def _product_to(x2, y, w, w_scales, flags, N, bias, keep_at, sums, ws, size):
    """gb_fp8_linear: y (P, N) of rows x2 and a weight's codes; keep_at: where x2's codes and exponents go, or None."""
    P, K = x2.shape
    _call("gb_fp8_linear", x2.device, x2.data_ptr(), _TYPES[x2.dtype], P, K, w, w_scales, flags, N, _lib.ptr(bias),
          y.data_ptr(), keep_at, None if keep_at is None else keep_at + _row_bytes(P, K)[0], _lib.ptr(sums), ws, size, _s(x2))


@functools.lru_cache(maxsize=1024)
def _fp8_workspace_bytes(what, P, N, K):
    size = ctypes.c_longlong()
    _lib.check(_lib.lib().gb_fp8_workspace(what, P, N, K, ctypes.byref(size)), "fp8_linear")
    return size.value


class _Codes:
    """Addresses of a weight's codes, transposed codes (None where nobody asked) and exponents, and what holds them."""
    __slots__ = ("N", "K", "codes", "codes_t", "scales", "held")

    @classmethod
    def of(cls, weight):
        """Of an Fp8Weight."""
        c = cls()
        c.N, c.K, c.held = weight.out_features, weight.in_features, (weight.codes, weight.scales, weight.codes_t)
        c.codes, c.scales, c.codes_t = (_lib.ptr(t) for t in c.held)
        return c

    @classmethod
    def quantise(cls, w, transposed):
        """Of a float weight (N, K), in one allocation (held) in that order."""
        c = cls()
        c.N, c.K = w.shape
        n, m = c.N * _up(c.K, 128), c.K * _up(c.N, 128) if transposed else 0
        c.held = torch.empty(n + m + _up(c.N, 128) // 128 * (_up(c.K, 128) // 128), dtype=torch.uint8, device=w.device)
        c.codes = c.held.data_ptr()
        c.codes_t, c.scales = c.codes + n if transposed else None, c.codes + n + m
        _call("gb_fp8_quant_weight", w.device, w.data_ptr(), _TYPES[w.dtype], c.N, c.K, c.codes, c.codes_t, c.scales, _s(w))
        return c

    def for_backward(self):
        """What the backward pass reads of it, as tensors for autograd to keep (and to watch)."""
        return (self.held,) if isinstance(self.held, torch.Tensor) else (self.held[2], self.held[1])

    @staticmethod
    def of_backward(kept, N, K):
        """(address of the transposed codes, of the exponents) in what for_backward gave."""
        if len(kept) == 2:
            return kept[0].data_ptr(), kept[1].data_ptr()
        n, m = N * _up(K, 128), K * _up(N, 128)
        return kept[0].data_ptr() + n, kept[0].data_ptr() + n + m


class Fp8Weight:
    """A weight (out_features, in_features) held in 8 bits for fp8_linear: ``codes`` (out_features, in_features up to whole
    blocks of 128, zeros behind) as torch.float8_e4m3fn, ``scales`` one biased exponent (1 .. 254; scale 2^(byte - 127)) per
    block of 128 x 128 as uint8, and for gradients of the input ``codes_t`` (in_features, out_features up to whole blocks).
    Make one from a float weight with ``Fp8Weight.quantize``."""

    def __init__(self, codes, scales, in_features, codes_t=None):
        what = "Fp8Weight"
        N, K = codes.shape[0], int(in_features)
        for name, t, shape, types in (
                ("codes", codes, (N, _up(K, 128)), (torch.float8_e4m3fn, torch.uint8)),
                ("scales", scales, (_up(N, 128) // 128, _up(K, 128) // 128), (torch.uint8,)),
                ("codes_t", codes_t, (K, _up(N, 128)), (torch.float8_e4m3fn, torch.uint8))):
            if t is None and name == "codes_t":
                continue
            if not t.is_cuda:
                _refuse(what, "CPU not supported (%s)" % name)
            if N <= 0 or K <= 0 or t.shape != shape or t.dtype not in types or t.device != codes.device \
                    or not t.is_contiguous() or (name != "scales" and t.data_ptr() % 16):
                _refuse(what, "%s must be a contiguous, 16-byte aligned %s tensor of %s" % (name, types[0], shape))
        self.codes, self.scales, self.codes_t = codes, scales, codes_t
        self.in_features, self.out_features = K, N

    @classmethod
    def quantize(cls, weight, input_gradients=False):
        """From a float weight (out_features, in_features); input_gradients: also what fp8_linear's backward pass needs."""
        w = _fp8_weight_tensor("Fp8Weight", weight.detach()).contiguous()
        N, K = w.shape
        held = _Codes.quantise(w, input_gradients).held
        n, m = N * _up(K, 128), K * _up(N, 128) if input_gradients else 0
        return cls(held[:n].view(N, -1).view(torch.float8_e4m3fn), held[n + m:].view(_up(N, 128) // 128, -1), K,
                   held[n:n + m].view(K, -1).view(torch.float8_e4m3fn) if input_gradients else None)


def _fp8_weight_tensor(what, w):
    _rows_tensor(what, "weight", w)
    if w.dim() < 2 or w.numel() == 0 or any(n != 1 for n in w.shape[2:]):
        _refuse(what, "weight must be (out_features, in_features) or that of a 1x1 convolution")
    return w.view(w.shape[0], w.shape[1]) if w.dim() > 2 else w


def _fp8_forward(x, weight, bias, flags, need_x, keep):
    """(y, the weight's _Codes, x's codes and exponents | None)"""
    dev = x.device
    P, K = x.shape
    w = _Codes.of(weight) if isinstance(weight, Fp8Weight) else _Codes.quantise(weight, need_x)
    if need_x and w.codes_t is None:
        _refuse("fp8_linear", "gradients of the input need Fp8Weight.quantize(weight, input_gradients=True)")
    y = torch.empty((P, w.N), dtype=x.dtype, device=dev)
    kept = torch.empty(sum(_row_bytes(P, K)), dtype=torch.uint8, device=dev) if keep else None
    size = _fp8_workspace_bytes(_WS_LINEAR + _KEEP * keep, P, w.N, K)
    ws = _bytes(size, dev)
    _product_to(x, y, w.codes, w.scales, flags, w.N, bias, _lib.ptr(kept), None, _lib.ptr(ws), size)
    return y, w, kept


class _Fp8Linear(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, held, flags):
        need_x, need_w = ctx.needs_input_grad[:2]
        y, w, kept = _fp8_forward(x, weight if held is None else held, bias, flags, need_x, need_w)
        # one byte per element of x stays for the backward pass
        ctx.save_for_backward(kept, *(w.for_backward() if need_x else ()))
        ctx.dims, ctx.flags = (w.N, w.K, None if held is not None else weight.dtype), flags
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        kept, *codes_w = ctx.saved_tensors
        N, K, wtype = ctx.dims
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = dy.contiguous()
        dev, P = dy.device, dy.shape[0]
        # dy's codes, then a workspace for one kernel after the other
        codes = sum(_row_bytes(P, N)) if need_w or not need_x else 0
        first = _fp8_workspace_bytes(_WS_LINEAR + _KEEP * (codes > 0) + _SUM * need_b, P, K, N) if need_x else \
            _fp8_workspace_bytes(_WS_COLSUM, P, N, 1) if need_b else 0
        second = _fp8_workspace_bytes(_WS_WGRAD, P, N, K) if need_w else 0
        room = _up(codes, 16)
        scratch = torch.empty(room + max(first, second), dtype=torch.uint8, device=dev)
        at = scratch.data_ptr()
        dx = dw = None
        db = torch.empty(N, dtype=torch.float32, device=dev) if need_b else None
        if need_x:
            dx = torch.empty((P, K), dtype=dy.dtype, device=dev)
            _product_to(dy, dx, *_Codes.of_backward(codes_w, N, K), ctx.flags | _TRANSPOSED, K, None, at if codes else None, db,
                        at + room, first)
        else:
            _quantise_rows_to(dy, at, db, at + room, first)
        if need_w:
            dw = torch.empty((N, K), dtype=torch.float32, device=dev)
            x_at = kept.data_ptr()
            _call("gb_fp8_wgrad", dev, at, at + _row_bytes(P, N)[0], x_at, x_at + _row_bytes(P, K)[0], dw.data_ptr(), P, N, K,
                  at + room, second, _s(dy))
            dw = dw if wtype == torch.float32 else dw.to(wtype)
        return dx, dw, db, None, None


def fp8_linear(x, weight, bias=None, short_sums=False):
    """x weight^T + bias with both operands in 8-bit floats (e4m3) under power-of-two scales: x (..., in_features) has one
    per 128 elements of a row, weight one per 128 x 128.  weight: (out_features, in_features) - a parameter, or that of a
    1x1 convolution - quantised in the call, or an Fp8Weight that is kept.  -> (..., out_features) like x; sums in fp32.

    Gradients are those of the products with the quantisers passed straight through: the incoming gradient is quantised
    like x, dx and dweight are products of the 8-bit operands, dbias sums the gradient as it came.  An element of x or
    weight that is not finite makes every output it takes part in NaN.  The codes are multiplied as bf16, which holds them
    exactly (what rounds to 2^128 counts as infinite, what is below 2^-126 as zero), with fp32 sums.  short_sums: for 16-bit
    x, y and dx come from the 8-bit matrix instructions instead: faster where the matrix cores bind, but a step of 64 or 128
    products keeps only about 14 bits below its largest (measured 5e-5 of the result's norm); fp32 x is computed as ever."""
    what = "fp8_linear"
    _rows_tensor(what, "x", x)
    held = weight if isinstance(weight, Fp8Weight) else None
    if held is None:
        weight = _fp8_weight_tensor(what, weight)
        N, K = weight.shape
        where = weight.device
    else:
        N, K, where = held.out_features, held.in_features, held.codes.device
    if where != x.device:
        _refuse(what, "weight must be on the input's device")
    if x.dim() < 1 or x.shape[-1] != K:
        _refuse(what, "x must be (..., %d)" % K)
    bias = _channel_vector(what, "bias", bias, N, x)
    rows = (x if x.dim() == 2 else x.reshape(-1, K)).contiguous()
    weight = None if held is not None else weight.contiguous()
    flags = _SHORT_SUMS if short_sums else 0
    if _grads(x, weight, bias):
        y = _Fp8Linear.apply(rows, weight, bias, held, flags)
    else:
        y = _fp8_forward(rows, weight if held is None else held, bias, flags, False, False)[0]
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (N,))


# ---- conv + group norm blocks ------------------------------------------------------------------------------------------

def activation_of(module):
    """(name, slope) of an activation module as group_norm_act takes it (None: no activation); None for any other."""
    if module is None or isinstance(module, nn.Identity):
        return "none", 0.0
    if isinstance(module, nn.ReLU):
        return "relu", 0.0
    if isinstance(module, nn.LeakyReLU):
        return "leaky_relu", float(module.negative_slope)
    if isinstance(module, nn.SiLU):
        return "silu", 0.0
    if isinstance(module, nn.GELU) and module.approximate == "none":
        return "gelu", 0.0
    return None


def conv_gn_act(x, conv, gn, act=("none", 0.0), fp8=False, residual=None, dropout=None):
    """A 1x1 ``conv`` (with or without bias), ``gn`` (nn.GroupNorm), an activation (activation_of) and optionally a Dropout on
    channel-last rows x (samples, rows, Cin) -> (samples, rows, Cout), with the modules' own parameters; residual joins
    in front of the activation.  fp8: the product in 8-bit floats; else x and the weight must be fp32 (linear_bias)."""
    W = conv.weight.view(conv.weight.shape[0], -1)
    if fp8:
        y = fp8_linear(x, W, conv.bias)
    else:
        y = linear_bias(x.reshape(-1, x.shape[-1]), conv).view(x.shape[:-1] + (W.shape[0],))
    drop = dropout is not None and dropout.training and dropout.p > 0
    return group_norm_act(y, gn.num_groups, gn.weight, gn.bias, gn.eps, act[0], act[1], residual,
                          dropout_p=dropout.p if drop else 0.0, rng=dropout.take() if drop else None)
