"""Channel-last row operators without a GPU: refusals (Python and C-ABI) and the generator of their oracle."""
import ctypes

import numpy as np
import pytest
import torch

from tests import row_truth


def test_generator_of_the_oracle_gives_the_published_vectors():
    """The known answers of Philox4x32-10 that go with the paper (counter, key all zeros / all ones / digits of pi)."""
    def run(c, k):
        return [int(v) for v in row_truth.philox(np.array([c], np.uint64), k)[0]]
    assert run([0] * 4, (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert run([0xffffffff] * 4, (0xffffffff, 0xffffffff)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert run([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], (0xa4093822, 0x299f31d0)) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_cpu_tensors_raise():
    from graspbalance_amd import fused_rows
    x = torch.randn(4, 16)
    with pytest.raises(RuntimeError, match="CPU not supported"):
        fused_rows.group_norm_act(x, 4)
    with pytest.raises(RuntimeError, match="CPU not supported"):
        fused_rows.dropout(x, 0.5, (1, 2))


def test_bad_rates_raise():
    from graspbalance_amd import fused_rows
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(RuntimeError, match="not in"):
            fused_rows.Dropout(p)


def _norm(**kw):
    from graspbalance_amd import _lib
    base = dict(x=64, weight=None, bias=None, mean=64, rstd=64, rows=8, samples=2, channels=16, groups=4, dtype=0, act=0, q=0,
                eps=1e-5)
    base.update(kw)
    return _lib.GroupNorm(**base)


@pytest.mark.parametrize("kw,rc", [
    ({"groups": 3}, -1), ({"groups": 0}, -1), ({"channels": 0}, -1), ({"samples": 0}, -1), ({"rows": -1}, -1),
    ({"rows": 7}, -1), ({"dtype": 3}, -1), ({"act": 5}, -1), ({"act": -1}, -1), ({"q": 65537}, -1), ({"q": -1}, -1),
    ({"eps": -1.0}, -1), ({"eps": float("nan")}, -1), ({"offsets": 4}, -1), ({"rng": 12}, -1), ({"used": 12}, -1),
    ({"channels": 4104, "groups": 1}, -3), ({"channels": 1025, "groups": 1}, -3), ({"channels": 2050, "groups": 1}, -3),
    ({"samples": 65535, "rows": 65535}, -3)])
def test_norm_refuses_on_the_host(kw, rc):
    from graspbalance_amd import _lib
    L, n = _lib.lib(), _norm(**kw)
    size = ctypes.c_longlong(-5)
    assert L.gb_group_norm_workspace(ctypes.byref(n), 0, ctypes.byref(size)) == rc and size.value == -5
    assert L.gb_group_norm_fwd(ctypes.byref(n), 64, 64, 1 << 20, None) == rc
    assert L.gb_group_norm_bwd(ctypes.byref(n), 64, 64, None, None, None, 64, 1 << 20, None) == rc


def test_norm_refuses_missing_pointers_and_small_workspaces():
    from graspbalance_amd import _lib
    L = _lib.lib()
    big = dict(rows=1 << 16, samples=1, channels=256, groups=8)
    for kw in ({"x": None}, {"mean": None}, {"rstd": None}):
        n = _norm(**kw)
        assert L.gb_group_norm_fwd(ctypes.byref(n), 64, 64, 1 << 30, None) == -1
        assert L.gb_group_norm_bwd(ctypes.byref(n), 64, 64, None, None, None, 64, 1 << 30, None) == -1
    n = _norm(**big)
    assert L.gb_group_norm_fwd(None, 64, 64, 1 << 30, None) == -1
    assert L.gb_group_norm_fwd(ctypes.byref(n), None, 64, 1 << 30, None) == -1
    for backward in (0, 1):
        size = ctypes.c_longlong()
        assert L.gb_group_norm_workspace(ctypes.byref(n), backward, ctypes.byref(size)) == 0 and size.value > 0
        assert L.gb_group_norm_workspace(ctypes.byref(n), backward, None) == -1
        for ws, have in ((64, size.value - 1), (None, size.value), (72, size.value)):
            if backward:
                assert L.gb_group_norm_bwd(ctypes.byref(n), 64, 64, None, None, None, ws, have, None) == -1
            else:
                assert L.gb_group_norm_fwd(ctypes.byref(n), 64, ws, have, None) == -1
    assert L.gb_group_norm_bwd(ctypes.byref(n), None, 64, None, None, None, 64, 1 << 30, None) == -1
    empty = _norm(rows=0, x=None)
    assert L.gb_group_norm_fwd(ctypes.byref(empty), None, None, 0, None) == 0     # nothing to do: nothing is launched


def test_dropout_refuses_on_the_host():
    from graspbalance_amd import _lib
    L = _lib.lib()
    ok = [64, None, 64, 8, 0, 100, None, 1, 2, None, None]
    for at, bad in ((0, None), (2, None), (3, -1), (4, 3), (4, -1), (5, -1), (5, 65537), (6, 12), (9, 12)):
        args = list(ok)
        args[at] = bad
        assert L.gb_dropout(*args) == -1, (at, bad)
    assert L.gb_dropout(None, None, None, 0, 0, 100, None, 1, 2, None, None) == 0


def test_fp8_cpu_tensors_raise():
    from graspbalance_amd import fused_rows
    with pytest.raises(RuntimeError, match="CPU not supported"):
        fused_rows.fp8_linear(torch.randn(4, 16), torch.randn(8, 16))
    with pytest.raises(RuntimeError, match="CPU not supported"):
        fused_rows.Fp8Weight.quantize(torch.randn(8, 16))


def test_fp8_refuses_on_the_host():
    from graspbalance_amd import _lib
    L = _lib.lib()
    size = ctypes.c_longlong(-5)

    def refused(fn, ok, bad):
        for at, value, rc in bad:
            args = list(ok)
            args[at] = value
            assert fn(*args) == rc, (fn.__name__, at, value)
    refused(L.gb_fp8_workspace, [1, 8, 8, 8, ctypes.byref(size)],
            [(0, 2, -1), (0, 3, -1), (0, 8, -1), (0, -1, -1), (1, -1, -1), (2, 0, -1), (3, 0, -1), (4, None, -1), (1, 1 << 41, -3), (2, 1 << 23, -3)])
    assert size.value == -5
    refused(L.gb_fp8_quant_rows, [64, 0, 8, 8, 64, 64, None, None, 0, None],
            [(0, None, -1), (1, 3, -1), (2, -1, -1), (3, 0, -1), (4, None, -1), (4, 72, -1), (5, None, -1), (5, 68, -1),
             (3, 1 << 23, -3), (2, 1 << 41, -3), (6, 64, -1)])
    refused(L.gb_fp8_quant_weight, [64, 0, 8, 8, 64, 64, 64, None],
            [(0, None, -1), (1, 9, -1), (2, 0, -1), (3, -2, -1), (4, None, -1), (4, 65, -1), (5, 72, -1), (6, None, -1),
             (2, 1 << 23, -3)])
    ok = [64, 0, 8, 8, 64, 64, 0, 8, None, 64, None, None, None, 64, 1 << 20, None]
    refused(L.gb_fp8_linear, ok,
            [(0, None, -1), (1, 5, -1), (2, -1, -1), (3, 0, -1), (4, None, -1), (4, 72, -1), (5, None, -1), (7, 0, -1), (9, None, -1),
             (10, 64, -1), (11, 64, -1), (13, 72, -1), (3, 1 << 23, -3), (7, 1 << 23, -3), (2, 1 << 41, -3)])
    # a shape whose codes need room: none, too little, and room that is not needed where the caller keeps the codes
    big = list(ok)
    big[2], big[3], big[7] = 1000, 1024, 1024
    assert L.gb_fp8_workspace(4, 1000, 1024, 1024, ctypes.byref(size)) == 0 and size.value == 1000 * (1024 + 8)
    refused(L.gb_fp8_linear, big, [(13, None, -1), (14, size.value - 1, -1)])
    assert L.gb_fp8_workspace(5, 1000, 1024, 1024, ctypes.byref(size)) == 0 and size.value == 0
    big[12] = 64      # column sums
    assert L.gb_fp8_workspace(6, 1000, 1024, 1024, ctypes.byref(size)) == 0 and size.value > 1000 * (1024 + 8)
    refused(L.gb_fp8_linear, big, [(14, size.value - 1, -1)])
    refused(L.gb_fp8_wgrad, [64, 64, 64, 64, 64, 8, 8, 8, None, 0, None],
            [(0, None, -1), (0, 72, -1), (1, None, -1), (2, None, -1), (2, 72, -1), (3, None, -1), (4, None, -1), (5, -1, -1),
             (6, 0, -1), (7, 0, -1), (7, 1 << 23, -3), (5, 100000, -1)])
    assert L.gb_fp8_linear(None, 0, 0, 8, None, None, 0, 8, None, None, None, None, None, None, 0, None) == 0
    assert L.gb_fp8_workspace(0, 100, 30, 1, ctypes.byref(size)) == 0 and size.value > 0 and size.value % (30 * 4) == 0


def test_the_oracle_of_8_bits_agrees_with_torchs_cast():
    """Codes of the oracle against torch's own float8_e4m3fn on values inside its range."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 256, generator=g) * torch.exp(3 * torch.randn(64, 256, generator=g))
    got = row_truth.in_8_bits(x.double(), 1)
    blocks = x.view(64, 2, 128)
    scale = got.new_ones(64, 2, 1)
    for i in range(64):
        for j in range(2):
            e = -126
            while blocks[i, j].abs().max().item() > 448 * 2.0 ** e:
                e += 1
            scale[i, j] = 2.0 ** e
    want = (blocks / scale.float()).to(torch.float8_e4m3fn).double() * scale
    assert torch.equal(got, want.view(64, 256))


def test_fp8_refuses_unknown_flags():
    from graspbalance_amd import _lib
    for dtype in (0, 1, 2):
        for flags in (4, 8, -1, 1 << 20):
            assert _lib.lib().gb_fp8_linear(64, dtype, 8, 8, 64, 64, flags, 8, None, 64, None, None, None, 64, 1 << 20, None) == -1
        for flags in (0, 1, 2, 3):      # (no rows: nothing is launched)
            assert _lib.lib().gb_fp8_linear(None, dtype, 0, 8, None, None, flags, 8, None, None, None, None, None, None, 0, None) == 0
