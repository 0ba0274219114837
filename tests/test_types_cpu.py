"""Types that a kernel would read wrongly are refused on the host, before anything is launched (no GPU: stand-ins that say
they are on one, and a library that records what reaches it)."""
import types

import pytest
import torch


class _Tensor:
    """A contiguous GPU tensor as far as a host check looks at one."""
    is_cuda, requires_grad = True, False
    device = torch.device("cuda:0")

    def __init__(self, dtype, *shape):
        self.dtype, self.shape = dtype, shape

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


@pytest.fixture
def launches(monkeypatch):
    """The names of what was launched; nothing is."""
    from graspbalance_amd import _lib
    seen = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or 0
    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(_lib, "current_stream", lambda device: None)
    monkeypatch.setattr(_lib, "device_ctx", lambda device: _lib._NO_CONTEXT)
    return seen


F, I = torch.float32, torch.int32
WRAPPERS = [("ball_query_wrapper", (1, 8, 8, 0.1, 4), (F, F, I)), ("group_points_wrapper", (1, 8, 8, 8, 4), (F, I, F)),
            ("group_points_grad_wrapper", (1, 8, 8, 8, 4), (F, I, F)), ("gather_points_wrapper", (1, 8, 8, 8), (F, I, F)),
            ("gather_points_grad_wrapper", (1, 8, 8, 8), (F, I, F)),
            ("furthest_point_sampling_wrapper", (1, 8, 8), (F, F, I)), ("three_nn_wrapper", (1, 8, 8), (F, F, F, I)),
            ("three_interpolate_wrapper", (1, 8, 8, 8), (F, I, F, F)),
            ("three_interpolate_grad_wrapper", (1, 8, 8, 8), (F, I, F, F))]


@pytest.mark.parametrize("name,sizes,kinds", WRAPPERS, ids=[w[0] for w in WRAPPERS])
def test_batch_wrappers_refuse_other_types(launches, name, sizes, kinds):
    from graspbalance_amd import pointnet2_batch_cuda as pb
    for at, kind in enumerate(kinds):
        for other in (torch.bfloat16, torch.float16, torch.float64, torch.int64, I if kind is F else F):
            tensors = [_Tensor(k, 8) for k in kinds]
            tensors[at] = _Tensor(other, 8)
            with pytest.raises(RuntimeError, match="float32"):
                getattr(pb, name)(*sizes, *tensors)
    assert launches == []
    getattr(pb, name)(*sizes, *[_Tensor(k, 8) for k in kinds])
    assert len(launches) == 1
