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


SIXTEEN = (torch.bfloat16, torch.float16)


@pytest.mark.parametrize("dtype", SIXTEEN + (torch.float64,))
def test_fused_rows_of_other_types_are_refused(dtype):
    """Every entry of the channel-last path that hands an address to an fp32 kernel."""
    import torch.nn as nn
    from graspbalance_amd import fused_mlp, fused_rows
    xyz, f, idx = torch.randn(1, 8, 3), torch.randn(1, 8, 4), torch.zeros(1, 8, 2, dtype=torch.int32)
    rows, odd = torch.randn(8, 4), torch.randn(8, 4).to(dtype)
    conv, bn, gn = nn.Conv1d(4, 4, 1, bias=False), nn.BatchNorm1d(4), nn.GroupNorm(2, 4)
    conv16, bn16 = nn.Conv1d(4, 4, 1, bias=False).to(dtype), nn.BatchNorm1d(4).to(dtype)
    geo = type("Geo", (), dict(xyz=xyz, centres=xyz, idx=idx, b=1, n=8, m=8, ns=2))
    agg = nn.Conv2d(7, 4, 1, bias=False)
    weight = torch.rand(1, 8, 3)
    for call in (lambda: fused_mlp.group_concat_cl(xyz, xyz, idx, f.to(dtype)),
                 lambda: fused_mlp.group_concat_cl(xyz.to(dtype), xyz, idx, f),
                 lambda: fused_mlp.group_concat_cl(xyz, xyz.to(dtype), idx, f),
                 lambda: fused_mlp.group_concat_cl(xyz, xyz, idx, None, mode=2, rot=torch.eye(3).expand(1, 8, 3, 3).to(dtype)),
                 lambda: fused_mlp.interp_concat_cl(f.to(dtype), idx, weight),
                 lambda: fused_mlp.interp_concat_cl(f, idx, weight.to(dtype)),
                 lambda: fused_mlp.interp_concat_cl(f, idx, weight, f.to(dtype)),
                 lambda: fused_mlp.linear_bias(odd, conv), lambda: fused_mlp.linear_bias(rows, conv16),
                 lambda: fused_mlp.conv_bn_act(odd, conv, bn), lambda: fused_mlp.conv_bn_act(rows, conv16, bn),
                 lambda: fused_mlp.conv_bn_act(rows, conv, bn16), lambda: fused_mlp.conv_bn_act(rows, conv, bn, residual=odd),
                 lambda: fused_mlp.conv_bn_act_chain(rows, [(conv, bn), (conv16, bn)]),
                 lambda: fused_mlp.LocalGeometry(xyz.to(dtype), xyz, idx), lambda: fused_mlp.LocalGeometry(xyz, xyz.to(dtype), idx),
                 lambda: fused_mlp.local_agg_pool(f.reshape(8, 4).to(dtype), agg, bn, geo),
                 lambda: fused_mlp.local_agg_pool(f.reshape(8, 4), agg, bn16, geo),
                 lambda: fused_rows.conv_gn_act(odd.unsqueeze(0), conv, gn), lambda: fused_rows.conv_gn_act(rows.unsqueeze(0), conv16, gn)):
        with pytest.raises(RuntimeError, match="must be float32"):
            call()


def test_rows_and_weight_have_to_match():
    import torch.nn as nn
    from graspbalance_amd import fused_mlp
    with pytest.raises(RuntimeError, match="input channels"):
        fused_mlp.linear_bias(torch.randn(8, 5), nn.Conv1d(4, 4, 1))
    with pytest.raises(RuntimeError, match="input channels"):
        fused_mlp.linear_bias(torch.randn(8, 4), nn.Conv1d(4, 4, 1, groups=2))


@pytest.mark.parametrize("norm", ["bn", "gn"])
@pytest.mark.parametrize("dtype", SIXTEEN)
def test_blocks_take_fp32_features_alone(launches, norm, dtype):
    """A block's fused path is for fp32 features; 16-bit ones reach the grouping's own check, and nothing of theirs is launched."""
    from graspbalance_amd.drp import InvResMLP
    blk = InvResMLP(in_channels=32, aggr_args={'feature_type': 'dp_fj', "reduction": 'max'},
                    norm_args={'norm': 'gn', 'num_groups': 4} if norm == "gn" else {'norm': 'bn'}, act_args={'act': 'relu'},
                    group_args={'NAME': 'ballquery', 'radius': 0.1, 'nsample': 16}, conv_args={'order': 'conv-norm-act'},
                    expansion=4, use_res=True)
    assert blk._fused_on(_Tensor(torch.float32, 1, 32, 64)) and not blk._fused_on(_Tensor(dtype, 1, 32, 64))
    from graspbalance_amd import pointnet2_batch_cuda as pb
    with pytest.raises(RuntimeError, match="float32"):
        pb.group_points_wrapper(1, 32, 64, 64, 16, _Tensor(dtype, 1, 32, 64), _Tensor(torch.int32, 1, 64, 16), _Tensor(torch.float32, 1, 32, 64, 16))
    assert launches == []


@pytest.mark.parametrize("norm", ["bn", "gn"])
@pytest.mark.parametrize("extra", [{'groups': 3}, {'padding': 1}, {'stride': 1}, {'padding': 'same'}, {}], ids=str)
def test_blocks_fuse_plain_products_alone(norm, extra):
    """Grouped or padded 1x1 convolutions are no product on rows: such a block runs its modules."""
    from graspbalance_amd.drp import InvResMLP
    blk = InvResMLP(in_channels=24, aggr_args={'feature_type': 'dp_fj', "reduction": 'max'},
                    norm_args={'norm': 'gn', 'num_groups': 3} if norm == "gn" else {'norm': 'bn'}, act_args={'act': 'relu'},
                    group_args={'NAME': 'ballquery', 'radius': 0.1, 'nsample': 16}, conv_args={'order': 'conv-norm-act', **extra},
                    expansion=4, use_res=True)
    fused = extra in ({}, {'stride': 1}, {'padding': 'same'})
    assert (blk.fusable() or blk.fusable_gn()) is fused and blk._fused_on(_Tensor(torch.float32, 1, 24, 64)) is fused
