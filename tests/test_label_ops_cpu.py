"""Refusals of group_norm_act and clip_grads_ that need no GPU, at the Python and at the C boundary; the layout rule of channels-last
operands."""
from array import array

import pytest
import torch

from image_segmentation_amd import GroupNormAct, LoRAGradReducer, _C, clip_grad_norm_, clip_grads_, group_norm_act, ops


def test_cpu_tensors_are_refused():
    with pytest.raises(_C.LsamError, match="MI355X only"):
        group_norm_act(torch.zeros(1, 8, 2, 2), 2)
    with pytest.raises(_C.LsamError, match="no CPU fallback"):
        clip_grads_([torch.zeros(3)], 1.0)
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0            # no gradient yet: nothing to clip, as in torch
    p.grad = torch.ones(3)
    with pytest.raises(_C.LsamError):
        clip_grad_norm_(p, 1.0)


@pytest.mark.parametrize("kw", [dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, grad_scale=float("nan"))])
def test_clip_values(kw):
    with pytest.raises(ValueError):
        clip_grads_([torch.zeros(3)], **kw)


def test_clip_arguments():
    g = [torch.zeros(3), torch.zeros(2)]
    for kw in (dict(norm_type=1.0), dict(norm_type=0.0), dict(out=[torch.zeros(3)]), dict(out=[torch.zeros(3), torch.zeros(3)])):
        with pytest.raises(_C.LsamError):
            clip_grads_(g, 1.0, **kw)


def _clip(src, dst, n, kind, max_norm=1.0, inf=0, scale=1.0, out=256, ws=256, ws_bytes=1 << 20):
    src, dst, n = array("Q", src), array("Q", dst), array("q", n)
    return _C.lib().lsam_clip_grads(src.buffer_info()[0], dst.buffer_info()[0], n.buffer_info()[0], bytes(kind), len(src), max_norm, inf, scale,
                                    out, ws, ws_bytes, 0)


@pytest.mark.parametrize("src, dst, n, kind, kw, rc", [
    # the addresses are never followed: every call ends at a check of the host's
    ([4096], [4096], [8], [4], {}, -1), ([4096], [4096], [-1], [0], {}, -1), ([0], [4096], [8], [0], {}, -1), ([4096], [0], [8], [0], {}, -1),
    ([4098], [4098], [8], [0], {}, -1), ([4097], [4097], [8], [3], {}, -1), ([4096], [4096], [8], [0], dict(max_norm=-1.0), -1),
    ([4096], [4096], [8], [0], dict(max_norm=float("nan")), -1), ([4096], [4096], [8], [0], dict(out=0), -1), ([4096], [4096], [8], [0], dict(ws=0), -1),
    ([4096], [4096], [8], [0], dict(ws=260), -1), ([4096], [4096], [8], [0], dict(ws_bytes=0), -4),
    ([4096, 4096], [4096, 4096], [8, 8], [0, 0], {}, -1),             # one tensor twice
    ([4096, 4112], [4096, 4112], [8, 8], [0, 0], {}, -1),             # the second begins inside the first
    ([4096, 8192], [12288, 12292], [8, 8], [0, 0], {}, -1),           # outputs overlap
    ([4096], [4100], [8], [0], {}, -1),                               # written over itself, shifted
    ([4096], [4096], [8], [1], {}, -1),                               # bf16 read where fp32 is written
    ([4096, 8192], [8192, 4096], [8, 8], [0, 0], {}, -1),             # each other's outputs
    ([4096], [4128], [8], [0], dict(max_norm=float("inf"), scale=2.0, ws_bytes=0), -4),
])
def test_clip_refuses(src, dst, n, kind, kw, rc):
    assert _clip(src, dst, n, kind, **kw) == rc
    assert _C.lib().lsam_last_error()


GN = dict(dtype=_C.BF16, x=256, sx=64, px=8, N=2, P=8, C=8, G=2, eps=1e-5, act=0, y=256, ws=256, ws_bytes=1 << 20)


@pytest.mark.parametrize("change, rc", [
    (dict(C=0), -1), (dict(G=0), -1), (dict(G=3), -1), (dict(N=-1), -1), (dict(P=-1), -1), (dict(act=4), -1), (dict(act=-1), -1), (dict(px=-8), -1),
    (dict(sx=-1), -1), (dict(x=0), -1), (dict(y=0), -1), (dict(ws=0), -1), (dict(ws=264), -1), (dict(ws_bytes=0), -4), (dict(C=8200, G=2), -2),
    (dict(dtype=9), -1), (dict(P=1 << 30), -2),
])
def test_group_norm_refuses(change, rc):
    a = dict(GN, **change)
    L = _C.lib()
    assert L.lsam_group_norm_act_fwd(a["dtype"], a["x"], a["sx"], a["px"], 0, 0, a["N"], a["P"], a["C"], a["G"], a["eps"], a["act"], a["y"], 0,
                                     a["ws"], a["ws_bytes"], 0) == rc
    assert L.lsam_group_norm_act_bwd(a["dtype"], a["x"], a["sx"], a["px"], 256, 64, 8, 0, 0, 256, a["N"], a["P"], a["C"], a["G"], a["act"],
                                     a["y"], 256, 256, a["ws"], a["ws_bytes"], 0) == rc


def test_channels_last_rows():
    cl = torch.zeros(2, 6, 4, 5).contiguous(memory_format=torch.channels_last)
    assert ops.channels_last_rows(cl) == (2, 20, 120, 6)
    assert ops.channels_last_rows(cl[:, 1:4]) == (2, 20, 120, 6)               # a channel slice
    assert ops.channels_last_rows(cl[1:]) == (1, 20, 120, 6)
    assert ops.channels_last_rows(cl[:, :, 1:3]) == (2, 10, 120, 6)            # whole rows of the map
    assert ops.channels_last_rows(cl[:, :, :, 1:3]) is None                    # pixels with gaps between the rows
    assert ops.channels_last_rows(torch.zeros(2, 6, 4, 5)) is None
    assert ops.channels_last_rows(torch.zeros(2, 6, 1, 1)) == (2, 1, 6, 6)
    assert ops.channels_last_rows(torch.zeros(2, 6)) == (2, 1, 6, 6)
    assert ops.channels_last_rows(torch.zeros(2, 1, 4, 5)) == (2, 20, 20, 1)
    assert ops.channels_last_rows(torch.zeros(1, 6, 1, 1).expand(3, 6, 4, 5)) is None   # broadcast: pixels on top of each other
    assert ops.channels_last_rows(torch.zeros(0, 6, 4, 5).contiguous(memory_format=torch.channels_last))[:2] == (0, 20)
    x = ops._channels_last_like(cl)
    assert x.shape == cl.shape and x.is_contiguous(memory_format=torch.channels_last)


def test_module_is_group_norm():
    m = GroupNormAct(4, 16, act="silu")
    assert sorted(m.state_dict()) == ["bias", "weight"] and "act=silu" in repr(m)
    m.load_state_dict(torch.nn.GroupNorm(4, 16).state_dict())
    with pytest.raises(_C.LsamError):
        GroupNormAct(4, 16, act="tanh")


def test_clip_of_copies_refuses_shared_memory():
    # tensors that are not contiguous go through copies; what they share is looked at before
    g = torch.ones(4, 6)
    for grads, kw in (([g.t(), g.t()], {}), ([g.t(), g], {}), ([g.t(), torch.ones(3).expand(2, 3)], {}),
                      ([g, g + 1], dict(out=[g.t().contiguous().t(), torch.zeros(4, 1).expand(4, 6)]))):
        with pytest.raises(_C.LsamError, match="share memory"):
            clip_grads_(grads, 1.0, **kw)


@pytest.mark.parametrize("max_norm", [1.0, -1.0, float("nan")])
def test_reducer_refuses_before_the_exchange(max_norm):
    p = torch.nn.Parameter(torch.zeros(3))
    red = LoRAGradReducer([p])
    with pytest.raises(_C.LsamError, match="max_norm"):
        red.reduce(max_norm)
    assert p.grad is None and red.stats["all_reduce"] == 0
    red.reduce()                                              # without it, as before
    assert p.grad is None


@pytest.mark.parametrize("change, rc", [
    (dict(C=0), -1), (dict(G=3), -1), (dict(act=4), -1), (dict(sx=-1), -1), (dict(x=0), -1), (dict(ws=0), -1), (dict(ws_bytes=0), -4),
    (dict(C=8200, G=2), -2), (dict(dtype=9), -1),
])
def test_group_norm_parameter_gradients_refuse(change, rc):
    a = dict(GN, **change)
    assert _C.lib().lsam_group_norm_act_bwd_params(a["dtype"], a["x"], a["sx"], a["px"], 256, 64, 8, 0, 0, 256, a["N"], a["P"], a["C"], a["G"],
                                                   a["act"], 256, 256, a["ws"], a["ws_bytes"], 0) == rc
