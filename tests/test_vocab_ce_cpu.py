"""Refusals of loss_fns.linear_cross_entropy and of its C entry points that need no GPU: arguments are checked on the host, before
anything is launched."""
import pytest
import torch

from image_segmentation_amd import _C
from image_segmentation_amd.loss_fns import linear_cross_entropy


def test_cpu_tensors_are_refused():
    with pytest.raises(_C.LsamError, match="MI355X only"):
        linear_cross_entropy(torch.zeros(2, 8), torch.zeros(3, 8), torch.zeros(2, dtype=torch.long))


@pytest.mark.parametrize("change, rc", [
    (dict(M=-1), -1), (dict(D=0), -1), (dict(V=0), -1), (dict(reduction=3), -1), (dict(smooth=1.5), -1), (dict(smooth=float("nan")), -1),
    (dict(ldx=7), -1), (dict(ldw=7), -1), (dict(x=0), -1), (dict(w=0), -1), (dict(target=0), -1), (dict(loss=0), -1), (dict(state=0), -1),
    (dict(ws=0), -1), (dict(ws=264), -1), (dict(ws_bytes=0), -4), (dict(dtype=7), -1), (dict(M=1 << 29), -2), (dict(M=1 << 28, V=1 << 28), -2),
])
def test_forward_refuses(change, rc):
    # the pointers are never followed: every call ends at a check of the host's
    a = dict(dtype=_C.BF16, x=256, ldx=8, w=256, ldw=8, bias=0, target=256, M=4, D=8, V=5, ignore=-100, smooth=0.0, reduction=1, loss=256,
             state=256, ws=256, ws_bytes=0)
    a.update(change)
    got = _C.lib().lsam_linear_ce_fwd(a["dtype"], a["x"], a["ldx"], a["w"], a["ldw"], a["bias"], a["target"], a["M"], a["D"], a["V"],
                                      a["ignore"], a["smooth"], a["reduction"], a["loss"], a["state"], a["ws"], a["ws_bytes"], 0)
    assert got == rc
    assert _C.lib().lsam_last_error()


@pytest.mark.parametrize("change, rc", [
    (dict(D=0), -1), (dict(ldw=7), -1), (dict(lddx=7), -1), (dict(lddw=7), -1), (dict(gout=0), -1), (dict(state=0), -1), (dict(ws=0), -1),
    (dict(ws_bytes=0), -4), (dict(reduction=-1), -1),
])
def test_backward_refuses(change, rc):
    a = dict(w=256, ldw=8, bias=0, gout=256, M=4, D=8, V=5, smooth=0.0, reduction=1, state=256, dx=256, lddx=8, dw=256, lddw=8, db=0, ws=256,
             ws_bytes=0)
    a.update(change)
    got = _C.lib().lsam_linear_ce_bwd(_C.BF16, a["w"], a["ldw"], a["bias"], a["gout"], a["M"], a["D"], a["V"], a["smooth"], a["reduction"],
                                      a["state"], a["dx"], a["lddx"], a["dw"], a["lddw"], a["db"], a["ws"], a["ws_bytes"], 0)
    assert got == rc


def test_workspace_of_a_piece_is_bounded():
    """Scores of 65,536 rows against 262,144 classes would be 34 GB in bf16; the backward's workspace stays far below."""
    got = _C.lib().lsam_linear_ce_ws_bytes(_C.BF16, 65536, 256, 262144, 256, 256, 0.0, 3)
    assert 0 < got < 3 << 30


def test_sizes_without_rows():
    L = _C.lib()
    for dtype in (_C.F32, _C.BF16):
        assert L.lsam_linear_ce_state_bytes(dtype, 0, 16) > 0
        for grads in range(8):
            assert L.lsam_linear_ce_ws_bytes(dtype, 0, 16, 40, 256, 16, 0.0, grads) > 0


@pytest.mark.parametrize("M, D, V, rc", [
    ((1 << 26) - 16, 8, 5, -4), ((1 << 26) - 15, 8, 5, -2), (1 << 26, 8, 5, -2), (1 << 28, 8, 5, -2),
    ((1 << 26) - 16, 1920, 5, -4), ((1 << 26) - 16, 1921, 5, -2),   # 2^19 x 15 tiles of 512 threads, and 2^19 x 16
])
def test_rows_of_a_launch(M, D, V, rc):
    # a launch may have 2^32 - 1 threads; the next check to fail is the workspace's
    L = _C.lib()
    assert L.lsam_linear_ce_fwd(_C.BF16, 256, D, 256, D, 0, 256, M, D, V, -100, 0.0, 1, 256, 256, 256, 0, 0) == rc
    assert L.lsam_linear_ce_bwd(_C.BF16, 256, D, 0, 256, M, D, V, 0.0, 1, 256, 256, D, 256, D, 0, 256, 0, 0) == rc


@pytest.mark.parametrize("dtype, row", [(_C.BF16, 512), (_C.F32, 1536)])
@pytest.mark.parametrize("M", [100_000, 1 << 20, 1 << 21, 1 << 22])
def test_workspace_of_many_rows(M, dtype, row):
    """The weight gradient's workspace: a piece of the scores' gradients (1 GiB, or 256 classes' worth), partial sums of 512 x 128 x 128 or 256 x 256 x 256
    fp32 values at most, in fp32 the table's three planes, and each part's alignment."""
    D, V = 256, 32000
    piece = max(1 << 30, M * row)
    got = _C.lib().lsam_linear_ce_ws_bytes(dtype, M, D, V, 256, D, 0.0, 2)
    assert piece - M * row < got <= piece + 4 * 256 ** 3 + (6 * V * D if dtype == _C.F32 else 0) + 4096
