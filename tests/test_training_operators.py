"""The training operators that keep no large tensor, without a GPU: what they refuse, in Python and at the C ABI, before anything is
launched, and the workspace sizes they ask for."""
import ctypes

import pytest
import torch

from mvs_amd import _lib, ops
from mvs_amd._lib import MvsHipError

OK, EINVAL, EUNSUPPORTED, EWORKSPACE = 0, -1, -2, -4
FAKE = ctypes.c_void_p(1 << 20)          # an aligned address that is never read: every call here is refused first
ODD = ctypes.c_void_p((1 << 20) + 2)


def _text():
    return _lib.load().mvs_last_error_string().decode()


def test_host_tensors_are_refused():
    x, w, t = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(MvsHipError, match="CPU tensor"):
        ops.act8_quantize(x)
    with pytest.raises(MvsHipError, match="CPU tensor"):
        ops.lookup_rows(w, t)
    with pytest.raises(MvsHipError, match="CPU tensor"):
        ops.linear_cross_entropy(x, w, t)
    with pytest.raises(MvsHipError, match="CPU tensor"):
        ops.bn_relu_cl(x, torch.nn.BatchNorm2d(8), act8=True)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.bool, torch.complex64])
def test_other_types_are_refused(dtype):
    x, w, t = torch.zeros(3, 8, dtype=dtype), torch.zeros(5, 8, dtype=dtype), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.act8_quantize(x), lambda: ops.lookup_rows(w, t), lambda: ops.linear_cross_entropy(x, w, t)):
        with pytest.raises(MvsHipError, match="float32, bfloat16 or float16"):
            call()


def test_lookup_rows_refuses_what_does_not_fit():
    w, t = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for table in (torch.zeros(5), torch.zeros(5, 2, 4), torch.zeros(0, 8), torch.zeros(5, 0)):
        with pytest.raises(MvsHipError, match="table"):
            ops.lookup_rows(table, t)
    for index in (t.float(), t.bool(), t.to(torch.uint8)):
        with pytest.raises(MvsHipError, match="index"):
            ops.lookup_rows(w, index)


def test_linear_cross_entropy_refuses_what_does_not_fit():
    x, w, t = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for bad, what in (((x, w.half(), t), "weight"), ((x, torch.zeros(5, 7), t), "weight"), ((x, torch.zeros(0, 8), t), "weight"),
                      ((x, torch.zeros(8), t), "weight"), ((x, w, t[:2]), "target"), ((x, w, t.float()), "target"),
                      ((x.view(3, 8, 1)[..., 0].unsqueeze(0), w, t), "target"), ((torch.zeros(3, 0), torch.zeros(5, 0), t), "weight")):
        with pytest.raises(MvsHipError, match=what):
            ops.linear_cross_entropy(*bad)
    with pytest.raises(MvsHipError, match="reduction"):
        ops.linear_cross_entropy(x, w, t, reduction="avg")


def test_act8_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    for n, dtype, x, codes, scales in ((-1, 0, FAKE, FAKE, FAKE), (5, 3, FAKE, FAKE, FAKE), (5, -1, FAKE, FAKE, FAKE), (5, 0, None, FAKE, FAKE),
                                       (5, 0, FAKE, None, FAKE), (5, 0, FAKE, FAKE, None), (5, 0, ODD, FAKE, FAKE)):
        assert lib.mvs_act8_quantize(x, dtype, n, codes, scales, None) == EINVAL and "mvs_act8_quantize" in _text()
        assert lib.mvs_act8_dequantize(codes, scales, n, dtype, x, None) == EINVAL and "mvs_act8_dequantize" in _text()
    assert lib.mvs_act8_quantize(FAKE, 0, (1 << 38) + 1, FAKE, FAKE, None) == EUNSUPPORTED
    assert lib.mvs_act8_quantize(None, 0, 0, None, None, None) == OK          # nothing to do
    assert lib.mvs_act8_dequantize(None, None, 0, 1, None, None) == OK


def _bn_fwd(**change):
    a = dict(x=FAKE, weight=FAKE, bias=FAKE, skip=None, G=1, N=4, C=8, relu=1, mean=FAKE, invstd=FAKE, y=FAKE, codes=FAKE, scales=FAKE, mask=FAKE,
             ws=FAKE, nbytes=1 << 20)
    a.update(change)
    return _lib.load().mvs_bn_train_fwd_act8_f32(a["x"], a["weight"], a["bias"], a["skip"], a["G"], a["N"], a["C"], 1e-5, 0.1, a["relu"], None, None,
                                                 None, a["mean"], a["invstd"], a["y"], a["codes"], a["scales"], a["mask"], a["ws"], a["nbytes"], None)


def _bn_bwd(**change):
    a = dict(gy=FAKE, codes=FAKE, scales=FAKE, mask=FAKE, weight=FAKE, mean=FAKE, invstd=FAKE, G=1, N=4, C=8, gx=FAKE, gw=FAKE, gb=FAKE, ws=FAKE,
             nbytes=1 << 20)
    a.update(change)
    return _lib.load().mvs_bn_train_bwd_act8_f32(a["gy"], a["codes"], a["scales"], a["mask"], a["weight"], a["mean"], a["invstd"], a["G"], a["N"],
                                                 a["C"], a["gx"], a["gw"], a["gb"], a["ws"], a["nbytes"], None)


def test_bn_act8_entry_points_refuse_bad_arguments():
    for change in (dict(x=None), dict(y=None), dict(codes=None), dict(scales=None), dict(mask=None), dict(relu=0), dict(ws=None), dict(N=0), dict(G=0),
                   dict(G=17), dict(x=ODD), dict(codes=ODD), dict(skip=ODD), dict(mask=ODD)):
        assert _bn_fwd(**change) == EINVAL, change
        assert "mvs_bn_train_fwd_act8_f32" in _text()
    for change in (dict(gy=None), dict(codes=None), dict(scales=None), dict(gx=None), dict(gw=None), dict(ws=None), dict(N=0), dict(G=17), dict(gy=ODD),
                   dict(gx=ODD), dict(mask=ODD)):
        assert _bn_bwd(**change) == EINVAL, change
        assert "mvs_bn_train_bwd_act8_f32" in _text()
    for call in (_bn_fwd, _bn_bwd):
        assert call(C=12) == EUNSUPPORTED and call(C=128) == EUNSUPPORTED
        assert call(nbytes=16) == EWORKSPACE


def test_lookup_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    need = lib.mvs_lookup_rows_workspace_bytes(10, 8, 5)
    assert need >= 5 * 8
    for table, dtype, rows, C, index, n, out in ((None, 0, 10, 8, FAKE, 5, FAKE), (FAKE, 7, 10, 8, FAKE, 5, FAKE), (FAKE, 0, 0, 8, FAKE, 5, FAKE),
                                                 (FAKE, 0, 10, 0, FAKE, 5, FAKE), (FAKE, 0, 10, 8, None, 5, FAKE), (FAKE, 0, 10, 8, FAKE, 5, None),
                                                 (FAKE, 0, 10, 8, FAKE, -1, FAKE)):
        assert lib.mvs_lookup_rows_fwd(table, dtype, rows, C, index, n, 1.0, out, None) == EINVAL
        assert lib.mvs_lookup_rows_bwd(out, dtype, index, n, rows, C, 1.0, table, FAKE, 1 << 30, None) == EINVAL
    assert lib.mvs_lookup_rows_fwd(FAKE, 0, 1 << 31, 8, FAKE, 5, 1.0, FAKE, None) == EUNSUPPORTED
    assert lib.mvs_lookup_rows_fwd(FAKE, 0, 10, (1 << 20) + 1, FAKE, 5, 1.0, FAKE, None) == EUNSUPPORTED
    assert lib.mvs_lookup_rows_workspace_bytes(10, (1 << 20) + 1, 5) == 0
    assert lib.mvs_lookup_rows_bwd(FAKE, 0, FAKE, 1 << 31, 10, 8, 1.0, FAKE, FAKE, 1 << 30, None) == EUNSUPPORTED
    for ws, nbytes in ((None, 1 << 30), (FAKE, need - 1), (ODD, 1 << 30)):
        assert lib.mvs_lookup_rows_bwd(FAKE, 0, FAKE, 5, 10, 8, 1.0, FAKE, ws, nbytes, None) == EWORKSPACE
    assert lib.mvs_lookup_rows_fwd(FAKE, 0, 10, 8, None, 0, 1.0, None, None) == OK
    assert lib.mvs_lookup_rows_workspace_bytes(0, 8, 5) == 0


def _ce(call="fwd", **change):
    a = dict(x=FAKE, w=FAKE, dtype=1, t=FAKE, n=4, V=9, C=8, reduction=1, loss=FAKE, lse=FAKE, kept=FAKE, g=FAKE, gx=FAKE, gw=FAKE, ws=FAKE, nbytes=1 << 30)
    a.update(change)
    lib = _lib.load()
    if call == "fwd":
        return lib.mvs_linear_ce_fwd(a["x"], a["w"], a["dtype"], a["t"], a["n"], a["V"], a["C"], 1.0, -100, a["reduction"], a["loss"], a["lse"],
                                     a["kept"], a["ws"], a["nbytes"], None)
    return lib.mvs_linear_ce_bwd(a["x"], a["w"], a["dtype"], a["t"], a["lse"], a["kept"], a["g"], a["n"], a["V"], a["C"], 1.0, -100, a["reduction"],
                                 a["gx"], a["gw"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("call", ["fwd", "bwd"])
def test_linear_ce_entry_points_refuse_bad_arguments(call):
    for change in (dict(x=None), dict(w=None), dict(t=None), dict(dtype=5), dict(n=-1), dict(V=0), dict(C=0), dict(reduction=3), dict(ws=None),
                   dict(x=ODD), dict(w=ODD), dict(ws=ODD), dict(lse=None), dict(kept=None)):
        assert _ce(call, **change) == EINVAL, change
        assert f"mvs_linear_ce_{call}" in _text()
    for change in (dict(n=1 << 31), dict(V=1 << 31), dict(C=1 << 21), dict(n=1 << 24, V=1 << 24), dict(n=(1 << 23) + 1, C=129)):
        assert _ce(call, nbytes=1 << 60, **change) == EUNSUPPORTED, change
    assert _ce(call, nbytes=64) == EWORKSPACE
    assert _ce("fwd", loss=None) == EINVAL
    assert _ce("bwd", g=None) == EINVAL and _ce("bwd", gx=None, gw=None) == EINVAL
    assert _ce("bwd", gx=ODD) == EINVAL and _ce("bwd", gw=ODD) == EINVAL and "gradients" in _text()


def test_linear_ce_workspace_keeps_no_logits():
    lib = _lib.load()
    ask = lib.mvs_linear_ce_workspace_bytes
    n, V, C = 8192, 128000, 2048
    assert ask(n, V, C, 1, 0, 0, 0) < n * V * 2 / 16
    assert ask(n, V, C, 1, 1, 1, 1) < n * V * 2 / 3
    assert ask(n, V, C, 1, 1, 1, 0) < ask(n, V, C, 1, 1, 1, 1)
    assert ask(n, V, C, 9, 0, 0, 0) == 0 and ask(-1, V, C, 0, 0, 0, 0) == 0 and ask(n, 0, C, 0, 0, 0, 0) == 0
    assert ask(0, 1, 1, 0, 1, 1, 1) > 0
