"""CPU tests of group norm and dropout: the generator against the published vectors, the entry
points' refusals, the layers' construction."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import random_np as R


def test_philox_known_answers():
    """Vectors published with the generator (zero, all ones, digits of pi)."""
    pi = [[0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]], (0xA4093822, 0x299F31D0)
    for (ctr, key), want in ((([[0, 0, 0, 0]], (0, 0)), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
                             (([[0xFFFFFFFF] * 4], (0xFFFFFFFF,) * 2), "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                             (pi, "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert " ".join("%08x" % w for w in R.philox4x32(np.array(ctr, np.uint64), key)[0]) == want
    assert np.array_equal(R.keep_mask(0, 64, 0.5, 3, 4)[5:20], R.keep_mask(5, 15, 0.5, 3, 4))


def test_group_norm_entry_points_validate_without_gpu():
    from yolo_amd import _lib
    L = _lib.lib()
    one, odd = ctypes.c_void_p(256), ctypes.c_void_p(260)

    def fwd(x=one, B=2, P=16, C=64, G=8, act=2, eps=1e-3, dtype=_lib.BF16, rate=0.0, state=None, ws=one, nb=1 << 20):
        return L.ymx_group_norm_forward(x, one, one, None, one, one, B, P, C, G, act, eps, dtype, rate, state, ws, nb, None)

    def bwd(dx=one, C=64, G=8, rate=0.0, state=None, nb=1 << 20):
        return L.ymx_group_norm_backward(one, one, one, one, one, dx, one, one, 2, 16, C, G, 2, _lib.BF16, rate, state, one, nb, None)
    need = L.ymx_group_norm_workspace_bytes(2, 16, 64, 8)
    assert need > 0 and L.ymx_group_norm_workspace_bytes(0, 16, 64, 8) == 0
    for call, code, text in ((lambda: fwd(x=None), -1, b"null"), (lambda: fwd(G=7), -1, b"do not split"), (lambda: fwd(B=0), -1, b"size"),
                             (lambda: fwd(act=3), -1, b"activation"), (lambda: fwd(eps=0.0), -1, b"epsilon"), (lambda: fwd(eps=float("nan")), -1, b"epsilon"),
                             (lambda: fwd(dtype=2), -1, b"dtype"), (lambda: fwd(rate=1.0, state=one), -1, b"rate"), (lambda: fwd(rate=float("nan"), state=one), -1, b"rate"),
                             (lambda: fwd(rate=0.5), -1, b"state"), (lambda: fwd(rate=0.5, state=odd), -1, b"state"), (lambda: fwd(ws=odd), -1, b"aligned"),
                             (lambda: fwd(nb=need - 1), -3, b"workspace"), (lambda: fwd(P=1 << 31), -2, b"pixels"), (lambda: fwd(B=1 << 21), -2, b"samples"),
                             (lambda: fwd(C=8192, G=8192), -2, b"groups"),
                             (lambda: bwd(dx=None), -1, b"null"), (lambda: bwd(G=0), -1, b"size"), (lambda: bwd(rate=-0.1), -1, b"rate"),
                             (lambda: bwd(nb=8), -3, b"workspace"),
                             (lambda: L.ymx_dropout(one, None, one, 8, _lib.BF16, 0.5, None, None), -1, b"null"),
                             (lambda: L.ymx_dropout(one, None, one, -1, _lib.BF16, 0.5, one, None), -1, b"negative"),
                             (lambda: L.ymx_dropout(one, None, one, 8, 2, 0.5, one, None), -1, b"dtype"),
                             (lambda: L.ymx_dropout(one, None, one, 8, _lib.F32, 1.0, one, None), -1, b"rate"),
                             (lambda: L.ymx_dropout(one, None, one, 8, _lib.F32, 0.5, odd, None), -1, b"state")):
        assert call() == code and text in L.ymx_last_error(), (code, text, L.ymx_last_error())
    assert L.ymx_dropout(one, None, one, 0, _lib.F32, 0.5, one, None) == 0


def test_sizes_beyond_a_grid_are_refused():
    """More workgroups than a launch has room for; the workspace may then be missing as well."""
    from yolo_amd import _lib
    L, one = _lib.lib(), ctypes.c_void_p(256)

    def fwd(B, P, C, G, ws=one):
        return L.ymx_group_norm_forward(one, one, one, None, one, one, B, P, C, G, 0, 1e-3, _lib.BF16, 0.0, None, ws, 1 << 50, None)
    for B, P, C, G in ((1 << 20, 1, 2048, 1), (1, 1 << 20, 1 << 20, 4096), (4096, 8, 1 << 19, 8), ((1 << 20) + 1, 4, 64, 8)):
        for ws in (one, None):
            assert fwd(B, P, C, G, ws) == -2 and b"samples" in L.ymx_last_error()
    assert fwd(2, 8, 64, 8, None) == -1 and b"null" in L.ymx_last_error()


def test_statistics_are_quadruples():
    from yolo_amd import _lib
    L, one, odd = _lib.lib(), ctypes.c_void_p(256), ctypes.c_void_p(264)
    assert L.ymx_group_norm_forward(one, one, one, None, one, odd, 2, 16, 64, 8, 0, 1e-3, _lib.BF16, 0.0, None, one, 1 << 30, None) == -1
    assert b"stats" in L.ymx_last_error()
    assert L.ymx_group_norm_backward(one, one, one, one, odd, one, one, one, 2, 16, 64, 8, 0, _lib.BF16, 0.0, None, one, 1 << 30, None) == -1
    assert b"stats" in L.ymx_last_error()


def test_functions_refuse_before_the_device():
    from yolo_amd import training as T
    x, v = torch.zeros(1, 2, 2, 8), torch.zeros(8)
    with pytest.raises(RuntimeError, match="GPU"):
        T.group_norm_act(x, v, v, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        T.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="rate"):
        T._check_dropout(x, 1.0, None, "dropout")
    for bad in (None, torch.zeros(2), torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)[::2], [1, 2]):
        with pytest.raises(ValueError, match="int64"):
            T._check_dropout(x, 0.5, bad, "dropout")
    with pytest.raises(ValueError, match="shortcut"):
        T._check_shortcut(x, torch.zeros(1, 2, 2, 4), "dropout")
    with pytest.raises(ValueError, match="activation"):
        T._activation_code("relu", "group_norm_act")


def test_layers_construct_and_refuse():
    from yolo_amd.backbones import Darknet53
    from yolo_amd.layers import Dropout, GroupNormalization, ResidialBlock, YOLOConv
    c = YOLOConv((3, 3, 64), groupNormalization=8, dropout=0.1, dropout_seed=4, in_channels=32)
    assert not hasattr(c, "bias") and c.bn is None and tuple(c.gn.gamma.shape) == (64,) and c.drop.state.tolist() == [4, 0]
    assert YOLOConv((3, 3, 64), in_channels=8).drop is None
    p = {"kernel": torch.randn(3, 3, 32, 64), "gamma": torch.randn(64), "beta": torch.randn(64)}
    c.load_reference_params(p)
    assert torch.equal(c.gn.gamma, p["gamma"]) and torch.equal(c.gn.beta, p["beta"])
    for kw, text in ((dict(groupNormalization=8, batchNormalization=True), "excludes"), (dict(groupNormalization=7), "split"),
                     (dict(groupNormalization=-1), "groups"), (dict(dropout=1.0), "rate"), (dict(dropout=-0.5), "rate"),
                     (dict(groupNormalization=8, activation=torch.relu), "activation"), (dict(dropout=0.5, activation=torch.relu), "activation")):
        with pytest.raises(ValueError, match=text):
            YOLOConv((1, 1, 64), **kw)
    with pytest.raises(ValueError, match="groups"):
        GroupNormalization(0)
    with pytest.raises(ValueError, match="split"):
        GroupNormalization(5, 64)
    with pytest.raises(ValueError, match="rate"):
        Dropout(1.5)
    with pytest.raises(TypeError):
        ResidialBlock(32, 64, groups=8)
    net = Darknet53(seed=1, groupNormalization=16, dropout=0.2)
    assert all(conv.gn.groups == 16 for conv in net.conv_layers())
    assert sum(conv.drop is not None for conv in net.conv_layers()) == 23
    plain = Darknet53(seed=1)
    assert all(torch.equal(a.kernel, b.kernel) for a, b in zip(net.conv_layers(), plain.conv_layers()))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("needs", [False, True])
def test_tangents_are_refused(grad, needs):
    """Forward mode: an error, whether or not the input requires a gradient and gradients are enabled.  (An empty map launches
    nothing; without a tangent the same call succeeds.)"""
    from torch.autograd import forward_ad
    from yolo_amd import _lib
    native = _lib.native()
    empty, v = torch.zeros(0, 2, 2, 8), torch.ones(8)
    state = torch.zeros(2, dtype=torch.int64)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone().requires_grad_(needs), torch.ones_like(t))
        assert native.group_norm_act(empty, v, v, None, None, 2, 0, 1e-3, 0.0).shape == empty.shape
        for args in ((empty, dual(v), v, None), (empty, v, dual(v), None), (dual(empty), v, v, None), (empty, v, v, dual(empty))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                native.group_norm_act(*args, None, 2, 0, 1e-3, 0.0)
        x = torch.ones(4)
        for args in ((dual(x), None), (x, dual(x))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                native.dropout(*args, state, 0.5)
