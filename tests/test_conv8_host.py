"""CPU tests of the 8-bit convolution blocks: the entry points' refusals and sizes, the layers' checks."""
import ctypes

import pytest
import torch

F8 = torch.float8_e4m3fn


def test_entry_points_validate_without_gpu():
    from yolo_amd import _lib
    L = _lib.lib()
    one, odd = ctypes.c_void_p(256), ctypes.c_void_p(260)
    assert L.ymx_packed_weight_bytes(3, 512, 1024, _lib.F8E4M3) == 1024 * 36 * (128 + 1)
    assert L.ymx_packed_weight_bytes(1, 1024, 255, _lib.F8E4M3) == 256 * 8 * (128 + 1)
    assert L.ymx_packed_weight_bytes(3, 144, 16, _lib.F8E4M3) == 256 * 18 * (128 + 1)
    assert L.ymx_packed_weight_bytes(3, 24, 16, _lib.F8E4M3) == 0 and L.ymx_packed_weight_bytes(5, 32, 16, _lib.F8E4M3) == 0
    assert L.ymx_quantized_bytes(10, 48) == 512 + 12 and L.ymx_quantized_bytes(1, 640) == 768 + 5 * 4
    assert L.ymx_quantized_bytes(0, 48) == 0

    def quant(x=one, q=one, n=4, c=32, dtype=_lib.BF16, ld=0):
        return L.ymx_quantize_blocks(x, q, n, c, dtype, ld, None)

    def conv(x=one, w=one, y=one, res=None, B=1, H=8, W=8, cin=32, cout=32, k=3, stride=1, act=0, dtype=_lib.F8E4M3, xd=_lib.F8E4M3, od=_lib.BF16, x_ld=0):
        return L.ymx_conv2d_fused_ex(x, w, None, None, res, y, B, H, W, cin, cout, k, stride, act, dtype, xd, od, x_ld, 0, 0, None)
    for call, code, text in ((lambda: quant(x=None), -1, b"null"), (lambda: quant(n=0), -1, b"size"), (lambda: quant(c=24), -2, b"multiples of 16"),
                             (lambda: quant(dtype=_lib.F8E4M3), -1, b"dtype"), (lambda: quant(ld=16), -1, b"stride"), (lambda: quant(ld=36), -1, b"stride"),
                             (lambda: quant(q=odd), -1, b"alignment"), (lambda: quant(n=1 << 31), -2, b"2^31"),
                             (lambda: L.ymx_pack_weights(one, one, 3, 24, 8, _lib.F8E4M3, None), -2, b"multiples of 16"),
                             (lambda: L.ymx_pack_weights(one, one, 5, 32, 8, _lib.F8E4M3, None), -2, b"3x3"),
                             (lambda: L.ymx_pack_weights(one, odd, 3, 32, 8, _lib.F8E4M3, None), -1, b"aligned"),
                             (lambda: conv(xd=_lib.BF16), -1, b"quantised map"), (lambda: conv(dtype=_lib.BF16), -1, b"8-bit kernel"),
                             (lambda: conv(dtype=_lib.F32, cin=3), -1, b"8-bit kernel"), (lambda: conv(od=_lib.F8E4M3), -1, b"out_dtype"),
                             (lambda: conv(cin=40), -2, b"multiples of 16"), (lambda: conv(k=5), -2, b"3x3"), (lambda: conv(x_ld=64), -1, b"dense"),
                             (lambda: conv(x=odd), -1, b"aligned"), (lambda: conv(y=ctypes.c_void_p(257)), -1, b"aligned"),
                             (lambda: conv(od=_lib.F32, res=ctypes.c_void_p(258)), -1, b"aligned"),
                             (lambda: conv(B=64, H=1024, W=1024, cin=32), -2, b"2^31"), (lambda: conv(H=0), -1, b"size")):
        assert call() == code and text in L.ymx_last_error(), (code, text, L.ymx_last_error())
    op = _lib.ymx_op()
    op.kind, op.B, op.H, op.W, op.Cin, op.Cout, op.k, op.stride = 1, 1, 8, 8, 32, 32, 3, 1
    op.dtype = op.x_dtype = _lib.F8E4M3
    op.out_dtype = _lib.BF16
    op.x = op.w = op.y = 256
    assert L.ymx_conv_kernel_label(ctypes.byref(op)) == b"f8"


def test_plain_maps_are_for_small_1x1_layers():
    from yolo_amd import _lib
    L, one = _lib.lib(), ctypes.c_void_p(256)

    def conv(B=1, H=8, W=8, cin=32, cout=32, k=1, xd=_lib.BF16, x_ld=0, x=one):
        return L.ymx_conv2d_fused_ex(x, one, None, None, None, one, B, H, W, cin, cout, k, 1, 0, _lib.F8E4M3, xd, _lib.BF16, x_ld, 0, 0, None)
    assert [L.ymx_conv2d_quantizes(n, c, k, _lib.BF16) for n, c, k in ((169, 512, 1), (11264, 64, 1), (11265, 64, 1), (169, 512, 3), (0, 64, 1), (1, 0, 1))] == [1, 1, 0, 0, 0, 0]
    assert [L.ymx_conv2d_quantizes(n, 64, 1, _lib.F32) for n in (11265, 49152, 49153)] == [1, 1, 0]
    for call, text in ((lambda: conv(B=200), b"quantised map"), (lambda: conv(xd=_lib.F32), b"quantised map"), (lambda: conv(x_ld=36), b"stride"),
                       (lambda: conv(x_ld=24), b"stride"), (lambda: conv(x=ctypes.c_void_p(264)), b"aligned")):
        assert call() == -1 and text in L.ymx_last_error(), L.ymx_last_error()


def test_layers_check_before_the_device():
    from yolo_amd import training as T
    from yolo_amd.layers import BlockQuantized, YOLOConv, quantize_blocks
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_blocks(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="1x1 or 3x3"):
        YOLOConv((5, 5, 32), dtype=F8)
    c = YOLOConv((3, 3, 32), dtype=F8, in_channels=32)
    assert c.is_8bit() and c.map_dtype(torch.zeros(1)) == torch.bfloat16
    assert not YOLOConv((3, 3, 32), dtype=F8, in_channels=3).is_8bit()
    assert not YOLOConv((3, 3, 32), dtype=torch.bfloat16, in_channels=32).is_8bit()
    q = BlockQuantized(torch.zeros(2 * 256 + 16, dtype=torch.uint8), (1, 4, 4, 32))
    assert tuple(q.values.shape) == (1, 4, 4, 32) and tuple(q.exponents.shape) == (1, 4, 4, 1)
    assert torch.equal(q.dequantize(), torch.zeros(1, 4, 4, 32))
    with pytest.raises(ValueError, match="quantised map"):
        YOLOConv((3, 3, 32), dtype=torch.bfloat16, in_channels=32)(q)
    with T.backprop():
        with pytest.raises(ValueError, match="quantised map"):
            c(q)
    with pytest.raises(ValueError, match="residual"):
        c(q, residual=q)
    with pytest.raises(ValueError, match="input channels"):
        YOLOConv((3, 3, 32), dtype=F8, in_channels=64)(q)


def test_quantised_maps_are_checked_against_their_buffer():
    """The kernels take a map's extent from its shape: a buffer that does not hold it is refused before the device is used."""
    from yolo_amd.layers import BlockQuantized, YOLOConv
    c = YOLOConv((3, 3, 32), dtype=F8, in_channels=32)
    need = 2 * 256 + 16                                       # 16 pixels of 32 bytes, one exponent each
    whole = torch.zeros(need + 16, dtype=torch.uint8)
    whole = whole[-whole.data_ptr() % 16:][:need]
    for buf in (whole[:-1], whole.view(2, -1), torch.zeros(2 * need, dtype=torch.uint8)[::2], whole.view(torch.int8),
                torch.zeros(need + 32, dtype=torch.uint8)[-whole.data_ptr() % 16 + 8:][:need]):
        with pytest.raises(ValueError, match="needs a flat"):
            c(BlockQuantized(buf, (1, 4, 4, 32)))
    with pytest.raises(ValueError, match="needs a flat"):
        c(BlockQuantized(whole, (2, 4, 4, 32)))
    with pytest.raises(RuntimeError, match="GPU"):            # the right one passes this check
        c(BlockQuantized(whole, (1, 4, 4, 32)))


def test_the_planned_program_refuses_what_it_has_no_kernels_for():
    import yolo_amd
    from yolo_amd.backbones import Darknet53
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        yolo_amd.Detector(num_classes=2, dtype=F8)
    for kw in (dict(groupNormalization=8), dict(dtype=F8)):
        det = yolo_amd.Detector(num_classes=2, dtype=torch.bfloat16)
        det.backbone = Darknet53(seed=0, **kw)
        for m in det.backbone.conv_layers():
            if m.in_channels is None:
                m.build(3)
        with pytest.raises(ValueError, match="run by module"):
            det._build_plan((1,), 64, torch.bfloat16, torch.device("cpu"))
