"""Every tile that an 8-bit convolution may be computed in: which layers take it (on the CPU), and those layers against the 64-bit
restatement in oracle/block8_torch.py.  Each tile meets input channels that are no multiple of 128, output channels and pixels off its
own size where it takes such layers, and the widths at which one gives way to another."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import block8_torch as Q

DEV = "cuda:0"
F8 = torch.float8_e4m3fn

CASES = [   # tile, B, H, W, Cin, Cout, k, stride, act, out, residual
    ("256x256 slab", 31, 55, 55, 48, 500, 3, 1, "mish", "bf16", True),              # rows of 55 pixels: the last that 256 have room for
    ("256x192 slab", 31, 55, 56, 48, 500, 3, 1, "leaky", "bf16", False),
    ("256x256 and 256x192 slab", 31, 53, 52, 48, 512, 3, 1, None, "bf16", False),
    ("256x192 slab", 16, 53, 52, 144, 256, 3, 1, "mish", "bf16", True),             # two blocks, the second of 16 channels
    ("256x192 slab", 6, 87, 87, 80, 256, 3, 1, "mish", "bf16", False),              # rows of 87 pixels: the last that 192 have room for
    ("256x192", 6, 87, 88, 80, 256, 3, 1, "leaky", "bf16", True),
    ("256x256", 1, 211, 260, 48, 252, 3, 1, None, "bf16", True),
    ("256x256", 18, 53, 52, 400, 256, 1, 1, "mish", "bf16", False),
    ("256x192", 16, 53, 52, 400, 255, 1, 1, "mish", "bf16", True),
    ("256x256 and 256x192", 31, 53, 52, 400, 500, 1, 1, "leaky", "bf16", True),
    ("256x256", 20, 105, 104, 144, 256, 3, 2, "mish", "bf16", True),
    ("256x192", 16, 104, 105, 144, 250, 3, 2, None, "bf16", False),
    ("256x256 and 256x192", 62, 53, 103, 48, 512, 3, 2, "mish", "bf16", False),
    ("128x128", 40, 61, 61, 144, 72, 1, 2, "mish", "bf16", True),
    ("128x128", 16, 52, 52, 64, 256, 1, 1, "mish", "bf16", True),
    ("64x128", 48, 53, 52, 144, 64, 1, 1, "leaky", "bf16", False),
    ("64x128", 26, 53, 52, 144, 61, 3, 1, "mish", "f32", True),
    ("32x128", 48, 53, 52, 144, 30, 1, 1, "mish", "bf16", True),
    ("32x128", 26, 53, 52, 48, 29, 3, 1, None, "bf16", False),
    ("32x128", 26, 53, 52, 48, 32, 3, 1, "mish", "f32", False),
    ("64x64, two stages", 11, 53, 52, 144, 100, 3, 1, "mish", "bf16", True),
    ("64x64", 4, 26, 27, 144, 200, 3, 1, "leaky", "bf16", False),
    ("64x32", 2, 27, 25, 64, 128, 3, 2, "mish", "bf16", True),
    ("64x32", 26, 53, 52, 144, 30, 3, 2, None, "f32", True),
]


def _tile(case, raw=False):
    from yolo_amd import _lib
    _, B, H, W, cin, cout, k, stride, act, out, _ = case
    op = _lib.ymx_op()
    op.kind, op.B, op.H, op.W, op.Cin, op.Cout, op.k, op.stride = 1, B, H, W, cin, cout, k, stride
    op.dtype, op.x_dtype, op.out_dtype = _lib.F8E4M3, _lib.BF16 if raw else _lib.F8E4M3, _lib.BF16 if out == "bf16" else _lib.F32
    op.x = op.w = op.y = 256
    label = _lib.lib().ymx_conv8_tile_label(ctypes.byref(op))
    return label.decode() if label else _lib.lib().ymx_last_error().decode()


def test_layers_take_the_tiles_they_are_listed_for():
    from yolo_amd import _lib
    assert [_tile(c) for c in CASES] == [c[0] for c in CASES]
    small = (None, 1, 13, 13, 1024, 512, 1, 1, None, "bf16", False)
    assert _tile(small, raw=True) == "64x32 raw" and _tile(small) == "64x32"
    assert "quantised map" in _tile(CASES[0], raw=True)
    op = _lib.ymx_op()
    op.kind, op.dtype = 1, _lib.BF16
    assert not _lib.lib().ymx_conv8_tile_label(ctypes.byref(op)) and b"8-bit" in _lib.lib().ymx_last_error()
    assert not _lib.lib().ymx_conv8_tile_label(None)


def _act(t, name):
    if name == "mish":
        return t * torch.tanh(torch.nn.functional.softplus(t))
    return torch.where(t > 0, t, 0.1 * t) if name == "leaky" else t


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_tile_against_64_bits(case):
    """Bounds: 32-bit outputs 64 units of 2^-24 of the summed magnitudes (blocks of 32 exact products added in fp32); bf16
    ones half a step, 2^-8, and what the 8-bit pipe drops of each group of eight products: seven times less than 2^-13 of the
    group's largest, times the activation's slope of at most 1.1.  The image by image results have the same bits."""
    from yolo_amd.layers import YOLOConv, quantize_blocks
    _, B, H, W, cin, cout, k, stride, act, out, use_res = CASES[case]
    odt = torch.bfloat16 if out == "bf16" else torch.float32
    g = torch.Generator(device=DEV).manual_seed(700 + case)

    def r(*s):
        return torch.randn(*s, device=DEV, generator=g)
    x = _act(r(B, H, W, cin) * (0.2 + torch.rand(cin, device=DEV, generator=g)), "mish").bfloat16()
    kernel, bias = r(k, k, cin, cout) / (k * k * cin) ** 0.5, 0.1 * r(cout)
    layer = YOLOConv((k, k, cout), downsample=stride == 2, activation=act, dtype=F8, in_channels=cin).to(DEV)
    layer.load_reference_params({"kernel": kernel, "bias": bias})
    oh, ow = layer.output_hw(H, W)
    res = r(B, oh, ow, cout).to(odt) if use_res else None
    q = quantize_blocks(x)                                    # (a plain map of few pixels may be quantised by a kernel of another tile)
    got = layer(q, residual=res, out_dtype=odt)
    total, mag = Q.conv(x, kernel, stride)
    want = _act(total + bias.double(), act) + (0.0 if res is None else res.double())
    units = 64 * 2.0 ** -24 * (mag + bias.abs().double() + want.abs())
    err = (got.double() - want).abs()
    n = B * oh * ow
    if odt == torch.float32:
        assert float((err / (2.0 ** -24 * want.abs() + units + 1e-30)).max()) <= 1.0
    else:
        assert float((err / (2.0 ** -8 * want.abs() + 1.1 * 7 * 2.0 ** -13 * mag + units + 1e-30)).max()) <= 1.0
        pix = torch.from_numpy(np.random.default_rng(case).choice(n, 32, replace=False)).to(DEV)
        peaks = Q.group_peaks(x, kernel, stride, pix)

        def some(v):
            return v.reshape(n, cout)[pix]
        assert float((some(err) / (2.0 ** -8 * some(want).abs() + 1.1 * 7 * 2.0 ** -13 * peaks + some(units) + 1e-30)).max()) <= 1.0
    for b in (0, B // 2, B - 1):
        one = layer(quantize_blocks(x[b:b + 1]), residual=None if res is None else res[b:b + 1], out_dtype=odt)
        assert torch.equal(got[b:b + 1], one)
