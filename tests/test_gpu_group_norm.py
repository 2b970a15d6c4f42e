"""Group norm + activation + dropout + shortcut and dropout alone, forward and backward, against the
64-bit restatement in oracle/group_norm_torch.py and the numpy Philox of oracle/random_np.py.

Bounds.  A result of type T is off by half a step, eps(T) / 2 relative, plus the fp32 arithmetic before
it.  The latter: t = gamma (x - mean) r + beta is made of terms of magnitude t_mag = |gamma| (|x| + |mean|) r
+ |beta|; a thread adds at most a few hundred of its values one after the other (sums about its first
value, then a tree), and exp / rcp of the activation add a few units and up to |t| <= 20 units through
the rounded argument: 512 units of 2^-24 of the magnitudes cover them.  The sums of the gradients run over
values of the magnitudes given by the oracle with the same count."""
import numpy as np
import pytest
import torch

from oracle import group_norm_torch as O
from oracle import random_np as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNITS = 512 * 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(shape, dtype, seed, mean=1.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = torch.randn(*shape, generator=g) * spread * (0.5 + torch.rand(c, generator=g)) + mean * torch.randn(c, generator=g)
    return (x.to(dtype), 1 + 0.3 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g),
            torch.randn(*shape, generator=g).to(dtype), torch.randn(*shape, generator=g).to(dtype))


def _within(name, got, want, mag, dtype):
    got = got.detach().double().cpu()
    err = (got - want).abs()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + UNITS * mag + 1e-30
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, "%s: %.3g of the bound, largest error %.3g" % (name, worst, float(err.max()))


def _keep(shape, rate, seed, call):
    n = int(np.prod(shape))
    return torch.from_numpy(R.keep_mask(0, n, rate, seed, call).copy()).reshape(shape)


CASES = [   # shape, groups, activation, shortcut, rate, type
    ((1, 13, 13, 1024), 32, "mish", False, 0.0, "bf16"),
    ((16, 13, 13, 512), 32, "mish", True, 0.0, "bf16"),
    ((3, 26, 26, 256), 32, "leaky", True, 0.2, "bf16"),
    ((2, 52, 52, 64), 16, "mish", True, 0.1, "bf16"),
    ((2, 52, 52, 128), 32, "mish", False, 0.0, "f32"),
    ((3, 19, 19, 255), 5, None, False, 0.0, "f32"),
    ((3, 19, 19, 255), 17, "mish", True, 0.5, "bf16"),
    ((2, 5, 7, 96), 32, "mish", True, 0.3, "bf16"),             # 3 channels per group
    ((1, 104, 104, 64), 32, "leaky", False, 0.0, "bf16"),
    ((2, 23, 31, 64), 1, "mish", True, 0.0, "bf16"),            # one group = layer statistics over the map
    ((4, 9, 9, 40), 40, "mish", False, 0.1, "f32"),             # one channel per group
    ((2, 6, 6, 1030), 5, "leaky", True, 0.1, "bf16"),           # channels in several blocks of scalar loads
    ((2, 3, 3, 2056), 8, None, True, 0.0, "bf16"),              # more than 256 vectors of channels
    ((1, 1, 1, 8), 8, "mish", False, 0.0, "bf16"),              # a group of one value: h = 0
    ((5, 1, 1, 32), 4, "mish", True, 0.0, "f32"),
    ((1, 2, 1, 1), 1, None, False, 0.0, "f32"),
    ((7, 48), 6, "leaky", False, 0.0, "bf16"),                  # [B, C]
    ((2, 4, 5, 6, 16), 2, "mish", True, 0.1, "bf16"),           # more than two pixel axes
    ((300, 4, 4, 32), 8, "mish", True, 0.1, "bf16"),            # many samples
    ((1, 208, 208, 32), 8, "mish", True, 0.1, "bf16"),
    ((2, 6, 7, 1023), 1, "mish", True, 0.1, "f32"),             # a group in four parts
    ((2, 40, 41, 771), 3, "leaky", False, 0.0, "bf16"),         # groups of 257: two parts each
    ((1, 9, 9, 4112), 1, "mish", False, 0.0, "bf16"),           # ... of vectors
    ((1, 4, 4, 6168), 8, "leaky", True, 0.0, "bf16"),           # 771 channels a group: no whole vectors
    ((1, 5, 5, 2400), 300, "mish", False, 0.1, "bf16"),         # more than 256 groups
    ((1, 77, 77, 1024), 1, "mish", True, 0.0, "bf16"),          # one wide group over many chunks
    ((2, 40, 41, 260), 13, "mish", True, 0.1, "bf16"),          # vectors of four
    ((3, 9, 11, 68), 17, "leaky", False, 0.3, "bf16"),
    ((2, 21, 20, 2052), 27, None, True, 0.0, "bf16"),           # ... in several blocks
    ((1, 30, 30, 1028), 1, "mish", True, 0.1, "bf16"),          # ... a group in parts of them
    ((5, 33, 31, 129), 43, "mish", True, 0.4, "f32"),           # single elements with dropout over several chunks
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_group_norm_act_forward_and_gradients(case):
    from yolo_amd import training as T
    shape, G, act, use_sc, rate, dt = CASES[case]
    dtype = DT[dt]
    x, ga, be, sc, dy = _case(shape, dtype, 100 + case)
    keep = _keep(shape, rate, 77, 2 ** 33 + case) if rate else None
    want = O.group_norm(x, ga, be, G, act, 1e-3, sc if use_sc else None, keep, rate, dy)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, ga, be)] + ([sc.to(DEV).requires_grad_(True)] if use_sc else [])
    state = torch.tensor([77, 2 ** 33 + case], device=DEV) if rate else None
    args = (G, act, leaves[3] if use_sc else None, 1e-3, rate, state)
    y = T.group_norm_act(*leaves[:3], *args)
    with torch.no_grad():
        plain = T.group_norm_act(*leaves[:3], *args)
    assert not plain.requires_grad and torch.equal(plain, y)
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    again = torch.autograd.grad(T.group_norm_act(*leaves[:3], *args), leaves, dy.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))                  # same bits every time
    assert y.dtype == dtype and grads[0].dtype == dtype and grads[1].dtype == torch.float32
    _within("y", y, want["y"], want["t_mag"] + want["y"].abs(), dtype)
    _within("dx", grads[0], want["dx"], want["dx_mag"], dtype)
    _within("dgamma", grads[1], want["dgamma"], want["dgamma_mag"], torch.float32)
    _within("dbeta", grads[2], want["dbeta"], want["dbeta_mag"], torch.float32)
    if use_sc:
        assert torch.equal(grads[3].cpu(), dy)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("mean,spread", [(300.0, 0.1), (0.0, 1e-4), (0.0, 1e4)])
def test_group_norm_far_mean_and_scales(dt, mean, spread):
    """A mean far from zero (the spread is then a few steps of bf16), values well below sqrt(eps), large values."""
    from yolo_amd import training as T
    x, ga, be, _, dy = _case((2, 40, 40, 64), DT[dt], 5, mean, spread)
    want = O.group_norm(x, ga, be, 8, "mish", 1e-3, dy=dy)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, ga, be)]
    y = T.group_norm_act(*leaves, 8, "mish")
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    _within("y", y, want["y"], want["t_mag"] + want["y"].abs(), DT[dt])
    for name, g in zip(("dx", "dgamma", "dbeta"), grads):
        _within(name, g, want[name], want[name + "_mag"], DT[dt] if name == "dx" else torch.float32)


def test_group_norm_constant_outlier_and_nan():
    from yolo_amd import training as T
    ga, be = torch.full((16,), 2.0, device=DEV), torch.linspace(-1, 1, 16, device=DEV)
    y = T.group_norm_act(torch.full((2, 9, 9, 16), 37.5, device=DEV), ga, be, 4)              # no spread: y = beta
    assert torch.equal(y, be.expand(2, 9, 9, 16))
    x = torch.randn(1, 40, 40, 16, generator=torch.Generator().manual_seed(1))
    x[0, 0, 0, 0] = 1e4                                                                         # the first value far off
    want = O.group_norm(x, ga.cpu(), be.cpu(), 4, None, 1e-3)
    _within("outlier", T.group_norm_act(x.to(DEV), ga, be, 4), want["y"], want["t_mag"], torch.float32)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z[0, 3, 5, 6] = bad
        y = T.group_norm_act(z.to(DEV), ga, be, 4, "mish").cpu()
        ok = T.group_norm_act(x.to(DEV), ga, be, 4, "mish").cpu()
        assert torch.isnan(y[..., 4:8]).any() and torch.equal(y[..., :4], ok[..., :4]) and torch.equal(y[..., 8:], ok[..., 8:])


@pytest.mark.parametrize("act", ["mish", None])
@pytest.mark.parametrize("size", [13, 40, 96])            # slabs, chunks, several chunks
def test_group_norm_non_finite_values_reach_their_group(size, act):
    """A NaN or an infinity makes the statistics of its sample and group NaN, hence y, dx and the parameters' gradients
    there (dbeta through the activation's derivative), and nothing else."""
    from yolo_amd import training as T
    g = torch.Generator().manual_seed(size)
    x, dy = torch.randn(2, size, size, 48, generator=g), torch.randn(2, size, size, 48, generator=g)
    ga, be = torch.ones(48), torch.zeros(48)

    def run(z):
        leaves = [t.to(DEV).requires_grad_() for t in (z, ga, be)]
        y = T.group_norm_act(*leaves, 6, act)
        return [t.detach().cpu() for t in (y, *torch.autograd.grad(y, leaves, dy.to(DEV)))]
    ok = run(x)
    for bad, pix in ((float("nan"), 0), (float("inf"), 1), (float("-inf"), size * size - 1), (float("inf"), size * size // 2)):
        z = x.clone()
        z.view(2, -1, 48)[1, pix, 19] = bad               # group 2 of sample 1: channels 16 ... 23
        y, dx, dga, dbe = run(z)
        for a, b in ((y, ok[0]), (dx, ok[1])):
            assert torch.isnan(a[1, ..., 16:24]).all()
            a[1, ..., 16:24] = b[1, ..., 16:24]
            assert torch.equal(a, b)
        assert torch.isnan(dga[16:24]).all() and torch.equal(dga[:16], ok[2][:16]) and torch.equal(dga[24:], ok[2][24:])
        assert (torch.isnan(dbe[16:24]).all() if act else torch.equal(dbe, ok[3])) and torch.equal(dbe[24:], ok[3][24:])


@pytest.mark.parametrize("samples,c,g", [(70000, 2048, 64), (1 << 20, 128, 4)])
def test_group_norm_many_samples_of_one_pixel(samples, c, g):
    """More channel slabs than a grid has room for: the chunked form takes them."""
    from yolo_amd import training as T
    x = torch.randn(samples, c, device=DEV).bfloat16()
    ga, be = torch.linspace(0.5, 1.5, c, device=DEV), torch.linspace(-1, 1, c, device=DEV)
    y = T.group_norm_act(x, ga, be, g)
    for part in (slice(0, 3), slice(samples // 2, samples // 2 + 3), slice(samples - 3, samples)):
        want = O.group_norm(x[part].float().cpu(), ga.cpu(), be.cpu(), g, None, 1e-3)
        _within("y", y[part], want["y"], want["t_mag"], torch.bfloat16)


@pytest.mark.parametrize("how", ["slice", "permuted", "offset", "expanded", "mixed"])
def test_group_norm_strides_and_alignment(how):
    """Inputs that are not dense or not 16-byte aligned give the bits of the dense copy."""
    from yolo_amd import training as T
    g = torch.Generator().manual_seed(3)
    base = torch.randn(2, 14, 15, 96, generator=g).bfloat16().to(DEV)
    ga, be = torch.randn(32, generator=g).to(DEV), torch.randn(32, generator=g).to(DEV)
    state = torch.tensor([1, 2], device=DEV)
    x = {"slice": base[..., 32:64], "permuted": base.permute(0, 2, 1, 3)[..., :32],
         "offset": torch.empty(2 * 14 * 15 * 32 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(2, 14, 15, 32).copy_(base[..., :32]),
         "expanded": base[:, :1, :, :32].expand(2, 14, 15, 32), "mixed": base[..., :32]}[how]
    sc = base[..., 64:].transpose(1, 2) if x.shape[1] == 15 else base[..., 64:]
    if how == "mixed":
        sc = sc.float()
    x, sc, gr = x.detach().requires_grad_(True), sc.detach().requires_grad_(True), ga[::1].detach().requires_grad_(True)
    y = T.group_norm_act(x, gr, be, 4, "mish", sc, rate=0.25, state=state)
    dy = torch.randn(1, 1, 1, 32, generator=g).bfloat16().to(DEV).expand_as(y)
    got = torch.autograd.grad(y, (x, gr, sc), dy)
    xc, scc, dyc = (t.detach().to(torch.bfloat16).contiguous().clone().requires_grad_(True) for t in (x, sc, dy))
    yc = T.group_norm_act(xc, gr, be, 4, "mish", scc, rate=0.25, state=state)
    want = torch.autograd.grad(yc, (xc, gr, scc), dyc.detach())
    assert y.is_contiguous() and torch.allclose(y, yc, rtol=2 ** -7, atol=1e-6)
    # (scalar accesses split the pixels among the threads otherwise: the sums differ in their last bits)
    for a, b in zip(got, want):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -7, atol=1e-4)
    if how != "offset":
        assert torch.equal(y, yc) and all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))


def test_group_norm_differences():
    """The gradients against central differences of the operator itself (fp32, the mask fixed by its state).
    Along v with step s the difference is off by s^2 / 6 times a third derivative (a few units here: h and mish
    are smooth, spread 1) and by 2^-24 * 512 / s of the summed magnitudes: at s = 2^-7 both stay below 1e-3 of the
    sum of |grad v|."""
    from yolo_amd import training as T
    x, ga, be, sc, dy = (t.to(DEV) for t in _case((2, 8, 8, 32), torch.float32, 11))
    state = torch.tensor([3, 4], device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, ga, be, sc)]

    def f(a, b, c, d):
        return T.group_norm_act(a, b, c, 4, "mish", d, rate=0.2, state=state)
    grads = torch.autograd.grad(f(*leaves), leaves, dy)
    s = 2.0 ** -7
    g = torch.Generator().manual_seed(1)
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=g).to(DEV)
        with torch.no_grad():
            hi, lo = [f(*[t + sign * s * v if j == i else t for j, t in enumerate(leaves)]).double() for sign in (1, -1)]
        diff = float(((hi - lo) * dy.double()).sum() / (2 * s))
        want = float((grads[i].double() * v.double()).sum())
        scale = float((grads[i].double() * v.double()).abs().sum())
        assert abs(diff - want) < 1e-3 * scale, (i, diff, want, scale)


def test_group_norm_beyond_32_bit_offsets():
    """More than 2^31 elements: the last group of the last sample against 64-bit arithmetic on that slice."""
    from yolo_amd import training as T
    P, C, G = 1050000, 1024, 32
    x = torch.empty((2, P, C), device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(1)
    for b in range(2):
        x[b].normal_(generator=g)
    ga, be = torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    y = T.group_norm_act(x, ga, be, G, "leaky")[1, :, -32:].double()
    t = x[1, :, -32:].double()
    del x
    t = (t - t.mean()) / torch.sqrt(t.var(unbiased=False) + 1e-3)
    want = torch.where(t > 0, t, 0.1 * t)
    assert float(((y - want).abs() / (2.0 ** -8 * want.abs() + UNITS * (1 + want.abs()))).max()) <= 1.0


def test_group_norm_backward_beyond_32_bit_offsets():
    """More than 2^31 elements, with dropout: dx of the last group of the last sample and the parameters' gradients of its channels,
    against 64-bit arithmetic on those slices (the mask as the forward pass shows it)."""
    from yolo_amd import training as T
    P, C, G, rate = 1050000, 1024, 32, 0.5
    g = torch.Generator(device=DEV).manual_seed(2)
    x, dy = (torch.empty((2, P, C), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    for b in range(2):
        x[b].normal_(generator=g)
        dy[b].normal_(generator=g)
    leaves = [x.requires_grad_(), torch.ones(C, device=DEV, requires_grad=True), torch.zeros(C, device=DEV, requires_grad=True)]
    y = T.group_norm_act(*leaves, G, "mish", rate=rate, state=torch.tensor([7, 8], device=DEV))
    keep = y.detach()[..., -32:] != 0
    dx, dgamma, dbeta = torch.autograd.grad(y, leaves, dy)
    del y
    sums = [0.0] * 4
    for b in range(2):
        h = x.detach()[b, :, -32:].double()
        h -= h.mean()
        r = 1.0 / torch.sqrt(h.square().mean() + 1e-3)
        h *= r
        m = torch.where(keep[b], dy[b, :, -32:].double() / (1 - rate), 0.0)
        dt = m * O.act_grad(h, "mish")
        mag = m.abs() * (1 + h.abs())
        for i, v in enumerate((dt * h, dt, mag * (1 + h.abs()), mag)):
            sums[i] = sums[i] + v.sum(0)
    want = r * (dt - dt.mean() - h * (dt * h).mean())
    mag = r * (1 + h.abs()) * (mag + mag.mean() + h.abs() * (mag * h.abs()).mean())
    err = (dx[1, :, -32:].double() - want).abs()
    assert float((err / (2.0 ** -8 * want.abs() + UNITS * mag)).max()) <= 1.0
    for got, want, mag in ((dgamma, sums[0], sums[2]), (dbeta, sums[1], sums[3])):
        assert float(((got[-32:].double() - want).abs() / (2.0 ** -24 * want.abs() + UNITS * mag)).max()) <= 1.0


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("n,dt,rate,use_sc", [(1, "f32", 0.5, False), (7, "bf16", 0.3, True), (4099, "bf16", 0.1, False),
                                              (8 * 19 * 19 * 255, "f32", 0.5, True), (1 << 20, "bf16", 0.25, True),
                                              (1001, "f32", 2.0 ** -32, False), (1001, "bf16", 0.9999, True)])
def test_dropout_values_and_gradients(n, dt, rate, use_sc):
    from yolo_amd import training as T
    dtype = DT[dt]
    g = torch.Generator().manual_seed(n)
    x, sc, dy = (torch.randn(n, generator=g).to(dtype) for _ in range(3))
    seed, call = -3, 2 ** 40 + 5                                                # every bit of both words counts
    keep = torch.from_numpy(R.keep_mask(0, n, rate, seed, call).copy())
    scale = np.float32(1.0 / (1.0 - rate))
    state = torch.tensor([seed, call], device=DEV)
    xg, sg = x.to(DEV).requires_grad_(True), sc.to(DEV).requires_grad_(True)
    y = T.dropout(xg, rate, state, shortcut=sg if use_sc else None)
    got = torch.autograd.grad(y, (xg, sg) if use_sc else (xg,), dy.to(DEV))
    kept = torch.where(keep, x.float() * float(scale), 0.0)                     # one fp32 product, (one fp32 sum,) one rounding
    want = (kept + sc.float() if use_sc else kept).to(dtype)
    assert torch.equal(y.detach().cpu(), want)
    assert torch.equal(got[0].cpu(), torch.where(keep, dy.float() * float(scale), 0.0).to(dtype))
    if use_sc:
        assert torch.equal(got[1].cpu(), dy)


def test_dropout_drops_non_finite_values_and_misaligned_views():
    from yolo_amd import training as T
    n = 4096
    state = torch.tensor([9, 1], device=DEV)
    keep = torch.from_numpy(R.keep_mask(0, n, 0.5, 9, 1).copy())
    x = torch.full((n,), float("inf"), device=DEV)
    x[1::2] = float("nan")
    y = T.dropout(x, 0.5, state).cpu()
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())
    z = torch.randn(n + 1, device=DEV)
    assert torch.equal(T.dropout(z[1:], 0.5, state), T.dropout(z[1:].clone(), 0.5, state))
    t = torch.randn(64, 64, device=DEV)
    assert torch.equal(T.dropout(t.t(), 0.5, state), T.dropout(t.t().contiguous(), 0.5, state))
    assert T.dropout(t[:0], 0.5, state).shape == (0, 64)


def test_dropout_beyond_32_bit_offsets():
    """Words behind element 2^32 use the counter's second word."""
    from yolo_amd import training as T
    n = 2 ** 32 + 1003
    x = torch.ones((n,), device=DEV, dtype=torch.bfloat16)
    y = T.dropout(x, 0.5, torch.tensor([5, 6], device=DEV))
    del x
    for a, b in ((0, 64), (2 ** 31 - 32, 2 ** 31 + 32), (2 ** 32 - 64, n)):
        assert np.array_equal(y[a:b].float().cpu().numpy() != 0, R.keep_mask(a, b - a, 0.5, 5, 6))


def test_dropout_layer_sequence():
    """Every active call draws another mask; inactive calls draw none; the state resumes from a state_dict."""
    from yolo_amd.layers import Dropout
    d = Dropout(0.5, seed=11).to(DEV)
    x = torch.ones(2, 8, 8, 64, device=DEV)
    assert d(x) is x and int(d.state[1]) == 0
    a = d(x, training=True)
    saved = {k: v.clone() for k, v in d.state_dict().items()}
    b = d(x, training=True)
    assert not torch.equal(a, b) and int(d.state[1]) == 2
    assert np.array_equal(a.cpu().numpy().reshape(-1) != 0, R.keep_mask(0, x.numel(), 0.5, 11, 0))
    assert np.array_equal(b.cpu().numpy().reshape(-1) != 0, R.keep_mask(0, x.numel(), 0.5, 11, 1))
    d.load_state_dict(saved)
    assert torch.equal(d(x, training=True), b)
    frac = float((a != 0).double().mean())
    assert abs(frac - 0.5) < 5 * 0.5 / x.numel() ** 0.5


# ---------------------------------------------------------------- layers, streams, graphs
def _block(drop=0.2):
    from yolo_amd.layers import ResidialBlock
    torch.manual_seed(5)
    blk = ResidialBlock(32, 64, groupNormalization=8, dropout=drop, dropout_seed=21, dtype=torch.bfloat16)
    blk.layer_stack[0].build(64)
    blk.layer_stack[1].build(32)
    with torch.no_grad():
        for conv in blk.layer_stack:
            conv.kernel.mul_(8.0)
            conv.gn.gamma.add_(0.1 * torch.randn(conv.filters))
            conv.gn.beta.add_(0.1 * torch.randn(conv.filters))
    return blk.to(DEV)


def _oracle_block(blk, x, call, dy, rate):
    """Convolutions in fp32 on the bf16 weights; every map that is stored is rounded to bf16 as stored."""
    from oracle import net_torch as N
    ps = []
    for conv in blk.layer_stack:
        ps.append([t.detach().float().cpu().clone().requires_grad_(True) for t in (conv.kernel, conv.gn.gamma, conv.gn.beta)])
    xo = x.float().cpu().clone().requires_grad_(True)

    class Round(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t.bfloat16().float()

        @staticmethod
        def backward(ctx, g):
            return g.bfloat16().float()
    t = xo
    for i, (kernel, ga, be) in enumerate(ps):
        k = kernel.shape[0]
        u = Round.apply(torch.nn.functional.conv2d(t.permute(0, 3, 1, 2), N.bf16_round(kernel).permute(3, 2, 0, 1), padding=k // 2).permute(0, 2, 3, 1))
        v = u.reshape(u.shape[0], -1, 8, u.shape[-1] // 8)
        h = (v - v.mean((1, 3), keepdim=True)) / torch.sqrt(v.var((1, 3), unbiased=False, keepdim=True) + 1e-3)
        t = O.act(h.reshape(u.shape) * ga + be, "mish")
        if i == 0:
            t = Round.apply(t)
    keep = torch.from_numpy(R.keep_mask(0, t.numel(), rate, 21, call).copy()).reshape(t.shape)
    y = torch.where(keep, t / (1 - rate), 0.0) + xo
    y.backward(dy.float().cpu())
    return y.detach(), xo.grad, ps


def test_residual_block_with_group_norm_and_dropout_trains():
    """conv -> group norm -> mish -> conv -> group norm -> mish -> dropout -> + x, forward and all gradients.
    2e-2 of each tensor's scale, the bar of the other block tests: stored maps are bf16, and a rounding that
    falls the other way (2^-8) passes through two normalisations and a sum over 9 x 32 taps."""
    from yolo_amd import training as T
    blk = _block()
    x = torch.randn(2, 12, 10, 64, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV).requires_grad_(True)
    dy = torch.randn(2, 12, 10, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    with T.backprop():
        y = blk(x)
    y.backward(dy)
    want, dx, ps = _oracle_block(blk, x.detach(), 0, dy, 0.2)

    def err(a, b):
        return float((a.detach().double().cpu() - b.double()).abs().max() / b.double().abs().max())
    errs = [err(y, want), err(x.grad, dx)]
    for conv, p in zip(blk.layer_stack, ps):
        errs += [err(conv.kernel.grad, p[0].grad), err(conv.gn.gamma.grad, p[1].grad), err(conv.gn.beta.grad, p[2].grad)]
    print("errors", errs)
    assert max(errs) < 2e-2
    # inference: no dropout, no graph, the same normalisation
    z = blk(x.detach())
    assert not z.requires_grad and int(blk.layer_stack[1].drop.state[1]) == 1
    with T.backprop():
        blk.layer_stack[1].drop.rate = 0.0
        assert err(blk(x), z.float().cpu()) < 2e-2


def test_dropout_after_plain_and_batch_norm_blocks():
    """YOLOConv(dropout=...) without group norm: the mask on act(conv) before the shortcut, in training only."""
    from yolo_amd import training as T
    from yolo_amd.layers import YOLOConv
    for bn in (False, True):
        torch.manual_seed(1)
        conv = YOLOConv((3, 3, 64), batchNormalization=bn, activation="leaky", dropout=0.4, dropout_seed=8, in_channels=64, dtype=torch.bfloat16).to(DEV)
        x = torch.randn(2, 9, 9, 64, device=DEV).bfloat16().requires_grad_(True)
        sc = torch.randn(2, 9, 9, 64, device=DEV).bfloat16().requires_grad_(True)
        rate, conv.drop.rate = conv.drop.rate, 0.0
        with T.backprop():
            plain = conv(x)
            conv.drop.rate = rate
            y = conv(x, residual=sc)
        keep = torch.from_numpy(R.keep_mask(0, y.numel(), rate, 8, 0).copy()).reshape(y.shape).to(DEV)
        want = (torch.where(keep, plain.float() * np.float32(1 / (1 - rate)), 0.0) + sc.float()).bfloat16()
        assert torch.equal(y, want)
        dy = torch.randn_like(y)
        got = torch.autograd.grad(y, (x, conv.kernel, sc), dy)
        ref = torch.autograd.grad(plain, (x, conv.kernel), torch.where(keep, dy.float() * np.float32(1 / (1 - rate)), 0.0).bfloat16())
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1]) and torch.equal(got[2], dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape,cin,cout,k", [((2, 12, 10), 64, 96, 3), ((1, 40, 41), 32, 64, 1)])
def test_group_norm_layer_with_a_32_bit_result(dtype, shape, cin, cout, k):
    """out_dtype=torch.float32: the normalisation of the convolution's own 32-bit result, not of one rounded to bf16 on the way."""
    from yolo_amd.layers import YOLOConv
    torch.manual_seed(3)
    conv = YOLOConv((k, k, cout), groupNormalization=8, activation="mish", in_channels=cin, dtype=dtype).to(DEV)
    linear = YOLOConv((k, k, cout), activation=None, in_channels=cin, dtype=dtype).to(DEV)
    with torch.no_grad():
        conv.kernel.mul_(8.0)
        conv.gn.gamma.add_(0.3 * torch.randn(cout, device=DEV))
        conv.gn.beta.add_(0.3 * torch.randn(cout, device=DEV))
        linear.kernel.copy_(conv.kernel)
    x = torch.randn(*shape, cin, device=DEV).bfloat16()
    sc = torch.randn(*shape, cout, device=DEV)
    u = linear(x, out_dtype=torch.float32)
    want = O.group_norm(u.cpu(), conv.gn.gamma.detach().cpu(), conv.gn.beta.detach().cpu(), 8, "mish", 1e-3, sc.cpu())
    y = conv(x, residual=sc, out_dtype=torch.float32)
    assert y.dtype == torch.float32
    _within("y", y, want["y"], want["t_mag"] + want["y"].abs() + sc.cpu().double().abs(), torch.float32)
    buf = torch.zeros(*shape, cout + 8, device=DEV)
    assert torch.equal(conv(x, residual=sc, out_dtype=torch.float32, out=buf[..., :cout]), y) and not buf[..., cout:].any()
    assert conv(x).dtype == torch.bfloat16                       # the default stays the map's type


def test_backbone_with_group_norm_and_dropout():
    """Darknet53(groupNormalization=, dropout=): one training step reaches every parameter, inference runs."""
    from yolo_amd import training as T
    from yolo_amd.backbones import Darknet53
    net = Darknet53(dtype=torch.bfloat16, seed=3, groupNormalization=32, dropout=0.1).to(DEV)
    x = torch.rand(1, 64, 64, 3, device=DEV)
    with T.backprop():
        ys = net(x)
    sum(y.float().square().mean() for y in ys).backward()
    ps = list(net.parameters())
    assert len(ps) == 52 * 3 and all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in ps)
    drops = [b.layer_stack[1].drop for s in (net.layer_stack_1, net.layer_stack_2, net.layer_stack_3) for b in s if hasattr(b, "layer_stack")]
    assert len(drops) == 23 and len({int(d.state[0]) for d in drops}) == 23 and all(int(d.state[1]) == 1 for d in drops)
    out = net(x)
    assert all(bool(torch.isfinite(o.float()).all()) for o in out) and not out[0].requires_grad


def test_second_stream_and_two_calls_at_once():
    from yolo_amd import training as T
    x, ga, be, sc, _ = (t.to(DEV) for t in _case((4, 52, 52, 128), torch.bfloat16, 1))
    want = T.group_norm_act(x, ga, be, 32, "mish", sc)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(T.group_norm_act(x, ga, be, 32, "mish", sc))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_training_step_in_a_graph():
    """Forward and backward of the block captured once and replayed with other inputs between eager work:
    every replay equals the eager step from the same state, and draws its own mask."""
    from yolo_amd import training as T
    blk = _block()
    params = list(blk.parameters())
    xs = [torch.randn(2, 12, 10, 64, generator=torch.Generator().manual_seed(40 + i)).bfloat16().to(DEV) for i in range(4)]
    dy = torch.randn(2, 12, 10, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)

    def step(x):
        with T.backprop():
            y = blk(x)
        return [y.detach()] + list(torch.autograd.grad(y, [x] + params, dy))
    eager = []
    for i, x in enumerate(xs):
        eager.append([t.clone() for t in step(x.clone().requires_grad_(True))])
    assert int(blk.layer_stack[1].drop.state[1]) == 4
    static = xs[0].clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(static)
    drop = blk.layer_stack[1].drop
    drop.state[1] = 0
    for i, x in enumerate(xs):
        with torch.no_grad():
            static.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert int(drop.state[1]) == i + 1
        for a, b in zip(out, eager[i]):
            assert torch.equal(a, b), i
        torch.ones(1000, device=DEV).sum().item()                    # eager work between the replays


@pytest.mark.parametrize("shape,groups,dt", [((1, 207, 207, 593), 1, "f32"), ((64, 26, 26, 512), 32, "f32"), ((16, 104, 104, 128), 32, "bf16"),
                                             ((4, 150, 150, 260), 13, "bf16")])
def test_leaky_derivative_is_taken_on_the_right_side_of_zero(shape, groups, dt):
    """dbeta for dy = 1 counts the elements on each side of t = 0 (weights 1 and 0.1): against 64-bit signs no channel of
    millions of elements is off by one of them, 0.9 (the sum of 43 thousand rounds to 0.004 at most)."""
    from yolo_amd import training as T
    c = shape[-1]
    g = torch.Generator().manual_seed(c)
    x = (torch.randn(shape, generator=g) + 0.25).to(DT[dt]).to(DEV)
    ga, be = torch.randn(c, generator=g).to(DEV), torch.randn(c, generator=g).to(DEV).requires_grad_()
    dbeta, = torch.autograd.grad(T.group_norm_act(x, ga, be, groups, "leaky").float().sum(), [be]) if dt == "f32" else \
        torch.autograd.grad(T.group_norm_act(x, ga, be, groups, "leaky"), [be], torch.ones_like(x))
    want = torch.zeros(c, dtype=torch.float64, device=DEV)
    for b in range(shape[0]):
        z = x[b].double().reshape(-1, groups, c // groups)
        mean, var = z.mean((0, 2), keepdim=True), z.var((0, 2), unbiased=False, keepdim=True)
        t = ((z - mean) / torch.sqrt(var + 1e-3)).reshape(-1, c) * ga.double() + be.detach().double()
        want += torch.where(t > 0, 1.0, 0.1).sum(0, dtype=torch.float64)
    assert float((dbeta.double() - want).abs().max()) < 0.45


@pytest.mark.parametrize("far", [1.0, 100.0, 1000.0])
@pytest.mark.parametrize("shape,groups,dt", [((2, 26, 26, 256), 16, "bf16"), ((2, 26, 26, 256), 16, "f32"), ((2, 104, 104, 64), 4, "bf16"),
                                             ((2, 40, 41, 260), 13, "bf16"), ((2, 52, 52, 128), 2, "f32"), ((2, 40, 41, 255), 5, "f32")])
def test_leaky_derivative_with_a_mean_far_from_zero(shape, groups, dt, far):
    """The sign of t where the mean is `far` spreads from zero.  beta is chosen, channel by channel, so that one value of the map
    has a t of about 1e-7: above what the kept statistics may be off by, below what fp32 ones would be off by (2^-24 far / sqrt 3
    a rounding: 3e-6 at 100).
    Their error, at its largest here (26^2, 16 channels a group): fp32 sums of a wave's 85 pixels of a channel about the first
    pixel's value, which is one spread off the mean, so that k values add up to k spreads and each addition rounds by 2^-24 /
    sqrt 3 of that: eleven in a row in each of eight lanes, then their tree, sqrt(8 * 11^3 / 3 + 4 * 22^2 + 2 * 44^2 + 88^2) = 131,
    4.5e-6 spreads.  128 of those sums make a group of 10816 values: 4.5e-6 sqrt(128) / 10816 = 5e-9 of a spread; the
    squares' sum is off by the same part of itself.  Eight times that, 4e-8 (|gamma| + |beta|), is not asked about."""
    from yolo_amd import training as T
    c, d = shape[-1], shape[-1] // groups
    g = torch.Generator().manual_seed(int(far) + c)
    x = (torch.randn(shape, generator=g) + far).to(DT[dt])
    ga = (0.5 + torch.rand(c, generator=g)) * torch.where(torch.rand(c, generator=g) < 0.5, -1.0, 1.0)
    xd = x.double().reshape(shape[0], -1, groups, d)
    mean = xd.mean((1, 3), keepdim=True)
    r = 1.0 / torch.sqrt((xd - mean).square().mean((1, 3), keepdim=True) + 1e-3)
    h = ((xd - mean) * r).reshape(shape[0], -1, c)
    near = h[0].abs().argmin(0)                                # one pixel a channel: the value of sample 0 next to the mean
    aim = -ga.double() * h[0, near, torch.arange(c)]
    be = (aim + (1.0 + aim.abs()) * 1e-7 * torch.where(torch.arange(c) % 2 == 0, 1.0, -1.0)).float()
    t = ga.double() * h + be.double()
    asked = t.abs() > 4e-8 * (ga.double().abs() + be.double().abs())
    assert int((asked & (t.abs() < 3e-7)).sum()) >= c // 2      # what the test is about
    leaves = [v.to(DEV).requires_grad_() for v in (x, ga, be)]
    y = T.group_norm_act(*leaves, groups, "leaky")
    dx, _, dbeta = torch.autograd.grad(y, leaves, torch.ones_like(y))
    dt_ = torch.where(t > 0, 1.0, 0.1).double()
    gd = (ga.double() * dt_).reshape(xd.shape)
    hg = h.reshape(xd.shape)
    want = r * (gd - gd.mean((1, 3), keepdim=True) - hg * (gd * hg).mean((1, 3), keepdim=True))
    off = ((dx.double().cpu().reshape(xd.shape) - want) / (r * ga.double().abs().reshape(1, 1, groups, d))).abs().reshape(t.shape)
    wrong = int((asked & (off > 0.45)).sum())                  # a wrong sign: 0.9
    assert wrong == 0, wrong
    whole = asked.all((0, 1))
    assert float((dbeta.double().cpu() - dt_.sum((0, 1)))[whole].abs().max()) < 0.45


def _zero_leaky(shape, kind, dtype):
    """Leaves with t = 0 in every element: gamma = beta = 0 (a residual branch that starts as zero), or an empty map with beta = 0."""
    c = shape[-1]
    g = torch.Generator(device=DEV).manual_seed(c)
    x = torch.zeros(shape, device=DEV) if kind == "map" else torch.randn(shape, device=DEV, generator=g)
    ga = torch.zeros(c, device=DEV) if kind == "parameters" else torch.randn(c, device=DEV, generator=g)
    return [x.to(dtype).requires_grad_(), ga.requires_grad_(), torch.zeros(c, device=DEV, requires_grad=True)]


@pytest.mark.parametrize("kind", ["parameters", "map"])
@pytest.mark.parametrize("shape,groups,dt", [((2, 13, 13, 256), 32, "bf16"), ((2, 104, 104, 64), 8, "bf16"), ((3, 19, 19, 255), 5, "f32")])
def test_leaky_derivative_at_zero(shape, groups, dt, kind):
    from yolo_amd import training as T
    leaves = _zero_leaky(shape, kind, DT[dt])
    dy = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(DT[dt])
    want = O.group_norm(*(t.detach().cpu() for t in leaves), groups, "leaky", 1e-3, dy=dy)
    got = torch.autograd.grad(T.group_norm_act(*leaves, groups, "leaky"), leaves, dy.to(DEV))
    for name, v in zip(("dx", "dgamma", "dbeta"), got):
        _within(name, v, want[name], want[name + "_mag"], DT[dt] if name == "dx" else torch.float32)


@pytest.mark.parametrize("shape,groups,dt", [((3, 13, 13, 256), 16, "bf16"), ((3, 13, 13, 128), 8, "f32"), ((2, 40, 41, 96), 32, "f32"),
                                             ((2, 104, 104, 64), 4, "bf16"), ((2, 19, 19, 255), 5, "f32"), ((1, 77, 77, 1024), 1, "f32")])
def test_leaky_derivative_of_a_constant_map(shape, groups, dt):
    """A map without spread is its own mean exactly, whatever the value (1 / n and sums of n values are not exact): with beta = 0 every
    t is 0, on the side of the slope 0.1."""
    from yolo_amd import training as T
    c = shape[-1]
    g = torch.Generator().manual_seed(c)
    value = torch.rand(groups, generator=g).repeat_interleave(c // groups)
    x = (torch.zeros(shape) + 10.0 * value).to(DT[dt]).to(DEV)
    be = torch.zeros(c, device=DEV, requires_grad=True)
    ga = torch.randn(c, generator=g).to(DEV)
    dbeta, = torch.autograd.grad(T.group_norm_act(x, ga, be, groups, "leaky"), [be], torch.ones_like(x))
    n = x.numel() // c
    assert torch.allclose(dbeta, torch.full_like(dbeta, 0.1 * n), rtol=1e-5), (dbeta / n)


@pytest.mark.parametrize("kind", ["parameters", "map"])
def test_leaky_backward_at_zero_is_as_fast(kind):
    """Signs of t = 0 need no second look: the backward step over such a map takes the time of any other (a factor of two
    leaves room for the clock)."""
    from yolo_amd import training as T
    shape = (16, 208, 208, 64)
    dy = torch.randn(shape, device=DEV).bfloat16()

    def micros(leaves):
        y = T.group_norm_act(*leaves, 32, "leaky")
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            torch.autograd.grad(y, leaves, dy, retain_graph=True)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 1e3)
        return sorted(times)[4]
    plain = [torch.randn(shape, device=DEV).bfloat16().requires_grad_()] + [torch.randn(64, device=DEV, requires_grad=True) for _ in range(2)]
    usual, zero = micros(plain), micros(_zero_leaky(shape, kind, torch.bfloat16))
    print("us: usual %.0f, t = 0 %.0f" % (usual, zero))
    assert zero < 2 * usual


def test_gradients_share_no_memory():
    """backward() into leaves, the shortcut among them: no .grad lies in the caller's dy or in another one, and a second
    backward() over the kept graph adds the same again."""
    from yolo_amd import training as T
    for use in (lambda x, s: T.group_norm_act(x, ga, be, 4, "mish", s), lambda x, s: T.dropout(x, 0.25, torch.tensor([1, 2], device=DEV), s)):
        ga, be = torch.ones(32, device=DEV, requires_grad=True), torch.zeros(32, device=DEV, requires_grad=True)
        x, s = (torch.randn(2, 5, 5, 32, device=DEV).requires_grad_() for _ in range(2))
        dy = torch.randn(2, 5, 5, 32, device=DEV)
        kept = dy.clone()
        y = use(x, s)
        y.backward(dy, retain_graph=True)
        assert len({t.data_ptr() for t in (dy, x.grad, s.grad, x, s, y)}) == 6 and torch.equal(s.grad, dy)
        first = x.grad.clone()
        s.grad.mul_(3.0)
        assert torch.equal(dy, kept)
        y.backward(dy)
        assert torch.equal(x.grad, first + first) and torch.equal(s.grad, 3.0 * kept + kept)
        with pytest.raises(RuntimeError, match="second time"):
            y.backward(dy)


def test_a_changed_state_is_noticed():
    """The backward pass computes the mask from the state again: autograd refuses one that was written to in between."""
    from yolo_amd import training as T
    x = torch.randn(2, 4, 4, 32, device=DEV, requires_grad=True)
    ga, be = torch.ones(32, device=DEV), torch.zeros(32, device=DEV)
    state = torch.tensor([1, 2], device=DEV)
    for y in (T.group_norm_act(x, ga, be, 4, None, rate=0.5, state=state), T.dropout(x, 0.5, state)):
        state.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.parametrize("size", [13, 60])
def test_inside_an_activation_checkpoint(size):
    """A segment run again in the backward pass, its state drawn outside: the gradients of the plain call."""
    from torch.utils.checkpoint import checkpoint
    from yolo_amd import training as T
    from yolo_amd.layers import Dropout
    x, ga, be, sc, dy = (t.to(DEV) for t in _case((2, size, size, 64), torch.float32, 3))
    drop = Dropout(0.3, seed=5).to(DEV)
    leaves = [t.requires_grad_() for t in (x, ga, be, sc)]
    one, two = drop.draw(), drop.draw()

    def segment(a, b, c, d):
        return T.dropout(T.group_norm_act(a, b, c, 8, "mish", d, rate=0.2, state=one), 0.3, two)
    want = torch.autograd.grad(segment(*leaves), leaves, dy)
    got = torch.autograd.grad(checkpoint(segment, *leaves, use_reentrant=False), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(drop.state[1]) == 2


def test_second_derivatives_are_refused():
    from yolo_amd import training as T
    x = torch.randn(2, 4, 4, 32, device=DEV, requires_grad=True)
    ga, be = torch.ones(32, device=DEV, requires_grad=True), torch.zeros(32, device=DEV, requires_grad=True)
    for y in (T.group_norm_act(x, ga, be, 4, "mish"), T.dropout(x, 0.5, torch.tensor([1, 2], device=DEV))):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_partial_gradients_and_empty_batches():
    from yolo_amd import training as T
    x = torch.randn(2, 6, 6, 32, device=DEV)
    ga, be = torch.randn(32, device=DEV, requires_grad=True), torch.randn(32, device=DEV, requires_grad=True)
    y = T.group_norm_act(x, ga, be.detach(), 4, "mish", shortcut=x)
    (only,) = torch.autograd.grad(y.sum(), ga)
    full = torch.autograd.grad(T.group_norm_act(x, ga, be, 4, "mish").sum(), (ga, be))
    assert torch.equal(only, full[0])
    s = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(T.group_norm_act(x, ga.detach(), be.detach(), 4, shortcut=s).sum(), s)[0], torch.ones_like(x))
    e = torch.empty(0, 6, 6, 32, device=DEV, requires_grad=True)
    y = T.group_norm_act(e, ga, be, 4, "mish")
    got = torch.autograd.grad(y.sum(), (e, ga, be))
    assert y.shape == e.shape and got[0].shape == e.shape and not got[1].any() and not got[2].any()
    half = T.group_norm_act(x, ga.to(torch.bfloat16), be, 4)                        # parameters of another type: gradients of theirs
    p = ga.detach().to(torch.bfloat16).requires_grad_(True)
    assert torch.autograd.grad(T.group_norm_act(x, p, be, 4).sum(), p)[0].dtype == torch.bfloat16 and half.dtype == torch.float32
