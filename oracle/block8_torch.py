"""Block-scaled e4m3 numbers and the convolution of them, in 64 bits."""
import torch


def quantise(x):
    """x [..., C] -> (values it is held as, in double; exponents k [..., ceil(C / 128)]).  e4m3: four significant
    bits, steps of 2^-9 below 2^-6, largest 448; NaN and infinities become NaN."""
    x = x.double()
    c = x.shape[-1]
    nb = -(-c // 128)
    p = torch.zeros(x.shape[:-1] + (nb * 128,), dtype=torch.float64, device=x.device)
    p[..., :c] = x
    p = p.reshape(x.shape[:-1] + (nb, 128))
    fin = torch.isfinite(p)
    top = torch.where(fin, p.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(top)                                   # top = m 2^e, 0.5 <= m < 1; 448 = 0.875 2^9
    k = torch.where(top > 0, e - 9 + (m > 0.875).int(), 0).clamp_min(-126)
    v = p * torch.exp2(-k.double())
    step = torch.exp2(torch.frexp(torch.where(fin, v, 1.0))[1].clamp_min(-5).double() - 4.0)
    q = torch.round(v / step) * step                          # halves to even
    q = torch.where(fin, q * torch.exp2(k.double()), float("nan"))
    return q.reshape(x.shape[:-1] + (nb * 128,))[..., :c], k[..., 0]


def taps(x, k, stride):
    """[taps][B, OH, OW, C]: the input pixel of every output pixel under each tap (layers.py:46-57)."""
    b, h, w, c = x.shape
    lo = 1 if stride == 2 else (k - 1) // 2
    hi = 0 if stride == 2 else (k - 1) // 2
    p = torch.nn.functional.pad(x, (0, 0, lo, hi, lo, hi))
    oh, ow = (h, w) if stride == 1 else ((h + 1 - k) // 2 + 1, (w + 1 - k) // 2 + 1)
    return [p[:, r:r + stride * (oh - 1) + 1:stride, s:s + stride * (ow - 1) + 1:stride] for r in range(k) for s in range(k)]


def conv(x, kernel, stride):
    """(sum, sum of magnitudes) of the quantised operands' products, [B, OH, OW, Cout] in double."""
    k, _, cin, cout = kernel.shape
    wq = quantise(kernel.permute(0, 1, 3, 2))[0].permute(0, 1, 3, 2).reshape(k * k, cin, cout)
    xq = quantise(x)[0]
    total = mag = None
    for t, xt in enumerate(taps(xq, k, stride)):
        rows = xt.reshape(-1, cin)
        a, m = rows @ wq[t], rows.abs() @ wq[t].abs()
        total, mag = (a, m) if total is None else (total + a, mag + m)
    b, oh, ow = taps(xq[..., :1], k, stride)[0].shape[:3]
    return total.reshape(b, oh, ow, cout), mag.reshape(b, oh, ow, cout)


def group_peaks(x, kernel, stride, pixels):
    """For the given output pixels (flat indexes): the sum over groups of eight neighbouring channels of one tap of
    the group's largest product magnitude, [len(pixels), Cout]."""
    k, _, cin, cout = kernel.shape
    wq = quantise(kernel.permute(0, 1, 3, 2))[0].permute(0, 1, 3, 2).reshape(k * k, cin, cout).abs()
    out = 0.0
    for t, xt in enumerate(taps(quantise(x)[0], k, stride)):
        rows = xt.reshape(-1, cin)[pixels].abs()
        out = out + (rows[:, :, None] * wq[t][None]).reshape(len(pixels), cin // 8, 8, cout).amax(2).sum(1)
    return out
