"""Calls of the training and 8-bit operators, for timing and for comparing their results.

    group_norm   training.group_norm_act: group norm over channels-last maps, activation, dropout and shortcut in one
                 operator; forward alone (a frozen network on single images) and with its gradients (a training step)
    dropout      training.dropout: dropout whose mask is computed from (seed, call number), alone or before a shortcut add,
                 with its gradient
    conv8        layers.YOLOConv(dtype=torch.float8_e4m3fn): the convolution block as a matrix product of 8-bit floating
                 point numbers with one power-of-two scale for each block of 128 channels; the input map is quantised
                 within the call

`own` chooses who computes: this package's kernels, or the plain torch form of the same formulas in 32 bits.
Map sizes and channel counts are those of Darknet53 / YoloV3 at 416 x 416 and 608 x 608.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-3


# ---------------------------------------------------------------- cases
def _gn(name, B, S, C, G, act, dtype="bf16", train=True, shortcut=False, rate=0.0):
    return dict(name=name, op="group_norm", B=B, S=S, C=C, G=G, act=act, dtype=dtype, train=train, shortcut=shortcut, rate=rate)


def _dr(name, B, S, C, rate, dtype="bf16", shortcut=False):
    return dict(name=name, op="dropout", B=B, S=S, C=C, rate=rate, dtype=dtype, shortcut=shortcut)


def _cv(name, B, S, Cin, Cout, k, stride, act, out="bf16", shortcut=False):
    return dict(name=name, op="conv8", B=B, S=S, Cin=Cin, Cout=Cout, k=k, stride=stride, act=act, out=out, shortcut=shortcut)


def listed():
    return [
        # one image through the deepest map of the backbone: a call that is all latency
        _gn("norm image 13", 1, 13, 1024, 32, "mish", train=False),
        # eight 608 x 608 images in inference, second half of a residual block
        _gn("norm images 76", 8, 76, 256, 32, "mish", train=False, shortcut=True),
        # training step of a residual block of the 52 x 52 stage, a small batch per GPU
        _gn("norm train 52", 16, 52, 256, 32, "mish", shortcut=True),
        # training step of the widest early map, regularised: the largest group norm
        _gn("norm train 208 dropout", 16, 208, 64, 32, "leaky", shortcut=True, rate=0.1),
        # channels that divide by neither 8 nor a power of two, 32-bit, as on the 255-channel maps of 80 classes
        _gn("norm train 255 f32", 3, 19, 255, 5, None, dtype="f32"),
        # dropout of one image's deepest map
        _dr("dropout 13", 1, 13, 512, 0.1),
        # dropout before the shortcut add of the 26 x 26 stage, a full training batch
        _dr("dropout 26 shortcut", 64, 26, 512, 0.2, shortcut=True),
        # 32-bit, an odd number of elements
        _dr("dropout 255 f32", 5, 19, 255, 0.5, dtype="f32"),
        # 1 x 1 block of the head for a single image: latency
        _cv("conv8 image 1x1", 1, 13, 1024, 512, 1, 1, "mish"),
        # linear output layer of the head, 3 * (80 + 5) channels, 32-bit logits
        _cv("conv8 logits 255", 8, 26, 1024, 255, 1, 1, None, out="f32"),
        # stage entry: stride 2
        _cv("conv8 3x3 stride 2", 16, 104, 128, 256, 3, 2, "mish"),
        # the head's widest layer at the benchmark's batch of 64: most of the detector's arithmetic
        _cv("conv8 3x3 wide", 64, 52, 512, 1024, 3, 1, "mish"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "dropout", "conv8", "conv8"])
    act = rng.choice(["mish", "mish", "leaky", None])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    B, S = _log_int(rng, 1, 64), _log_int(rng, 7, 208)
    if op == "conv8":
        k, stride = rng.choice([(1, 1), (1, 1), (3, 1), (3, 1), (3, 2)])
        Cin = 16 * _log_int(rng, 2, 64)
        Cout = rng.choice([_log_int(rng, 32, 1024), 32 * rng.randint(1, 32), 128 * rng.randint(1, 8), 255])
        while B > 1 and (B * S * S * Cin > 64 * 52 * 52 * 512 or B * S * S * Cout > 64 * 52 * 52 * 512):
            B = (B + 1) // 2
        return dict(op=op, B=B, S=S, Cin=Cin, Cout=Cout, k=k, stride=stride, act=act, out=rng.choice(["bf16", "bf16", "f32"]),
                    shortcut=rng.random() < 0.3)
    if op == "dropout":
        C = _log_int(rng, 16, 1024)
        while B > 1 and B * S * S * C > 64 * 26 * 26 * 512:
            B = (B + 1) // 2
        while B * S * S * C > 64 * 26 * 26 * 512:
            C = (C + 1) // 2
        return dict(op=op, B=B, S=S, C=C, rate=rng.choice([0.1, 0.2, 0.5]), dtype=dtype, shortcut=rng.random() < 0.5)
    G = rng.choice([1, 4, 8, 16, 32, 5, 17])
    C = G * max(1, _log_int(rng, 16, 1024) // G)
    while B > 1 and B * S * S * C > 16 * 208 * 208 * 64:
        B = (B + 1) // 2
    while B * S * S * C > 16 * 208 * 208 * 64:
        C = G * max(1, C // G // 2)
    return dict(op=op, B=B, S=S, C=C, G=G, act=act, dtype=dtype, train=rng.random() < 0.7, shortcut=rng.random() < 0.5,
                rate=rng.choice([0.0, 0.0, 0.1, 0.3]))


def _out_size(c):
    return c["S"] if c["stride"] == 1 else (c["S"] + 1 - c["k"]) // 2 + 1


# ---------------------------------------------------------------- inputs
def _inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device=DEV, generator=gen)

    if c["op"] == "conv8":
        B, S, ci, co, k = c["B"], c["S"], c["Cin"], c["Cout"], c["k"]
        u = randn(B, S, S, ci)
        u.mul_(0.5 + rand(ci)).add_(0.5 * randn(ci))
        x = (u * torch.tanh(torch.nn.functional.softplus(u))).to(torch.bfloat16)          # what a mish layer leaves
        w = randn(k, k, ci, co) * (1.0 / math.sqrt(k * k * ci))
        bias = 0.05 * randn(co)
        out = DTYPES[c["out"]]
        oh = _out_size(c)
        sc = randn(B, oh, oh, co).to(out) if c["shortcut"] else None
        return dict(x=x, kernel=w, bias=bias, shortcut=sc)
    dt = DTYPES[c["dtype"]]
    B, S, C = c["B"], c["S"], c["C"]
    x = randn(B, S, S, C)
    x.mul_(0.5 + rand(C)).add_(randn(C))                                                    # channels differ in mean and spread
    d = dict(x=x.to(dt), dy=(0.1 * randn(B, S, S, C)).to(dt))
    d["shortcut"] = randn(B, S, S, C).to(dt) if c["shortcut"] else None
    if c["op"] == "group_norm":
        d["gamma"] = 1.0 + 0.2 * randn(C)
        d["beta"] = 0.2 * randn(C)
    d["state"] = torch.tensor([seed * 7919 + 12345, seed + 3], dtype=torch.int64, device=DEV)   # (seed, call number)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if own and case["op"] == "conv8":
        from yolo_amd.layers import YOLOConv
        k = case["k"]
        layer = YOLOConv((k, k, case["Cout"]), downsample=case["stride"] == 2, activation=case["act"],
                         dtype=torch.float8_e4m3fn, in_channels=case["Cin"]).to(DEV)
        layer.load_reference_params({"kernel": d["kernel"], "bias": d["bias"]})
        d["layer"] = layer
    if own and case["op"] != "conv8":
        for name in ("x", "shortcut", "gamma", "beta"):
            if d.get(name) is not None and (case["op"] == "dropout" or case["train"]):
                d[name].requires_grad_(True)
    return d


# ---------------------------------------------------------------- plain forms
def _act(t, act):
    if act == "mish":
        return t * torch.tanh(torch.log1p(torch.exp(-t.abs())) + t.clamp_min(0))
    if act == "leaky":
        return torch.where(t > 0, t, 0.1 * t)
    return t


def _act_grad(t, act):
    if act == "mish":
        w = torch.tanh(torch.log1p(torch.exp(-t.abs())) + t.clamp_min(0))
        return w + t * (1 - w * w) / (1 + torch.exp(-t))
    if act == "leaky":
        return torch.where(t > 0, 1.0, 0.1)
    return torch.ones_like(t)


def _philox(n, state):
    """n 32-bit words (in int64) of Philox4x32-10: words 4 j .. 4 j + 3 belong to counter (j, call), the key is the seed."""
    M, LOW = (0xD2511F53, 0xCD9E8D57), 0xFFFFFFFF
    j = torch.arange((n + 3) // 4, device=state.device, dtype=torch.int64)
    seed, call = state[0], state[1]
    c0, c1, c2, c3 = j & LOW, j >> 32, (call & LOW).expand_as(j), ((call >> 32) & LOW).expand_as(j)
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        p0, p1 = c0 * M[0], c2 * M[1]                       # the low 64 bits of the product, as the wrapped int64 holds them
        c0, c1, c2, c3 = ((p1 >> 32) & LOW) ^ c1 ^ k0, p1 & LOW, ((p0 >> 32) & LOW) ^ c3 ^ k1, p0 & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]


def _keep(shape, rate, state):
    n = 1
    for s in shape:
        n *= s
    return (_philox(n, state) >= int(rate * 2 ** 32)).reshape(shape)


def _plain_group_norm(s):
    c = s["case"]
    dt, act, rate = DTYPES[c["dtype"]], c["act"], c["rate"]
    B, C, G = c["B"], c["C"], c["G"]
    x = s["x"].float().reshape(B, -1, G, C // G)
    mean = x.double().mean((1, 3), keepdim=True).float()
    var = (x - mean).square().mean((1, 3), keepdim=True)
    r = 1.0 / torch.sqrt(var + EPS)
    h = (x - mean) * r
    gamma, beta = s["gamma"].reshape(G, -1), s["beta"].reshape(G, -1)
    t = gamma * h + beta
    y = _act(t, act)
    if rate > 0:
        keep = _keep(x.shape, rate, s["state"])
        y = torch.where(keep, y * (1.0 / (1.0 - rate)), 0.0)
    y = y.reshape(s["x"].shape)
    if s["shortcut"] is not None:
        y = y + s["shortcut"].float()
    y = y.to(dt)
    if not c["train"]:
        return y
    d = s["dy"].float().reshape(x.shape)
    if rate > 0:
        d = torch.where(keep, d * (1.0 / (1.0 - rate)), 0.0)
    d = d * _act_grad(t, act)
    dbeta = d.sum((0, 1), dtype=torch.float64).float().reshape(-1)
    dgamma = (d * h).sum((0, 1), dtype=torch.float64).float().reshape(-1)
    gd = gamma * d
    n = x.shape[1] * x.shape[3]
    dx = r * (gd - (gd.sum((1, 3), keepdim=True) + h * (gd * h).sum((1, 3), keepdim=True)) / n)
    out = [y, dx.reshape(s["x"].shape).to(dt), dgamma, dbeta]
    return out + [s["dy"]] if s["shortcut"] is not None else out


def _plain_dropout(s):
    c = s["case"]
    dt, rate = DTYPES[c["dtype"]], c["rate"]
    keep = _keep(s["x"].shape, rate, s["state"])
    y = torch.where(keep, s["x"].float() * (1.0 / (1.0 - rate)), 0.0)
    if s["shortcut"] is not None:
        y = y + s["shortcut"].float()
    out = [y.to(dt), torch.where(keep, s["dy"].float() * (1.0 / (1.0 - rate)), 0.0).to(dt)]
    return out + [s["dy"]] if s["shortcut"] is not None else out


def _quantised(x):
    """x [..., C] in 32 bits -> the values its 8-bit form stands for: q * 2^k with, for each block of 128 channels, the
    smallest integer k (>= -126) for which the largest magnitude is at most 448 * 2^k, and q = x / 2^k rounded to e4m3."""
    C = x.shape[-1]
    out = torch.empty_like(x)
    for c0 in range(0, C, 128):
        b = x[..., c0:c0 + 128]
        m, e = torch.frexp(b.abs().amax(-1, keepdim=True))              # largest = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
        k = torch.where(m > 0, e - 9 + (m > 0.875), 0).clamp_min(-126)
        q = torch.ldexp(b, -k).to(torch.float8_e4m3fn).float()
        out[..., c0:c0 + 128] = torch.ldexp(q, k)
    return out


def _taps(c, x):
    """The input pixel of every output pixel, tap by tap: [B, OH, OW, Cin] for tap (r, s) of the k x k kernel."""
    k, stride, S = c["k"], c["stride"], c["S"]
    lo = 1 if stride == 2 else (k - 1) // 2
    hi = 0 if stride == 2 else (k - 1) // 2
    oh = _out_size(c)
    if lo or hi:
        p = torch.zeros((x.shape[0], S + lo + hi, S + lo + hi, x.shape[3]), device=x.device, dtype=x.dtype)
        p[:, lo:lo + S, lo:lo + S] = x
        x = p
    for r in range(k):
        for q in range(k):
            yield r, q, x[:, r:r + stride * (oh - 1) + 1:stride, q:q + stride * (oh - 1) + 1:stride]


def _plain_conv8(s):
    c = s["case"]
    x = _quantised(s["x"].float())
    w = _quantised(s["kernel"].transpose(2, 3).contiguous()).transpose(2, 3).contiguous()     # blocks along the input channels
    acc = None
    for r, q, xt in _taps(c, x):
        part = torch.matmul(xt.reshape(-1, c["Cin"]), w[r, q])
        acc = part if acc is None else acc.add_(part)
    y = _act(acc + s["bias"], c["act"]).reshape(c["B"], _out_size(c), _out_size(c), c["Cout"])
    if s["shortcut"] is not None:
        y = y + s["shortcut"].float()
    return y.to(DTYPES[c["out"]])


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"group_norm": _plain_group_norm, "dropout": _plain_dropout, "conv8": _plain_conv8}[op](s)
    if op == "conv8":
        return s["layer"](s["x"], residual=s["shortcut"], out_dtype=DTYPES[c["out"]])
    from yolo_amd import training
    sc = s["shortcut"]
    if op == "dropout":
        y = training.dropout(s["x"], c["rate"], s["state"], shortcut=sc)
        leaves = [s["x"]]
    else:
        y = training.group_norm_act(s["x"], s["gamma"], s["beta"], c["G"], activation=c["act"], shortcut=sc, epsilon=EPS,
                                    rate=c["rate"], state=s["state"] if c["rate"] > 0 else None)
        if not c["train"]:
            return y
        leaves = [s["x"], s["gamma"], s["beta"]]
    if sc is not None:
        leaves.append(sc)
    return [y.detach()] + list(torch.autograd.grad(y, leaves, s["dy"]))


# ---------------------------------------------------------------- what a pass cannot do without
def work(c):
    if c["op"] == "conv8":
        oh = _out_size(c)
        P, ob = c["B"] * oh * oh, 2 if c["out"] == "bf16" else 4
        K = c["k"] * c["k"] * c["Cin"]
        return {"bytes": c["B"] * c["S"] * c["S"] * c["Cin"] * 2 + K * c["Cout"] + P * c["Cout"] * ob * (2 if c["shortcut"] else 1),
                "flops": 2 * P * K * c["Cout"]}
    n, eb = c["B"] * c["S"] * c["S"] * c["C"], 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "dropout":
        return {"bytes": n * eb * (4 + (1 if c["shortcut"] else 0)), "flops": n * 4}
    maps = 2 + (2 if c["train"] else 0) + (1 if c["shortcut"] else 0)
    return {"bytes": n * eb * maps + c["C"] * 4 * (4 if c["train"] else 2), "flops": n * (45 if c["train"] else 20)}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_keep(shape, rate, state):
    """Philox4x32-10 with 16-bit limbs: no product here passes 64 bits."""
    n = math.prod(shape)
    seed, call = int(state[0]), int(state[1])
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]

    def hilo(a, m):
        al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
        mid = al * mh + ((al * ml) >> 16)
        mid2 = ah * ml + (mid & 0xFFFF)
        return ah * mh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((al * ml) & 0xFFFF)

    words = (n + 3) // 4
    ctr = [torch.arange(words, device=state.device), torch.zeros(words, dtype=torch.int64, device=state.device),
           torch.full((words,), call & 0xFFFFFFFF, dtype=torch.int64, device=state.device),
           torch.full((words,), (call >> 32) & 0xFFFFFFFF, dtype=torch.int64, device=state.device)]
    for i in range(10):
        h0, l0 = hilo(ctr[0], 0xD2511F53)
        h1, l1 = hilo(ctr[2], 0xCD9E8D57)
        a = (key[0] + i * 0x9E3779B9) % 2 ** 32
        b = (key[1] + i * 0xBB67AE85) % 2 ** 32
        ctr = [h1 ^ ctr[1] ^ a, l1, h0 ^ ctr[3] ^ b, l0]
    flat = torch.empty(words * 4, dtype=torch.int64, device=state.device)
    for i in range(4):
        flat[i::4] = ctr[i]
    return ~(flat[:n] < math.floor(rate * 2.0 ** 32)).reshape(shape)


def _exact_act(t, act):
    if act == "mish":
        e = torch.exp(t.clamp_max(40.0))
        u = e * (e + 2.0)
        return t * u / (u + 2.0)                                        # tanh(log(1 + e)) = e (e + 2) / (e (e + 2) + 2)
    if act == "leaky":
        return torch.maximum(t, 0.1 * t)
    return t


def _exact_quantised(x):
    """The same rule as _quantised, from the format's definition: 3 bits behind the leading one, steps of 2^-9 at the least."""
    C = x.shape[-1]
    nb = (C + 127) // 128
    p = torch.zeros(x.shape[:-1] + (nb * 128,), dtype=torch.float64, device=x.device)
    p[..., :C] = x
    p = p.reshape(x.shape[:-1] + (nb, 128))
    top = p.abs().max(-1, keepdim=True).values
    k = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0)).clamp_min(-126)
    k = torch.where(top > 448.0 * torch.exp2(k), k + 1, k)               # (log2 may be off next to a power of two)
    k = torch.where((top <= 448.0 * torch.exp2(k - 1)) & (top > 0) & (k > -126), k - 1, k)
    v = p * torch.exp2(-k)
    step = torch.exp2(torch.frexp(v)[1].clamp_min(-5).double() - 4.0)    # v = m 2^e, 0.5 <= m < 1: four significant bits
    q = torch.round(v / step) * step                                     # torch.round: halves to even
    return (q * torch.exp2(k)).reshape(x.shape[:-1] + (nb * 128,))[..., :C]


def exact(c, seed):
    d = _inputs(c, seed)
    if c["op"] == "conv8":
        B, S, ci, co, k, stride, oh = c["B"], c["S"], c["Cin"], c["Cout"], c["k"], c["stride"], _out_size(c)
        w = _exact_quantised(d["kernel"].permute(0, 1, 3, 2).double()).permute(0, 1, 3, 2).reshape(k * k * ci, co)
        lo = 1 if stride == 2 else (k - 1) // 2
        x = torch.nn.functional.pad(d["x"], (0, 0, lo, k - 1 - lo if stride == 1 else 0, lo, k - 1 - lo if stride == 1 else 0))
        ys = []
        for b in range(B):                                               # one image at a time: rows of k * k * Cin numbers
            xq = _exact_quantised(x[b].double())
            rows = xq.unfold(0, k, stride).unfold(1, k, stride)[:oh, :oh]        # [OH, OW, Cin, k, k]
            rows = rows.permute(0, 1, 3, 4, 2).reshape(oh * oh, k * k * ci)
            y = _exact_act(rows @ w + d["bias"].double(), c["act"]).reshape(oh, oh, co)
            if d["shortcut"] is not None:
                y = y + d["shortcut"][b].double()
            ys.append(y)
        return torch.stack(ys)
    keep = _exact_keep(d["x"].shape, c["rate"], d["state"]) if c["rate"] > 0 else None
    x = d["x"].double()
    if c["op"] == "dropout":
        y = torch.where(keep, x / (1.0 - c["rate"]), 0.0)
        if d["shortcut"] is not None:
            y = y + d["shortcut"].double()
        out = [y, torch.where(keep, d["dy"].double() / (1.0 - c["rate"]), 0.0)]
        return out + [d["dy"].double()] if d["shortcut"] is not None else out
    B, C, G = c["B"], c["C"], c["G"]
    leaves = [t.double().requires_grad_(c["train"]) for t in (x, d["gamma"], d["beta"])]
    u = leaves[0].reshape(B, -1, G, C // G)
    centred = u - u.mean((1, 3), keepdim=True)
    t = centred / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + EPS)
    y = _exact_act(t.reshape(x.shape) * leaves[1] + leaves[2], c["act"])
    if keep is not None:
        y = torch.where(keep, y / (1.0 - c["rate"]), 0.0)
    full = y if d["shortcut"] is None else y + d["shortcut"].double()
    if not c["train"]:
        return full.detach()
    out = [full.detach()] + list(torch.autograd.grad(y, leaves, d["dy"].double()))
    return out + [d["dy"].double()] if d["shortcut"] is not None else out
