"""Group norm with activation, dropout mask and shortcut, and its gradients, in 64 bits on the CPU."""
import torch


def act(t, name):
    if name == "mish":
        return t * torch.tanh(torch.nn.functional.softplus(t))
    if name == "leaky":
        return torch.where(t > 0, t, 0.1 * t)
    return t


def act_grad(t, name):
    if name == "mish":
        w = torch.tanh(torch.nn.functional.softplus(t))
        return w + t * (1 - w * w) * torch.sigmoid(t)
    if name == "leaky":
        return torch.where(t > 0, 1.0, 0.1).double()
    return torch.ones_like(t)


def group_norm(x, gamma, beta, groups, name, eps, shortcut=None, keep=None, rate=0.0, dy=None):
    """A dict of doubles: y, and with dy also dx, dgamma, dbeta, dshortcut; and the magnitudes error
    bounds are made of: t_mag >= |t| before cancellation, dt and its sums' magnitudes."""
    b, c = x.shape[0], x.shape[-1]
    xd = x.double().reshape(b, -1, groups, c // groups)
    ga, be = gamma.double().reshape(groups, -1), beta.double().reshape(groups, -1)
    mean = xd.mean((1, 3), keepdim=True)
    r = 1.0 / torch.sqrt((xd - mean).square().mean((1, 3), keepdim=True) + eps)
    h = (xd - mean) * r
    t = ga * h + be
    y = act(t, name)
    k = 1.0 if keep is None else keep.reshape(xd.shape).double() / (1.0 - rate)
    y = y * k
    h_mag = (xd.abs() + mean.abs()) * r
    out = {"act": y.reshape(x.shape), "t_mag": ((ga.abs() * h_mag + be.abs()) * k).reshape(x.shape)}
    out["y"] = out["act"] if shortcut is None else out["act"] + shortcut.double()
    if dy is None:
        return out
    n = xd.shape[1] * xd.shape[3]
    dt = dy.double().reshape(xd.shape) * k * act_grad(t, name)
    gd = ga * dt
    s1, s2 = gd.sum((1, 3), keepdim=True), (gd * h).sum((1, 3), keepdim=True)
    out["dx"] = (r * (gd - (s1 + h * s2) / n)).reshape(x.shape)
    out["dgamma"], out["dbeta"] = (dt * h).sum((0, 1)).reshape(-1), dt.sum((0, 1)).reshape(-1)
    # magnitudes: |dy k| (a derivative of the activation is at most 1.1 and changes by at most 1.1 per unit of t)
    m = (dy.double().reshape(xd.shape) * k).abs()
    tm = 1.0 + ga.abs() * h_mag + be.abs()
    out["dgamma_mag"] = (m * tm * (1 + h_mag)).sum((0, 1)).reshape(-1)
    out["dbeta_mag"] = (m * tm).sum((0, 1)).reshape(-1)
    gm = ga.abs() * m * tm
    out["dx_mag"] = (r * (1 + h_mag) * (gm + gm.mean((1, 3), keepdim=True) + h_mag * (gm * h_mag).mean((1, 3), keepdim=True))).reshape(x.shape)
    return out
