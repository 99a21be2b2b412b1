"""Group norm with an activation, channels last, and its gradients in 64 bits.  TEST INFRASTRUCTURE ONLY.

Sample by sample from the definition; tests/test_groupnorm_oracle.py holds it against torch's group norm and autograd."""
import torch


def _parts(x, lengths):
    """(index, frames [n, C]) of every sample: utterances, or single rows."""
    if x.dim() == 2:
        return [(i, x[i:i + 1]) for i in range(x.shape[0])]
    T = x.shape[1]
    n = [T] * x.shape[0] if lengths is None else [min(max(int(v), 0), T) for v in lengths]
    return [((i, slice(0, n[i])), x[i, :n[i]]) for i in range(x.shape[0]) if n[i] > 0]


def _normalised(part, groups, eps):
    p = part.reshape(part.shape[0], groups, -1)
    mean = p.mean(dim=(0, 2), keepdim=True)
    rstd = ((p - mean) ** 2).mean(dim=(0, 2), keepdim=True).add(eps).rsqrt()
    return (p - mean) * rstd, rstd


def group_norm(x, groups, weight, bias, eps=1e-5, activation=None, lengths=None):
    x, w, b = x.double(), weight.double(), bias.double()
    y = torch.zeros_like(x)
    for at, part in _parts(x, lengths):
        z = _normalised(part, groups, eps)[0].reshape(part.shape) * w + b
        z = z.clamp(min=0) if activation == "relu" else z * torch.sigmoid(z) if activation == "silu" else z
        y[at] = z.reshape(y[at].shape)
    return y


def group_norm_backward(x, groups, weight, bias, dy, eps=1e-5, activation=None, lengths=None):
    """(dx, dweight, dbias)."""
    x, w, b, dy = x.double(), weight.double(), bias.double(), dy.double()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for at, part in _parts(x, lengths):
        hat, rstd = _normalised(part, groups, eps)
        z = hat.reshape(part.shape) * w + b
        s = torch.sigmoid(z)
        slope = {None: torch.ones_like(z), "relu": (z > 0).double(), "silu": s * (1 + z * (1 - s))}[activation]
        dz = dy[at].reshape(part.shape) * slope
        dw += (dz * hat.reshape(part.shape)).sum(0)
        db += dz.sum(0)
        g = (dz * w).reshape(hat.shape)
        m = lambda t: t.mean(dim=(0, 2), keepdim=True)  # noqa: E731
        dx[at] = (rstd * (g - m(g) - hat * m(g * hat))).reshape(dx[at].shape)
    return dx, dw, db
