"""The gated linear recurrence and its gradients in 64 bits, step by step from their definitions, and bounds on what float32
arithmetic may be off by."""
import torch

U = 2.0 ** -24          # half a float32 step, relative


def _wide(t):
    return None if t is None else t.to(torch.float64)


def forward(f, x, h0=None, resets=None, bias=None):
    """(h [T, E, H], last state, states each step starts from) in float64."""
    f, x = _wide(f), _wide(x)
    zf = f if bias is None else f + _wide(bias)
    a, om = torch.sigmoid(zf), torch.sigmoid(-zf)
    h = torch.zeros(x.shape[1:], dtype=torch.float64, device=x.device) if h0 is None else _wide(h0)
    hs, ps = [], []
    for t in range(x.shape[0]):
        if resets is not None:
            h = torch.where(resets[t].bool().unsqueeze(-1), 0.0, h)
        ps.append(h)
        h = a[t] * h + om[t] * x[t]
        hs.append(h)
    empty = x.new_zeros((0,) + tuple(x.shape[1:]))
    return torch.stack(hs) if hs else empty, h, torch.stack(ps) if ps else empty


def backward(f, x, h0, resets, bias, dy, dh_last=None):
    f, x = _wide(f), _wide(x)
    zf = f if bias is None else f + _wide(bias)
    a, om = torch.sigmoid(zf), torch.sigmoid(-zf)
    p = forward(f, x, h0, resets, bias)[2]
    g = torch.zeros(x.shape[1:], dtype=torch.float64, device=x.device) if dh_last is None else _wide(dh_last)
    df, dx = torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[0] - 1, -1, -1):
        g = g + _wide(dy[t])
        dx[t] = om[t] * g
        df[t] = g * (p[t] - x[t]) * a[t] * om[t]
        g = a[t] * g
        if resets is not None:
            g = torch.where(resets[t].bool().unsqueeze(-1), 0.0, g)
    return df, dx, g, df.sum((0, 1))


class Bounds:
    """Worst-case float32 errors, one number per column where it matters.

    A step h = big + s (other - big), s = min(a, 1 - a): the distance and the sum round once each (U times a value of at most
    2 M and M, M the largest |x| and |h0|), and s itself is off by at most 8 U of its value (exp, its argument's two
    roundings, the sum, reciprocal and product of the sigmoid).  An error that entered k steps ago has shrunk by the gates
    since, so K = min(T, 1 / smallest (1 - a)) of them count in full; the gates' own errors enter times s and add up to
    16 U M at most.  The sum f + bias rounds by U |f + bias|, which moves the gate by as much relative to s: times Z, the
    largest |f + bias|.  A scan in spans carries at most three more roundings per span, again counted by K."""

    def __init__(self, f, x, h0, resets, bias):
        zf = _wide(f) if bias is None else _wide(f) + _wide(bias)
        T = x.shape[0]
        self.K = torch.clamp(1 / torch.sigmoid(-zf).amin(0), max=float(T))
        self.Z = zf.abs().amax(0)
        self.M = _wide(x).abs().amax(0)
        if h0 is not None:
            self.M = torch.maximum(self.M, _wide(h0).abs())
        self.h = U * self.M * (16 + 2 * self.Z + 6 * self.K)

    def grads(self, g_abs):
        """Bounds for g (and dh0), dx and df, from the largest |g| of each column: the same argument with g for h; df multiplies
        g's error by |p - x| <= 2 M and the state's by |g|, both by a (1 - a) <= 1/4, and rounds a few times itself."""
        tg = U * g_abs * (16 + 2 * self.Z + 6 * self.K)
        df = 0.25 * (tg * 2 * self.M + g_abs * self.h + (24 + 2 * self.Z) * U * g_abs * 2 * self.M)
        return tg, tg + (24 + 2 * self.Z) * U * g_abs, df


def largest_g(f, bias, resets, dy, dh_last):
    """Largest |g| of each column, from the recursion over |dy| (no cancellation)."""
    zf = _wide(f) if bias is None else _wide(f) + _wide(bias)
    a = torch.sigmoid(zf)
    g = torch.zeros(dy.shape[1:], dtype=torch.float64, device=dy.device) if dh_last is None else _wide(dh_last).abs()
    top = g
    for t in range(dy.shape[0] - 1, -1, -1):
        g = g + _wide(dy[t]).abs()
        top = torch.maximum(top, g)
        g = a[t] * g
        if resets is not None:
            g = torch.where(resets[t].bool().unsqueeze(-1), 0.0, g)
    return top
