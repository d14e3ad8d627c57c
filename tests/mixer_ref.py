"""Plain float64 forms of the mixer calls (causal convolution, state space scan, gated and residual norms), on
the CPU, and bounds of the kernels' rounding errors.

A rounding to a type is off by at most half a step, HALF[type] of the value. Sums run in 32 bits: n products
of partial sums below S (the sum of the terms' magnitudes) are off by at most n 2^-24 S; the exponential, the
logarithm and the quotient of a term by a few steps of 2^-24 more, counted as 2^-21 of it.
"""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# below a type's normal numbers a step is no smaller: half of the smallest one
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
U = 2.0 ** -24


def f64(t):
    return None if t is None else t.detach().cpu().double()


def spans(n, batch, starts=None):
    if starts is None:
        return [(b * (n // batch), (b + 1) * (n // batch)) for b in range(batch)]
    s = [int(v) for v in starts]
    return list(zip(s[:-1], s[1:]))


def start_of(state, b, offsets, slots):
    """(slot or None, whether the sequence begins with what it holds)."""
    slot = b if slots is None else int(slots[b])
    if not 0 <= slot < state.shape[0]:
        return None, False
    return slot, offsets is None or int(offsets[b]) > 0


def conv(x, w, bias, state, batch, starts=None, offsets=None, slots=None, silu=True):
    """y, the pool afterwards, and sum |terms| of each value before the activation."""
    x, w, bias = f64(x), f64(w), f64(bias)
    n, C = x.shape
    W = w.shape[1]
    pool = None if state is None else f64(state).clone()
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    for b, (lo, hi) in enumerate(spans(n, batch, starts)):
        if lo == hi:
            continue
        slot, kept = (None, False) if pool is None else start_of(pool, b, offsets, slots)
        before = pool[slot].clone() if kept else torch.zeros(W - 1, C, dtype=torch.float64)
        rows = torch.cat([before, x[lo:hi]])
        for t in range(hi - lo):
            terms = rows[t:t + W].T * w
            y[lo + t] = terms.sum(1) + (0 if bias is None else bias)
            mag[lo + t] = terms.abs().sum(1) + (0 if bias is None else bias.abs())
        if slot is not None:
            pool[slot] = rows[hi - lo:]
    return (y * torch.sigmoid(y) if silu else y), pool, mag


def scan(x, dt, B, C, A, state, batch, D=None, dt_bias=None, starts=None, offsets=None, slots=None, softplus=True,
         limit=(0.0, float("inf"))):
    """y, the pool afterwards, and the same with the magnitudes of all terms."""
    x, dt, B, C, A, D, dt_bias = (f64(t) for t in (x, dt, B, C, A, D, dt_bias))
    n, H, P = x.shape
    rep = H // B.shape[1]
    pool = f64(state).clone()
    pool_mag = pool.abs()
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    d = dt if dt_bias is None else dt + dt_bias
    if softplus:
        d = torch.where(d > 40, d, torch.log1p(torch.exp(d.clamp(max=40))))
    d = d.clamp(*limit)
    decay = torch.exp(d * A)
    B, C = B.repeat_interleave(rep, 1), C.repeat_interleave(rep, 1)
    for b, (lo, hi) in enumerate(spans(n, batch, starts)):
        if lo == hi:
            continue
        slot, kept = start_of(pool, b, offsets, slots)
        h = pool[slot].clone() if kept else torch.zeros(H, P, B.shape[2], dtype=torch.float64)
        m = h.abs()
        for t in range(lo, hi):
            add = (d[t][:, None] * x[t])[:, :, None] * B[t][:, None]
            h = h * decay[t][:, None, None] + add
            m = m * decay[t][:, None, None] + add.abs()
            y[t] = (h * C[t][:, None]).sum(-1)
            mag[t] = (m * C[t][:, None].abs()).sum(-1)
            if D is not None:
                y[t] += D[:, None] * x[t]
                mag[t] += (D[:, None] * x[t]).abs()
        if slot is not None:
            pool[slot], pool_mag[slot] = h, m
    return y, pool, mag, pool_mag


def norm(u, w, eps, unit=False):
    u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + eps)
    return u if w is None else u * (1 + w if unit else w)


def gated(x, gate, w, eps, group, first=False, sigmoid=False, unit=False):
    x, gate, w = f64(x), f64(gate), f64(w)
    n, dim = x.shape
    k = torch.ones_like(x) if gate is None else torch.sigmoid(gate) if sigmoid else gate * torch.sigmoid(gate)
    w = None if w is None else w.view(-1, group)
    x, k = x.view(n, -1, group), k.view(n, -1, group)
    return (norm(x * k, w, eps, unit) if first else norm(x, w, eps, unit) * k).view(n, dim)


def residual(branch, res, pre_w, eps, post_w=None, gate=None, scale=1.0, unit=False):
    """h, out and the magnitudes of h's two terms."""
    u = f64(branch)
    if post_w is not None:
        u = norm(u, f64(post_w), eps, unit)
    if gate is not None:
        u = u * f64(gate)
    r = f64(res)
    h = r + scale * u
    return h, None if pre_w is None else norm(h, f64(pre_w), eps, unit), r.abs() + abs(scale) * u.abs()


def check(got, want, tol, what):
    """|got - want| <= tol everywhere; where want is not finite the kernel's value is not either."""
    g, d = got.detach().cpu().double(), None
    assert g.shape == want.shape, (what, g.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(g), fine), f"{what}: finite values where the definition has none, or the reverse"
    d = (g - want).abs()[fine]
    tol = tol.expand_as(want)[fine]
    bad = d > tol
    worst = float((d / tol.clamp(min=1e-300)).max()) if d.numel() else 0.0
    print(f"  {what}: max {float(d.max()) if d.numel() else 0:.3e}, {worst:.3f} of the bound", flush=True)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {d.numel()} values beyond the bound (worst {worst:.2f})"
