"""float64 restatements of the sequence-layer operators, one loop over time each, with their gradients from the formulas.

``absolute=True`` replaces every factor of every sum by its magnitude: the same expressions then bound what rounding in the
kernels' float32 sums can do (each result is off by at most the number of roundings on its way times 2^-24 of that)."""

import torch


def rows_of(lengths, b, steps):
    return torch.full((b,), steps) if lengths is None else lengths.cpu().long().clamp(0, steps)


def d64(t):
    return None if t is None else t.detach().cpu().double()


def conv(x, w, b=None, act="none", state=None, lengths=None, dy=None, dstate_out=None, absolute=False):
    """dict of y, state and, with dy, dx / dw / db / dstate."""
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    x, w = d64(x), d64(w)
    bsz, steps, ch = x.shape
    taps = w.shape[1]
    n = rows_of(lengths, bsz, steps)
    live = (torch.arange(steps) < n[:, None])[:, :, None]
    x = torch.where(live, x, torch.zeros_like(x))
    head = d64(state) if state is not None else torch.zeros(bsz, taps - 1, ch, dtype=torch.float64)
    full = torch.cat([head, x], 1)
    z = sum(full[:, j:j + steps] * w[:, j] for j in range(taps)) + (0 if b is None else d64(b))
    za = sum(f(full[:, j:j + steps]) * f(w[:, j]) for j in range(taps)) + (0 if b is None else f(d64(b)))
    s = torch.sigmoid(z)
    # (absolute: an error e of z moves silu by at most 1.1 e, its slope by at most 0.5 e)
    y = (za * 1.1 if absolute else z * s) if act == "silu" else za
    zero = torch.zeros_like(y)
    out = {"y": torch.where(live, y, zero),
           "state": torch.stack([full[i, n[i]:n[i] + taps - 1] for i in range(bsz)])}
    if dy is None:
        return out
    g = torch.where(live, d64(dy), zero)
    slope = s * (1 + z * (1 - s)) if act == "silu" else torch.ones_like(z)
    if absolute:
        slope = 1.1 + 0.5 * za if act == "silu" else slope
    dz = f(g) * slope
    dfull, dw = torch.zeros_like(full), torch.zeros_like(w)
    for j in range(taps):
        dfull[:, j:j + steps] += dz * f(w[:, j])
        dw[:, j] = (dz * f(full[:, j:j + steps])).sum((0, 1))
    if dstate_out is not None:
        for i in range(bsz):
            dfull[i, n[i]:n[i] + taps - 1] += f(d64(dstate_out)[i])
    dx = dfull[:, taps - 1:]
    out.update(dx=torch.where(live, dx, torch.zeros_like(dx)), dw=dw, db=dz.sum((0, 1)), dstate=dfull[:, :taps - 1])
    return out


def scan(x, dt, a, b, c, d=None, gate=None, dt_bias=None, softplus=False, state=None, lengths=None, dy=None,
         dstate_out=None, absolute=False):
    """dict of y, state and, with dy, the gradients dx, ddt, da, db, dc, dd, dgate, ddt_bias, dstate."""
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    x, dt, a, b, c = d64(x), d64(dt), d64(a), d64(b), d64(c)
    bsz, steps, ch = x.shape
    n_st = a.shape[1]
    n = rows_of(lengths, bsz, steps)
    live = (torch.arange(steps) < n[:, None])[:, :, None]

    def clean(t):
        return torch.where(live, t, torch.zeros_like(t))

    x, dt, b, c = clean(x), clean(dt), clean(b), clean(c)
    raw = dt + (0 if dt_bias is None else d64(dt_bias))
    delta = clean(torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw)
    sp = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    skip = torch.zeros(ch, dtype=torch.float64) if d is None else d64(d)
    if gate is None:
        sg, dsg, gt = torch.ones_like(x), None, None
    else:
        gt = clean(d64(gate))
        s = torch.sigmoid(gt)
        # the slope is a sum itself, 1 + gate (1 - s), and cancels near gate = -1.28: its magnitudes are 1 and |gate| (1 - s)
        sg, dsg = gt * s, s * (1 + f(gt) * (1 - s))
    h = torch.zeros(bsz, ch, n_st, dtype=torch.float64) if state is None else f(d64(state))
    first = h
    hs, es = [], []
    for t in range(steps):
        e = torch.exp(delta[:, t, :, None] * a)
        h = e * h + f(delta[:, t] * x[:, t])[:, :, None] * f(b[:, t])[:, None, :]
        hs.append(h)
        es.append(e)
    H = torch.stack(hs, 1) if steps else torch.zeros(bsz, 0, ch, n_st, dtype=torch.float64)
    y0 = (H * f(c)[:, :, None, :]).sum(-1) + f(skip) * f(x)
    out = {"y": clean(y0 * f(sg)), "state": h}
    if dy is None:
        return out
    dyv = clean(d64(dy))
    g = f(dyv) * f(sg)
    X = torch.zeros_like(h) if dstate_out is None else f(d64(dstate_out))
    dx, ddt = torch.zeros_like(x), torch.zeros_like(x)
    db, dc, da = torch.zeros_like(b), torch.zeros_like(c), torch.zeros_like(a)
    for t in range(steps - 1, -1, -1):
        G = f(c[:, t])[:, None, :] * g[:, t, :, None] + X
        prev = hs[t - 1] if t else first
        X = es[t] * G
        W = X * prev
        s1 = (G * f(b[:, t])[:, None, :]).sum(-1)
        dx[:, t] = g[:, t] * f(skip) + f(delta[:, t]) * s1
        ddt[:, t] = ((W * f(a)).sum(-1) + f(x[:, t]) * s1) * sp[:, t]
        da += (W * f(delta[:, t])[:, :, None]).sum(0)
        db[:, t] = (G * f(delta[:, t] * x[:, t])[:, :, None]).sum(1)
        dc[:, t] = (H[:, t] * g[:, t, :, None]).sum(1)
    ddt = clean(ddt)
    out.update(dx=clean(dx), ddt=ddt, da=da, db=clean(db), dc=clean(dc), dd=(g * f(x)).sum((0, 1)), ddt_bias=ddt.sum((0, 1)),
               dstate=X)
    if gate is not None:
        out["dgate"] = clean(f(dyv) * y0 * f(dsg))
    return out


HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def close(got, ref, bound, roundings, what=""):
    """|got - ref| <= half a step of got's type (relative) + roundings 2^-24 bound, element by element."""
    assert got.shape == ref.shape, (what, tuple(got.shape), tuple(ref.shape))
    g = got.detach().cpu().double()
    assert bool(torch.isfinite(g).all()), f"{what}: not finite"
    tol = HALF_STEP[got.dtype] * ref.abs() + roundings * 2.0 ** -24 * bound.abs() * (1 + HALF_STEP[got.dtype])
    tol = tol + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)  # half of the smallest number of the type
    over = (g - ref).abs() - tol
    if over.numel() and float(over.max()) > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {over.numel()} outside; worst at {i}: "
                             f"got {float(g.flatten()[i])!r}, ref {float(ref.flatten()[i])!r}, "
                             f"allowed {float(tol.flatten()[i])!r}")


def linear(x, w, b=None, act="none", residual=None, dy=None, absolute=False):
    """dict of y and, with dy, dx / dw / db; x [M, K].  absolute: the sums of magnitudes, through slopes of at most 1.13 and
    the change of the slope (at most 1 per unit of z) under an error of z."""
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    x, w = d64(x), d64(w)
    z = x @ w.t() + (0 if b is None else d64(b))
    za = f(x) @ f(w).t() + (0 if b is None else f(d64(b)))
    s, cdf = torch.sigmoid(z), 0.5 * torch.erfc(-z * 0.5 ** 0.5)
    y, slope = {"none": (z, torch.ones_like(z)), "relu": (z.clamp(min=0), (z > 0).double()), "silu": (z * s, s + z * s * (1 - s)),
                "gelu": (z * cdf, cdf + z * torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5)}[act]
    if absolute:
        y, slope = 1.13 * za, 1.13 + za
    out = {"y": y if residual is None else y + f(d64(residual)), "z": z}
    if dy is not None:
        dz = f(d64(dy)) * slope
        out.update(dx=dz @ f(w), dw=dz.t() @ f(x), db=dz.sum(0), dz=dz)
    return out
