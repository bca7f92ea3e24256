"""The operators of rlfluidcontrol_amd.ops written out in 64 bits, with bounds on what arithmetic in 32 bits may add.

`magnitude=True` evaluates the same formulas with every factor replaced by its absolute value (decays are positive anyway):
the size M of the sums of products that a value is made of.  A value computed in 32 bits is off by at most k u M, u = 2^-24,
where k counts the roundings on the longest way from an input to it, plus half a step of the output's type (half an eps)
relative to the value itself.  The counts:

 * softplus, sigmoid, exp: 8 roundings, and |v| for the argument's own (exp of an argument off by |v| u is off by |v| u);
 * a decay exp(delta A): |delta A| (12 + |v|) + 2 (delta off by (8 + |v|) u, two products, the exp itself);
 * a state: one decay, a product and a sum each position: L times that; a sum over n values: n.
"""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def keep_mask(lengths, B, L):
    if lengths is None:
        return torch.ones(B, L, dtype=torch.bool)
    return torch.arange(L)[None, :] < lengths.cpu().clamp(0, L)[:, None]


def d(t):
    return None if t is None else t.detach().cpu().double()


def conv(x, weight, bias, silu, state, lengths, dy=None, dlast=None, magnitude=False):
    """dict of y, last and, with dy, dx, dweight, dbias, dstate"""
    x, weight, bias, state, dy, dlast = (d(t) for t in (x, weight, bias, state, dy, dlast))
    B, L, W = x.shape
    K = weight.shape[1]
    keep = keep_mask(lengths, B, L)[:, :, None]
    zero = torch.zeros((), dtype=torch.float64)
    size = torch.abs if magnitude else (lambda t: t)
    x = torch.where(keep, x, zero)
    state = torch.zeros(B, K - 1, W, dtype=torch.float64) if state is None else state
    rows = torch.cat([state, x], 1)
    pre = sum(rows[:, k:k + L] * weight[:, k] for k in range(K))
    pre = pre + bias if bias is not None else pre
    pre_size = sum(rows[:, k:k + L].abs() * weight[:, k].abs() for k in range(K)) + (bias.abs() if bias is not None else 0)
    sig = torch.sigmoid(pre)
    if silu:  # an error of pre reaches silu with a slope of at most 1.1, and its slope with one of at most 0.5
        y, slope = pre * sig, sig * (1 + pre * (1 - sig))
        y_size, slope_size = 1.1 * pre_size, 1.1 + 0.5 * pre_size
    else:
        y, slope, y_size, slope_size = pre, torch.ones_like(pre), pre_size, torch.ones_like(pre)
    n = keep.sum(1)[:, 0]
    last = torch.stack([rows[b, int(n[b]):int(n[b]) + K - 1] for b in range(B)]) if B else state.clone()
    r = dict(y=torch.where(keep, y_size if magnitude else y, zero), last=size(last))
    if dy is None:
        return r
    dp = torch.where(keep, dy.abs() * slope_size if magnitude else dy * slope, zero)
    drows = torch.zeros(B, L + K - 1, W, dtype=torch.float64)
    for k in range(K):
        drows[:, k:k + L] += dp * size(weight[:, k])
    for b in range(B):
        if dlast is not None:
            drows[b, int(n[b]):int(n[b]) + K - 1] += size(dlast[b])
    r.update(dx=torch.where(keep, drows[:, K - 1:], zero), dstate=drows[:, :K - 1].clone(),
             dweight=torch.stack([(dp * size(rows[:, k:k + L])).sum((0, 1)) for k in range(K)], 1), dbias=dp.sum((0, 1)))
    return r


def conv_bounds(m, dtype, x, taps, silu):
    """how far each output of the kernel may be from the reference `r`: k u M, added to half a step of its type"""
    B, L, W = x.shape
    top = float(m["y"].max()) if m["y"].numel() else 0.0
    k = 2 * taps + 4 + ((8 + top) if silu else 0)
    return dict(y=k, last=0, dx=2 * k + 2 * taps, dstate=2 * k + 2 * taps, dweight=2 * k + B * L + 4, dbias=2 * k + B * L + 4)


def scan(x, dt, A, B, C, D, z, dt_bias, softplus, state, lengths, dy=None, dlast=None, magnitude=False):
    """dict of y, last and, with dy, dx, ddt, dA, dB, dC, dD, dz, dbias, dstate; B and C [batch, length, groups, state]"""
    x, dt, A, B, C, D, z, dt_bias, state, dy, dlast = (d(t) for t in (x, dt, A, B, C, D, z, dt_bias, state, dy, dlast))
    Bn, L, W = x.shape
    G, N = B.shape[2:]
    keep = keep_mask(lengths, Bn, L)
    zero = torch.zeros((), dtype=torch.float64)
    size = torch.abs if magnitude else (lambda t: t)
    x, dt = (torch.where(keep[..., None], t, zero) for t in (x, dt))
    B, C = (torch.where(keep[..., None, None], t, zero).repeat_interleave(W // G, 2) for t in (B, C))
    v = dt + dt_bias if dt_bias is not None else dt
    delta = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v
    slope = torch.sigmoid(v) if softplus else torch.ones_like(v)
    if z is not None:
        z = torch.where(keep[..., None], z, zero)
        sig = torch.sigmoid(z)
        gate, gate_slope = z * sig, sig * (1 + z * (1 - sig))
    else:
        gate, gate_slope = torch.ones_like(x), torch.zeros_like(x)
    decay = [torch.exp(delta[:, l, :, None] * A) for l in range(L)]  # (of the signed values in either form)
    x, B, C, delta, gate = size(x), size(B), size(C), size(delta), size(gate)
    gate_slope = gate_slope.abs() + 1.1 if magnitude else gate_slope
    A = size(A)
    D = torch.zeros(W, dtype=torch.float64) if D is None else size(D)
    h = torch.zeros(Bn, W, N, dtype=torch.float64) if state is None else size(state)
    hs, ys = [h], []
    for l in range(L):
        on = keep[:, l, None, None]
        h = torch.where(on, decay[l] * h + (delta[:, l] * x[:, l])[..., None] * B[:, l], h)
        hs.append(h)
        ys.append((C[:, l] * h).sum(-1) + D * x[:, l])
    y0 = torch.stack(ys, 1) if ys else torch.zeros(Bn, 0, W, dtype=torch.float64)
    r = dict(y=torch.where(keep[..., None], y0 * gate, zero), last=h, delta_A=delta[..., None] * A.abs(), v=v)
    if dy is None:
        return r
    dout = torch.where(keep[..., None], size(dy), zero)
    r["dz"] = dout * y0 * gate_slope
    dy = dout * gate
    g = torch.zeros(Bn, W, N, dtype=torch.float64) if dlast is None else size(dlast)
    dx, ddt, dB, dC = (torch.zeros(Bn, L, W, *s, dtype=torch.float64) for s in ((), (), (N,), (N,)))
    dA = torch.zeros(W, N, dtype=torch.float64)
    for l in range(L - 1, -1, -1):
        on = keep[:, l, None, None]
        g = g + dy[:, l, :, None] * C[:, l]
        now = torch.where(on, g, zero)
        t = now * decay[l] * hs[l]
        du = (now * B[:, l]).sum(-1)
        dx[:, l] = du * delta[:, l] + D * dy[:, l]
        ddt[:, l] = (du * x[:, l] + (t * A).sum(-1)) * slope[:, l]
        dB[:, l] = now * (delta[:, l] * x[:, l])[..., None]
        dC[:, l] = dy[:, l, :, None] * hs[l + 1]
        dA += (t * delta[:, l, :, None]).sum(0)
        g = torch.where(on, g * decay[l], g)
    ddt = torch.where(keep[..., None], ddt, zero)
    r.update(dx=torch.where(keep[..., None], dx, zero), ddt=ddt, dA=dA, dB=dB.unflatten(2, (G, W // G)).sum(3), dC=dC.unflatten(2, (G, W // G)).sum(3),
             dD=(dy * x).sum((0, 1)), dbias=ddt.sum((0, 1)), dstate=g)
    return r


def scan_bounds(r, x, N, G):
    B, L, W = x.shape
    v = float(r["v"].abs().max()) if r["v"].numel() else 0.0
    da = float(r["delta_A"].max()) if r["delta_A"].numel() else 0.0
    state = L * (da * (12 + v) + 4) + 2 * (8 + v) + 4
    y = state + N + 16
    back = 2 * (state + 16) + 2 * N + 16 + v
    total = back + B * L + 4
    return dict(y=y, last=state, dx=back, ddt=back + 8 + v, dz=y + 16, dB=back + W // G, dC=back + W // G, dA=total, dD=total, dbias=total + 8 + v,
                dstate=back)


def off(got, want, size, k, dtype):
    """largest excess of |got - want| over its bound, as a multiple of the bound (1 and less is within it)"""
    got, want = got.detach().cpu().double(), want
    assert got.shape == want.shape, (got.shape, want.shape)
    if not got.numel():
        return 0.0
    assert bool(torch.isfinite(got).all())
    err = (got - want).abs()
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}[dtype]  # half the smallest step; 32 bits may flush
    bound = half_step(dtype) * (want.abs() + k * U * size) + k * U * size + tiny
    return float((err / bound).max())
