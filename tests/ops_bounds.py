"""The selective scan in 64 bits with a bound for every element of every output on what arithmetic in 32 bits may add.

ops_reference multiplies the largest decay term of any position by the length, which is easy to read and wide for long rows.  Here the
bounds follow the recurrence: what a rounding adds decays as the state that it was made on does.  They are in units of u = 2^-24, of
first order (check() allows one part in a hundred for the rest), with ops_reference's counts for the activations: exp, sigmoid and
softplus of v are off by (8 + |v|) u of themselves.

 * a decay exp(delta A) is off by |delta A| (12 + |v|) + 2, and by |delta A| (part + 3) where parts of `part` positions are joined
   by the decay across them: its exponent is a sum of that many step sizes, whose terms share its error by their size;
 * a state: E[l] = a (E[l-1] + (that of a) M[l-1]) + |delta x B| (11 + |v|) + M[l], M its size with all terms positive; an adjoint alike;
 * a sum over n values: n + 4 roundings of its size, whatever its order.
"""
import torch

from tests import ops_reference as ref

U = 2.0 ** -24


def scan(c, softplus=True, part=256, carried=None):
    """(values, bounds) of y, last, dx, ddt, dA, dB, dC, dD, dz, dbias and dstate for a case as tests.test_ops.scan_case makes it (all
    operands given).  carried: what every 32 positions is done to the state, to see what a bound notices"""
    x, dt, A, B, C, D, z, bias, h0, dout, dlast = (ref.d(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state", "dy", "dlast"))
    Bn, L, W = x.shape
    G, N = B.shape[2:]
    keep = ref.keep_mask(c["lengths"], Bn, L).to(x)
    k3, k4 = keep[..., None], keep[..., None, None]
    x, z, dout = x * k3, z * k3, dout * k3
    B, C = ((t * k4).repeat_interleave(W // G, 2) for t in (B, C))
    v = dt + bias
    delta = (torch.logaddexp(v, torch.zeros_like(v)) if softplus else v) * k3
    slope = torch.sigmoid(v) if softplus else torch.ones_like(v)
    v, za, Aa = v.abs(), z.abs(), A.abs()
    sig = torch.sigmoid(z)
    gate, gate_slope = z * sig, sig * (1 + z * (1 - sig))
    gate_off = gate.abs() * (9 + za)
    gate_slope_off = (1 + za) * (12 + za)
    decay = torch.exp(delta[..., None] * A)
    decay_off = (delta[..., None] * Aa) * (15 + part + v[..., None]) + 2
    drive = (delta * x)[..., None] * B
    hs, Ms, Es = [h0], [h0.abs()], [torch.zeros_like(h0)]
    for l in range(L):
        a, h, M, E = decay[:, l], hs[-1], Ms[-1], Es[-1]
        if carried and l % 32 == 0:
            h = carried(h)
        live = k3[:, l, :, None]
        M2 = a * M + drive[:, l].abs()
        E2 = a * (E + decay_off[:, l] * M) + drive[:, l].abs() * (11 + v[:, l, :, None]) + M2
        hs.append(torch.where(live > 0, a * h + drive[:, l], h))
        Ms.append(torch.where(live > 0, M2, M))
        Es.append(torch.where(live > 0, E2, E))
    H, M, E = (torch.stack(t, 1) for t in (hs, Ms, Es))  # [batch, length + 1, ...]: in front of every position, and at the end
    Ca, Ba = C.abs(), B.abs()
    y0 = (C * H[:, 1:]).sum(-1) + D * x
    y0_size = (Ca * M[:, 1:]).sum(-1) + (D * x).abs()
    y0_off = (Ca * E[:, 1:]).sum(-1) + (N + 6) * y0_size
    val = dict(y=y0 * gate * k3, last=H[:, -1])
    off = dict(y=(y0_off * gate.abs() + y0_size * (gate_off + 2 * gate.abs())) * k3, last=E[:, -1])
    val["dz"] = dout * y0 * gate_slope
    off["dz"] = dout.abs() * (y0_off * gate_slope.abs() + y0_size * (gate_slope_off + 3 * gate_slope.abs()))
    dy = dout * gate
    dya, dy_off = dy.abs(), dout.abs() * (gate_off + 2 * gate.abs())
    g, Gm, Eg = dlast, dlast.abs(), torch.zeros_like(dlast)
    new = lambda *s: torch.zeros(Bn, L, W, *s, dtype=torch.float64)  # noqa: E731
    dx, ddt, dB, dC, dx_off, ddt_off, dB_off, dC_off = new(), new(), new(N), new(N), new(), new(), new(N), new(N)
    dB_size, dC_size, ddt_size = new(N), new(N), new()
    dA, dA_off, dA_size = (torch.zeros(W, N, dtype=torch.float64) for _ in range(3))
    for l in range(L - 1, -1, -1):
        live = k3[:, l, :, None]
        de, a, ao, Hp, Mp, Ep = delta[:, l], decay[:, l], decay_off[:, l], H[:, l], M[:, l], E[:, l]
        g2, Gm2 = g + dy[:, l, :, None] * C[:, l], Gm + dya[:, l, :, None] * Ca[:, l]
        Eg2 = Eg + dy_off[:, l, :, None] * Ca[:, l] + Gm2
        du, du_size = (g2 * B[:, l]).sum(-1), (Gm2 * Ba[:, l]).sum(-1)
        du_off = (Eg2 * Ba[:, l]).sum(-1) + (N + 4) * du_size
        t, t_size = g2 * a * Hp, Gm2 * a * Mp
        t_off = a * (Eg2 * Mp + Gm2 * Ep) + t_size * (ao + 3)
        ta, ta_size = (t * A).sum(-1), (t_size * Aa).sum(-1)
        ta_off = (t_off * Aa).sum(-1) + (N + 7) * ta_size
        w8 = 11 + v[:, l]
        dx[:, l] = du * de + D * dy[:, l]
        dx_off[:, l] = du_off * de + du_size * de * w8 + D.abs() * (dy_off[:, l] + 2 * dya[:, l])
        ddt[:, l] = (du * x[:, l] + ta) * slope[:, l]
        ddt_size[:, l] = (du_size * x[:, l].abs() + ta_size) * slope[:, l]
        ddt_off[:, l] = (du_off * x[:, l].abs() + ta_off) * slope[:, l] + ddt_size[:, l] * w8
        dxa = (de * x[:, l].abs())[..., None]
        dB[:, l] = g2 * (de * x[:, l])[..., None]
        dB_size[:, l] = Gm2 * dxa
        dB_off[:, l] = Eg2 * dxa + dB_size[:, l] * w8[..., None]
        dC[:, l] = dy[:, l, :, None] * H[:, l + 1]
        dC_size[:, l] = dya[:, l, :, None] * M[:, l + 1]
        dC_off[:, l] = dya[:, l, :, None] * E[:, l + 1] + dy_off[:, l, :, None] * M[:, l + 1] + dC_size[:, l]
        on = live * de[..., None]
        dA += (t * on).sum(0)
        dA_size += (t_size * on).sum(0)
        dA_off += ((t_off + t_size * w8[..., None]) * on).sum(0)
        g, Gm, Eg = (torch.where(live > 0, p, q) for p, q in ((a * g2, g), (a * Gm2, Gm), (a * (Eg2 + Gm2 * (ao + 1)), Eg)))
    group = lambda t: t.unflatten(2, (G, W // G)).sum(3)  # noqa: E731
    # sums over positions: those of a part one after the other, then over parts of 32 positions and more and rows
    many = part + Bn * L // 32 + 32
    val.update(dx=dx * k3, ddt=ddt * k3, dB=group(dB * k4), dC=group(dC * k4), dA=dA, dD=(dy * x).sum((0, 1)), dbias=(ddt * k3).sum((0, 1)), dstate=g)
    off.update(dx=dx_off * k3, ddt=ddt_off * k3, dB=group((dB_off + (W // G + 4) * dB_size) * k4), dC=group((dC_off + (W // G + 4) * dC_size) * k4), dA=dA_off + many * dA_size,
               dD=(dy_off * x.abs()).sum((0, 1)) + many * (dya * x.abs()).sum((0, 1)), dbias=((ddt_off + many * ddt_size) * k3).sum((0, 1)), dstate=Eg)
    return val, off


def excess(got, want, bound, dtype):
    """largest |got - want| as a multiple of its bound"""
    got = got.detach().cpu().double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    add = 1.01 * U * bound
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -120}[dtype]  # (32 bits may flush what it adds to others)
    return float(((got - want).abs() / (ref.half_step(dtype) * (want.abs() + add) + add + tiny)).max()) if got.numel() else 0.0
