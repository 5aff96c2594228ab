"""Plain float64 implementations of the training and streaming operators, and
the error their fp32 kernels are allowed, derived per element from the
operations a kernel does (u = 2^-24 is half a step of fp32).

An output stored in type t is off by half a step of t more:
|y| finfo(t).eps / 2, plus half a subnormal step."""
import torch

U = 2.0 ** -24
TINY = 2.0 ** -149  # the spacing of fp32 below 2^-126


def stored(err, value, dtype):
    """The allowed error of a result stored in `dtype` whose fp32 value is off by `err`."""
    fi = torch.finfo(dtype)
    half = fi.eps / 2 * (value.abs() + err) + fi.smallest_normal * fi.eps / 2
    return err + (half if dtype != torch.float32 else TINY / 2)


def assert_within(got, want, err, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= err)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{(off / err.clamp_min(1e-300))[bad].max().item():.3g} times the allowed error")


# ---------------------------------------------------------------------- recurrence
class Recurrence:
    """x, gate [B, L, D], state [B, D], lengths [B] or None (CPU, any type).

    Error of a state: a step rounds the weight s = min(a, 1 - a) (expf 2u, the
    sum u, the quotient 4u), the difference of input and state, and the result:
    9 u s (|x| + |h|) + u |h|.  In a split scan the decay of a step enters up to
    three states that are joined (its own step, a warp's part, a tile), each
    with the same relative error and a rounding of the join, so at most three
    times that, and 4 u |h| for the roundings of the joins.  Errors decay like
    the state itself: e_t = |a_t| e_{t-1} + the step's.  In the gate form a is
    exact and its products are rounded once each.

    Relative errors end where fp32 does: a weight s below 2^-126 (a leaky gate
    beyond +-87) is a multiple of TINY, and both expf's result and the quotient
    may be one such spacing off, so s is off by 2 TINY at least, and what it
    multiplies carries that: 2 TINY (|x| + |h|) in a step, 2 TINY |g| in dx
    and in what passes to the step before, 2 TINY |g| (|h| + |x|) in dgate."""

    def __init__(self, x, gate, state, form, lengths=None, gh=None, glast=None):
        x, gate, h = x.double(), gate.double(), state.double()
        B, L, D = x.shape
        lens = torch.full((B,), L) if lengths is None else lengths.long().clamp(0, L)
        leaky = form == "leaky"
        a = torch.sigmoid(gate) if leaky else gate
        q = torch.sigmoid(-gate) if leaky else None
        s = torch.minimum(a, q) if leaky else None
        e, m = torch.zeros_like(h), h.abs()
        self.h, self.h_err = torch.zeros(B, L, D).double(), torch.zeros(B, L, D).double()
        before, before_err = torch.zeros(B, L, D).double(), torch.zeros(B, L, D).double()
        for t in range(L):
            on = (lens > t).unsqueeze(1)
            before[:, t], before_err[:, t] = h, e
            xt = torch.where(on, x[:, t], 0.0)
            at = torch.where(on, a[:, t], 1.0)
            if leaky:
                st, qt = torch.where(on, s[:, t], 0.0), torch.where(on, q[:, t], 0.0)
                new, mag = at * h + qt * xt, at * m + qt * xt.abs()
                step = (27 * U * st + 2 * TINY) * (xt.abs() + m) + 4 * U * mag
            else:
                new = at * h + torch.where(on, xt, 0.0)
                mag = at.abs() * m + torch.where(on, xt.abs(), 0.0)
                step = 6 * U * mag
            h, m, e = (torch.where(on, new, h), torch.where(on, mag, m), torch.where(on, at.abs() * e + step, e))
            self.h[:, t] = torch.where(on, h, 0.0)
            self.h_err[:, t] = torch.where(on, e, 0.0)
        self.last, self.last_err = h, e
        if gh is None:
            return
        c = glast.double()
        ce, cm = torch.zeros_like(c), c.abs()
        self.dx, self.dgate = torch.zeros_like(self.h), torch.zeros_like(self.h)
        self.dx_err, self.dgate_err = torch.zeros_like(self.h), torch.zeros_like(self.h)
        for t in range(L - 1, -1, -1):
            on = (lens > t).unsqueeze(1)
            ght = torch.where(on, gh[:, t].double(), 0.0)
            xt, at = torch.where(on, x[:, t], 0.0), torch.where(on, a[:, t], 1.0)
            hb, he = before[:, t], before_err[:, t]
            g, ge, gm = c + ght, ce + U * (cm + ght.abs()), cm + ght.abs()
            if leaky:
                qt = torch.where(on, q[:, t], 0.0)
                st = torch.where(on, s[:, t], 0.0)
                dx, dg = qt * g, g * (hb - xt) * at * qt
                dxe = qt * ge + ((8 * st + U + qt) * 2 * U + 2 * TINY) * gm
                w = at * qt  # rounded: s 7u, 1 - s, products
                dge = w * ((hb - xt).abs() * ge + gm * he + 24 * U * gm * (hb.abs() + xt.abs()))
                dge = dge + 2 * TINY * gm * (hb.abs() + xt.abs())
                back = (27 * U * st + 2 * TINY) * gm + 4 * U * at * gm
            else:
                dx, dg, dxe = g, g * hb, ge
                dge = hb.abs() * ge + gm * he + 2 * U * gm * hb.abs()
                back = 6 * U * at.abs() * gm
            c, ce, cm = (torch.where(on, at * g, c), torch.where(on, at.abs() * ge + back, ce),
                         torch.where(on, at.abs() * gm, cm))
            for buf, v in ((self.dx, dx), (self.dgate, dg), (self.dx_err, dxe), (self.dgate_err, dge)):
                buf[:, t] = torch.where(on, v, 0.0)
        self.dstate, self.dstate_err = c, ce


# ---------------------------------------------------------------------- group norm
class GroupNorm:
    """x [S, P, C], weight and bias [C] (CPU, any type).

    Errors: a sum over a group is made of parts of at most 64 terms added one
    after the other and a tree over the parts (at most 64 roundings more), so it
    is off by at most 128 u times the sum of magnitudes; every term that was
    computed adds its own error."""

    def __init__(self, x, groups, weight, bias, eps, act, thr=0.0, gy=None):
        x = x.double()
        S, P, C = x.shape
        cg, n = C // groups, P * (C // groups)
        w = torch.ones(C).double() if weight is None else weight.double()
        b = torch.zeros(C).double() if bias is None else bias.double()

        def group_mean(v):  # [S, P, C] -> the mean over the group, spread over its channels [S, 1, C]
            return v.reshape(S, P, groups, cg).sum((1, 3)).div(n).repeat_interleave(cg, 1).unsqueeze(1)

        mean = group_mean(x)
        mean_err = 128 * U * group_mean(x.abs())
        xc = x - mean
        xc_err = mean_err + 2 * U * (x.abs() + mean.abs())
        var = group_mean(xc * xc)
        var_err = 128 * U * var + group_mean(2 * xc.abs() * xc_err + xc_err ** 2)
        rstd = (var + eps).rsqrt()
        rstd_rel = 0.5 * var_err / (var + eps) + 4 * U
        rstd_rel = rstd_rel * (1 + rstd_rel)
        self.mean, self.rstd = mean[:, 0, ::cg], rstd[:, 0, ::cg]
        xhat = xc * rstd
        xhat_err = xc_err * rstd * (1 + rstd_rel) + xhat.abs() * (rstd_rel + 2 * U)
        z = xhat * w + b
        z_err = xhat_err * w.abs() + 4 * U * ((xhat * w).abs() + b.abs())
        self.z, self.z_err = z, z_err
        if act == "silu":
            sig = torch.sigmoid(z)
            self.y = z * sig
            self.y_err = 1.1 * z_err + 12 * U * (1 + z.abs()) * self.y.abs()  # |silu'| < 1.1; expf of a rounded z
            d = sig * (1 + z * (1 - sig))
            d_err = 0.5 * z_err + 16 * U * (1 + z.abs()) * (sig * (1 + (z * (1 - sig)).abs()))  # |silu''| <= 0.5
        elif act == "heaviside":
            self.y = (z - thr > 0).double()
            self.y_err = torch.where((z - thr).abs() > z_err + U * (z.abs() + abs(thr)), 0.0, 1.0)
            sig = torch.sigmoid(10 * (z - thr))
            d = 10 * sig * (1 - sig)
            arg = 10 * (z_err + 2 * U * (z.abs() + abs(thr)))
            d_err = d * (2 * arg + 16 * U) + 16 * U  # 1 - sig: rounded at 1
        else:
            self.y, self.y_err, d, d_err = z, z_err, torch.ones_like(z), torch.zeros_like(z)
        if gy is None:
            return
        gy = gy.double()
        dz, dz_err = gy * d, gy.abs() * d_err + 2 * U * (gy * d).abs()
        prod, prod_err = dz * xhat, dz_err * xhat.abs() + dz.abs() * xhat_err + 2 * U * (dz * xhat).abs()
        total = lambda v: v.sum((0, 1))  # noqa: E731
        self.dbias, self.dbias_err = total(dz), total(dz_err) + 128 * U * total(dz.abs())
        self.dweight, self.dweight_err = total(prod), total(prod_err) + 128 * U * total(prod.abs())
        m1, m2 = group_mean(dz * w), group_mean(prod * w)
        m1_err = group_mean(dz_err * w.abs()) + 130 * U * group_mean((dz * w).abs())
        m2_err = group_mean(prod_err * w.abs()) + 130 * U * group_mean((prod * w).abs())
        inner = dz * w - m1 - xhat * m2
        size = (dz * w).abs() + m1.abs() + (xhat * m2).abs()
        inner_err = dz_err * w.abs() + m1_err + xhat_err * m2.abs() + xhat.abs() * m2_err + 4 * U * size
        self.dx = rstd * inner
        self.dx_err = rstd * (1 + rstd_rel) * inner_err + self.dx.abs() * (rstd_rel + 2 * U)


# ---------------------------------------------------------------------- dropout
def philox(counter, key, rounds=7):
    """Philox4x32 (Salmon et al., 2011) of one counter (four words) under a key (two words)."""
    c, k = [int(v) for v in counter], [int(v) for v in key]
    for _ in range(rounds):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_words(n, seed, offset):
    """The n words of a dropout call, one per element (Python integers)."""
    words = []
    for i in range((n + 3) // 4):
        words += philox((i & 0xFFFFFFFF, i >> 32, offset & 0xFFFFFFFF, (offset >> 32) & 0xFFFFFFFF),
                        (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    return words[:n]
