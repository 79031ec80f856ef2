"""numpy restatement, in 64 bits, of the feedback operators (label-path log-probabilities, preference loss, clipped policy loss) and of the
4-bit microscaled form -- test infrastructure only.  Written from the definitions, class by class; nothing here is fast."""
import numpy as np


def level_slices(levels):
    s = 0
    for n in levels:
        yield s, s + n
        s += n


def log_softmax(z):
    """Row-wise; a row with nothing finite, a NaN or a +inf is NaN, as the definition has it."""
    with np.errstate(all='ignore'):
        m = z.max(axis=-1, keepdims=True)
        return (z - m) - np.log(np.exp(z - m).sum(axis=-1, keepdims=True))


def path_log_probs(z, paths, levels):
    """z [R, C], paths [R, G, L] -> logp [R, G, L]; 0 where paths < 0, NaN where a class is not in its level."""
    z = np.asarray(z, dtype=np.float64)
    out = np.zeros(paths.shape)
    for l, (a, b) in enumerate(level_slices(levels)):
        ls = log_softmax(z[:, a:b])
        for r in range(paths.shape[0]):
            for g in range(paths.shape[1]):
                y = int(paths[r, g, l])
                if y >= b - a:
                    out[r, g, l] = np.nan
                elif y >= 0:
                    out[r, g, l] = ls[r, y]
    return out


def path_grad(z, paths, levels, coef):
    """d/dz of sum(coef * logp): dz, and the two non-negative parts it is the difference of summed (for error bounds)."""
    z = np.asarray(z, dtype=np.float64)
    dz, size = np.zeros(z.shape), np.zeros(z.shape)
    for l, (a, b) in enumerate(level_slices(levels)):
        with np.errstate(all='ignore'):
            p = np.exp(log_softmax(z[:, a:b]))
        for r in range(paths.shape[0]):
            y = paths[r, :, l]
            on = y >= 0
            if not on.any():
                continue                                        # nothing counted: exactly zero, whatever the level holds
            if (y >= b - a).any():
                dz[r, a:b] = np.nan
                continue
            c = np.where(on, coef[r, :, l], 0.0)
            A = c.sum()
            dz[r, a:b] = -A * p[r] if A != 0 else 0.0
            size[r, a:b] = np.abs(c).sum() * p[r]
            for g in np.nonzero(on)[0]:
                dz[r, a + y[g]] += c[g]; size[r, a + y[g]] += abs(c[g])
    return dz, size


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


def sigmoid(x):
    return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def preference_loss(z, paths, ref, levels, beta, smooth):
    """paths [P, 2, L] (both on row p) or [2P, L] (the chosen rows first) -> loss, rewards [P, 2], coef of paths' shape."""
    shared = paths.ndim == 3
    p3 = paths if shared else paths[:, None]
    lp = path_log_probs(z, p3, levels)
    r = beta * np.where(p3 >= 0, lp - np.where(p3 >= 0, ref if shared else ref[:, None], 0.0), 0.0).sum(2)
    P = r.shape[0] if shared else r.shape[0] // 2
    r = r if shared else np.stack([r[:P, 0], r[P:, 0]], 1)
    d = r[:, 0] - r[:, 1]
    loss = ((1 - smooth) * softplus(-d) + smooth * softplus(d)).mean()
    g = (smooth * sigmoid(d) - (1 - smooth) * sigmoid(-d)) * beta / P
    c = np.stack([g, -g], 1)
    c = (c[:, :, None] if shared else c.T.reshape(2 * P, 1, 1)) * (p3 >= 0)
    return loss, r, c.reshape(paths.shape)


def policy_loss(z, paths, adv, old, ref, levels, low, high, kl, reduction):
    """paths [R, G, L], adv [R, G] -> loss, stats (mean k3, clipped share), coef [R, G, L]."""
    on = paths >= 0
    lp = path_log_probs(z, paths, levels)
    A = np.asarray(adv, dtype=np.float64)[:, :, None]
    rho = np.ones(lp.shape) if old is None else np.exp(np.where(on, lp - np.where(on, old, 0.0), 0.0))
    clipped = on & (((A > 0) & (rho > 1 + high)) | ((A < 0) & (rho < 1 - low)))
    gain = np.minimum(rho * A, np.clip(rho, 1 - low, 1 + high) * A)
    q = np.zeros(lp.shape) if ref is None else np.where(on, np.where(on, ref, 0.0) - lp, 0.0)
    k3 = np.expm1(q) - q
    if reduction == 'level':
        w = on / max(on.sum(), 1)
    else:
        w = on / np.maximum(on.sum(2, keepdims=True), 1) / (on.shape[0] * on.shape[1])
    loss = (w * (kl * k3 - gain)).sum()
    coef = w * (np.where(clipped, 0.0, -rho * A) - kl * np.expm1(q))
    return loss, np.array([(w * k3).sum(), (w * clipped).sum()]), coef


# ------------------------------------------------------------------------------------------------ 4-bit microscaled form
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mxfp4_values(x):
    """The values the 4-bit form of x [rows, k] stands for: per block of 32 the power of two, then the nearest of the eight magnitudes (the one
    with the even code on a tie), 6 beyond the last."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    out = np.empty((rows, k))
    for a in range(0, k, 32):
        v = x[:, a:a + 32]
        top = np.abs(v).max(1)
        bad = ~np.isfinite(top)
        _, e = np.frexp(np.where(bad | (top == 0), 1.0, top))
        X = np.where(top == 0, -127, np.clip(e - 3, -127, 127))
        s = np.ldexp(1.0, X)[:, None]
        q = np.abs(np.where(bad[:, None], 0.0, v)) / s
        d = np.abs(q[:, :, None] - E2M1)
        best = d.min(2, keepdims=True)
        near = d == best                                        # one code, or two neighbours of which one is even
        code = np.where(near.sum(2) > 1, (near * (np.arange(8) % 2 == 0)).argmax(2), near.argmax(2))
        out[:, a:a + 32] = np.where(bad[:, None], np.nan, np.copysign(E2M1[code] * s, v))
    return out
