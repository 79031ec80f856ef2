"""Feedback operators on the MI355X against the 64-bit oracle: values, gradients, masks, strides, streams, graphs.

Tolerances, from the arithmetic (u = 2^-24, one rounding to 32 bits):
  * a softmax term exp(z - m): the difference, its product with log2 e and the constant round by u each, relative error 3 |z - m| u, plus 2 u of the exponential;
    the mean of |z - m| under the softmax is at most log n, the sum's chain is at most 40 + 6 + 24 additions: relative error of the sum below (3 log n + 80) u;
  * logp in 64 bits from that sum, rounded once: LT(n) = (3 log n + 90) u, plus u |logp|;
  * a probability: (3 |z - m| + 3 log n + 90) u relative;
  * a coefficient follows from logp in 64 bits: its error is the formula's derivative times LT, plus u of itself;
  * the gradient's elements round once to the logits' type: half a step, eps / 2 relative (fp16 also 2^-25 absolute below its normal range)."""
import numpy as np
import pytest
import torch

from oracle import feedback_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
ETHEC = [6, 21, 135, 561]
S5 = [2, 8, 32, 128, 512, 2048, 8192, 39078]
LEVELS = {'one': [1], 'two': [2], 'ones': [1, 1, 1], 'odd': [3, 5], 'ethec': ETHEC, 'sixteen': list(range(1, 17)), 'run32': [2303, 2304, 2305], 'run16': [2559, 2560, 2561],
          'wide': [4608, 5121, 7], 's5': S5}


def LT(levels):
    return np.array([(3 * np.log(n) + 90) * U for n in levels])


def make(levels, R, G, dtype, seed=0, known=0.8):
    """z in the type under test (as float64 too), paths, old, ref, adv: an entry's ratio stays off both clip bounds by 1e-3."""
    rs = np.random.RandomState(seed)
    z = torch.from_numpy((rs.randn(R, sum(levels)) * 2.5).astype(np.float32)).to(DT[dtype])
    zd = z.double().numpy()
    paths = np.stack([rs.randint(0, n, size=(R, G)) for n in levels], 2)
    paths[rs.rand(*paths.shape) > known] = -1
    if R > 2:
        paths[1] = -1                                           # a row with nothing known
        paths[2] = paths[2, :1]                                 # a row whose paths are all the same
    lp = O.path_log_probs(zd, paths, levels)
    d = 0.25 * rs.randn(*lp.shape)
    for b in (0.8, 1.2):
        d[np.abs(np.exp(d) - b) < 1e-3] += 0.004
    old, ref = (lp - d), lp + 0.3 * rs.randn(*lp.shape)
    old, ref = old.astype(np.float32), ref.astype(np.float32)
    return z, zd, paths, old, ref, rs.randn(R, G).astype(np.float32)


def dev(a):
    return (torch.from_numpy(a) if isinstance(a, np.ndarray) else a).cuda()


def check_grad(got, z, zd, paths, levels, coef, coef_err, dtype):
    want, size = O.path_grad(zd, paths, levels, coef)
    _, err = O.path_grad(zd, paths, levels, coef_err)
    tol = np.zeros_like(want)
    for l, (a, b) in enumerate(O.level_slices(levels)):
        span = zd[:, a:b].max(1, keepdims=True) - zd[:, a:b]
        tol[:, a:b] = (3 * span + 3 * np.log(b - a) + 100) * U * size[:, a:b] + err[:, a:b]
    tol += torch.finfo(DT[dtype]).eps / 2 * (np.abs(want) + tol) + (2.0 ** -25 if dtype == 'fp16' else 1e-37)
    g = got.double().cpu().numpy()
    assert g.shape == want.shape and got.dtype == DT[dtype]
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), 'max error / tolerance %.3g at %s' % ((np.abs(g - want) / tol).max(), np.argwhere(bad)[0])
    return g


SHAPES = [('one', 1, 1), ('two', 3, 1), ('ones', 4, 2), ('odd', 5, 3), ('ethec', 1, 1), ('ethec', 37, 8), ('sixteen', 9, 5), ('run32', 3, 2), ('run16', 3, 2), ('wide', 4, 3),
          ('ethec', 3, 64), ('s5', 3, 2)]


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('name,R,G', SHAPES)
def test_path_log_probs(name, R, G, dtype):
    from learning_embeddings_amd import loss
    lv = LEVELS[name]
    z, zd, paths, _, _, _ = make(lv, R, G, dtype)
    zt = dev(z).requires_grad_()
    lp = loss.path_log_probs(zt, dev(paths), lv)
    want = O.path_log_probs(zd, paths, lv)
    assert lp.dtype == torch.float32 and lp.shape == paths.shape
    assert (np.abs(lp.detach().cpu().numpy() - want) <= LT(lv) + U * np.abs(want)).all()
    assert (lp.detach().cpu().numpy()[paths < 0] == 0).all()
    up = np.random.RandomState(9).randn(*paths.shape).astype(np.float32)
    lp.backward(dev(up))
    check_grad(zt.grad, z, zd, paths, lv, up.astype(np.float64), 2 * U * G * np.abs(up), dtype)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('shared', [True, False])
@pytest.mark.parametrize('name,P', [('one', 1), ('odd', 5), ('ethec', 1), ('ethec', 33), ('sixteen', 9), ('wide', 4), ('s5', 2)])
@pytest.mark.parametrize('smooth', [0.0, 0.1])
def test_preference_loss(name, P, shared, dtype, smooth):
    from learning_embeddings_amd import loss
    lv = LEVELS[name]
    R, G = (P, 2) if shared else (2 * P, 1)
    z, zd, paths, _, ref, _ = make(lv, R, G, dtype, seed=3)
    p, rf = (paths, ref) if shared else (paths[:, 0], ref[:, 0])
    beta = 0.5
    zt = dev(z).requires_grad_()
    l, rewards = loss.PreferenceLoss(lv, beta=beta, label_smoothing=smooth)(zt, dev(p), dev(rf))
    assert not rewards.requires_grad
    want, r, coef = O.preference_loss(zd, p, rf.astype(np.float64), lv, beta, smooth)
    ed = beta * 2 * LT(lv).sum()
    assert abs(float(l) - want) <= ed + 2 * U * abs(want)
    assert (np.abs(rewards.cpu().numpy() - r) <= ed + U * np.abs(r)).all()
    l.backward()
    cerr = (beta / P * (ed / 4 + 2 * U) + 4 * U * np.abs(coef)) * (p >= 0)
    full = (lambda a: a) if shared else (lambda a: a[:, None])
    check_grad(zt.grad, z, zd, paths, lv, full(coef), full(cerr), dtype)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('name,R,G', SHAPES)
@pytest.mark.parametrize('reduction,kl,with_old', [('level', 0.1, True), ('path', 0.0, True), ('path', 0.1, False)])
def test_policy_loss(name, R, G, dtype, reduction, kl, with_old):
    from learning_embeddings_amd import loss
    lv = LEVELS[name]
    z, zd, paths, old, ref, adv = make(lv, R, G, dtype, seed=5)
    zt = dev(z).requires_grad_()
    crit = loss.ClippedPolicyLoss(lv, clip_low=0.2, clip_high=0.2, kl_coef=kl, reduction=reduction)
    l, stats = crit(zt, dev(paths), dev(adv), dev(old) if with_old else None, dev(ref) if kl else None)
    o64, r64 = (old.astype(np.float64) if with_old else None), (ref.astype(np.float64) if kl else None)
    want, st, coef = O.policy_loss(zd, paths, adv, o64, r64, lv, 0.2, 0.2, kl, reduction)
    on = paths >= 0
    w = on / max(on.sum(), 1) if reduction == 'level' else on / np.maximum(on.sum(2, keepdims=True), 1) / (R * G)
    lp = O.path_log_probs(zd, paths, lv)
    rho = np.exp(np.where(on, lp - old, 0)) if with_old else np.ones(lp.shape)
    q = np.where(on, ref - lp, 0) if kl else np.zeros(lp.shape)
    A = np.abs(adv.astype(np.float64))[:, :, None]
    e_t = w * LT(lv) * (rho * A + kl * (np.exp(q) + 1))
    mag = (w * (rho * A + kl * np.abs(np.expm1(q) - q))).sum()
    assert abs(float(l) - want) <= e_t.sum() + 4 * U * mag
    assert abs(float(stats[0]) - st[0]) <= (w * LT(lv) * (np.exp(q) + 1)).sum() + 4 * U * st[0]
    assert abs(float(stats[1]) - st[1]) <= 4 * U
    l.backward()
    cerr = w * LT(lv) * (rho * A + kl * np.exp(q)) + 8 * U * G * np.abs(coef)
    check_grad(zt.grad, z, zd, paths, lv, coef, cerr, dtype)


def test_gradient_against_differences_of_the_kernels_own_loss():
    """Directional derivative, h = 2^-6: truncation h^2 / 6 times the third derivative along v (|v| <= 1 element-wise, 4 levels, beta 0.5: below 4, so 2e-4), and the two
    losses' errors (LT of four levels, beta 0.5: 4e-5) over 2 h: 3e-3.  The derivative itself is of order 0.1."""
    from learning_embeddings_amd import loss
    z, zd, paths, _, ref, _ = make(ETHEC, 6, 2, 'fp32', seed=11, known=1.0)
    crit = loss.PreferenceLoss(ETHEC, beta=0.5)
    v = torch.from_numpy(np.random.RandomState(12).uniform(-1, 1, size=z.shape).astype(np.float32)).cuda()
    zt = dev(z).requires_grad_()
    crit(zt, dev(paths), dev(ref))[0].backward()
    h = 2.0 ** -6
    with torch.no_grad():
        d = (float(crit(zt + h * v, dev(paths), dev(ref))[0]) - float(crit(zt - h * v, dev(paths), dev(ref))[0])) / (2 * h)
    assert abs(d - float((zt.grad * v).sum())) < 4e-3


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_levels_nobody_counts_may_hold_anything(dtype):
    from learning_embeddings_amd import loss
    z, zd, paths, old, ref, adv = make(ETHEC, 7, 3, dtype, seed=7, known=1.0)
    paths[:, :, 2] = -1; paths[3] = -1
    clean = dev(z).requires_grad_()
    dirty_z = z.clone()
    dirty_z[:, 27:162] = float('nan'); dirty_z[3] = float('inf')
    dirty = dev(dirty_z).requires_grad_()
    old2, ref2 = old.copy(), ref.copy()
    old2[paths < 0] = np.nan; ref2[paths < 0] = np.inf
    crit = loss.ClippedPolicyLoss(ETHEC, kl_coef=0.1)
    a, sa = crit(clean, dev(paths), dev(adv), dev(old), dev(ref)); a.backward()
    b, sb = crit(dirty, dev(paths), dev(adv), dev(old2), dev(ref2)); b.backward()
    assert torch.isfinite(a) and torch.equal(a, b) and torch.equal(sa, sb)
    assert torch.equal(clean.grad, dirty.grad)
    assert (dirty.grad[:, 27:162] == 0).all() and (dirty.grad[3] == 0).all()


def test_nothing_counted_at_all():
    from learning_embeddings_amd import loss
    z = torch.full((4, sum(ETHEC)), float('nan'), device='cuda', requires_grad=True)
    none = torch.full((4, 2, 4), -1, device='cuda')
    e = torch.full((4, 2, 4), float('nan'), device='cuda')
    for red in ('level', 'path'):
        z.grad = None
        l, st = loss.ClippedPolicyLoss(ETHEC, kl_coef=0.1, reduction=red)(z, none, torch.ones(4, 2, device='cuda'), e, e)
        l.backward()
        assert float(l) == 0 and (st == 0).all() and (z.grad == 0).all()
    z.grad = None
    l, r = loss.PreferenceLoss(ETHEC)(z, none, e)
    l.backward()
    assert abs(float(l) - np.log(2)) <= 2 * U and (r == 0).all() and (z.grad == 0).all()


def test_excluded_classes_and_special_values():
    """-inf (or the type's lowest value) takes a class out of its softmax; a counted class that is out has logp -inf; a level with nothing in, a NaN or a +inf gives NaN;
    a class that the level does not have gives NaN and reads nothing; other rows are as without."""
    from learning_embeddings_amd import loss
    lv = [4, 700]
    z, zd, _, _, _, _ = make(lv, 8, 1, 'fp32', seed=1)
    z[0, 1:4] = -float('inf'); z[1, 4:704] = -float('inf'); z[2, 5] = float('nan'); z[3, 6] = float('inf'); z[4, 1:3] = torch.finfo(torch.float32).min
    zd = z.double().numpy()
    paths = np.zeros((8, 1, 2), dtype=np.int64)
    paths[5, 0, 1] = 700; paths[6, 0, 0] = 2 ** 40; paths[7, 0, 1] = -2 ** 40
    zt = dev(z).requires_grad_()
    lp = loss.path_log_probs(zt, dev(paths), lv)
    lp.backward(torch.ones_like(lp))
    got, g = lp.detach().cpu().numpy()[:, 0], zt.grad.cpu().numpy()
    want = O.path_log_probs(zd, paths, lv)[:, 0]
    nan = np.zeros((8, 2), dtype=bool); nan[[1, 2, 3, 5], 1] = True; nan[6, 0] = True
    assert (np.isnan(got) == nan).all() and (np.abs(got - want)[~nan] <= (LT(lv) + U * np.abs(want))[~nan]).all()
    assert got[7, 1] == 0 and got[0, 0] == 0
    for r in range(8):
        for l, (a, b) in enumerate(O.level_slices(lv)):
            assert np.isfinite(g[r, a:b]).all() == (not nan[r, l]), (r, l)
    assert (g[0, 1:4] == 0).all() and (g[4, 1:3] == 0).all() and (g[7, 4:] == 0).all()
    out = torch.zeros(1, 704, device='cuda'); out[0, 0] = -float('inf')
    assert float(loss.path_log_probs(out, torch.zeros(1, 2, dtype=torch.int64, device='cuda'), lv)[0, 0]) == -float('inf')


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_levels_full_of_the_lowest_or_highest_value_are_uniform(dtype):
    """Every class at the type's lowest (highest) value: the softmax is uniform; one class apart from the rest takes it all.  Offsets that no difference shows change nothing."""
    from learning_embeddings_amd import loss
    lv = [4, 700, 3000]
    f = torch.finfo(DT[dtype])
    z = torch.zeros(4, 3704, dtype=DT[dtype])
    z[0] = f.min; z[1] = f.max; z[2] = f.min; z[2, 4:8] = 0.0; z[3] = 1000.0
    paths = np.full((4, 1, 3), 2, dtype=np.int64)
    zt = dev(z).requires_grad_()
    lp = loss.path_log_probs(zt, dev(paths), lv)
    lp.backward(torch.ones_like(lp))
    want = -np.log(np.array([[4, 700, 3000], [4, 700, 3000], [4, 4, 3000], [4, 700, 3000]], dtype=np.float64))
    assert (np.abs(lp.detach().cpu().numpy()[:, 0] - want) <= LT(lv) + U * np.abs(want)).all()
    check_grad(zt.grad, z, z.double().numpy(), paths, lv, np.ones(paths.shape), np.full(paths.shape, 2 * U), dtype)


@pytest.mark.parametrize('offset', [2.0 ** 10, 2.0 ** 19, 2.0 ** 20, 2.0 ** 24, 2.0 ** 34, 2.0 ** 60, 2.0 ** 125])
@pytest.mark.parametrize('sign', [1, -1])
def test_logits_far_from_zero(offset, sign):
    """Logits a few units in the last place apart at any distance from zero: their differences are exact, and so are the softmaxes'."""
    from learning_embeddings_amd import loss
    lv = [4, 700, 3000]
    rs = np.random.RandomState(3)
    step = max(offset * 2.0 ** -23, 0.25)
    z = torch.from_numpy((sign * offset + step * rs.randint(-8, 9, size=(5, 3704))).astype(np.float32))
    paths = np.stack([rs.randint(0, n, size=(5, 2)) for n in lv], 2)
    zt = dev(z).requires_grad_()
    lp = loss.path_log_probs(zt, dev(paths), lv)
    lp.backward(torch.ones_like(lp))
    want = O.path_log_probs(z.double().numpy(), paths, lv)
    assert (np.abs(lp.detach().cpu().numpy() - want) <= LT(lv) + U * np.abs(want)).all()
    check_grad(zt.grad, z, z.double().numpy(), paths, lv, np.ones(paths.shape), np.full(paths.shape, 4 * U), 'fp32')


@pytest.mark.parametrize('name,dtype', [('ethec', 'fp32'), ('ethec', 'bf16'), ('run32', 'fp32'), ('s5', 'fp16')])
def test_ratios_next_to_the_clip_bounds_are_decided_exactly(name, dtype):
    """The gradient jumps at the bound, so the decision has to be the formula's own, not that of a sum with 32 bits: every 16th row has an entry whose old log-probability
    puts log rho within half a step of a float of the bound (about 1e-7, where the error of a softmax's sum in 32 bits is as large)."""
    from learning_embeddings_amd import loss
    levels = LEVELS[name]
    R = 512 if name == 'ethec' else 256
    g = torch.Generator(device='cuda').manual_seed(21)
    z = (torch.randn(R, sum(levels), generator=g, device='cuda') * 2.5).to(DT[dtype])
    y = torch.stack([torch.randint(0, n, (R,), generator=g, device='cuda') for n in levels], 1)
    exact = torch.stack([torch.log_softmax(zl.double(), 1).gather(1, yl[:, None])[:, 0] for zl, yl in zip(z.split(levels, 1), y.unbind(1))], 1)
    adv = torch.where(torch.arange(R, device='cuda') % 32 < 16, 1.0, -1.0) * (1 + torch.rand(R, generator=g, device='cuda'))
    hi, lo = 0.25, 0.25                                          # 1 + hi and 1 - lo are floats
    bound = torch.where(adv > 0, 1 + hi, 1 - lo).double().log()[:, None]
    old = (exact - bound / 2).float()                            # well inside
    edge = torch.zeros(R, len(levels), dtype=torch.bool, device='cuda')
    rows = torch.arange(0, R, 16, device='cuda')
    edge[rows, rows // 16 % len(levels)] = True
    old = torch.where(edge, (exact - bound).float(), old)
    off = exact - old.double() - bound                           # log rho - log bound
    hit = torch.where(adv[:, None] > 0, off > 0, off < 0) & edge
    assert off[edge].abs().max() < 2e-6 and off[edge].abs().min() > 1e-12 and 0 < hit.sum() < edge.sum()      # near, but no ties
    zz = z.requires_grad_()
    l, st = loss.ClippedPolicyLoss(levels, clip_low=lo, clip_high=hi)(zz, y, adv, old)
    grad, = torch.autograd.grad(l, zz)
    n = R * len(levels)
    assert round(st[1].item() * n) == hit.sum().item() and abs(st[1].item() * n - hit.sum().item()) < 1e-3
    c = torch.where(hit, 0.0, -(exact - old.double()).exp() * adv.double()[:, None] / n)                        # d loss / d logp
    want, s = torch.zeros_like(z, dtype=torch.float64), 0
    for k, m in enumerate(levels):
        p = torch.softmax(z[:, s:s + m].detach().double(), 1)
        want[:, s:s + m] = -c[:, k:k + 1] * p
        want[:, s:s + m].scatter_add_(1, y[:, k:k + 1], c[:, k:k + 1])
        s += m
    # a wrong decision moves a row's level by |c| = 0.75 / n or more; a right one by its rounding and by the 32-bit softmax's error, (3 span + 3 log(classes) + 100) 2^-24 of
    # |c| <= 2.5 / n: with a span of 30 below 4e-5 / n (fp16's smallest step, 2^-25, is below 4e-5 / n too)
    tol = torch.finfo(DT[dtype]).eps / 2 * want.abs() + 1e-4 / n
    assert ((grad.double() - want).abs() <= tol).all()


def test_every_ratio_at_its_bound():
    """Bounds of 0 and the model's own log-probabilities: every ratio is 1 within a rounding, more of them next to the bound than are summed again.  Whatever is decided is
    one of the two gradients, the loss is -mean A within the roundings, and the bits are the same every time."""
    from learning_embeddings_amd import loss
    z, zd, paths, _, _, adv = make(ETHEC, 300, 3, 'fp32', seed=4)
    y, a = dev(paths), dev(adv)
    zz = dev(z).requires_grad_()
    old = loss.path_log_probs(zz, y, ETHEC).detach()
    crit = loss.ClippedPolicyLoss(ETHEC, clip_low=0.0, clip_high=0.0)
    runs = []
    for _ in range(3):
        l, st = crit(zz, y, a, old)
        runs.append((l.detach(), st, torch.autograd.grad(l, zz)[0]))
    assert all(torch.equal(u, v) for r in runs[1:] for u, v in zip(runs[0], r))
    on = paths >= 0
    want = -(adv[:, :, None] * on).sum() / on.sum()
    # rho = 1 within a rounding of logp (2^-24 of at most 16) and the sum's own error (below 2^-20): 2e-6 of mean |A|; the share is a proper one
    assert abs(runs[0][0].item() - want) <= 2e-6 * np.abs(adv).mean() + U and 0.0 <= runs[0][1][1].item() <= 1.0
    assert torch.isfinite(runs[0][2]).all()


@pytest.mark.parametrize('old', [-0.25, -0.18, 0.1, 0.31])
@pytest.mark.parametrize('step', [1e-10, -1e-10])
def test_clip_bounds_keep_64_bits(old, step):
    """One class a level: log p is 0 exactly and rho = exp(-old).  A bound 1e-10 beyond rho does not clip, one 1e-10 short of it does; rounded to 32 bits (steps of 1e-8) it
    would be either."""
    from learning_embeddings_amd import loss
    old = float(np.float32(old))
    away = abs(np.expm1(-old)) + step
    crit = loss.ClippedPolicyLoss([1], clip_low=away, clip_high=away)
    z = torch.zeros(1, 1, device='cuda', requires_grad=True)
    l, st = crit(z, torch.zeros(1, 1, dtype=torch.int64, device='cuda'), torch.tensor([1.0 if old < 0 else -1.0], device='cuda'), torch.tensor([[old]], device='cuda'))
    assert st[1].item() == (1.0 if step < 0 else 0.0)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_strided_transposed_and_broadcast_logits(dtype):
    from learning_embeddings_amd import loss
    lv = [3, 5, 600]
    z, zd, paths, _, _, _ = make(lv, 6, 2, dtype, seed=2)
    y = dev(paths)
    base = dev(z)
    plain = base.clone().requires_grad_()
    ref = loss.path_log_probs(plain, y, lv); ref.sum().backward()
    for off in (0, 1, 3):                                       # a slice of columns: odd offset, odd row stride
        big = torch.full((6, 613 + off), float('nan'), dtype=z.dtype, device='cuda')
        big[:, off:off + 608] = base
        big.requires_grad_()
        lp = loss.path_log_probs(big[:, off:off + 608], y, lv); lp.sum().backward()
        assert torch.equal(lp, ref) and torch.equal(big.grad[:, off:off + 608], plain.grad) and (big.grad[:, :off] == 0).all() and (big.grad[:, off + 608:] == 0).all()
    tr = base.t().contiguous().requires_grad_()
    lp = loss.path_log_probs(tr.t(), y, lv); lp.sum().backward()
    assert torch.equal(lp, ref) and torch.equal(tr.grad, plain.grad.t())
    every = base.flip(0)[::2].contiguous()                      # strided rows and strided paths
    big = base.flip(0)
    lp = loss.path_log_probs(big[::2], y[::2], lv)
    assert torch.equal(lp, loss.path_log_probs(every, y[::2].contiguous(), lv))
    row = base[:1].clone().requires_grad_()                     # one row for all paths: its gradient is the sum over the rows
    lp = loss.path_log_probs(row.expand(6, -1), y, lv); lp.sum().backward()
    want, size = O.path_grad(np.repeat(zd[:1], 6, 0), paths, lv, np.ones(paths.shape))
    half = torch.finfo(z.dtype).eps / 2
    assert (np.abs(row.grad.double().cpu().numpy()[0] - want.sum(0)) <= (200 * U + 7 * half) * size.sum(0) + 2.0 ** -22).all()


def test_scaled_and_summed_upstream_and_two_uses_of_one_tensor():
    from learning_embeddings_amd import loss
    z, zd, paths, old, ref, adv = make(ETHEC, 9, 2, 'fp32', seed=8)
    crit = loss.PreferenceLoss(ETHEC); pol = loss.ClippedPolicyLoss(ETHEC, kl_coef=0.05)
    a = dev(z).requires_grad_(); crit(a, dev(paths), dev(ref))[0].backward()
    b = dev(z).requires_grad_(); pol(b, dev(paths), dev(adv), dev(old), dev(ref))[0].backward()
    c = dev(z).requires_grad_()
    l = 0.5 * crit(c, dev(paths), dev(ref))[0] + 2.0 * pol(c, dev(paths), dev(adv), dev(old), dev(ref))[0]
    l.backward(retain_graph=True)
    want = 0.5 * a.grad + 2.0 * b.grad
    tol = 8 * U * (0.5 * a.grad.abs() + 2.0 * b.grad.abs())
    assert ((c.grad - want).abs() <= tol + 1e-30).all()
    first = c.grad.clone(); c.grad = None
    l.backward()                                                # a second backward of the same graph
    assert torch.equal(first, c.grad)
    l, _ = crit(c, dev(paths), dev(ref))
    l += 1.0                                                    # the value may be changed in place, the inputs of the backward may not
    l.backward()
    l, _ = crit(c * 1.0, dev(paths), dev(ref))
    y = c * 1.0
    l, _ = crit(y, dev(paths), dev(ref))
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match='inplace'):
        l.backward()


def test_empty_batches_and_int32_paths():
    from learning_embeddings_amd import loss
    z = torch.zeros(0, sum(ETHEC), device='cuda', requires_grad=True)
    lp = loss.path_log_probs(z, torch.zeros(0, 4, dtype=torch.int64, device='cuda'), ETHEC)
    assert lp.shape == (0, 4)
    lp.sum().backward()
    assert z.grad.shape == z.shape
    z = torch.randn(3, sum(ETHEC), device='cuda', requires_grad=True)
    lp = loss.path_log_probs(z, torch.zeros(3, 0, 4, dtype=torch.int64, device='cuda'), ETHEC)
    assert lp.shape == (3, 0, 4)
    lp.sum().backward()
    assert (z.grad == 0).all()
    y = torch.tensor([[0, 1, 2, 3]] * 3, device='cuda')
    assert torch.equal(loss.path_log_probs(z, y, ETHEC), loss.path_log_probs(z, y.int(), ETHEC))
    with pytest.raises(ValueError, match='logits on'):
        loss.path_log_probs(z, y.cpu(), ETHEC)
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        loss.path_log_probs(z.double(), y, ETHEC)


def test_many_rows_give_the_same_bits_every_time_and_on_another_stream():
    from learning_embeddings_amd import loss
    g = torch.Generator(device='cuda').manual_seed(0)
    z = torch.randn(3001, sum(ETHEC), generator=g, device='cuda').requires_grad_()
    y = torch.stack([torch.randint(-1, n, (3001, 5), generator=g, device='cuda') for n in ETHEC], 2)
    e = torch.randn(3001, 5, 4, generator=g, device='cuda') - 5
    adv = torch.randn(3001, 5, generator=g, device='cuda')
    crit = loss.ClippedPolicyLoss(ETHEC, kl_coef=0.01)
    def once():
        z.grad = None
        l, st = crit(z, y, adv, e, e); l.backward()
        return l.detach().clone(), st.clone(), z.grad.clone()
    a, b = once(), once()
    s = torch.cuda.Stream(); s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = once()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for other in (b, c):
        assert all(torch.equal(u, v) for u, v in zip(a, other))


@pytest.mark.parametrize('which', ['pref', 'policy', 'logp'])
def test_captured_and_replayed(which):
    """Two graphs captured on one stream share no buffer: replayed in turn and out of order, between eager work, each equals the eager result."""
    from learning_embeddings_amd import loss
    z, zd, paths, old, ref, adv = make(ETHEC, 40, 2, 'fp32', seed=13)
    y, o, r, a = dev(paths), dev(old), dev(ref), dev(adv)
    pref, pol = loss.PreferenceLoss(ETHEC), loss.ClippedPolicyLoss(ETHEC, kl_coef=0.1)
    def step(zz):
        zz = zz.detach().requires_grad_()
        if which == 'pref':
            v = pref(zz, y, r)[0]
        elif which == 'policy':
            v = pol(zz, y, a, o, r)[0]
        else:
            v = (loss.path_log_probs(zz, y, ETHEC) * o).sum(2).amax()
        g, = torch.autograd.grad(v, zz)
        return v.detach(), g
    inputs = [dev(z).clone(), dev(z).clone()]
    s = torch.cuda.Stream(); s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(inputs[0])
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for x in inputs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs.append(step(x))
        graphs.append(gr)
    gen = torch.Generator(device='cuda').manual_seed(5)
    for k in range(4):
        for x in inputs:
            x.normal_(generator=gen)
        want = [step(x) for x in inputs]
        for i in ((0, 1), (1, 0), (1, 1), (0, 0))[k]:
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in set(((0, 1), (1, 0), (1, 1), (0, 0))[k]):
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_a_level_of_more_runs_than_a_wave_has_lanes(dtype):
    from learning_embeddings_amd import loss
    lv = [5, 200001]
    z, zd, paths, old, ref, adv = make(lv, 3, 2, dtype, seed=21, known=1.0)
    paths[0] = [[4, 200000], [0, 0]]
    zt = dev(z).requires_grad_()
    lp = loss.path_log_probs(zt, dev(paths), lv)
    want = O.path_log_probs(zd, paths, lv)
    slack = (200001 / 2304 + 1) * U                             # the runs are more than the 24 that LT counts
    assert (np.abs(lp.detach().cpu().numpy() - want) <= LT(lv) + slack + U * np.abs(want)).all()
    old = (want - 0.1).astype(np.float32)
    l, _ = loss.ClippedPolicyLoss(lv, kl_coef=0.1)(zt, dev(paths), dev(adv), dev(old), dev(ref))
    ref[0] = want[0] + 0.1
    l, _ = loss.ClippedPolicyLoss(lv, kl_coef=0.1)(zt, dev(paths), dev(adv), dev(old), dev(ref))
    w_loss, _, coef = O.policy_loss(zd, paths, adv, old.astype(np.float64), ref.astype(np.float64), lv, 0.2, 0.2, 0.1, 'level')
    q = np.abs(ref - want)
    err = (LT(lv) + slack) * (1.3 * np.abs(adv)[:, :, None] + 0.1 * (np.exp(q) + 1)) / coef.size
    assert abs(float(l.detach()) - w_loss) <= err.sum() + 8 * U * (np.abs(adv).max() + np.exp(q).max())
    l.backward()
    check_grad(zt.grad, z, zd, paths, lv, coef, err + slack * np.abs(coef) + 16 * U * np.abs(coef), dtype)


def test_more_logits_than_31_bits_count():
    """45 000 rows of 50 000 classes: 2.25e9 logits.  A row's result does not depend on the rows beside it, so the last rows equal the same rows alone, bit for bit."""
    from learning_embeddings_amd import loss
    R, C = 45000, sum(S5)
    z = torch.empty(R, C, dtype=torch.bfloat16, device='cuda')
    for r in range(0, R, 3000):
        z[r:r + 3000].normal_()
    y = torch.stack([torch.randint(0, n, (R, 2), device='cuda') for n in S5], 2)
    ref = torch.randn(R, 2, 8, device='cuda') - 5
    z.requires_grad_()
    crit = loss.PreferenceLoss(S5)
    l, rewards = crit(z, y, ref)
    l.backward()
    last = z.detach()[-7:].clone().requires_grad_()
    l2, r2 = crit(last, y[-7:].contiguous(), ref[-7:].contiguous())
    assert torch.equal(rewards[-7:], r2)
    lp = loss.path_log_probs(z.detach(), y, S5)
    assert torch.equal(lp[-7:], loss.path_log_probs(last.detach(), y[-7:].contiguous(), S5))
    (l2 * (7.0 / R)).backward()                                 # 1 / P of the mean: 7 / 45 000 is not exact, so to a rounding of the coefficient and of bf16
    assert ((z.grad[-7:].float() - last.grad.float()).abs() <= 2.0 ** -7 * last.grad.float().abs() + 1e-12).all() and last.grad.abs().max() > 0
