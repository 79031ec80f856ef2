"""The operators of the feedback path -- log-probabilities of label paths, the preference loss, the clipped policy loss -- and of the
4-bit classifier head -- microscaled quantisation, product -- each as a user's program calls it (`own`) and in its plain form:
elementary torch operations in 32 bits, 64 where 32 lose what matters, rounded once at the end.

A classifier over a label hierarchy answers an image with a label PATH, one class a level; its logits row [n_classes] is cut into the
levels' slices, each with a softmax of its own.  An entry of a path that is not known is -1 and counts nowhere.  Sizes are this
repository's: the ETHEC hierarchy (723 labels), the 2 000-label and the 50 000-label synthetic ones, ResNet-18 / -50 features
(512 / 2048), batches of 1 to 7 424 rows."""
import math

import torch

own = False                     # set from outside: the framework's operators (True) or the plain forms (False)

ETHEC = [6, 21, 135, 561]
S3 = [8, 64, 384, 1544]
S5 = [2, 8, 32, 128, 512, 2048, 8192, 39078]
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def _levels(case):
    return [int(v) for v in case['levels'].split(',')]


def _lv(levels):
    return ','.join(str(v) for v in levels)


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the log-probabilities of a batch's annotated paths under a frozen classifier: one path an image (a validation batch over ETHEC), ...
        {'name': 'logp_ethec_250', 'op': 'logp', 'levels': _lv(ETHEC), 'rows': 250, 'paths': 1, 'dtype': 'fp32', 'grad': False},
        # ... and eight sampled paths an image over the 50 000-label hierarchy, trained through (their gradient is an input of its own)
        {'name': 'logp_s5_512_g8_train', 'op': 'logp', 'levels': _lv(S5), 'rows': 512, 'paths': 8, 'dtype': 'bf16', 'grad': True},
        # preference training, forward and backward: pairs of images of their own (the preferred one's path, the other one's path), ETHEC
        {'name': 'pref_ethec_128_pairs', 'op': 'pref', 'levels': _lv(ETHEC), 'rows': 128, 'shared': False, 'dtype': 'fp32', 'smooth': 0.0},
        # an annotator's two paths for the same image, 50 000 labels, a large batch
        {'name': 'pref_s5_2048_shared', 'op': 'pref', 'levels': _lv(S5), 'rows': 2048, 'shared': True, 'dtype': 'fp32', 'smooth': 0.1},
        # policy training on a path-level reward, forward and backward: eight paths an image over ETHEC with the KL term, ...
        {'name': 'policy_ethec_512_g8', 'op': 'policy', 'levels': _lv(ETHEC), 'rows': 512, 'paths': 8, 'dtype': 'fp32', 'kl': 0.05, 'mean': 'level'},
        # ... over the 2 000-label hierarchy with an odd batch and fp16 logits, no KL term, ...
        {'name': 'policy_s3_333_g5', 'op': 'policy', 'levels': _lv(S3), 'rows': 333, 'paths': 5, 'dtype': 'fp16', 'kl': 0.0, 'mean': 'path'},
        # ... and the largest step: 4 096 images of the 50 000-label hierarchy, sixteen paths each
        {'name': 'policy_s5_4096_g16', 'op': 'policy', 'levels': _lv(S5), 'rows': 4096, 'paths': 16, 'dtype': 'bf16', 'kl': 0.05, 'mean': 'level'},
        # 4-bit quantisation and back: pooled ResNet-50 features of a batch, odd row length
        {'name': 'mxfp4_features_515', 'op': 'quant', 'rows': 723, 'k': 515, 'dtype': 'fp16', 'out': 'fp32'},
        # the weights of a 50 000-label head
        {'name': 'mxfp4_head_50000', 'op': 'quant', 'rows': 50000, 'k': 2048, 'dtype': 'bf16', 'out': 'bf16'},
        # the head of the 50 000-label hierarchy for ONE image (serving), ...
        {'name': 'head_1x50000', 'op': 'head', 'm': 1, 'n': 50000, 'k': 2048, 'dtype': 'bf16', 'out': 'bf16', 'bias': True},
        # ... the ETHEC head on a ResNet-18 batch of odd size, ...
        {'name': 'head_ethec_131', 'op': 'head', 'm': 131, 'n': 723, 'k': 512, 'dtype': 'fp32', 'out': 'fp32', 'bias': True},
        # ... and the largest: every row of the 50 000-label hierarchy's step
        {'name': 'head_7424x50000', 'op': 'head', 'm': 7424, 'n': 50000, 'k': 2048, 'dtype': 'bf16', 'out': 'bf16', 'bias': True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_levels(rng, total):
    """A hierarchy of 1 to 8 levels that widens downwards to about `total` labels."""
    n = rng.randint(1, 8)
    f = rng.uniform(1.6, 6.0)
    w = [f ** i * rng.uniform(0.7, 1.4) for i in range(n)]
    s = sum(w)
    return [max(1, int(total * v / s)) for v in w]


def draw(rng):
    op = rng.choice(['logp', 'pref', 'policy', 'quant', 'head'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if op == 'quant':
        k = _log_int(rng, 31, 4500)
        return {'op': op, 'rows': min(_log_int(rng, 1, 50000), 100_000_000 // k), 'k': k, 'dtype': dtype, 'out': 'bf16' if dtype == 'bf16' else 'fp32'}
    if op == 'head':
        n = _log_int(rng, 5, 50000)
        k = rng.choice([512, 2048, _log_int(rng, 31, 2048)])
        return {'op': op, 'm': _log_int(rng, 1, 7424), 'n': n, 'k': k, 'dtype': dtype, 'out': 'fp32' if dtype == 'fp32' else rng.choice([dtype, 'fp32']),
                'bias': rng.random() < 0.7}
    total = _log_int(rng, 20, 49000)
    levels = _lv(_draw_levels(rng, total))
    rows = min(_log_int(rng, 1, 4096), 200_000_000 // total)
    if op == 'logp':
        return {'op': op, 'levels': levels, 'rows': min(rows, 25_000_000 // total + 1), 'paths': rng.randint(1, 8), 'dtype': dtype, 'grad': rng.random() < 0.5}
    if op == 'pref':
        shared = rng.random() < 0.5
        cap = 100_000_000 // total
        return {'op': op, 'levels': levels, 'rows': max(1, min(rows, cap) // (1 if shared else 2)), 'shared': shared, 'dtype': dtype,
                'smooth': rng.choice([0.0, 0.05, 0.1])}
    return {'op': op, 'levels': levels, 'rows': rows, 'paths': rng.randint(1, 16), 'dtype': dtype, 'kl': rng.choice([0.0, 0.02, 0.05]),
            'mean': rng.choice(['level', 'path'])}


# ----------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed))


def _path_inputs(case, seed):
    """Logits and label paths as a classifier in training meets them: peaked softmaxes, paths drawn from the classifier itself, about a
    tenth of them known only down to some level and a few not at all; log-probabilities of the sampling classifier and of the
    reference a little away from the present ones."""
    g = _gen(seed)
    lv, C = _levels(case), sum(_levels(case))
    op = case['op']
    R = case['rows'] * (2 if op == 'pref' and not case['shared'] else 1)
    G = 1 if op == 'pref' and not case['shared'] else (2 if op == 'pref' else case['paths'])
    z = (torch.randn(R, C, generator=g, device='cuda') * 2.5).to(DTYPES[case['dtype']])
    paths = torch.empty(R, G, len(lv), dtype=torch.int64, device='cuda')
    logp = torch.empty(R, G, len(lv), dtype=torch.float32, device='cuda')
    s = 0
    for l, n in enumerate(lv):
        for r in range(0, R, 512):                              # (slices of rows: the cumulative sums stay small)
            p = torch.softmax(z[r:r + 512, s:s + n].float(), 1)
            u = torch.rand(p.shape[0], G, generator=g, device='cuda')
            c = torch.searchsorted(p.cumsum(1), u).clamp_(max=n - 1)
            paths[r:r + 512, :, l] = c
            logp[r:r + 512, :, l] = p.gather(1, c).clamp_(min=1e-30).log()
        s += n
    depth = torch.full((R, G, 1), len(lv), device='cuda')
    cut = torch.rand(R, G, 1, generator=g, device='cuda') < 0.1
    depth = torch.where(cut, torch.randint(0, len(lv) + 1, (R, G, 1), generator=g, device='cuda'), depth)
    paths = torch.where(torch.arange(len(lv), device='cuda') < depth, paths, torch.full_like(paths, -1))
    old = logp + 0.1 * torch.randn(logp.shape, generator=g, device='cuda')
    ref = logp + 0.3 * torch.randn(logp.shape, generator=g, device='cuda')
    adv = torch.randn(R, G, generator=g, device='cuda')
    if G == 1 and op in ('pref', 'logp'):
        paths, old, ref = paths[:, 0].contiguous(), old[:, 0].contiguous(), ref[:, 0].contiguous()
    up = torch.randn(paths.shape, generator=g, device='cuda')
    return {'z': z, 'paths': paths, 'old': old, 'ref': ref, 'adv': adv, 'up': up}


def _matrix_inputs(case, seed):
    """Pooled features (non-negative, some channels much larger than others) and a trained head's weights."""
    g = _gen(seed)
    rows = case['m'] if case['op'] == 'head' else case['rows']
    x = torch.randn(rows, case['k'], generator=g, device='cuda')
    x *= torch.exp(torch.randn(case['k'], generator=g, device='cuda'))
    if case['op'] == 'quant':
        return {'x': x.to(DTYPES[case['dtype']])}
    x = x.abs_().to(DTYPES[case['dtype']])
    w = torch.randn(case['n'], case['k'], generator=g, device='cuda') * (1.0 / math.sqrt(case['k']))
    b = torch.randn(case['n'], generator=g, device='cuda') * 0.1 if case['bias'] else None
    return {'x': x, 'w': w, 'b': b}


def prepare(case, seed):
    op = case['op']
    if op in ('quant', 'head'):
        st = _matrix_inputs(case, seed)
        st['out'] = DTYPES[case['out']]
        if op == 'head':                                        # the head is laid out once, when it is frozen
            if own:
                from learning_embeddings_amd import quant
                st['head'] = quant.MXFP4Linear(st.pop('w'), st['b'], out_dtype=st['out'])
            else:
                st['w'] = _plain_mxfp4(st['w'])
    else:
        st = _path_inputs(case, seed)
        if op != 'logp' or case['grad']:
            st['z'].requires_grad_(True)
        if own:
            from learning_embeddings_amd import hierarchy, loss
            lm = hierarchy.SyntheticLabelMap(_levels(case), edges=[])
            st['labelmap'] = lm
            if op == 'pref':
                st['criterion'] = loss.PreferenceLoss(lm, beta=0.1, label_smoothing=case['smooth'])
            elif op == 'policy':
                st['criterion'] = loss.ClippedPolicyLoss(lm, clip_low=0.2, clip_high=0.2, kl_coef=case['kl'], reduction=case['mean'])
    st['case'] = case
    return st


# ------------------------------------------------------------------------------------------------------------- plain forms
def _plain_mxfp4(x):
    """The values that x's 4-bit form stands for, in 32 bits: blocks of 32 along the row share a power of two, 2^(floor(log2 max|x|) - 2)
    clamped to [2^-127, 2^127]; elements round to nearest, ties to even, into {0, 0.5, 1, 1.5, 2, 3, 4, 6} times it and saturate.  A block
    that holds a NaN or an infinity is NaN."""
    rows, k = x.shape
    out = torch.empty(rows, k, dtype=torch.float32, device=x.device)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float32, device=x.device)
    step = max(1, (1 << 25) // k)
    for r in range(0, rows, step):                              # (slices of rows: the 64-bit intermediates stay small)
        v = x[r:r + step].float()
        n = v.shape[0]
        pad = -k % 32
        if pad:
            v = torch.cat([v, v.new_zeros(n, pad)], 1)
        v = v.view(n, -1, 32)
        top = v.abs().amax(2, keepdim=True)
        e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
        e = torch.where(top > 0, e, torch.full_like(e, -127))
        scale = torch.exp2(e.double())
        a = v.abs().double() / scale
        code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
        q = grid[code] * scale * torch.sign(v)
        q = torch.where(torch.isfinite(top), q, torch.full_like(q, float('nan')))
        out[r:r + step] = q.float().view(n, -1)[:, :k]
    return out


def _plain_logp(z, paths, levels):
    """Log-probability of every entry of every path, 0 where the entry is -1; z [R, C] in 32 bits, paths [R, G, L] -> [R, G, L]."""
    out = []
    for zl, y in zip(z.split(levels, 1), paths.unbind(2)):
        m = zl.detach().amax(1, keepdim=True)
        lse = (zl - m).exp().sum(1, keepdim=True).log()
        lp = zl.gather(1, y.clamp(min=0)) - m - lse
        out.append(torch.where(y >= 0, lp, torch.zeros_like(lp)))
    return torch.stack(out, 2)


def _plain_softplus(x):
    return x.clamp(min=0) + (1 + (-x.abs()).exp()).log()


def _plain_pref(z, paths, ref, levels, beta, smooth, shared):
    y = paths if shared else paths.unsqueeze(1)
    rf = ref if shared else ref.unsqueeze(1)
    lp = _plain_logp(z.float(), y, levels).double()
    reward = beta * (lp - torch.where(y >= 0, rf, torch.zeros_like(rf)).double()).sum(2)        # [R, 1 or 2]
    reward = reward if shared else torch.stack(list(reward[:, 0].chunk(2)), 1)                  # [P, 2]
    d = reward[:, 0] - reward[:, 1]
    loss = ((1 - smooth) * _plain_softplus(-d) + smooth * _plain_softplus(d)).mean()
    return loss.float(), reward.detach().float()


def _plain_policy(z, paths, adv, old, ref, levels, low, high, kl, mean):
    lp = _plain_logp(z.float(), paths, levels).double()
    on = paths >= 0
    zero = torch.zeros_like(lp)
    ratio = torch.where(on, lp - old.double(), zero).exp()
    a = adv.double().unsqueeze(2)
    gain = torch.minimum(ratio * a, ratio.clamp(1 - low, 1 + high) * a)
    d = torch.where(on, ref.double() - lp, zero)
    k3 = torch.expm1(d) - d
    clipped = (((a > 0) & (ratio > 1 + high)) | ((a < 0) & (ratio < 1 - low))).double()
    if mean == 'level':
        w = on.double() / on.sum().clamp(min=1)
    else:
        w = on.double() / on.sum(2, keepdim=True).clamp(min=1) / (on.shape[0] * on.shape[1])
    klm = (w * k3).sum()
    loss = -(w * gain).sum() + (kl * klm if kl else 0.0)
    return loss.float(), torch.stack([klm.detach(), (w * clipped).sum()]).float()


# --------------------------------------------------------------------------------------------------------------------- run
def run(state):
    case = state['case']
    op = case['op']
    if op == 'quant':
        if own:
            from learning_embeddings_amd import quant
            return quant.mxfp4_quantize(state['x']).dequantize(state['out'])
        return _plain_mxfp4(state['x']).to(state['out'])
    if op == 'head':
        if own:
            return state['head'](state['x'])
        y = _plain_mxfp4(state['x']) @ state['w'].t()
        if state['b'] is not None:
            y += state['b']
        return y.to(state['out'])
    z, paths, lv = state['z'], state['paths'], _levels(case)
    z.grad = None
    if op == 'logp':
        if own:
            from learning_embeddings_amd import loss
            lp = loss.path_log_probs(z, paths, state['labelmap'])
        else:
            y = paths if paths.dim() == 3 else paths.unsqueeze(1)
            lp = _plain_logp(z.float(), y, lv).view(paths.shape)
        if not case['grad']:
            return lp
        lp.backward(state['up'])
        return lp.detach(), z.grad
    if op == 'pref':
        if own:
            loss_, reward = state['criterion'](z, paths, state['ref'])
        else:
            loss_, reward = _plain_pref(z, paths, state['ref'], lv, 0.1, case['smooth'], case['shared'])
        loss_.backward()
        return loss_.detach(), reward, z.grad
    ref = state['ref']
    if own:
        loss_, stats = state['criterion'](z, paths, state['adv'], state['old'], ref)
    else:
        loss_, stats = _plain_policy(z, paths, state['adv'], state['old'], ref, lv, 0.2, 0.2, case['kl'], case['mean'])
    loss_.backward()
    return loss_.detach(), stats, z.grad


# -------------------------------------------------------------------------------------------------------------------- work
_SIZE = {'bf16': 2, 'fp16': 2, 'fp32': 4}


def work(case):
    op, b = case['op'], _SIZE[case['dtype']]
    if op == 'quant':
        n = case['rows'] * case['k']
        return {'bytes': n * (b + _SIZE[case['out']]), 'flops': 2 * n}
    if op == 'head':
        m, n, k = case['m'], case['n'], case['k']
        return {'bytes': m * k * b + n * k * 17 // 32 + (4 * n if case['bias'] else 0) + m * n * _SIZE[case['out']], 'flops': 2 * m * n * k}
    lv = _levels(case)
    R = case['rows'] * (2 if op == 'pref' and not case['shared'] else 1)
    G = 1 if op == 'pref' and not case['shared'] else (2 if op == 'pref' else case['paths'])
    z, t = R * sum(lv), R * G * len(lv)
    train = op != 'logp' or case['grad']
    per_entry = 8 + {'logp': 4 + (4 if train else 0), 'pref': 4, 'policy': 8}[op]            # the path, its log-probabilities in and out
    return {'bytes': z * b * (2 if train else 1) + t * per_entry + R * G * 4, 'flops': z * (7 if train else 3)}


# ------------------------------------------------------------------------------------------------------------------- exact
def _exact_mxfp4(x):
    """The same definition by another route: the spacing of the 4-bit numbers in each binade, rounded half to even."""
    rows, k = x.shape
    out = torch.empty(rows, k, dtype=torch.float64, device=x.device)
    for r in range(0, rows, max(1, (1 << 24) // k)):
        v = x[r:r + max(1, (1 << 24) // k)].double()
        n = v.shape[0]
        v = torch.nn.functional.pad(v, (0, -k % 32)).view(n, -1, 32)
        top = v.abs().max(2, keepdim=True).values
        mant, ex = torch.frexp(top)
        s = torch.ldexp(torch.ones_like(top), torch.where(top == 0, torch.full_like(ex, -124), ex).sub(3).clamp(-127, 127))
        a = (v / s).abs()
        h = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0).double())
        q = torch.copysign(((a / h).round() * h).clamp(max=6.0) * s, v)
        q[~torch.isfinite(top).expand_as(q)] = float('nan')
        out[r:r + n] = q.view(n, -1)[:, :k]
    return out


def _exact_scores(z, paths, levels):
    """Per level: (first class, softmax [R, n], logp [R, G]) in 64 bits."""
    s = 0
    for l, n in enumerate(levels):
        zl = z[:, s:s + n].double()
        lsm = zl - torch.logsumexp(zl, 1, keepdim=True)
        y = paths[:, :, l]
        yield l, s, lsm, torch.where(y < 0, torch.zeros((), dtype=torch.float64, device=z.device), lsm.gather(1, y.clamp(min=0)))
        s += n


def _exact_grad(z, paths, levels, coef):
    """d/dz of sum(coef * logp), coef [R, G, L] in 64 bits."""
    out = torch.empty(z.shape, dtype=torch.float64, device=z.device)
    for l, s, lsm, _ in _exact_scores(z, paths, levels):
        y = paths[:, :, l]
        c = torch.where(y < 0, torch.zeros_like(coef[:, :, l]), coef[:, :, l])
        gl = lsm.exp_().mul_(-c.sum(1, keepdim=True))
        gl.scatter_add_(1, y.clamp(min=0), c)
        out[:, s:s + lsm.shape[1]] = gl
    return out


def exact(case, seed):
    op = case['op']
    if op == 'quant':
        return _exact_mxfp4(_matrix_inputs(case, seed)['x'])
    if op == 'head':
        t = _matrix_inputs(case, seed)
        y = torch.mm(_exact_mxfp4(t['x']), _exact_mxfp4(t['w']).t())
        return y if t['b'] is None else y.add_(t['b'].double())
    t = _path_inputs(case, seed)
    z, lv = t['z'], _levels(case)
    y = t['paths'] if t['paths'].dim() == 3 else t['paths'].unsqueeze(1)
    logp = torch.stack([p for _, _, _, p in _exact_scores(z, y, lv)], 2)
    on = (y >= 0).double()
    if op == 'logp':
        if not case['grad']:
            return logp.view(t['paths'].shape)
        return logp.view(t['paths'].shape), _exact_grad(z, y, lv, t['up'].double().view(y.shape))
    if op == 'pref':
        beta, eps = 0.1, case['smooth']
        P = case['rows']
        r = beta * ((logp - t['ref'].double().view(y.shape)) * on).sum(2)
        r = r if case['shared'] else r.view(2, P).t()
        d = r[:, 0] - r[:, 1]
        loss = -(1 - eps) * torch.nn.functional.logsigmoid(d) - eps * torch.nn.functional.logsigmoid(-d)
        dd = (eps * torch.sigmoid(d) - (1 - eps) * torch.sigmoid(-d)) * beta / P
        c = torch.stack([dd, -dd], 1)
        c = c if case['shared'] else c.t().reshape(2 * P, 1)
        return loss.mean(), r, _exact_grad(z, y, lv, c.unsqueeze(2).expand(y.shape))
    low = high = 0.2
    a = t['adv'].double().unsqueeze(2)
    if case['mean'] == 'level':
        w = on / max(float(on.sum()), 1.0)
    else:
        w = on / on.sum(2, keepdim=True).clamp(min=1.0) / (y.shape[0] * y.shape[1])
    ratio = torch.exp((logp - t['old'].double()) * on)
    hit = ((a > 0) & (ratio > 1 + high)) | ((a < 0) & (ratio < 1 - low))
    gain = torch.where(hit, torch.where(a > 0, (1 + high) * a, (1 - low) * a), ratio * a)
    d = (t['ref'].double() - logp) * on
    k3 = torch.special.expm1(d) - d
    klm = (w * k3).sum()
    loss = case['kl'] * klm - (w * gain).sum()
    coef = w * (torch.where(hit, torch.zeros_like(ratio), -ratio * a) - case['kl'] * torch.special.expm1(d))
    return loss, torch.stack([klm, (w * hit.double()).sum()]), _exact_grad(z, y, lv, coef)
