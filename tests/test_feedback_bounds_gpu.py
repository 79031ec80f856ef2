"""Clipped policy loss next to its clip bounds, on the MI355X: every entry is decided as 64 bits decide it, however many share a level and however wrong a level's 32-bit
sum is.

The decisions are read off twice: the clipped share times the number of entries is a whole number that has to be the right one, and an entry that is clipped contributes
nothing to the gradient, one that is not contributes -rho A / n.  The gradient's tolerance counts u = 2^-24: (3 span + 3 log(classes) + 100) u of the sum of |coefficients|
(span <= 30, so below 250 u), and half a step of the logits' type (fp16: 2^-25 below its normal range)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
ETHEC = [6, 21, 135, 561]
S5 = [2, 8, 32, 128, 512, 2048, 8192, 39078]


def exact_logp(z, y, levels):
    """z [R, C], y [R, G, L] -> [R, G, L] in 64 bits"""
    return torch.stack([torch.log_softmax(zl.double(), 1).gather(1, yl) for zl, yl in zip(z.split(levels, 1), y.unbind(2))], 2)


def off_the_tie(old, target):
    """old (fp32) moved by one step -- near 0, by 1e-9 -- wherever it is so near target (64 bits) that the last bits of a 64-bit sum could decide"""
    tie = lambda o: (o.double() - target).abs() < 1e-10
    old = torch.where(tie(old), torch.nextafter(old, torch.full_like(old, -1e9)), old)
    return torch.where(tie(old), (target - 1e-9).float(), old)


def check_decisions(levels, z, y, adv, old, low, high, softmax_off=250):
    """z of the type under test, y [R, G, L], adv [R, G], old [R, G, L] fp32 -> the share of clipped entries.  softmax_off: a probability's error in u (250: (3 span +
    3 log(classes) + 100) of levels of up to 40 000 classes)"""
    from learning_embeddings_amd import loss
    exact = exact_logp(z, y, levels)
    bound = torch.where(adv > 0, 1 + high, 1 - low).double().log()[:, :, None]
    off = exact - old.double() - bound                           # log rho - log bound
    assert off.abs().min() > 5e-11                               # (far above a 64-bit sum's rounding)
    hit = torch.where(adv[:, :, None] > 0, off > 0, off < 0)
    n = y.numel()
    zz = z.clone().requires_grad_()
    l, st = loss.ClippedPolicyLoss(levels, clip_low=low, clip_high=high)(zz, y, adv, old)
    grad, = torch.autograd.grad(l, zz)
    assert abs(st[1].item() * n - hit.sum().item()) < 0.25, '%g entries clipped, %d have to be' % (st[1].item() * n, hit.sum().item())
    c = torch.where(hit, 0.0, -(exact - old.double()).exp() * adv.double()[:, :, None] / n)
    want, size, s = torch.zeros_like(z, dtype=torch.float64), torch.zeros_like(z, dtype=torch.float64), 0
    for k, m in enumerate(levels):
        p = torch.softmax(z[:, s:s + m].double(), 1)
        want[:, s:s + m] = -c[:, :, k].sum(1, keepdim=True) * p
        size[:, s:s + m] = c[:, :, k].abs().sum(1, keepdim=True) * p
        want[:, s:s + m].scatter_add_(1, y[:, :, k], c[:, :, k])
        size[:, s:s + m].scatter_add_(1, y[:, :, k], c[:, :, k].abs())
        s += m
    tol = softmax_off * U * size + torch.finfo(z.dtype).eps / 2 * want.abs() + (2.0 ** -25 if z.dtype == torch.float16 else 1e-37)
    bad = (grad.double() - want).abs() > tol
    assert not bad.any(), 'gradient off at %s' % bad.nonzero()[:4].tolist()
    again, st2 = loss.ClippedPolicyLoss(levels, clip_low=low, clip_high=high)(zz, y, adv, old)
    assert torch.equal(again, l) and torch.equal(st2, st) and torch.equal(torch.autograd.grad(again, zz)[0], grad)
    return hit.double().mean().item()


@pytest.mark.parametrize('levels,R,G', [(ETHEC, 256, 16), (ETHEC, 50, 64), (S5, 24, 16), ([2, 3], 333, 5), ([3], 7, 2), (list(range(2, 18)), 40, 9), (list(range(2, 18)), 333, 1),
                                           (ETHEC, 9000, 16), ([2], 70000, 8)])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_paths_that_share_a_class_are_decided_alike(levels, R, G, dtype):
    """All paths of a row name the same classes with the same log-probabilities of the sampler, every one of them next to its bound: many entries of few levels.
    (The last two: more paths than the grid's blocks take in one round.)"""
    g = torch.Generator(device='cuda').manual_seed(5)
    z = (torch.randn(R, sum(levels), generator=g, device='cuda') * 2.5).to(DT[dtype])
    y = torch.stack([torch.randint(0, n, (R, 1), generator=g, device='cuda') for n in levels], 2).expand(R, G, len(levels)).contiguous()
    sign = torch.where(torch.arange(R, device='cuda') % 2 == 0, 1.0, -1.0)[:, None]
    adv = sign * (1 + torch.rand(R, G, generator=g, device='cuda'))
    target = exact_logp(z, y, levels) - torch.where(adv > 0, 1.25, 0.75).double().log()[:, :, None]
    share = check_decisions(levels, z, y, adv, off_the_tie(target.float(), target), 0.25, 0.25)
    assert R * len(levels) < 100 or 0.2 < share < 0.8


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_every_entry_at_its_bound_is_decided(dtype):
    """Bounds of 0 and the model's own log-probabilities, rounded to 32 bits: every entry's ratio is 1 within a rounding, paths and advantages differ."""
    g = torch.Generator(device='cuda').manual_seed(6)
    R, G = 300, 3
    z = (torch.randn(R, sum(ETHEC), generator=g, device='cuda') * 2.5).to(DT[dtype])
    y = torch.stack([torch.randint(0, n, (R, G), generator=g, device='cuda') for n in ETHEC], 2)
    adv = torch.randn(R, G, generator=g, device='cuda')
    target = exact_logp(z, y, ETHEC)
    assert 0.2 < check_decisions(ETHEC, z, y, adv, off_the_tie(target.float(), target), 0.0, 0.0) < 0.8


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('steps', [1.5, 20.0, 40.0, 80.0])
@pytest.mark.parametrize('side', [1, -1])
def test_levels_whose_sums_round_one_way(dtype, steps, side):
    """One class at 0 and the rest together at -d: a lane that starts with 1 loses or gains up to half a step with every one of its 35 or 39 small terms, always in the same
    direction (measured: log-probabilities off by up to 44 u for d of 11 to 13).  The ratio lies `steps` u beside its bound."""
    R, n = 96, 39078
    d = 11 + torch.arange(R, device='cuda') / 48 if dtype == 'fp32' else 8 + torch.arange(R, device='cuda') / 16
    z = (-d[:, None]).expand(R, n).contiguous().to(DT[dtype])
    z[:, 0] = 0
    y = torch.zeros(R, 1, 1, dtype=torch.int64, device='cuda')
    adv = torch.where(torch.arange(R, device='cuda') % 2 == 0, 1.0, -1.0)[:, None]
    target = exact_logp(z, y, [n]) - torch.where(adv > 0, 1.25, 0.75).double().log()[:, :, None] + side * steps * U
    check_decisions([n], z, y, adv, target.float(), 0.25, 0.25)


@pytest.mark.parametrize('steps', [20.0, 100.0, 300.0])
@pytest.mark.parametrize('side', [1, -1])
def test_a_level_of_a_million_classes(steps, side):
    """456 runs, merged one after the other by a single lane: its sum was measured 152 u off."""
    R, n = 32, 1 << 20
    z = -(11 + torch.arange(R, device='cuda') / 16)[:, None].expand(R, n).contiguous()
    z[:, 0] = 0
    y = torch.zeros(R, 1, 1, dtype=torch.int64, device='cuda')
    adv = torch.where(torch.arange(R, device='cuda') % 2 == 0, 1.0, -1.0)[:, None]
    target = exact_logp(z, y, [n]) - torch.where(adv > 0, 1.25, 0.75).double().log()[:, :, None] + side * steps * U
    check_decisions([n], z, y, adv, target.float(), 0.25, 0.25, softmax_off=2000)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_near_entries_beside_unknown_ones_and_empty_levels(dtype):
    """A row's unknown entries, rows without a known entry and levels that hold no number stay out of it."""
    from learning_embeddings_amd import loss
    levels, R, G = ETHEC, 64, 8
    g = torch.Generator(device='cuda').manual_seed(7)
    z = (torch.randn(R, sum(levels), generator=g, device='cuda') * 2.5).to(DT[dtype])
    y = torch.stack([torch.randint(0, n, (R, 1), generator=g, device='cuda') for n in levels], 2).expand(R, G, 4).contiguous()
    adv = 1 + torch.rand(R, G, generator=g, device='cuda')
    exact = exact_logp(z, y, levels)
    target = exact - np.log(1.25)
    old = off_the_tie(target.float(), target)
    hit = exact - old.double() > np.log(1.25)
    known = torch.rand(R, G, 4, generator=g, device='cuda') < 0.6
    known[3] = False
    known[5, :, 1] = False
    z[5, levels[0]:levels[0] + levels[1]] = float('nan')
    zz = z.requires_grad_()
    l, st = loss.ClippedPolicyLoss(levels, clip_low=0.25, clip_high=0.25)(zz, torch.where(known, y, -1), adv, old)
    grad, = torch.autograd.grad(l, zz)
    assert abs(st[1].item() * known.sum().item() - (hit & known).sum().item()) < 0.25
    moved = torch.stack([gl.abs().sum(1) > 0 for gl in grad.float().split(levels, 1)], 1)                       # [R, L]: a level moves where an unclipped entry counts it
    assert torch.isfinite(grad).all() and torch.equal(moved, (known & ~hit).any(1))
