"""The feedback operators together, as ETHECExperiment uses them: a frozen reference with its head in 4 bits, its log-probabilities, a preference or policy step of the
trainable model -- loss and gradient of the classifier against the 64-bit oracle on the very logits of the step."""
import numpy as np
import pytest
import torch

from oracle import feedback_oracle as O

pytestmark = pytest.mark.gpu
LEVELS = [3, 5, 9, 40]
U = 2.0 ** -24


def experiment(dtype=torch.float32):
    from learning_embeddings_amd import experiment as ex, hierarchy, loss
    torch.manual_seed(0)
    lm = hierarchy.SyntheticLabelMap(LEVELS)
    e = ex.ETHECExperiment({}, lm, loss.MultiLevelCELoss(lm), lr=1e-3, batch_size=8, model_name='resnet18', experiment_dir='/tmp/lec_exp', compute_dtype=dtype)
    e.model.train()
    return e, lm


def batch(n, shape, seed=0):
    rs = np.random.RandomState(seed)
    x = torch.from_numpy(rs.rand(n, 3, 32, 32).astype(np.float32)).cuda()
    paths = np.stack([rs.randint(0, m, size=shape) for m in LEVELS], -1)
    paths[rs.rand(*paths.shape) > 0.85] = -1
    return x, paths


def record_outputs(e):
    seen = {}
    def keep(module, args, out):
        seen['x'], seen['z'] = args[0].detach().clone(), out.detach().clone()
    return seen, e.model.fc.register_forward_hook(keep)


def check_fc_gradients(e, seen, dz, size):
    """fc.bias.grad is the sum of dz over the rows, fc.weight.grad = dz^T x: fp32 products of at most 16 terms by torch's own linear, whose dz is within (200 u) of the oracle's
    size; 64 u for the products and sums."""
    x = seen['x'].double().cpu().numpy()
    gb, gw = e.model.fc.bias.grad.double().cpu().numpy(), e.model.fc.weight.grad.double().cpu().numpy()
    assert (np.abs(gb - dz.sum(0)) <= 300 * U * size.sum(0) + 1e-12).all()
    assert (np.abs(gw - dz.T @ x) <= 300 * U * (size.T @ np.abs(x)) + 1e-12).all()


@pytest.mark.parametrize('head', ['mxfp4', 'full'])
@pytest.mark.parametrize('shared', [True, False])
def test_preference_step(head, shared):
    from learning_embeddings_amd import loss
    e, lm = experiment()
    ref_model = e.freeze_reference(head)
    assert not any(p.requires_grad for p in ref_model.parameters()) and not ref_model.training
    x, paths = batch(8, (8, 2) if shared else (8,))
    crit = loss.PreferenceLoss(lm, beta=0.5, label_smoothing=0.05)
    ref = e.reference_log_probs(x, torch.from_numpy(paths)).cpu().numpy()
    before = e.arena.data.clone()
    seen, hook = record_outputs(e)
    l, rewards = e.preference_step(x, torch.from_numpy(paths), crit)
    hook.remove()
    z = seen['z'].double().cpu().numpy()
    want, r, coef = O.preference_loss(z, paths, ref.astype(np.float64), LEVELS, 0.5, 0.05)
    assert abs(float(l) - want) <= 500 * U * (1 + abs(want)) and (np.abs(rewards.cpu().numpy() - r) <= 500 * U * (1 + np.abs(r))).all()
    p3, c3 = (paths, coef) if shared else (paths[:, None], coef[:, None])
    check_fc_gradients(e, seen, *O.path_grad(z, p3, LEVELS, c3))
    assert not torch.equal(before, e.arena.data) and torch.isfinite(e.arena.data).all()
    again = e.reference_log_probs(x, torch.from_numpy(paths)).cpu().numpy()
    assert (again == ref).all()                                 # the reference did not move with the model


def test_policy_step_with_the_frozen_reference():
    from learning_embeddings_amd import loss
    e, lm = experiment()
    e.freeze_reference()
    x, paths = batch(8, (8, 4), seed=1)
    adv = np.random.RandomState(2).randn(8, 4).astype(np.float32)
    crit = loss.ClippedPolicyLoss(lm, kl_coef=0.1)
    ref = e.reference_log_probs(x, torch.from_numpy(paths)).cpu().numpy()
    seen, hook = record_outputs(e)
    l, stats = e.policy_step(x, torch.from_numpy(paths), torch.from_numpy(adv), crit)
    hook.remove()
    z = seen['z'].double().cpu().numpy()
    want, st, coef = O.policy_loss(z, paths, adv, None, ref.astype(np.float64), LEVELS, 0.2, 0.2, 0.1, 'level')
    assert abs(float(l) - want) <= 500 * U * (1 + np.abs(adv).max()) and np.abs(stats.cpu().numpy() - st).max() <= 500 * U * (1 + st[0])
    check_fc_gradients(e, seen, *O.path_grad(z, paths, LEVELS, coef))
    for k in range(3):                                          # off-policy steps against the sampling model's log-probabilities
        old = ref if k == 0 else old
        l, stats = e.policy_step(x, torch.from_numpy(paths), torch.from_numpy(adv), crit, old_log_probs=torch.from_numpy(old))
        assert torch.isfinite(l) and torch.isfinite(stats).all()


def test_bf16_model_and_refusals():
    from learning_embeddings_amd import loss
    e, lm = experiment(torch.bfloat16)
    x, paths = batch(8, (8, 2), seed=3)
    crit = loss.PreferenceLoss(lm)
    with pytest.raises(RuntimeError, match='freeze_reference'):
        e.preference_step(x, torch.from_numpy(paths), crit)
    with pytest.raises(ValueError, match='head must be'):
        e.freeze_reference('int8')
    e.freeze_reference()
    l, rewards = e.preference_step(x, torch.from_numpy(paths), crit)
    assert torch.isfinite(l) and rewards.shape == (8, 2) and torch.isfinite(e.arena.data).all()
    l, _ = e.policy_step(x, torch.from_numpy(paths), torch.ones(8, 2), loss.ClippedPolicyLoss(lm))       # no KL term: no reference needed
    assert torch.isfinite(l)


def test_the_4_bit_reference_is_close_to_the_full_one():
    """The head's logits: every weight is off by at most a quarter of its block's step ... of 2 X, X = 2^(floor(log2 max) - 2): at most max / 4 a weight (saturation included),
    the features the same; so |dz| <= sum_k (|x| max_w / 4 + |w| max_x / 4 + max_x max_w / 16) over the block, and a log-probability moves by at most twice the largest dz of its level."""
    e, lm = experiment()
    e.model.eval()
    x, paths = batch(8, (8,), seed=4)
    seen, hook = record_outputs(e)
    with torch.no_grad():
        e.model(x)
    hook.remove()
    e.freeze_reference('full'); full = e.reference_log_probs(x, torch.from_numpy(paths)).double().cpu().numpy()
    e.freeze_reference('mxfp4'); four = e.reference_log_probs(x, torch.from_numpy(paths)).double().cpu().numpy()
    f, w = seen['x'].abs().double().cpu().numpy(), e.model.fc.weight.detach().abs().double().cpu().numpy()
    top = lambda a: np.repeat(a.reshape(a.shape[0], -1, 32).max(2), 32, 1)
    dz = (f @ top(w).T + top(f) @ w.T) / 4 + top(f) @ top(w).T / 16
    worst = np.stack([dz[:, a:b].max(1) for a, b in O.level_slices(LEVELS)], 1)
    assert (np.abs(full - four) <= 2 * worst + 1e-5).all() and not (full == four).all()


def test_calls_in_flight_on_two_streams_and_from_two_threads():
    """A criterion and a head are one object each; their calls share no buffer, so calls in flight together give what they give one after the other."""
    import threading
    from learning_embeddings_amd import loss, quant
    levels, R, G, K = [6, 21, 135, 561], 700, 3, 512
    g = torch.Generator(device='cuda').manual_seed(3)
    y = torch.stack([torch.randint(-1, n, (R, G, 1), generator=g, device='cuda') for n in levels], 3).squeeze(2)
    adv, old = torch.randn(R, G, generator=g, device='cuda'), torch.randn(R, G, 4, generator=g, device='cuda') - 5
    feats = [torch.randn(R, K, generator=g, device='cuda') for _ in range(8)]
    logits = [torch.randn(R, sum(levels), generator=g, device='cuda') for _ in range(8)]
    head = quant.MXFP4Linear(torch.randn(sum(levels), K, generator=g, device='cuda') / K ** 0.5, out_dtype=torch.float32)
    crit = loss.ClippedPolicyLoss(levels, kl_coef=0.1)
    def step(i):
        ref = loss.path_log_probs(head(feats[i]), y, levels)
        z = logits[i].detach().requires_grad_()
        l, st = crit(z, y, adv, old, ref)
        dz, = torch.autograd.grad(l, z)
        return l.detach(), st, dz, ref
    want = [step(i) for i in range(8)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None] * 8
    for i in range(8):                                           # one thread, nothing waited for in between
        with torch.cuda.stream(streams[i & 1]):
            got[i] = step(i)
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for w, h in zip(want, got) for u, v in zip(w, h))
    again, errors = [None] * 8, []
    def work(k):
        try:
            with torch.cuda.stream(streams[k]):
                for i in range(k, 8, 2):
                    again[i] = step(i)
        except BaseException as e:                               # (an assertion in a thread is not the test's)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and all(torch.equal(u, v) for w, h in zip(want, again) for u, v in zip(w, h))
