"""The 4-bit product in the forms for large products -- rings of 128 x 128 and 192 x 192 tiles --, on the MI355X: every output type, remainders, streams, threads, captured
graphs, blocks without a value.  Each case says which form it is for and the choice is restated here, so that another rule shows as a failure and not as a form untested.

Tolerance: products are exact in 32 bits, K additions of up to 2 u each (u = 2^-24) against the sum of |x_4 w_4|, the bias's addition, one rounding to the output's type of half
a step."""
import threading

import numpy as np
import pytest
import torch

from oracle import feedback_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def form(M, N, K):
    up = lambda a, b: -(-a // b)
    tiles = up(N, 32) * up(M, 32)
    if M <= 4 and up(K, 64) * 1024 + up(K, 256) * 256 <= 56 * 1024:
        return 'few'
    if up(M, 32) == 1 or tiles <= 1024 or (tiles <= 2048 and up(N, 32) * up(K, 64) * 1024 <= 4 << 20):
        return 'rows'
    return 'ring3' if up(N, 192) * up(M, 192) >= 3000 else 'ring2'


def inputs(M, N, K, dtype, seed=0):
    rs = np.random.RandomState(seed)
    x = torch.from_numpy((rs.randn(M, K) * np.exp(rs.randn(1, K))).astype(np.float32)).to(DT[dtype])
    w = torch.from_numpy((rs.randn(N, K) * np.exp(rs.randn(N, 1))).astype(np.float32))
    return x, w, torch.from_numpy(rs.randn(N).astype(np.float32))


def check(y, x, w, b, out):
    f64 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    xq, wq = f64(O.mxfp4_values(x.double().numpy())), f64(O.mxfp4_values(w.double().numpy()))
    want, size = torch.mm(xq, wq.t().contiguous()), torch.mm(xq.abs(), wq.abs().t().contiguous())
    if b is not None:
        want += b.double().cuda(); size += b.double().abs().cuda()
    tol = size.mul_(2 * (x.shape[1] + 4) * U)
    tol += torch.finfo(DT[out]).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if out == 'fp16' else 0)
    assert y.dtype == DT[out] and y.shape == want.shape
    err = (y.double() - want).abs_()
    assert (err <= tol).all(), 'error / tolerance %.3g at %s' % (float((err / tol).max()), (err > tol).nonzero()[:4].tolist())


@pytest.mark.parametrize('which,M,N,K', [('ring2', 2100, 2101, 5000), ('ring2', 700, 5003, 512), ('ring2', 129, 30001, 97), ('ring3', 11800, 9501, 130), ('ring3', 5800, 19201, 33),
                                         ('ring3', 9600, 11520, 64)])
@pytest.mark.parametrize('dtype,out', [('fp32', 'fp32'), ('fp16', 'fp16'), ('bf16', 'bf16'), ('bf16', 'fp32'), ('fp32', 'fp16')])
@pytest.mark.parametrize('bias', [True, False])
def test_output_types(which, M, N, K, dtype, out, bias):
    from learning_embeddings_amd import quant
    assert form(M, N, K) == which
    x, w, b = inputs(M, N, K, dtype, seed=8)
    h = quant.MXFP4Linear(w.cuda(), b.cuda() if bias else None, out_dtype=DT[out])
    y = h(x.cuda())
    check(y, x, w, b if bias else None, out)
    assert torch.equal(y, h(x.cuda()))


@pytest.mark.parametrize('which,M,N,K', [('ring2', 700, 5003, 512), ('ring3', 11800, 9501, 130)])
@pytest.mark.parametrize('out', ['fp16', 'fp32'])
def test_captured_and_on_other_streams(which, M, N, K, out):
    """The graph is captured before anything else has run this form (its kernel's LDS is allowed on the first call), then replayed between eager calls."""
    from learning_embeddings_amd import quant
    assert form(M, N, K) == which
    x, w, b = inputs(M, N, K, out, seed=9)
    h = quant.MXFP4Linear(w.cuda(), b.cuda(), out_dtype=DT[out])
    xs = [x.cuda(), x.cuda().flip(0).contiguous()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs, outs = [], []
    for v in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(h(v))
        graphs.append(g)
    want = [h(v) for v in xs]
    check(want[0], x, w, b, out)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = [h(v) for v in xs]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(again, want))
    for k in range(3):
        for v in xs:
            v.copy_(torch.roll(v, 1, 0))
        want = [h(v) for v in xs]
        for i in ((0, 1), (1, 0), (1, 1, 0))[k]:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want))


def test_two_threads_on_two_streams():
    from learning_embeddings_amd import quant
    M, N, K = 700, 5003, 512
    assert form(M, N, K) == 'ring2'
    g = torch.Generator(device='cuda').manual_seed(3)
    h = quant.MXFP4Linear(torch.randn(N, K, generator=g, device='cuda'), torch.randn(N, generator=g, device='cuda'), out_dtype=torch.bfloat16)
    xs = [torch.randn(M, K, generator=g, device='cuda') for _ in range(8)]
    want = [h(x) for x in xs]
    torch.cuda.synchronize()
    streams, got, errors = [torch.cuda.Stream(), torch.cuda.Stream()], [None] * 8, []

    def work(k):
        try:
            with torch.cuda.stream(streams[k]):
                for i in range(k, 8, 2):
                    got[i] = h(xs[i])
        except BaseException as e:                               # (an assertion in a thread is not the test's)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('which,M,N,K', [('ring2', 700, 5003, 512), ('ring3', 11800, 9501, 130)])
@pytest.mark.parametrize('out', ['fp32', 'bf16'])
def test_blocks_without_a_value_stay_in_their_row_and_column(which, M, N, K, out):
    """In the first tiles and in the last, incomplete ones."""
    from learning_embeddings_amd import quant
    assert form(M, N, K) == which
    x, w, b = inputs(M, N, K, 'fp32', seed=10)
    clean = quant.MXFP4Linear(w.cuda(), b.cuda(), out_dtype=DT[out])(x.cuda())
    rows, cols = [3, M // 2, M - 1], [7, N - 1]
    for r in rows:
        x[r, K - 1] = float('nan')
    for c in cols:
        w[c, 1] = float('inf')
    y = quant.MXFP4Linear(w.cuda(), b.cuda(), out_dtype=DT[out])(x.cuda())
    nan = torch.zeros(M, N, dtype=torch.bool, device='cuda')
    nan[rows] = True
    nan[:, cols] = True
    assert torch.equal(torch.isnan(y), nan) and torch.equal(y[~nan], clean[~nan])
