"""The 4-bit form and the head held in it, on the MI355X, against the 64-bit oracle.

Quantisation has one right answer, so it is compared for equality.  A product: x_4 w_4 is exact in 32 bits (two 2-bit significands), K additions of up to 2 u each
(u = 2^-24; the matrix core may truncate) against the sum of |x_4 w_4|, the bias's addition, one rounding to the output's type of half a step."""
import numpy as np
import pytest
import torch

from oracle import feedback_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def same(a, b):
    return ((a == b) | (np.isnan(a) & np.isnan(b))).all()


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('rows,k', [(1, 1), (1, 31), (2, 32), (15, 33), (16, 128), (17, 129), (3, 512), (5, 513), (33, 515), (64, 2048), (200, 1000)])
def test_quantize_and_back(rows, k, dtype):
    from learning_embeddings_amd import quant
    rs = np.random.RandomState(rows * 1000 + k)
    x = torch.from_numpy((rs.randn(rows, k) * np.exp(2 * rs.randn(rows, 1))).astype(np.float32)).to(DT[dtype])
    x[0, 0] = 0.0
    q = quant.mxfp4_quantize(x.cuda())
    want = O.mxfp4_values(x.double().numpy())
    assert same(q.dequantize().double().cpu().numpy(), want) and same(q.dequantize(torch.bfloat16).double().cpu().numpy(), want)
    wide = torch.full((rows, k + 3), float('nan'), dtype=x.dtype, device='cuda')                # odd offset and row stride
    wide[:, 1:k + 1] = x.cuda()
    q2 = quant.mxfp4_quantize(wide[:, 1:k + 1])
    assert torch.equal(q2.codes, q.codes) and torch.equal(q2.scales, q.scales)
    if rows > 1:
        assert torch.equal(quant.mxfp4_quantize(x.cuda().t().contiguous().t()).codes, q.codes)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('order', ['bits', 'shuffled'])
def test_every_16_bit_value(dtype, order):
    from learning_embeddings_amd import quant
    bits = np.arange(65536)
    if order == 'shuffled':
        bits = np.random.RandomState(0).permutation(bits)
    x = torch.from_numpy(bits.astype(np.uint16).view(np.int16)).view(DT[dtype]).view(64, 1024)
    assert same(quant.mxfp4_quantize(x.cuda()).dequantize().double().cpu().numpy(), O.mxfp4_values(x.double().numpy()))


def test_every_threshold_at_every_scale():
    """For each exponent a block holds: the thresholds between neighbouring magnitudes, the next float below and above each, and the block's maximum; with the smallest
    and largest floats, subnormals among them."""
    from learning_embeddings_amd import quant
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
    t = np.concatenate([mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(9)), -mid, [0.0, -0.0, 6.0]]).astype(np.float32)
    assert len(t) == 31
    rows = []
    for e in range(-149, 126):
        for top in (4.0, 7.9999995):
            with np.errstate(under='ignore'):
                rows.append(np.concatenate([np.ldexp(t, e), [np.ldexp(np.float32(top), e)]]).astype(np.float32))
    x = np.stack(rows)
    got = quant.mxfp4_quantize(torch.from_numpy(x).cuda()).dequantize().double().cpu().numpy()
    assert same(got, O.mxfp4_values(x))


def test_blocks_without_a_value():
    from learning_embeddings_amd import quant
    x = torch.ones(4, 96)
    x[0, 5] = float('nan'); x[1, 40] = float('inf'); x[2, 95] = -float('inf'); x[3] = 0.0
    got = quant.mxfp4_quantize(x.cuda()).dequantize().cpu().numpy()
    assert same(got, O.mxfp4_values(x.numpy())) and np.isnan(got).sum() == 96 and (got[3] == 0).all()


def head(M, N, K, dtype, out, bias, seed=0):
    rs = np.random.RandomState(seed)
    x = torch.from_numpy((rs.randn(M, K) * np.exp(rs.randn(1, K))).astype(np.float32)).to(DT[dtype])
    w = torch.from_numpy((rs.randn(N, K) * np.exp(rs.randn(N, 1))).astype(np.float32))
    b = torch.from_numpy(rs.randn(N).astype(np.float32)) if bias else None
    return x, w, b


def check(y, x, w, b, out):
    f64 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.float64)).cuda()          # (the products of the oracle's values, in 64 bits)
    xq, wq = f64(O.mxfp4_values(x.double().numpy())), f64(O.mxfp4_values(w.double().numpy()))
    want, size = xq @ wq.T.contiguous(), xq.abs() @ wq.abs().T.contiguous()
    if b is not None:
        want += b.double().cuda(); size += b.double().abs().cuda()
    tol = 2 * (x.shape[1] + 4) * U * size
    tol += torch.finfo(DT[out]).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if out == 'fp16' else 0)
    assert y.dtype == DT[out] and y.shape == want.shape
    err = (y.double() - want).abs()
    assert (err <= tol).all(), 'error / tolerance %.3g at %s' % (float((err / tol).max()), (err > tol).nonzero()[:4].tolist())


# (M <= 4: one launch; up to 32 rows or 1 024 tiles of 32 x 32: wave pairs; beyond: the ring of 128 x 128; from 3 000 tiles of 192 x 192: that ring)
HEADS = [(1, 1, 1), (4, 33, 4000), (4, 40, 3328), (5, 31, 64), (1, 5, 31), (1, 723, 512), (2, 17, 33), (3, 50, 515), (8, 16, 127), (15, 100, 128), (16, 64, 129), (17, 63, 512), (31, 200, 513), (33, 129, 640), (64, 128, 2048),
         (65, 257, 256), (127, 130, 384), (128, 723, 512), (131, 723, 512), (200, 1000, 1100), (256, 256, 2048), (257, 300, 2047), (300, 2000, 160), (513, 777, 300)]


@pytest.mark.parametrize('M,N,K', HEADS)
@pytest.mark.parametrize('dtype,out,bias', [('fp32', 'fp32', True), ('bf16', 'bf16', True), ('fp16', 'fp16', False), ('bf16', 'fp32', False)])
def test_head(M, N, K, dtype, out, bias):
    from learning_embeddings_amd import quant
    x, w, b = head(M, N, K, dtype, out, bias)
    h = quant.MXFP4Linear(w.cuda(), None if b is None else b.cuda(), out_dtype=DT[out])
    check(h(x.cuda()), x, w, b, out)


@pytest.mark.parametrize('M,N', [(1, 50000), (7, 20011), (40, 50000), (700, 5003), (2300, 1500), (4, 50000), (90, 30000)])
def test_large_heads(M, N):
    from learning_embeddings_amd import quant
    x, w, b = head(M, N, 512, 'bf16', 'bf16', True, seed=3)
    check(quant.MXFP4Linear(w.cuda(), b.cuda())(x.cuda()), x, w, b, 'bf16')


@pytest.mark.parametrize('M,N,K,dtype,out', [(2300, 5003, 640, 'bf16', 'bf16'), (4096, 2048, 512, 'fp32', 'fp32'), (2049, 4100, 130, 'fp16', 'fp16'), (300, 17000, 1300, 'bf16', 'fp32'),
                                               (9000, 1001, 33, 'bf16', 'bf16'), (2561, 3001, 2048, 'bf16', 'bf16'),
                                               (5800, 19201, 200, 'bf16', 'bf16'), (11600, 9300, 130, 'fp32', 'fp32'), (1400, 1200, 5000, 'fp16', 'fp32')])
def test_products_large_enough_for_the_ring(M, N, K, dtype, out):
    from learning_embeddings_amd import quant
    x, w, b = head(M, N, K, dtype, out, True, seed=5)
    h = quant.MXFP4Linear(w.cuda(), b.cuda(), out_dtype=DT[out])
    y = h(x.cuda())
    check(y, x, w, b, out)
    assert torch.equal(y, h(x.cuda()))


@pytest.mark.parametrize('M', [1, 20, 300])
def test_blocks_without_a_value_poison_their_row_and_column_only(M):
    from learning_embeddings_amd import quant
    x, w, b = head(M, 70, 200, 'fp32', 'fp32', True, seed=1)
    clean = quant.MXFP4Linear(w.cuda(), b.cuda())(x.cuda())
    w[7, 150] = float('inf')
    if M > 1:
        x[M // 2, 3] = float('nan')
    y = quant.MXFP4Linear(w.cuda(), b.cuda())(x.cuda())
    nan = torch.zeros(M, 70, dtype=torch.bool)
    nan[:, 7] = True
    if M > 1:
        nan[M // 2] = True
    assert torch.equal(torch.isnan(y).cpu(), nan) and torch.equal(y.cpu()[~nan], clean.cpu()[~nan])


def test_far_apart_scales_and_zero_rows():
    from learning_embeddings_amd import quant
    x, w, b = head(20, 40, 256, 'fp32', 'fp32', True, seed=2)
    x[:, 64:96] *= 2.0 ** 60; w[:, 64:96] *= 2.0 ** -60; x[:, 128:160] *= 2.0 ** -100; w[3] = 0.0; x[5] = 0.0
    y = quant.MXFP4Linear(w.cuda(), b.cuda())(x.cuda())
    check(y, x, w, b, 'fp32')
    assert (y[5].cpu() == b).all() and (y[:, 3] == float(b[3])).all()


def test_leading_dimensions_strides_empty_and_module_life():
    import torch.nn as nn
    from learning_embeddings_amd import quant
    lin = nn.Linear(96, 33).cuda()
    h = quant.MXFP4Linear.from_linear(lin)
    x = torch.randn(2, 3, 96, device='cuda')
    y = h(x)
    assert y.shape == (2, 3, 33) and torch.equal(y.view(6, 33), h(x.view(6, 96)))
    big = torch.randn(6, 101, device='cuda')
    assert torch.equal(h(big[:, 2:98]), h(big[:, 2:98].contiguous())) and torch.equal(h(big[::2, 2:98]), h(big[:, 2:98])[::2])
    assert h(x[:0]).shape == (0, 3, 33) and h(x[0, 0]).shape == (33,)
    assert torch.equal(h.dequantize(), quant.mxfp4_quantize(lin.weight.detach()).dequantize())
    other = quant.MXFP4Linear.from_linear(nn.Linear(96, 33).cuda())
    other.load_state_dict(h.state_dict())
    assert torch.equal(other(x), y)
    half = quant.MXFP4Linear.from_linear(lin).half()
    assert half(x.half()).dtype == torch.float16
    with pytest.raises(RuntimeError, match='no gradient'):
        h(x.requires_grad_())
    with torch.no_grad():
        h(x)
    with pytest.raises(ValueError, match='x must be'):
        h(torch.randn(2, 95, device='cuda'))
    with pytest.raises(ValueError, match='on cpu'):
        h(torch.randn(2, 96))
    with pytest.raises(ValueError, match='bias'):
        quant.MXFP4Linear(lin.weight, torch.zeros(32, device='cuda'))


@pytest.mark.parametrize('M,N,K', [(1, 5000, 512), (200, 723, 512), (600, 3000, 2048)])
def test_same_bits_on_another_stream_and_captured(M, N, K):
    from learning_embeddings_amd import quant
    x, w, b = head(M, N, K, 'bf16', 'bf16', True, seed=4)
    h = quant.MXFP4Linear(w.cuda(), b.cuda())
    xs = [x.cuda(), x.cuda().flip(0).contiguous()]
    want = [h(v) for v in xs]
    s = torch.cuda.Stream(); s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = [h(v) for v in xs]
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for v in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(h(v))
        graphs.append(g)
    for k in range(4):
        for v in xs:
            v.copy_(torch.roll(v, 1, 0))
        want_k = [h(v) for v in xs]
        order = ((0, 1), (1, 0), (0, 1), (1, 1, 0))[k]
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want_k))
    assert all(torch.equal(a, c) for a, c in zip(again, want))


def test_more_outputs_than_31_bits_count():
    """45 000 rows x 50 000 classes: 2.25e9 outputs.  The ring sums every output's products in the same order wherever it lies: the last rows equal the same rows alone."""
    from learning_embeddings_amd import quant
    g = torch.Generator(device='cuda').manual_seed(0)
    w, b = torch.randn(50000, 192, generator=g, device='cuda'), torch.randn(50000, generator=g, device='cuda')
    x = torch.randn(45000, 192, generator=g, device='cuda').bfloat16()
    h = quant.MXFP4Linear(w, b)
    y = h(x)
    assert torch.equal(y[-5000:], h(x[-5000:]))
    check(y[-3:, -300:].contiguous(), x[-3:].cpu(), w[-300:].cpu(), b[-300:].cpu(), 'bf16')
