"""The 4-bit head's host side without a GPU: states, sizes, alignment."""
import copy
import io

import pytest
import torch


@pytest.fixture
def quant(monkeypatch):
    """The module with a quantisation that fills its buffers with numbers that tell heads apart (the real one runs on the GPU)."""
    from learning_embeddings_amd import quant as q
    made = []

    def numbered(w):
        made.append(w)
        e = lambda n: torch.full((n,), len(made), dtype=torch.uint8)
        return q.MXFP4Tensor(e(q.codes_bytes(*w.shape)), e(q.scales_bytes(*w.shape)), w.shape)
    monkeypatch.setattr(q, 'mxfp4_quantize', numbered)
    return q


@pytest.mark.parametrize('mine,other', [((33, 80), (40, 96)), ((40, 96), (33, 80)), ((33, 80), (64, 80)), ((33, 80), (33, 128)), ((5, 31), (5, 32))])
def test_a_state_of_other_sizes_is_refused_and_changes_nothing(quant, mine, other):
    """Both heads have the same number of 32 x 64 tiles: their buffers are of one length."""
    a, b = quant.MXFP4Linear(torch.zeros(*mine)), quant.MXFP4Linear(torch.zeros(*other))
    assert a.codes.shape == b.codes.shape and a.scales.shape == b.scales.shape
    before = {k: v.clone() for k, v in a.state_dict().items()}
    for strict in (True, False):
        with pytest.raises(RuntimeError, match='%d x %d' % other):
            a.load_state_dict(b.state_dict(), strict=strict)
    with pytest.raises(RuntimeError, match='%d x %d' % other):
        torch.nn.Sequential(a).load_state_dict(torch.nn.Sequential(b).state_dict())
    assert all(torch.equal(v, before[k]) for k, v in a.state_dict().items())


@pytest.mark.parametrize('bias', [False, True])
def test_a_state_of_the_same_sizes_loads(quant, bias):
    make = lambda: quant.MXFP4Linear(torch.zeros(33, 80), torch.randn(33) if bias else None)
    a, b = make(), make()
    f = io.BytesIO()
    torch.save(b.state_dict(), f)
    f.seek(0)
    assert not any(a.load_state_dict(torch.load(f, weights_only=True)))
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and (not bias or torch.equal(a.bias, b.bias))
    c = copy.deepcopy(b).half()
    assert (c.out_features, c.in_features) == (33, 80) and not any(a.load_state_dict(c.state_dict()))
    old = {k: v for k, v in make().state_dict().items() if k in ('codes', 'scales', 'bias')}        # a state without its sizes
    assert not any(a.load_state_dict(old)) and torch.equal(a.codes, old['codes'])
    with pytest.raises(RuntimeError, match='size mismatch'):
        a.load_state_dict(quant.MXFP4Linear(torch.zeros(65, 80), torch.zeros(65) if bias else None).state_dict() | {'shape': torch.tensor([33, 80])})


def test_buffers_that_do_not_hold_the_matrix_are_refused():
    """The kernels take codes and scales by their sizes in whole tiles: shorter buffers would be read past their end."""
    from learning_embeddings_amd import quant
    codes, scales = torch.zeros(4096, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    assert quant.MXFP4Tensor(codes, scales, (33, 128)).nbytes() == 4608 and quant.MXFP4Tensor(codes[:0], scales[:0], (0, 32)).dequantize().shape == (0, 32)
    for c, s, shape in ((codes[:-1], scales, (33, 128)), (codes, scales[:-1], (33, 128)), (codes, scales, (65, 128)), (codes, scales, (33, 129)), (codes[:0], scales[:0], (1, 1)),
                        (codes, scales[:256], (33, 1)), (codes, scales, (2 ** 31, 128))):
        with pytest.raises(ValueError, match='bytes|too large'):
            quant.MXFP4Tensor(c, s, shape)
    for shape in ((33,), (33, 128, 1), (-1, 128), (33, -128)):
        with pytest.raises(ValueError, match='shape'):
            quant.MXFP4Tensor(codes, scales, shape)
    with pytest.raises(TypeError, match='uint8'):
        quant.MXFP4Tensor(codes.view(torch.int8), scales, (33, 128))
    with pytest.raises(ValueError, match='contiguous'):
        quant.MXFP4Tensor(torch.zeros(8192, dtype=torch.uint8)[::2], scales, (33, 128))
    with pytest.raises(ValueError, match='on meta'):
        quant.MXFP4Tensor(codes, scales.to('meta'), (33, 128))


def test_buffers_in_host_memory_are_refused(quant):
    q = quant.MXFP4Tensor(torch.zeros(1024, dtype=torch.uint8), torch.zeros(256, dtype=torch.uint8), (5, 31))
    head = quant.MXFP4Linear(torch.zeros(5, 31))
    for call in (q.dequantize, head.dequantize, lambda: head(torch.zeros(2, 31))):
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            call()


@pytest.mark.parametrize('off', [1, 4, 8])
def test_misaligned_buffers_are_refused_at_the_c_entries(off):
    """A wave's request is a contiguous kilobyte of 16 bytes a lane.  Never dereferenced: every call is refused before its launch."""
    import ctypes
    from learning_embeddings_amd import _lib
    lib, p, q = _lib.lib, ctypes.c_void_p(256), ctypes.c_void_p(256 + off)
    for call in (lambda: lib.lec_mxfp4_quantize(p, 0, 32, 1, 32, q, p, None), lambda: lib.lec_mxfp4_quantize(p, 0, 32, 1, 32, p, q, None),
                 lambda: lib.lec_mxfp4_dequantize(q, p, 1, 32, p, 0, 32, None), lambda: lib.lec_mxfp4_dequantize(p, q, 1, 32, p, 0, 32, None),
                 lambda: lib.lec_mxfp4_linear(p, 0, 32, 8, q, p, 4, 32, None, p, 0, 4, p, 1 << 20, None), lambda: lib.lec_mxfp4_linear(p, 0, 32, 8, p, q, 4, 32, None, p, 0, 4, p, 1 << 20, None),
                 lambda: lib.lec_mxfp4_linear(p, 0, 32, 8, p, p, 4, 32, None, p, 0, 4, q, 1 << 20, None)):
        assert call() == _lib.E_ARG and b'aligned' in lib.lec_last_error()
