"""Microscaled 4-bit floating point (MXFP4) and a classifier head held in it.  No counterpart in the reference.

Blocks of 32 elements along a row share a power of two, 2^(floor(log2 max|v|) - 2) within [2^-127, 2^127]; an element is one of
{0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign times it, rounded to nearest with ties to even, saturating.  A block that holds a NaN or an
infinity stands for NaN.  17/32 bytes an element (rows padded to 32, elements to 64, scale words to 256).

    head = MXFP4Linear.from_linear(model.fc)          # quantises the weights once
    logits = head(features)                           # quantises the features row by row, multiplies on the 4-bit matrix cores, sums in 32 bits

The head is frozen -- a reference model's, or one that serves: its weights take no gradient and it passes none to its input."""
import torch
import torch.nn as nn

from ._lib import lib, check, dptr, raw_stream
from .ops import DTYPE_CODE, on_device_of


def _matrix(x, name):
    """(row-major 2-D view, dtype code, row stride)"""
    code = DTYPE_CODE.get(x.dtype)
    if code is None:
        raise TypeError('%s must be float32, bfloat16 or float16, got %s' % (name, x.dtype))
    if not x.is_cuda:
        dptr(x)                                                                  # raises: there is no CPU fallback
    if x.is_contiguous():
        return x, code, x.shape[1]
    if x.stride(1) != 1 and x.shape[1] > 1 or x.stride(0) < x.shape[1] and x.shape[0] > 1:
        x = x.contiguous()
    return x, code, (x.stride(0) if x.shape[0] > 1 else x.shape[1])


class MXFP4Tensor:
    """A matrix [rows, k] in 4 bits: `codes` and `scales` (uint8, in the matrix instruction's tile order -- see include/lecone.h) on one device, codes_bytes(rows, k) and
    scales_bytes(rows, k) long at least."""

    def __init__(self, codes, scales, shape):
        self.codes, self.scales, self.shape = codes, scales, tuple(int(v) for v in shape)
        if len(self.shape) != 2 or min(self.shape) < 0:
            raise ValueError('shape must be (rows, k), got %s' % (self.shape,))
        for t, name, need in ((codes, 'codes', codes_bytes(*self.shape)), (scales, 'scales', scales_bytes(*self.shape))):
            if t.dtype != torch.uint8:
                raise TypeError('%s must be uint8, got %s' % (name, t.dtype))
            if t.numel() < need or not t.is_contiguous():
                raise ValueError('%s of a %d x %d matrix are %d contiguous bytes, got %d%s' % (name, *self.shape, need, t.numel(), '' if t.is_contiguous() else ', strided'))
        if scales.device != codes.device:
            raise ValueError('codes are on %s, scales on %s' % (codes.device, scales.device))

    @classmethod
    def _made(cls, codes, scales, shape):
        """Of buffers that were made for it: nothing to check."""
        q = cls.__new__(cls)
        q.codes, q.scales, q.shape = codes, scales, shape
        return q

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def dequantize(self, dtype=torch.float32):
        """The values it stands for, [rows, k]; float32 and bfloat16 hold every one of them exactly."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError('the values are exact in float32 and bfloat16 only, got %s' % dtype)
        rows, k = self.shape
        if rows == 0 or k == 0:
            return torch.empty(rows, k, dtype=dtype, device=self.device)
        return _dequantize(self.codes, self.scales, rows, k, dtype)


@on_device_of(0)
def _dequantize(codes, scales, rows, k, dtype):
    if not codes.is_cuda:
        dptr(codes)                                                              # raises: there is no CPU fallback
    out = torch.empty((rows, k), dtype=dtype, device=codes.device)
    check(lib.lec_mxfp4_dequantize(codes.data_ptr(), scales.data_ptr(), rows, k, out.data_ptr(), DTYPE_CODE[dtype], k, raw_stream(codes.device.index)))
    return out


@on_device_of(0)
def _quantize(z, code, ld, rows, k):
    codes = torch.empty(codes_bytes(rows, k), dtype=torch.uint8, device=z.device)
    scales = torch.empty(scales_bytes(rows, k), dtype=torch.uint8, device=z.device)
    check(lib.lec_mxfp4_quantize(z.data_ptr(), code, ld, rows, k, codes.data_ptr(), scales.data_ptr(), raw_stream(z.device.index)))
    return codes, scales


@on_device_of(0)
def _linear(z, code, ld, codes, scales, N, k, bias, dtype):
    M = z.shape[0]
    y = torch.empty((M, N), dtype=dtype, device=z.device)
    ws = torch.empty(codes_bytes(M, k) + scales_bytes(M, k), dtype=torch.uint8, device=z.device)      # this call's own
    check(lib.lec_mxfp4_linear(z.data_ptr(), code, ld, M, codes.data_ptr(), scales.data_ptr(), N, k, bias if bias is None else bias.data_ptr(), y.data_ptr(), DTYPE_CODE[dtype],
                               N, ws.data_ptr(), ws.numel(), raw_stream(z.device.index)))
    return y


def codes_bytes(rows, k):
    """As lec_mxfp4_codes_bytes: tiles of 32 rows x 64 elements, a kilobyte each."""
    if rows > (1 << 31) - 32 or k > 1 << 24:
        raise ValueError('matrix too large for the 4-bit form (at most 2^31 - 32 rows of 2^24 elements): %d x %d' % (rows, k))
    return (rows + 31 >> 5) * (k + 63 >> 6) << 10


def scales_bytes(rows, k):
    """As lec_mxfp4_scales_bytes: a word a lane for four tiles."""
    return (rows + 31 >> 5) * (k + 255 >> 8) << 8


def mxfp4_quantize(x):
    """x [rows, k] (float32 / bfloat16 / float16) -> MXFP4Tensor.  Carries no gradient."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError('x must be [rows, k] with k > 0, got %s' % (tuple(x.shape),))
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError('mxfp4_quantize passes no gradient to its input: detach it, or call it under torch.no_grad()')
    z, code, ld = _matrix(x, 'x')
    rows, k = z.shape
    if rows == 0:
        e = torch.empty(0, dtype=torch.uint8, device=z.device)
        return MXFP4Tensor._made(e, e, (0, k))
    return MXFP4Tensor._made(*_quantize(z, code, ld, rows, k), (rows, k))


class MXFP4Linear(nn.Module):
    """y = x_4 W_4^T + b with the weights held, and x quantised on the way in, in 4 bits; sums in 32 bits, one rounding to the output's type.
    weight [out_features, in_features], bias [out_features] or None; out_dtype None: the input's.  Frozen: see above.
    A state holds its sizes (`shape`) and loads into a head of the same sizes only: the buffers are padded to whole tiles and do not tell 33 x 80 from 40 x 96."""

    def __init__(self, weight, bias=None, out_dtype=None):
        super().__init__()
        if out_dtype is not None and out_dtype not in DTYPE_CODE:
            raise TypeError('out_dtype must be float32, bfloat16 or float16, got %s' % out_dtype)
        q = mxfp4_quantize(weight.detach())
        if q.shape[0] == 0:
            raise ValueError('weight must have at least one row')
        self.out_features, self.in_features = q.shape
        self.out_dtype = out_dtype
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError('bias must be [%d], got %s' % (self.out_features, tuple(bias.shape)))
        self.register_buffer('codes', q.codes)
        self.register_buffer('scales', q.scales)
        self.register_buffer('shape', torch.cat([torch.full((1,), v, dtype=torch.int64, device=q.device) for v in q.shape]))
        self.register_buffer('bias', None if bias is None else bias.detach().to(device=q.device, dtype=torch.float32).contiguous().clone())

    @classmethod
    def from_linear(cls, linear, out_dtype=None):
        return cls(linear.weight, linear.bias, out_dtype)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        saved = state_dict.get(prefix + 'shape')
        if saved is not None and tuple(saved.tolist()) != (self.out_features, self.in_features):
            error_msgs.append('%s: the state is of a head of %s, this one is %d x %d' % (prefix[:-1] or 'MXFP4Linear', ' x '.join(str(v) for v in saved.tolist()), self.out_features,
                                                                                         self.in_features))
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if saved is None and prefix + 'shape' in missing_keys and prefix + 'codes' in state_dict:       # (saved by a version that did not keep the sizes)
            missing_keys.remove(prefix + 'shape')

    def extra_repr(self):
        return 'in_features=%d, out_features=%d, bias=%s, out_dtype=%s' % (self.in_features, self.out_features, self.bias is not None, self.out_dtype)

    def dequantize(self, dtype=torch.float32):
        return MXFP4Tensor(self.codes, self.scales, (self.out_features, self.in_features)).dequantize(dtype)

    def forward(self, x):
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError('MXFP4Linear is a frozen head and passes no gradient to its input: call it under torch.no_grad(), or on a detached input')
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise ValueError('x must be [..., %d], got %s' % (self.in_features, tuple(x.shape)))
        if x.device != self.codes.device:
            raise ValueError('x is on %s, the head on %s' % (x.device, self.codes.device))
        z, code, ld = _matrix(x if x.dim() == 2 else x.reshape(-1, self.in_features), 'x')
        dtype = self.out_dtype or x.dtype
        bias = self.bias
        if bias is not None and bias.dtype != torch.float32:
            bias = bias.float()                                                  # (.half() on a model converts its buffers)
        if z.shape[0] == 0:
            y = torch.empty(0, self.out_features, dtype=dtype, device=z.device)
        else:
            y = _linear(z, code, ld, self.codes, self.scales, self.out_features, self.in_features, bias, dtype)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], self.out_features)
