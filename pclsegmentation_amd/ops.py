"""Row operators on device tensors: the 8-bit linear layer and the log probabilities of labels with their gradient.

  quantize_rows(x) -> Int8Rows              8-bit codes and one scale per row (weights: one per output channel)
  matmul_i8(a, b, ...) -> y                 product of two Int8Rows with op_conv2d's bias / activation / residual epilogue
  linear_i8(x, weight, ...) -> y            the layer on float rows: quantize_rows(x), then matmul_i8
  label_logprobs(logits, labels, ...)       log probability of a label, entropy, log-sum-exp and top alternatives of every row
  label_logprobs_grad(...) -> d logits      their gradient

A 1x1 convolution of NHWC activations is linear_i8 on their last axis (``Int8Rows.from_kernel`` takes the Keras kernel); the
logits of a model go into label_logprobs as they are, [..., classes].  Tensors are float32, bfloat16 or float16 on one MI355X;
rows may have any stride as long as their elements are adjacent (others are copied).  Calls are asynchronous on torch's current
stream of the tensors' device, allocate their outputs and workspace through torch and keep nothing, so they can be captured
into a graph.  Like the rest of the package they compute outside of autograd: results carry no history, and a call that is
given a tensor that requires a gradient while gradients are recorded warns of it.  All arithmetic is in libpclseg.so."""
import ctypes
import functools
import sys
import warnings
from collections import namedtuple

import torch

from . import engine as _engine

LabelLogprobs = namedtuple("LabelLogprobs", "logprob entropy lse top_ids top_logprobs")


_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # pclseg_dtype


def _fail(what):
  raise ValueError("pclseg: " + what)


def _dtype(t, name):
  d = _DTYPES.get(t.dtype)
  if d is None:
    _fail("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
  return d


def _on(t, dev, name):
  if not isinstance(t, torch.Tensor) or (t.device != dev if dev is not None else not _engine.on_device(t)):
    _fail("%s must be a tensor on %s" % (name, dev or "the device"))
  if t.requires_grad and torch.is_grad_enabled():
    depth = 1
    while sys._getframe(depth).f_globals is globals():      # to the caller's line
      depth += 1
    warnings.warn("pclseg: %s requires a gradient, but the row operators compute outside of autograd and none flows back to it (call "
                  "them under torch.no_grad() or on detached tensors; label_logprobs_grad is the gradient of label_logprobs)" % name,
                  stacklevel=depth + 1)


def _rows(t, cols):
  """[..., cols] as two axes with adjacent elements and rows that do not overlap (a copy where the strides say otherwise)."""
  if t.is_contiguous():
    return (t if t.dim() == 2 else t.view(-1, cols)), cols
  r = t if t.dim() == 2 else t.reshape(-1, cols)
  if cols > 1 and r.stride(1) != 1 or r.shape[0] > 1 and r.stride(0) < cols:
    r = r.contiguous()
  return r, (r.stride(0) if r.shape[0] > 1 else cols)


def _vector(t, dev, n, name):
  _on(t, dev, name)
  if t.dtype != torch.float32 or t.numel() != n:
    _fail("%s must hold %d float32 values, got %s of shape %s" % (name, n, t.dtype, tuple(t.shape)))
  return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
  return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=None)
def _several_devices():
  return torch.cuda.device_count() > 1


def _call(dev, fn, *args):
  """fn(*args, stream) with `dev` current: kernels are launched on the current device."""
  if _several_devices() and torch.cuda.current_device() != dev.index:
    with torch.cuda.device(dev):
      rc = fn(*args, _engine.stream_handle(dev))
  else:
    rc = fn(*args, _engine.stream_handle(dev))
  if rc:
    _engine.check(rc)


@functools.lru_cache(maxsize=4096)
def _workspace(name, *sizes):
  """Bytes of workspace a call of these sizes takes."""
  size = ctypes.c_size_t()
  _engine.check(getattr(_engine.load_library(), name)(*sizes, ctypes.byref(size)))
  return size.value


class Int8Rows:
  """8-bit codes of the rows of a matrix with one scale per row: row i stands for ``codes[i] * scale[i]``.

  ``data`` int8 [rows, pclseg_i8_row_bytes(k)] holds the codes with zeros behind column k (the layout the product reads),
  ``scale`` float32 [rows].  Made by quantize_rows, from_codes or from_kernel."""
  __slots__ = ("data", "scale", "k")

  def __init__(self, data, scale, k):
    if (data.dtype != torch.int8 or data.dim() != 2 or data.shape[1] != _row_bytes(k) or not data.is_contiguous() or
        scale.dtype != torch.float32 or tuple(scale.shape) != (data.shape[0],) or not scale.is_contiguous() or
        scale.device != data.device):
      _fail("Int8Rows holds contiguous int8 [rows, %d] (k %d) and float32 [rows] on one device, got %s %s and %s %s; "
            "codes of another layout go through from_codes" % (_row_bytes(k), k, data.dtype, tuple(data.shape), scale.dtype,
                                                              tuple(scale.shape)))
    self.data, self.scale, self.k = data, scale, int(k)

  @classmethod
  def from_codes(cls, codes, scale):
    """Codes int8 [rows, k] and scales float32 [rows] from elsewhere, laid out once."""
    _on(codes, None, "codes")
    if codes.dtype != torch.int8 or codes.dim() != 2:
      _fail("codes must be int8 [rows, k], got %s of shape %s" % (codes.dtype, tuple(codes.shape)))
    rows, k = codes.shape
    scale = _vector(scale, codes.device, rows, "scale")
    data = torch.zeros((rows, _row_bytes(k)), dtype=torch.int8, device=codes.device)
    data[:, :k] = codes
    return cls(data, scale, k)

  @classmethod
  def from_kernel(cls, kernel):
    """A Keras kernel (1,1,Cin,Cout) or (Cin,Cout) -> one row and scale per output channel."""
    if kernel.dim() == 4 and tuple(kernel.shape[:2]) != (1, 1) or kernel.dim() not in (2, 4):
      _fail("the kernel of an 8-bit layer is (1,1,Cin,Cout) or (Cin,Cout), got %s" % (tuple(kernel.shape),))
    return quantize_rows(kernel.reshape(kernel.shape[-2:]).t().contiguous())

  @property
  def rows(self):
    return self.data.shape[0]

  @property
  def codes(self):
    return self.data[:, :self.k]

  def dequantize(self):
    return self.codes.float() * self.scale[:, None]


def _row_bytes(k):
  b = _engine.load_library().pclseg_i8_row_bytes(k)
  if not b:
    _fail("rows of 8-bit codes have 1 to 131071 columns, got %d" % k)
  return b


def quantize_rows(x):
  """Symmetric 8-bit codes of x [..., k]: scale = max|row| / 127, code = round(x / scale), ties to even.  A row of zeros has
  the scale 0 (and so does one whose scale is too small for a float32); a row with an infinity or a NaN has the scale NaN, and so are the products it takes part in."""
  _on(x, None, "x")
  dt = _dtype(x, "x")
  if x.dim() < 1:
    _fail("x must have rows")
  k = x.shape[-1]
  kp = _row_bytes(k)
  r, stride = _rows(x, k)
  m = r.shape[0]
  data = torch.empty((m, kp), dtype=torch.int8, device=x.device)
  scale = torch.empty(m, dtype=torch.float32, device=x.device)
  if m:
    _call(x.device, _engine.load_library().pclseg_op_quantize_rows, r.data_ptr(), dt, m, k, stride, data.data_ptr(),
          scale.data_ptr())
  return Int8Rows(data, scale, k)


def _epilogue(dev, m, n, shape, weight, bias, act, residual, dtype):
  if act not in _engine.ACT:
    _fail("unknown activation %r" % (act,))
  if dtype not in _DTYPES:
    _fail("out_dtype must be float32, bfloat16 or float16, got %s" % (dtype,))
  if not isinstance(weight, Int8Rows) or weight.data.device != dev:
    _fail("weight must be Int8Rows on %s" % (dev,))
  if bias is not None:
    bias = _vector(bias, dev, n, "bias")
  rstride = 0
  if residual is not None:
    _on(residual, dev, "residual")
    if residual.dtype != dtype or tuple(residual.shape) != shape:
      _fail("residual must be %s of shape %s, got %s of shape %s" % (dtype, shape, residual.dtype, tuple(residual.shape)))
    if m and n:
      residual, rstride = _rows(residual, n)
  return bias, residual, rstride


def matmul_i8(a, b, bias=None, act="none", residual=None, out_dtype=torch.float32):
  """act(a b^T scaled by both sides' scales + bias) + residual: [a.rows, b.rows].  The int8 products are summed exactly."""
  if not isinstance(a, Int8Rows) or not isinstance(b, Int8Rows) or a.k != b.k:
    _fail("a and b must be Int8Rows with the same number of columns")
  dev, m, n = a.data.device, a.rows, b.rows
  bias, residual, rstride = _epilogue(dev, m, n, (m, n), b, bias, act, residual, out_dtype)
  y = torch.empty((m, n), dtype=out_dtype, device=dev)
  if m and n:
    _call(dev, _engine.load_library().pclseg_op_matmul_i8, a.data.data_ptr(), a.scale.data_ptr(), b.data.data_ptr(),
          b.scale.data_ptr(), m, n, a.k, _ptr(bias), _engine.ACT[act], _ptr(residual), rstride, y.data_ptr(), n,
          _DTYPES[out_dtype])
  return y


def linear_i8(x, weight, bias=None, act="none", residual=None, out_dtype=None):
  """The 8-bit linear layer: x [..., k] is quantised row by row (quantize_rows) and multiplied with weight [n, k] (Int8Rows);
  act(... + bias[n]) + residual[..., n].  out_dtype defaults to x's."""
  _on(x, None, "x")
  dt = _dtype(x, "x")
  out_dtype = out_dtype or x.dtype
  if not isinstance(weight, Int8Rows) or x.dim() < 1 or x.shape[-1] != weight.k:
    _fail("weight must be Int8Rows with as many columns as x")
  dev, k, n = x.device, weight.k, weight.rows
  shape = tuple(x.shape[:-1]) + (n,)
  r, stride = _rows(x, k)
  m = r.shape[0]
  bias, residual, rstride = _epilogue(dev, m, n, shape, weight, bias, act, residual, out_dtype)
  y = x.new_empty(shape, dtype=out_dtype)
  if m and n:
    size = _workspace("pclseg_op_linear_i8_workspace", m, n, k)
    work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _call(dev, _engine.load_library().pclseg_op_linear_i8, r.data_ptr(), dt, stride, weight.data.data_ptr(), weight.scale.data_ptr(), m, n, k,
          _ptr(bias), _engine.ACT[act], _ptr(residual), rstride, y.data_ptr(), n, _DTYPES[out_dtype],
          _ptr(work), size)
  return y


def _labels(labels, dev, m):
  _on(labels, dev, "labels")
  if labels.dtype not in (torch.int32, torch.int64) or labels.numel() != m:
    _fail("labels must hold %d int32 or int64 values, got %s of shape %s" % (m, labels.dtype, tuple(labels.shape)))
  return labels if labels.is_contiguous() else labels.contiguous()


def _mask(allowed, logits):
  """-> (tensor, row stride): [classes] for every row, or one row per row of the logits."""
  _on(allowed, logits.device, "allowed")
  v = logits.shape[-1]
  if allowed.dtype not in (torch.bool, torch.uint8) or tuple(allowed.shape) not in ((v,), tuple(logits.shape)):
    _fail("allowed must be bool or uint8 of shape (%d,) or %s, got %s of shape %s" % (
      v, tuple(logits.shape), allowed.dtype, tuple(allowed.shape)))
  if allowed.dim() == 1:
    return (allowed if allowed.is_contiguous() else allowed.contiguous()), 0
  return _rows(allowed, v)


def _logits(logits):
  _on(logits, None, "logits")
  dt = _dtype(logits, "logits")
  if logits.dim() < 1 or logits.shape[-1] < 1:
    _fail("logits must be [..., classes], got shape %s" % (tuple(logits.shape),))
  return (dt,) + _rows(logits, logits.shape[-1])


def label_logprobs(logits, labels=None, top_k=0, allowed=None):
  """logits [..., classes] -> LabelLogprobs(logprob, entropy, lse, top_ids, top_logprobs), float32 (ids int32).

  labels [...] int32 / int64: a label outside [0, classes) is not counted, its logprob is 0; without labels logprob is None.
  allowed bool / uint8 [classes] or like logits: excluded classes take no part, whatever their logit holds; a logit of -inf
  is an excluded class, an excluded label has the logprob -inf.  top_k <= 64 alternatives, most probable first, the lowest
  class first among equals, -1 and -inf where fewer are allowed.  A row without an allowed class has the lse -inf and the
  entropy 0; a row whose allowed logits hold a NaN or +inf has NaN throughout and ids -1."""
  dt, r, stride = _logits(logits)
  dev, shape, (m, v) = logits.device, tuple(logits.shape[:-1]), r.shape
  top_k = int(top_k)
  if labels is not None:
    labels = _labels(labels, dev, m)
  mstride = 0
  if allowed is not None:
    allowed, mstride = _mask(allowed, logits)
  size = _workspace("pclseg_op_label_logprobs_workspace", m, v, top_k)
  logprob, entropy, lse = logits.new_empty((3,) + shape, dtype=torch.float32).unbind(0)
  if labels is None:
    logprob = None
  ids = logits.new_empty(shape + (top_k,), dtype=torch.int32) if top_k else None
  tops = logits.new_empty(shape + (top_k,), dtype=torch.float32) if top_k else None
  if m:
    work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _call(dev, _engine.load_library().pclseg_op_label_logprobs, r.data_ptr(), dt, m, v, stride, _ptr(labels),
          labels.element_size() if labels is not None else 0, _ptr(allowed), mstride, top_k, _ptr(logprob), entropy.data_ptr(),
          lse.data_ptr(), _ptr(ids), _ptr(tops), _ptr(work), size)
  return LabelLogprobs(logprob, entropy, lse, ids, tops)


def label_logprobs_grad(logits, labels, lse, d_logprob=None, entropy=None, d_entropy=None, top_ids=None, d_top=None,
                        allowed=None, logprob=None, top_logprobs=None):
  """Gradient with respect to the logits (their shape and dtype) of a loss whose gradients with respect to label_logprobs'
  logprob, entropy and top_logprobs are d_logprob, d_entropy and d_top (float32; each may be None, one is given).  lse, entropy
  and top_ids are what label_logprobs returned for the same logits and mask; entropy is needed for d_entropy, top_ids for
  d_top.  Excluded classes, rows without an allowed class and labels that are not counted get 0.

  logprob (with labels) and top_logprobs (with top_ids) are what label_logprobs returned too.  Without them ln p is logit - lse,
  right to the rounding of lse; with them the gradient of a label or alternative that has nearly all of a row's probability
  is right to its own last bits (with d_entropy alone as well, where they name the decided class)."""
  dt, r, stride = _logits(logits)
  dev, (m, v) = logits.device, r.shape
  if d_logprob is None and d_entropy is None and d_top is None:
    _fail("one of d_logprob, d_entropy and d_top must be given")
  lse = _vector(lse, dev, m, "lse")
  if d_logprob is not None or logprob is not None:
    if labels is None:
      _fail("d_logprob and logprob need labels")
    labels = _labels(labels, dev, m)
    d_logprob = None if d_logprob is None else _vector(d_logprob, dev, m, "d_logprob")
    logprob = None if logprob is None else _vector(logprob, dev, m, "logprob")
  else:
    labels = None
  if d_entropy is not None:
    if entropy is None:
      _fail("d_entropy needs entropy")
    entropy, d_entropy = _vector(entropy, dev, m, "entropy"), _vector(d_entropy, dev, m, "d_entropy")
  top_k = 0
  if d_top is not None or top_logprobs is not None:
    if top_ids is None:
      _fail("d_top and top_logprobs need top_ids")
    _on(top_ids, dev, "top_ids")
    top_k = top_ids.shape[-1] if top_ids.dim() else 0
    if top_ids.dtype != torch.int32 or top_ids.numel() != m * top_k:
      _fail("top_ids must be int32 [..., top_k], got %s of shape %s" % (top_ids.dtype, tuple(top_ids.shape)))
    top_ids = top_ids.contiguous()
    d_top = None if d_top is None else _vector(d_top, dev, m * top_k, "d_top")
    top_logprobs = None if top_logprobs is None else _vector(top_logprobs, dev, m * top_k, "top_logprobs")
  mstride = 0
  if allowed is not None:
    allowed, mstride = _mask(allowed, logits)
  grad = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty(logits.shape)
  if m:
    _call(dev, _engine.load_library().pclseg_op_label_logprobs_grad_ex, r.data_ptr(), dt, m, v, stride, _ptr(labels),
          0 if labels is None else labels.element_size(), _ptr(allowed), mstride, lse.data_ptr(),
          _ptr(entropy) if d_entropy is not None else None, _ptr(logprob), _ptr(top_ids) if top_k else None,
          _ptr(top_logprobs) if top_k else None, _ptr(d_logprob), _ptr(d_entropy), _ptr(d_top) if top_k else None, top_k,
          grad.data_ptr(), v)
  return grad
