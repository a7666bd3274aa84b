"""Row operators without a GPU: every refusal of the C entry points and of pclsegmentation_amd.ops (a refused call launches
nothing), the layout helper, the exception barrier."""
import ctypes
import os
import re

import pytest
import torch

from pclsegmentation_amd import engine as E
from pclsegmentation_amd import ops

BUF = (ctypes.c_uint8 * 4096)()
P = (ctypes.addressof(BUF) + 255) // 256 * 256        # an aligned address that a refused call must not touch


def _refused(fn, args, code, word):
  lib = E.load_library()
  assert getattr(lib, fn)(*args) == code
  assert word in lib.pclseg_last_error(None).decode(), lib.pclseg_last_error(None)


def test_row_bytes():
  f = E.load_library().pclseg_i8_row_bytes
  assert [f(k) for k in (0, -1, 131072, 1 << 40)] == [0, 0, 0, 0]
  assert [f(k) for k in (1, 64, 65, 128, 129, 1000, 131071)] == [64, 64, 128, 128, 256, 1024, 131072]


QUANT = dict(x=P, dtype=0, rows=2, cols=8, x_stride=8, q=P, scale=P, stream=None)


@pytest.mark.parametrize("change,code,word", [
  (dict(dtype=3), -1, "dtype"), (dict(rows=-1), -2, "rows"), (dict(rows=1 << 31), -2, "rows"), (dict(cols=0), -2, "cols"),
  (dict(cols=131072), -2, "cols"), (dict(x_stride=7), -2, "stride"), (dict(x=None), -1, "NULL"), (dict(q=None), -1, "NULL"),
  (dict(scale=None), -1, "NULL"), (dict(x=P + 2), -1, "misaligned"), (dict(q=P + 4), -1, "misaligned"),
])
def test_quantize_rows_refuses(change, code, word):
  _refused("pclseg_op_quantize_rows", list({**QUANT, **change}.values()), code, word)


MATMUL = dict(a=P, a_scale=P, b=P, b_scale=P, m=2, n=3, k=8, bias=None, act=0, residual=None, residual_stride=0, y=P, y_stride=3,
              dtype=1, stream=None)


@pytest.mark.parametrize("change,code,word", [
  (dict(dtype=-1), -1, "dtype"), (dict(act=4), -1, "activation"), (dict(m=-1), -2, "m must"), (dict(n=0), -2, "n must"),
  (dict(n=1 << 31), -2, "n must"), (dict(k=0), -2, "k must"), (dict(k=131072), -2, "k must"), (dict(a=None), -1, "NULL"),
  (dict(b=None), -1, "NULL"), (dict(y=None), -1, "NULL"), (dict(a=P + 8), -1, "aligned"), (dict(b=P + 8), -1, "aligned"),
  (dict(y_stride=2), -2, "stride"), (dict(residual=P, residual_stride=2), -2, "stride"), (dict(y=P + 1), -1, "misaligned"),
  (dict(m=1 << 40, n=1 << 20, y_stride=1 << 20), -2, "tiles"), (dict(m=(1 << 40) + 1), -2, "m must"),
  (dict(n=(1 << 30) + 1, y_stride=1 << 31), -2, "n must"),
])
def test_matmul_i8_refuses(change, code, word):
  _refused("pclseg_op_matmul_i8", list({**MATMUL, **change}.values()), code, word)


LINEAR = dict(x=P, dtype=0, x_stride=8, weight=P, weight_scale=P, m=33, n=3, k=8, bias=None, act=0, residual=None,
              residual_stride=0, y=P, y_stride=3, y_dtype=1, workspace=P, workspace_bytes=33 * 68, stream=None)


@pytest.mark.parametrize("change,code,word", [
  (dict(dtype=7), -1, "dtype"), (dict(y_dtype=7), -1, "dtype"), (dict(x_stride=7), -2, "stride"), (dict(x=None), -1, "NULL"),
  (dict(workspace=None), -1, "workspace"), (dict(workspace_bytes=33 * 68 - 1), -1, "workspace"), (dict(workspace=P + 8), -1, "misaligned"),
  (dict(m=1 << 31), -2, "m must"), (dict(x=P + 1), -1, "misaligned"),
])
def test_linear_i8_refuses(change, code, word):
  _refused("pclseg_op_linear_i8", list({**LINEAR, **change}.values()), code, word)


def test_workspace_sizes():
  lib, size = E.load_library(), ctypes.c_size_t()
  assert lib.pclseg_op_linear_i8_workspace(33, 7, 65, ctypes.byref(size)) == 0 and size.value >= 33 * (128 + 4)
  assert lib.pclseg_op_linear_i8_workspace(4, 7, 8192, ctypes.byref(size)) == 0 and size.value == 0      # one launch
  assert lib.pclseg_op_linear_i8_workspace(4, 7, 8193, ctypes.byref(size)) == 0 and size.value >= 4 * 8320
  assert lib.pclseg_op_linear_i8_workspace(5, 7, 0, ctypes.byref(size)) == -2
  assert lib.pclseg_op_linear_i8_workspace(5, 7, 8, None) == -1
  for rows, classes in ((1, 20), (1, 2048), (1, 32768), (1 << 20, 50000)):
    assert lib.pclseg_op_label_logprobs_workspace(rows, classes, 5, ctypes.byref(size)) == 0 and size.value == 0
  assert lib.pclseg_op_label_logprobs_workspace(1, 1 << 20, 5, ctypes.byref(size)) == 0 and size.value > 0
  assert lib.pclseg_op_label_logprobs_workspace(0, 1 << 20, 5, ctypes.byref(size)) == 0 and size.value == 0
  assert lib.pclseg_op_label_logprobs_workspace(1, 0, 5, ctypes.byref(size)) == -2
  assert lib.pclseg_op_label_logprobs_workspace(1, 5, 65, ctypes.byref(size)) == -1


SCORE = dict(logits=P, dtype=0, rows=2, classes=4, stride=4, labels=P, label_bytes=4, allowed=None, allowed_stride=0, top_k=0,
             logprob=P, entropy=P, lse=P, top_ids=None, top_logprobs=None, workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize("change,code,word", [
  (dict(dtype=9), -1, "dtype"), (dict(rows=-1), -2, "rows"), (dict(classes=0), -2, "classes"), (dict(classes=1 << 31), -2, "classes"),
  (dict(classes=(1 << 30) + 1, stride=1 << 31), -2, "classes"), (dict(rows=(1 << 40) + 1), -2, "rows"),
  (dict(stride=3), -2, "stride"), (dict(top_k=65), -1, "top_k"), (dict(top_k=-1), -1, "top_k"), (dict(logits=None), -1, "NULL"),
  (dict(label_bytes=2), -1, "int32"), (dict(labels=P + 2), -1, "misaligned"), (dict(labels=None), -1, "labels"),
  (dict(top_k=2), -1, "top_ids"), (dict(allowed=P, allowed_stride=3), -2, "mask"), (dict(logits=P + 2), -1, "misaligned"),
  (dict(classes=1 << 20, stride=1 << 20, rows=1), -1, "workspace"),
])
def test_label_logprobs_refuses(change, code, word):
  _refused("pclseg_op_label_logprobs", list({**SCORE, **change}.values()), code, word)


GRAD = dict(logits=P, dtype=0, rows=2, classes=4, stride=4, labels=P, label_bytes=4, allowed=None, allowed_stride=0, lse=P,
            entropy=P, d_logprob=P, d_entropy=P, top_ids=P, d_top=P, top_k=2, grad=P + 1024, grad_stride=4, stream=None)


@pytest.mark.parametrize("change,code,word", [
  (dict(dtype=9), -1, "dtype"), (dict(stride=3), -2, "stride"), (dict(grad_stride=3), -2, "gradient stride"),
  (dict(d_logprob=None, d_entropy=None, d_top=None), -1, "no gradient"), (dict(labels=None), -1, "labels"),
  (dict(entropy=None), -1, "entropy"), (dict(top_ids=None), -1, "top_ids"), (dict(top_k=0), -1, "top_ids"),
  (dict(lse=None), -1, "NULL"), (dict(grad=None), -1, "NULL"), (dict(grad=P), -1, "overlaps"), (dict(grad=P + 28), -1, "overlaps"),
  (dict(grad=P + 1025), -1, "misaligned"), (dict(rows=1 << 40), -2, "blocks"),
])
def test_label_logprobs_grad_refuses(change, code, word):
  if "rows" in change:
    change = dict(change, grad=P + (1 << 46))      # 2^40 rows of 16 bytes: do not overlap
  _refused("pclseg_op_label_logprobs_grad", list({**GRAD, **change}.values()), code, word)


FAR = P + (1 << 46)      # a gradient that does not overlap the logits


# a launch has fewer than 2^32 threads along an axis: a size that does not fit, for each way of sharing rows out
@pytest.mark.parametrize("fn,call", [
  ("pclseg_op_quantize_rows", dict(QUANT, rows=(1 << 29) + 1)),                                     # 8 lanes a row
  ("pclseg_op_quantize_rows", dict(QUANT, rows=(1 << 26) + 1, cols=257, x_stride=257)),             # 64
  ("pclseg_op_quantize_rows", dict(QUANT, rows=1 << 24, cols=2049, x_stride=2049)),                 # 256
  ("pclseg_op_matmul_i8", dict(MATMUL, m=1, n=1 << 27, y_stride=1 << 27)),                          # 512 threads, 16 channels
  ("pclseg_op_matmul_i8", dict(MATMUL, m=1 << 30, k=65)),                                           # 256 threads, 64 rows
  ("pclseg_op_matmul_i8", dict(MATMUL, m=1 << 31)),                                                 # 256 threads, 128 rows
  ("pclseg_op_matmul_i8", dict(MATMUL, m=1 << 30, n=256, y_stride=256)),                            # 256 threads, 128x128
  ("pclseg_op_linear_i8", dict(LINEAR, m=1, n=1 << 27, y_stride=1 << 27)),
  ("pclseg_op_linear_i8", dict(LINEAR, m=(1 << 29) + 1, workspace_bytes=1 << 40)),                  # the quantisation
  ("pclseg_op_linear_i8", dict(LINEAR, m=1 << 28, n=1024, y_stride=1024, workspace_bytes=1 << 40)),   # the product
  ("pclseg_op_label_logprobs", dict(SCORE, rows=(1 << 32) + 1)),                                    # a thread a row
  ("pclseg_op_label_logprobs", dict(SCORE, rows=(1 << 29) + 1, classes=33, stride=33)),             # 8 lanes
  ("pclseg_op_label_logprobs", dict(SCORE, rows=1 << 26, classes=2049, stride=2049)),               # a wave
  ("pclseg_op_label_logprobs_grad", dict(GRAD, rows=1 << 40, grad=FAR)),
  ("pclseg_op_label_logprobs_grad", dict(GRAD, rows=1 << 24, classes=4096, stride=4096, grad=FAR, grad_stride=4096)),
])
def test_more_than_a_launch_holds_is_refused(fn, call):
  _refused(fn, list(call.values()), -2, "launch")


def test_no_rows_is_no_work():
  lib = E.load_library()
  assert lib.pclseg_op_quantize_rows(*{**QUANT, "rows": 0, "x": None}.values()) == 0
  assert lib.pclseg_op_matmul_i8(*{**MATMUL, "m": 0, "a": None, "y": None}.values()) == 0
  assert lib.pclseg_op_linear_i8(*{**LINEAR, "m": 0, "x": None, "y": None, "workspace": None}.values()) == 0
  assert lib.pclseg_op_label_logprobs(*{**SCORE, "rows": 0, "logits": None}.values()) == 0
  assert lib.pclseg_op_label_logprobs_grad(*{**GRAD, "rows": 0, "logits": None}.values()) == 0


def test_every_entry_point_is_behind_the_exception_barrier():
  src = open(os.path.join(os.path.dirname(E.__file__), "csrc", "pclseg_ops.hip")).read()
  body = src[src.index('extern "C" {'):src.index('}  // extern "C"')]
  defs = re.findall(r"^int (pclseg_\w+)\([^;{]*\)( try)? \{$", body, re.M)
  assert len(defs) == 7 and all(t for _, t in defs) and body.count("OP_CATCH") == 7


# ---- the Python layer: with on_device answered as if host tensors were device tensors, every refusal comes before a launch

@pytest.fixture
def host_as_device(monkeypatch):
  monkeypatch.setattr(E, "on_device", lambda x: True)


def _rows8(n=3, k=8):
  return ops.Int8Rows(torch.zeros((n, 64), dtype=torch.int8), torch.ones(n), k)


def test_host_tensors_are_refused():
  x = torch.zeros(2, 8)
  for call in (lambda: ops.quantize_rows(x), lambda: ops.linear_i8(x, _rows8()), lambda: ops.label_logprobs(x),
               lambda: ops.label_logprobs_grad(x, None, x[:, 0]), lambda: ops.Int8Rows.from_codes(x.to(torch.int8), x[:, 0])):
    with pytest.raises(ValueError, match="on the device"):
      call()


def test_python_layer_refuses(host_as_device):
  x, i = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
  v = torch.zeros(2)
  bad = [
    lambda: ops.quantize_rows(x.double()), lambda: ops.quantize_rows(torch.zeros(())), lambda: ops.quantize_rows(torch.zeros(2, 0)),
    lambda: ops.Int8Rows.from_codes(x, v), lambda: ops.Int8Rows.from_codes(x.to(torch.int8), torch.zeros(3)),
    lambda: ops.Int8Rows.from_kernel(torch.zeros(3, 3, 8, 4)),
    lambda: ops.Int8Rows(torch.zeros((3, 8), dtype=torch.int8), torch.ones(3), 8), lambda: ops.Int8Rows(torch.zeros(3, 64), torch.ones(3), 8),
    lambda: ops.Int8Rows(torch.zeros((3, 64), dtype=torch.int8), torch.ones(2), 8),
    lambda: ops.Int8Rows(torch.zeros((3, 64), dtype=torch.int8), torch.ones(3), 65),
    lambda: ops.Int8Rows(torch.zeros((3, 128), dtype=torch.int8)[:, :64], torch.ones(3), 8),
    lambda: ops.linear_i8(x, _rows8(k=9)), lambda: ops.linear_i8(x, x), lambda: ops.linear_i8(x, _rows8(), act="tanh"),
    lambda: ops.linear_i8(x, _rows8(), bias=torch.zeros(4)), lambda: ops.linear_i8(x, _rows8(), bias=torch.zeros(3).half()),
    lambda: ops.linear_i8(x, _rows8(), residual=torch.zeros(2, 4)), lambda: ops.linear_i8(x, _rows8(), residual=torch.zeros(2, 3).half()),
    lambda: ops.linear_i8(x, _rows8(), out_dtype=torch.float64), lambda: ops.matmul_i8(_rows8(), _rows8(k=9)),
    lambda: ops.matmul_i8(x, _rows8()),
    lambda: ops.label_logprobs(x.long()), lambda: ops.label_logprobs(torch.zeros(2, 0)), lambda: ops.label_logprobs(x, i[:1]),
    lambda: ops.label_logprobs(x, i.float()), lambda: ops.label_logprobs(x, i, top_k=65),
    lambda: ops.label_logprobs(x, i, top_k=-1), lambda: ops.label_logprobs(x, allowed=torch.ones(7, dtype=torch.bool)),
    lambda: ops.label_logprobs(x, allowed=torch.ones(8)), lambda: ops.label_logprobs_grad(x, i, v),
    lambda: ops.label_logprobs_grad(x, None, v, d_logprob=v), lambda: ops.label_logprobs_grad(x, i, v, d_entropy=v),
    lambda: ops.label_logprobs_grad(x, i, v, d_top=v), lambda: ops.label_logprobs_grad(x, i, v[:1], d_logprob=v),
    lambda: ops.label_logprobs_grad(x, i, v, d_logprob=v.double()),
    lambda: ops.label_logprobs_grad(x, i, v, d_top=torch.zeros(2, 3), top_ids=torch.zeros((2, 2), dtype=torch.int32)),
    lambda: ops.label_logprobs_grad(x, i, v, d_top=torch.zeros(2, 2), top_ids=torch.zeros((2, 2), dtype=torch.int64)),
  ]
  for n, call in enumerate(bad):
    with pytest.raises(ValueError):
      call()
      pytest.fail("call %d was accepted" % n)


def test_calls_run_with_the_tensors_device_current(monkeypatch):
  """With several devices the launch is made under the tensors' device, and the caller's is restored."""
  class Dev:
    index = 1
  state = {"current": 0, "during": None}

  class Guard:
    def __init__(self, dev):
      self.dev = dev

    def __enter__(self):
      self.was, state["current"] = state["current"], self.dev.index

    def __exit__(self, *a):
      state["current"] = self.was

  def launch(x, stream):
    state["during"] = (state["current"], x, stream)
    return 0
  monkeypatch.setattr(ops, "_several_devices", lambda: True)
  monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
  monkeypatch.setattr(torch.cuda, "device", Guard)
  monkeypatch.setattr(E, "stream_handle", lambda dev: 77)
  ops._call(Dev, launch, 5)
  assert state == {"current": 0, "during": (1, 5, 77)}
  state["current"] = 1
  ops._call(Dev, launch, 6)
  assert state == {"current": 1, "during": (1, 6, 77)}


# ---- outputs that share memory with inputs: one block stores while another still reads
BIG = (ctypes.c_uint8 * (1 << 16))()
Q = (ctypes.addressof(BIG) + 255) // 256 * 256


@pytest.mark.parametrize("m", [1, 2, 32, 33, 70])
@pytest.mark.parametrize("x,x_stride,y,y_stride,y_dtype", [
  (Q, 8, Q, 8, 0),                        # in place
  (Q, 8, Q + 16, 8, 0),                   # y begins inside x's first row
  (Q + 16, 8, Q, 8, 0),
  (Q, 20, Q + 28, 20, 0),                 # rows of one buffer, x in columns 0..7, y in 7..14
  (Q + 28, 20, Q, 20, 0),
  (Q, 20, Q + 56, 20, 0),                 # y in columns 14..21: its end is the next row's x (one row: behind it)
  (Q, 20, Q, 40, 1),                      # 16-bit outputs over float inputs, the same bytes a row
  (Q, 8, Q + 12, 9, 0),                   # different strides
])
def test_linear_i8_refuses_an_output_over_its_input(m, x, x_stride, y, y_stride, y_dtype):
  if m == 1 and y == Q + 56:
    pytest.skip("one row: y lies behind x")
  change = dict(x=x, x_stride=x_stride, y=y, y_stride=y_stride, y_dtype=y_dtype, m=m, n=8, workspace=P, workspace_bytes=1 << 20)
  _refused("pclseg_op_linear_i8", list({**LINEAR, **change}.values()), -1, "overlaps x")


@pytest.mark.parametrize("fn,base", [("pclseg_op_matmul_i8", MATMUL), ("pclseg_op_linear_i8", dict(LINEAR, x=P + 2048, k=8))])
@pytest.mark.parametrize("residual,stride", [(Q + 4, 3), (Q + 36, 3), (Q, 4), (Q + 28, 9), (Q + 4, 9)])
def test_products_refuse_a_residual_partly_under_the_output(fn, base, residual, stride):
  """y may be the residual; shifted or with another stride an element's residual may be gone before it is read."""
  change = dict(m=4, n=3, y=Q, y_stride=9 if stride == 9 else 3, residual=residual, residual_stride=stride)
  change["y_dtype" if "y_dtype" in base else "dtype"] = 0
  if residual == Q + 36:
    change.update(y=Q + 32)
  if (residual, stride) == (Q + 28, 9):
    change.update(n=8, y=Q)               # columns 7..14 of the residual under columns 0..7 of y
  _refused(fn, list({**base, **change}.values()), -1, "overlaps the residual")


def test_quantize_rows_refuses_codes_over_its_input():
  for x, q in ((Q, Q), (Q + 32, Q), (Q, Q + 8), (Q, Q + 56)):
    _refused("pclseg_op_quantize_rows", list({**QUANT, "x": x, "q": q}.values()), -1, "codes overlap")


@pytest.mark.parametrize("grad", [Q + 12, Q + 20, Q + 8, Q - 12 + 32])
def test_label_logprobs_grad_refuses_a_gradient_over_the_logits(grad):
  """Rows of 4 floats, 8 apart: a gradient that begins anywhere but 16 bytes into the logits' rows shares some of them."""
  _refused("pclseg_op_label_logprobs_grad", list({**GRAD, "logits": Q, "stride": 8, "grad": grad, "grad_stride": 8, "rows": 5}.values()),
           -1, "overlaps the logits")


def test_label_logprobs_grad_far_strides():
  """Strides whose products with the rows pass 64 bits are compared as they are: this gradient lies 2^46 bytes behind the logits'
  first row, inside their range."""
  _refused("pclseg_op_label_logprobs_grad", list({**GRAD, "stride": 1 << 60, "rows": 1 << 39, "grad": FAR, "grad_stride": 4}.values()),
           -1, "overlaps the logits")


GRAD_EX = dict(logits=P, dtype=0, rows=2, classes=4, stride=4, labels=P, label_bytes=4, allowed=None, allowed_stride=0, lse=P,
               entropy=P, logprob=P, top_ids=P, top_logprobs=P, d_logprob=P, d_entropy=P, d_top=P, top_k=2, grad=P + 1024, grad_stride=4,
               stream=None)


@pytest.mark.parametrize("change,code,word", [
  (dict(dtype=9), -1, "dtype"), (dict(stride=3), -2, "stride"), (dict(grad_stride=3), -2, "gradient stride"),
  (dict(d_logprob=None, d_entropy=None, d_top=None), -1, "no gradient"), (dict(labels=None), -1, "labels"),
  (dict(labels=None, d_logprob=None), -1, "logprob needs labels"), (dict(entropy=None), -1, "entropy"), (dict(top_ids=None), -1, "top_ids"),
  (dict(top_ids=None, d_top=None), -1, "top_logprobs needs"), (dict(top_k=0, d_top=None), -1, "top_logprobs needs"), (dict(lse=None), -1, "NULL"),
  (dict(grad=P), -1, "overlaps"), (dict(grad=P + 1025), -1, "misaligned"), (dict(rows=1 << 40, grad=FAR), -2, "blocks"),
])
def test_label_logprobs_grad_ex_refuses(change, code, word):
  _refused("pclseg_op_label_logprobs_grad_ex", list({**GRAD_EX, **change}.values()), code, word)


def test_entry_points_of_the_second_block_are_behind_the_exception_barrier():
  src = open(os.path.join(os.path.dirname(E.__file__), "csrc", "pclseg_ops.hip")).read()
  defs = re.findall(r"^int (pclseg_\w+)\([^;{]*\)( try)? \{$", src, re.M)
  assert len(defs) == 8 and all(t for _, t in defs) and src.count("} OP_CATCH\n") == 8


def test_python_layer_refuses_log_probabilities_without_names(host_as_device):
  x, i, v = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
  two, ids = torch.zeros(2, 2), torch.zeros((2, 2), dtype=torch.int32)
  for call in (lambda: ops.label_logprobs_grad(x, i, v, logprob=v),                       # no gradient arrives
               lambda: ops.label_logprobs_grad(x, None, v, entropy=v, d_entropy=v, logprob=v),
               lambda: ops.label_logprobs_grad(x, i, v, entropy=v, d_entropy=v, logprob=v[:1]),
               lambda: ops.label_logprobs_grad(x, i, v, entropy=v, d_entropy=v, logprob=v.double()),
               lambda: ops.label_logprobs_grad(x, i, v, entropy=v, d_entropy=v, top_logprobs=two),
               lambda: ops.label_logprobs_grad(x, i, v, entropy=v, d_entropy=v, top_ids=ids, top_logprobs=two[:, :1])):
    with pytest.raises(ValueError):
      call()


def test_inputs_that_require_a_gradient_are_warned_of(host_as_device, recwarn):
  """Results carry no history: a call that would drop a gradient says so, and nothing is said where none is recorded.  (Each call
  is refused for something else afterwards, so that none is launched.)"""
  x, p, i = torch.zeros(2, 8), torch.zeros(2, 8, requires_grad=True), torch.zeros(3, dtype=torch.int32)
  b = torch.zeros(4, requires_grad=True)
  calls = [("x", lambda t: ops.quantize_rows(t.double())), ("x", lambda t: ops.linear_i8(t, _rows8(k=9))),
           ("logits", lambda t: ops.label_logprobs(t, i)), ("logits", lambda t: ops.label_logprobs_grad(t, i, x[:, 0]))]
  for name, call in calls:
    with pytest.warns(UserWarning, match=name + " requires a gradient, but") as seen, pytest.raises(ValueError):
      call(p)
    assert seen[0].filename == __file__
    with torch.no_grad(), pytest.raises(ValueError):
      call(p)
    for quiet in (x, p.detach()):
      with pytest.raises(ValueError):
        call(quiet)
  for call in (lambda: ops.linear_i8(x, _rows8(), bias=b), lambda: ops.matmul_i8(_rows8(), _rows8(), bias=b)):
    with pytest.warns(UserWarning, match="outside of autograd"), pytest.raises(ValueError):
      call()
  assert not recwarn.list


def test_workspace_of_few_rows_goes_by_the_channels_too():
  """One launch (no workspace) quantises every row in every block of 16 channels: not beyond 512 blocks or 2^14 items of 512
  elements in all, but for one or two rows of 4096 columns and more."""
  lib, size = E.load_library(), ctypes.c_size_t()

  def need(m, n, k):
    assert lib.pclseg_op_linear_i8_workspace(m, n, k, ctypes.byref(size)) == 0
    return size.value
  for m, n, k in ((1, 8192, 1024), (16, 8192, 1024), (32, 4096, 1024), (8, 4096, 4096), (1, 1 << 20, 4096), (2, 131072, 16384)):
    assert need(m, n, k) == 0
  for m, n, k in ((1, 8193, 1024), (16, 8193, 1024), (32, 4097, 1024), (8, 4097, 4096), (1, 1 << 20, 4095), (3, 16384, 4096), (33, 16, 16)):
    assert need(m, n, k) == m * (lib.pclseg_i8_row_bytes(k) + 4)
