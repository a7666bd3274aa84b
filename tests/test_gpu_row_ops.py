"""Row operators on the MI355X against float64 restatements of their formulas (tensors are copied to the CPU first).

Tolerances count roundings: u = 2^-24 for each float32 operation, half a step of the output type for the final one
(finfo(t).eps / 2 relative).  `chain` is the longest chain of additions a sum can pass through."""
import math

import pytest
import torch

from pclsegmentation_amd import ops

pytestmark = [pytest.mark.gpu, pytest.mark.needs_hip]
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def half_step(t):
  return torch.finfo(t).eps / 2


def tiny(t):
  return torch.finfo(t).smallest_normal * torch.finfo(t).eps      # half a subnormal step and more


def rnd(seed, *shape):
  return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def close(got, want, bound):
  """|got - want| <= bound elementwise; the same infinities and NaNs."""
  got = got.detach().cpu().double()
  assert got.shape == want.shape, (got.shape, want.shape)
  fin = torch.isfinite(want)
  assert torch.equal(torch.nan_to_num(got[~fin], nan=7e77), torch.nan_to_num(want[~fin], nan=7e77))
  excess = ((got - want).abs() - bound)[fin]
  assert excess.numel() == 0 or excess.max() <= 0, "off by %g over the bound" % excess.max()


# ---------------------------------------------------------------------------------------------- quantisation

def quant64(x):
  """codes and scales by the definition: the scale is a float32, the quotient exact to 2^-53."""
  x = x.double()
  scale = (x.abs().amax(-1).double() / 127.0).float()
  s = scale.double().unsqueeze(-1)
  q = torch.where(s > 0, torch.round(x / torch.where(s > 0, s, 1.0)), 0.0).clamp(-127, 127)
  return q.to(torch.int8), scale


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (33, 65), (7, 250), (9, 256), (4, 257), (6, 1000), (3, 2048),
                                       (3, 2049), (2, 8192), (2, 9001), (300, 16), (1, 131071)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows_is_exact(cuda, rows, cols, dtype):
  x = (rnd(rows * cols, rows, cols) * torch.exp(rnd(5, rows, 1) * 3).clamp(1e-3, 1e3)).to(dtype)
  x[0] = 0
  got = ops.quantize_rows(x.to(cuda))
  q, scale = quant64(x)
  assert torch.equal(got.scale.cpu(), scale) and torch.equal(got.codes.cpu(), q)
  assert not got.data[:, cols:].any()


def test_quantize_rows_half_steps_and_extremes(cuda):
  # a row whose maximum is 127 * 2^e has the scale 2^e: multiples of half a step are exact ties
  ties = torch.cat([torch.arange(-253, 254) / 2.0, torch.tensor([127.0, -127.0])])
  x = torch.stack([ties, ties * 2.0 ** 60, ties * 2.0 ** -100, ties * 2.0 ** -140])
  got = ops.quantize_rows(x.to(cuda))
  want = torch.round(ties).to(torch.int8)          # torch rounds halves to even
  for r in range(3):
    assert torch.equal(got.codes[r].cpu(), want)
  # a subnormal scale: the row itself is a subnormal number of steps, codes times scale stay within its half step
  assert (got.dequantize()[3].cpu() - x[3]).abs().max() <= 2.0 ** -141 + 127 * 2.0 ** -150
  x = torch.ones(5, 40)
  x[0, 3], x[1, 39], x[2, 0] = math.nan, math.inf, -math.inf
  x[3, :] = torch.finfo(F32).max
  got = ops.quantize_rows(x.to(cuda))
  assert torch.isnan(got.scale[:3]).all() and not got.codes[:3].any()
  assert (got.codes[3:] == 127).all() and torch.isfinite(got.scale[3:]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows_layouts(cuda, dtype):
  base = rnd(1, 6, 5, 40).to(dtype).to(cuda)
  for view in (base[..., 3:36], base[:, 1], base.transpose(0, 1), base[..., ::2], base[0, :1].expand(4, 40), base.permute(2, 0, 1)):
    q, scale = quant64(view.cpu().reshape(-1, view.shape[-1]))
    got = ops.quantize_rows(view)
    assert torch.equal(got.codes.cpu(), q) and torch.equal(got.scale.cpu(), scale)


# ---------------------------------------------------------------------------------------------- product

ACT64 = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "leaky": lambda v: torch.where(v > 0, v, 0.1 * v),
         "sigmoid": torch.sigmoid}


def product64(qa, sa, qb, sb, bias, act, residual):
  p = (qa.double() @ qb.double().t().contiguous()) * sa.double()[:, None] * sb.double()[None, :]
  v = p + (bias.double() if bias is not None else 0.0)
  y = ACT64[act](v)
  # float32: the int32 sum, two scales, the bias, the activation; the sigmoid has slope <= 1/4 and |v| s(1-s) <= 1/4
  bound = 4 * U * p.abs() + 2 * U * v.abs() + (8 * U if act == "sigmoid" else 0.0)
  if residual is not None:
    y = y + residual.double()
    bound = bound + U * y.abs()
  return y, bound


def check_product(got, want, bound, dtype):
  close(got, want, bound + half_step(dtype) * (want.abs() + bound) + tiny(dtype))


PRODUCTS = [  # m, n, k
  (1, 1, 1), (1, 8, 16), (1, 4096, 512), (2, 17, 63), (5, 100, 65), (16, 33, 128), (17, 257, 1000), (32, 16, 4096), (33, 70, 300),
  (64, 511, 257), (65, 1, 5), (65, 129, 64), (127, 300, 40), (130, 64, 129), (200, 1000, 1000), (257, 513, 384), (3000, 4100, 200),
  (4100, 3001, 64), (5000, 2600, 256), (70001, 1000, 200), (20000, 64, 50), (20001, 50, 200), (13000, 33, 64), (9000, 1100, 384), (9000, 3000, 640),
  (1, 40, 131071), (70, 40, 20000)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_i8(cuda, m, n, k):
  act = ["none", "relu", "leaky", "sigmoid"][(m + n) % 4]
  dtype = TYPES[(m + k) % 3]
  g = torch.Generator().manual_seed(m * 7 + n * 3 + k)
  qa = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
  qb = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
  sa, sb = torch.rand(m, generator=g) * 1e-2 + 1e-4, torch.rand(n, generator=g) * 1e-2 / k ** 0.5 + 1e-6
  bias = rnd(1, n).float() if n % 2 else None
  residual = rnd(2, m, n).to(dtype) if m % 2 else None
  a, b = ops.Int8Rows.from_codes(qa.to(cuda), sa.to(cuda)), ops.Int8Rows.from_codes(qb.to(cuda), sb.to(cuda))
  got = ops.matmul_i8(a, b, bias=None if bias is None else bias.to(cuda), act=act,
                      residual=None if residual is None else residual.to(cuda), out_dtype=dtype)
  assert got.dtype == dtype
  want, bound = product64(qa, sa, qb, sb, bias, act, residual)
  check_product(got, want, bound, dtype)


def test_matmul_i8_sums_are_exact(cuda):
  """The largest sum int32 holds, unit scales, float32 out: one rounding."""
  k = 131071
  a = torch.full((3, k), -128, dtype=torch.int8)
  b = torch.full((70, k), -128, dtype=torch.int8)
  b[1] = 127
  a[2, ::2] = 127
  ra = ops.Int8Rows.from_codes(a.to(cuda), torch.ones(3, device=cuda))
  rb = ops.Int8Rows.from_codes(b.to(cuda), torch.ones(70, device=cuda))
  want = (a.double() @ b.double().t().contiguous())
  assert torch.equal(ops.matmul_i8(ra, rb).cpu(), want.float())
  assert torch.equal(ops.matmul_i8(rb, ra).cpu(), want.t().float())


@pytest.mark.parametrize("m,k,n", [(1, 333, 260), (7, 333, 260), (48, 333, 260), (100, 333, 260), (600, 333, 260),
                                   # up to 32 rows of together 64 stretches of 512 columns take one launch
                                   (1, 1, 1), (2, 64, 5), (3, 65, 16), (4, 4097, 33), (4, 8192, 20), (4, 8193, 20), (1, 32768, 40),
                                   (1, 32769, 9), (5, 1, 3), (16, 2048, 7), (16, 2049, 7), (17, 1536, 40), (17, 1537, 40), (31, 1000, 300),
                                   (32, 1024, 65), (32, 1025, 65), (33, 64, 20)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_i8(cuda, m, k, n, dtype):
  x = rnd(m, m, k).to(dtype)
  w = ops.quantize_rows((rnd(3, n, k) * 0.05).float().to(cuda))
  bias, residual = rnd(4, n).float(), rnd(5, m, n).to(dtype)
  got = ops.linear_i8(x.to(cuda), w, bias=bias.to(cuda), act="leaky", residual=residual.to(cuda))
  q, s = quant64(x)
  want, bound = product64(q, s, w.codes.cpu(), w.scale.cpu(), bias, "leaky", residual)
  check_product(got, want, bound, dtype)
  # the same numbers in two calls, another output type, batched axes, strided rows
  assert torch.equal(ops.matmul_i8(ops.quantize_rows(x.to(cuda)), w, bias=bias.to(cuda), act="leaky",
                                   residual=residual.to(cuda), out_dtype=dtype), got)
  plain = ops.linear_i8(x.to(cuda), w, out_dtype=F32)
  check_product(plain, *product64(q, s, w.codes.cpu(), w.scale.cpu(), None, "none", None), F32)
  wide = torch.zeros(m, k + 9, dtype=dtype, device=cuda)
  wide[:, 5:5 + k] = x.to(cuda)
  assert torch.equal(ops.linear_i8(wide[:, 5:5 + k], w, out_dtype=F32), plain)
  assert torch.equal(ops.linear_i8(x.to(cuda).view(1, m, 1, k), w, out_dtype=F32), plain.view(1, m, 1, n))


def test_linear_i8_bad_rows_stay_in_their_row(cuda):
  x = rnd(1, 70, 100).float()
  x[3, 5], x[60, 99] = math.nan, math.inf
  w = ops.quantize_rows(rnd(2, 40, 100).float().to(cuda))
  for rows in (70, 8):
    y = ops.linear_i8(x[:rows].to(cuda), w, act="relu").cpu()
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[3] = True
    if rows > 60:
      bad[60] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


def test_linear_i8_matches_a_1x1_convolution(cuda):
  """Int8Rows.from_kernel takes the Keras kernel of op_conv2d: the two layers agree to the 8-bit codes' half steps."""
  import numpy as np
  from pclsegmentation_amd import engine as E
  n, h, w, cin, cout = 1, 4, 16, 64, 32
  x = rnd(1, n, h, w, cin).float().to(cuda)
  kernel = (rnd(2, 1, 1, cin, cout) * 0.1).float()
  bias = rnd(3, cout).float()
  y = torch.empty((n, h, w, cout), dtype=F32, device=cuda)
  E.op_conv2d(x, n, h, w, cin, kernel.numpy(), 1, bias.numpy(), None, "leaky", None, y, math="f32")
  torch.cuda.synchronize()
  weight = ops.Int8Rows.from_kernel(kernel.to(cuda))
  got = ops.linear_i8(x, weight, bias=bias.to(cuda), act="leaky")
  sx = x.abs().amax(-1, keepdim=True).double() / 127
  sw = kernel.abs().amax(2).double().view(1, 1, 1, cout).to(cuda) / 127
  # each factor is off by half a step: sum |x| sw/2 + |w| sx/2 + sx sw / 4
  bound = x.abs().double().sum(-1, keepdim=True) * sw / 2 + (sx / 2) * kernel.abs().double().sum(2).view(1, 1, 1, cout).to(cuda)
  bound = (bound + cin * sx * sw / 4).cpu() * (1 + 1e-4) + 1e-5
  close(got, y.cpu().double(), bound)
  assert isinstance(np.asarray(bias), np.ndarray)


# ---------------------------------------------------------------------------------------------- log probabilities

def score64(x, labels, top_k, allowed):
  x = x.double()
  v = x.shape[-1]
  if allowed is not None:
    x = torch.where(allowed.bool(), x, torch.full((), -math.inf, dtype=torch.float64))
  m = x.amax(-1)
  bad = torch.isnan(x).any(-1) | (m == math.inf)
  empty = (m == -math.inf) & ~bad
  mm = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
  z = x - mm[:, None]
  e = torch.exp(z)
  s = e.sum(-1)
  lse = mm + torch.log(s)
  p = torch.where(empty[:, None], torch.zeros_like(e), e / s[:, None])
  zz = torch.where(p > 0, z, torch.zeros_like(z))
  h = torch.where(empty, torch.zeros_like(s), torch.log(s) - (p * zz).sum(-1))
  nan = torch.full_like(lse, math.nan)
  out = {"x": x, "p": p, "empty": empty, "bad": bad, "a": (p * zz.abs()).sum(-1), "b": (p * zz * zz).sum(-1), "m": mm,
         "logs": torch.log(s)}
  if labels is not None:
    lab = labels.long()
    known = (lab >= 0) & (lab < v)
    at = x.gather(1, lab.clamp(0, v - 1)[:, None])[:, 0]
    # (x - m) - ln s: x - lse would lose ln s beside the extremes of the types
    lp = torch.where(at == -math.inf, at, (at - mm) - torch.log(s))
    out["logprob"] = torch.where(known, torch.where(bad, nan, lp), torch.zeros_like(lse))
  out["entropy"] = torch.where(bad, nan, h)
  out["lse"] = torch.where(bad, nan, torch.where(empty, torch.full_like(lse, -math.inf), lse))
  xs = torch.where(bad[:, None], torch.full_like(x, -math.inf), x) + 0.0
  order = torch.sort(xs, dim=-1, descending=True, stable=True)
  k = min(top_k, v)
  ids, best = order.indices[:, :k], order.values[:, :k]
  gone = best == -math.inf
  ids = torch.where(gone, -1, ids).to(torch.int32)
  best = torch.where(gone, best, (best - mm[:, None]) - torch.log(s)[:, None])
  best = torch.where(bad[:, None], nan[:, None], best)
  pad = top_k - k
  if pad:
    ids = torch.cat([ids, torch.full((len(ids), pad), -1, dtype=torch.int32)], 1)
    best = torch.cat([best, torch.full((len(ids), pad), -math.inf, dtype=torch.float64)], 1)
    best = torch.where(bad[:, None], nan[:, None], best)
  out["top_ids"], out["top_logprobs"] = ids, best
  return out


def check_score(got, ref, v, top_k):
  chain = 64 + 32 * (v // 8192 + 1)
  a, b, logs, m = ref["a"], ref["b"], ref["logs"].abs(), ref["m"].abs()
  a, b, logs = [torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (a, b, logs)]
  rel_s = U * (chain + 4 + 4 * a)
  log_s = rel_s + 2 * U * logs                                      # logf
  lse, h = [torch.nan_to_num(ref[t], 0.0, 0.0, 0.0).abs() for t in ("lse", "entropy")]
  close(got.lse, ref["lse"], log_s + U * (m + lse))
  close(got.entropy, ref["entropy"], log_s + rel_s * a + U * (4 * b + (8 + chain) * a + h))
  if got.logprob is not None:
    lp = torch.nan_to_num(ref["logprob"], 0.0, 0.0, 0.0).abs()
    close(got.logprob, ref["logprob"], log_s + U * (lp + logs) + U * lp)      # |x - M| <= |logprob| + |ln S|
  if top_k:
    assert torch.equal(got.top_ids.cpu(), ref["top_ids"])
    lp = torch.nan_to_num(ref["top_logprobs"], 0.0, 0.0, 0.0).abs()
    close(got.top_logprobs, ref["top_logprobs"], log_s[:, None] + U * (lp + logs[:, None]) + U * lp)
  else:
    assert got.top_ids is None and got.top_logprobs is None


def labels_for(rows, v, seed, dtype=torch.int32):
  return torch.randint(-2, v + 2, (rows,), generator=torch.Generator().manual_seed(seed)).to(dtype)


SCORES = [(1, 1, 1), (5, 2, 3), (300, 3, 2), (257, 8, 8), (1000, 20, 3), (513, 31, 5), (70, 32, 32), (65, 33, 2), (40, 64, 64), (33, 100, 4),
          (31, 256, 20), (17, 257, 3), (9, 511, 32), (10, 513, 1), (6, 1031, 64), (5, 2048, 20), (7, 2049, 20), (3, 4097, 5), (4, 8193, 64),
          (2, 30001, 20), (600, 2500, 3), (1, 131072, 20), (3, 131071, 32), (1, 300000, 64), (3, 131073, 7), (2, 1000003, 20), (40, 40001, 20), (33, 131072, 3), (9000, 60, 9), (300, 56, 40), (600, 9001, 33), (1000, 5000, 0),
          (2100, 4099, 6), (2100, 2049, 0), (2, 9000, 0), (50, 77, 0)]


@pytest.mark.parametrize("rows,v,top_k", SCORES)
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs(cuda, rows, v, top_k, dtype):
  x = (rnd(v + rows, rows, v) * 3).to(dtype)
  x[0] += 50
  labels = labels_for(rows, v, v, torch.int64 if rows % 2 else torch.int32)
  got = ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=top_k)
  check_score(got, score64(x, labels, top_k, None), v, top_k)
  again = ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=top_k)
  assert all(u is None or torch.equal(u, w) for u, w in zip(got, again))


@pytest.mark.parametrize("rows,v,top_k", [(40, 5, 3), (40, 20, 3), (20, 33, 7), (20, 300, 64), (20, 2000, 9), (12, 2100, 20), (12, 20003, 33)])
@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_masks(cuda, rows, v, top_k, per_row, dtype):
  """Excluded classes hold whatever: NaN, infinities, the type's extremes.  Rows with nothing, one, or a few left."""
  g = torch.Generator().manual_seed(v)
  x = (rnd(v, rows, v) * 2).to(dtype)
  allowed = torch.rand((rows, v) if per_row else (v,), generator=g) < 0.6
  if per_row:
    allowed[0] = False
    allowed[1] = False
    allowed[1, v - 1] = True
    allowed[2] = torch.arange(v) < 2
  else:
    allowed[0], allowed[v - 1] = False, True
  full = allowed.expand(rows, v)
  fill = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max])
  junk = fill[torch.randint(0, 5, (rows, v), generator=g)].to(dtype)
  x = torch.where(full, x, junk)
  labels = labels_for(rows, v, 3)
  ref = score64(x, labels, top_k, full)
  got = ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=top_k, allowed=allowed.to(cuda))
  check_score(got, ref, v, top_k)
  # the same mask as bytes, as a strided view, and its effect spelled as logits of -inf
  wide = torch.zeros((rows, 2 * v + 3), dtype=torch.uint8, device=cuda)
  wide[:, 1:1 + v] = full.to(cuda)
  same = ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=top_k, allowed=wide[:, 1:1 + v])
  inf = ops.label_logprobs(torch.where(full, x, torch.full((), -math.inf, dtype=dtype)).to(cuda), labels.to(cuda), top_k=top_k)
  for other in (same, inf):
    assert all(torch.equal(u, w) for u, w in zip(got, other))


@pytest.mark.parametrize("v", [7, 32, 40, 500, 2048, 2049, 20000, 131072])
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_odd_rows(cuda, v, dtype):
  """Equal logits (ids ascend), rising, falling, the lowest value throughout, all -inf, signed zeros, far outliers, NaN, +inf."""
  lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
  ramp = torch.arange(v, dtype=torch.float64) * (8.0 / v)
  rows = [torch.full((v,), 1.5), ramp, -ramp, torch.full((v,), lo), torch.full((v,), -math.inf), torch.zeros(v),
          torch.where(torch.arange(v) == v // 2, 1e4, 0.0), torch.where(torch.arange(v) == 1, lo, 0.5), torch.full((v,), hi),
          torch.where(torch.arange(v) == v - 1, math.nan, 1.0), torch.where(torch.arange(v) == 0, math.inf, 1.0),
          torch.where(torch.arange(v) % 3 == 1, -math.inf, 2.0), torch.where(torch.arange(v) == v - 1, 1.0, -math.inf)]
  x = torch.stack([r.double() for r in rows]).to(dtype)
  x[5, ::2] = -0.0
  labels = torch.arange(len(x), dtype=torch.int32) % v
  k = min(v, 40)
  ref = score64(x, labels, k, None)
  check_score(ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=k), ref, v, k)
  # one row at a time takes the split path of long rows
  for r in range(len(x)):
    one = {n: t[r:r + 1] for n, t in ref.items()}
    check_score(ops.label_logprobs(x[r:r + 1].to(cuda), labels[r:r + 1].to(cuda), top_k=k), one, v, k)


@pytest.mark.parametrize("width", [90, 25, 3001])
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_layouts(cuda, width, dtype):
  base = rnd(1, 6, 4, width).to(dtype).to(cuda)
  for view in (base[..., 3:width - 4], base[:, 2], base.transpose(0, 1), base[..., ::3], base[:1, :1].expand(5, 2, width), base[0, 0]):
    v = view.shape[-1]
    flat = view.cpu().reshape(-1, v)
    labels = labels_for(len(flat), v, 1).view(view.shape[:-1])
    got = ops.label_logprobs(view, labels.to(cuda), top_k=2)
    assert got.lse.shape == view.shape[:-1] and got.top_ids.shape == view.shape[:-1] + (2,)
    ref = score64(flat, labels.reshape(-1), 2, None)
    check_score(ops.LabelLogprobs(*[t.reshape(-1, *t.shape[view.dim() - 1:]) for t in got]), ref, v, 2)
  assert ops.label_logprobs(base).logprob is None
  none = ops.label_logprobs(base[:0], top_k=3)      # no rows
  assert none.lse.shape == (0, 4) and none.top_ids.shape == (0, 4, 3)


# ---------------------------------------------------------------------------------------------- gradient

def grad64(ref, labels, lse, entropy, d_lp, d_h, ids, d_top, dtype):
  x = ref["x"]
  v = x.shape[1]
  lse = torch.where(ref["empty"], torch.zeros_like(lse), lse)
  z = torch.where(x == -math.inf, torch.zeros_like(x), x - lse[:, None])
  p = torch.where(x == -math.inf, torch.zeros_like(x), torch.exp(z))
  named, named_abs = torch.zeros_like(p), torch.zeros_like(p)
  if d_lp is not None:
    lab = labels.long()
    known = (lab >= 0) & (lab < v)
    g = torch.where(known, d_lp, torch.zeros_like(d_lp))
    named.scatter_add_(1, lab.clamp(0, v - 1)[:, None], g[:, None])
    named_abs.scatter_add_(1, lab.clamp(0, v - 1)[:, None], g.abs()[:, None])
  k = 1
  if d_top is not None:
    g = torch.where(ids >= 0, d_top, torch.zeros_like(d_top))
    named.scatter_add_(1, ids.long().clamp(min=0), g)
    named_abs.scatter_add_(1, ids.long().clamp(min=0), g.abs())
    k += ids.shape[1]
  w, w_abs = named.sum(1, keepdim=True), named_abs.sum(1, keepdim=True)
  ge = d_h[:, None] if d_h is not None else torch.zeros_like(w)
  h = (entropy if d_h is not None else torch.zeros_like(lse))[:, None]
  grad = named - p * (w + ge * (z + h))
  # p: x - lse, the product with log2 e, the exponential; the bracket: k + 1 sums and one fma
  inner = w_abs + ge.abs() * (z.abs() + (h - lse[:, None]).abs() + lse[:, None].abs())
  bound = p * inner * U * (3 * z.abs() + k + 10) + U * (k + 1) * (named_abs + p * inner)
  off = (x == -math.inf) | ref["empty"][:, None]
  grad, bound = [torch.where(off, torch.zeros_like(t), t) for t in (grad, bound)]
  bound = bound + half_step(dtype) * (grad.abs() + bound) + tiny(dtype) + 2.0 ** -140
  return grad, bound


@pytest.mark.parametrize("rows,v,top_k", [(1, 1, 1), (700, 20, 3), (300, 3, 2), (9, 33, 40), (64, 100, 5), (33, 1031, 32), (5, 4099, 20),
                                          (3, 8192, 2), (3, 8193, 3), (2, 50001, 20), (1, 131072, 64), (2000, 2, 1), (300, 4099, 2), (40001, 20, 3),
                                          (9000, 129, 1)])
@pytest.mark.parametrize("parts", ["lp", "h", "top", "lp+h+top"])
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_grad(cuda, rows, v, top_k, parts, dtype):
  x = (rnd(v, rows, v) * 2).to(dtype)
  g = torch.Generator().manual_seed(v)
  allowed = torch.rand((rows, v), generator=g) < 0.8 if v > 1 and rows % 2 else None
  if allowed is not None:
    allowed[0] = False
    x[1 % rows][~allowed[1 % rows]] = math.nan
  labels = labels_for(rows, v, 9, torch.int64 if v % 2 else torch.int32)
  ref = score64(x, labels, top_k, allowed)
  dev = lambda t: None if t is None else t.to(cuda)
  fwd = ops.label_logprobs(dev(x), dev(labels), top_k=top_k, allowed=dev(allowed))
  d_lp = rnd(1, rows).float() if "lp" in parts else None
  d_h = rnd(2, rows).float() if "h" in parts.split("+") else None
  d_top = rnd(3, rows, top_k).float() if "top" in parts else None
  got = ops.label_logprobs_grad(dev(x), dev(labels), fwd.lse, d_logprob=dev(d_lp), entropy=fwd.entropy, d_entropy=dev(d_h),
                                top_ids=fwd.top_ids, d_top=dev(d_top), allowed=dev(allowed))
  assert got.dtype == dtype and got.shape == x.shape
  d64 = [None if t is None else t.double() for t in (d_lp, d_h, d_top)]
  want, bound = grad64(ref, labels, fwd.lse.cpu().double(), fwd.entropy.cpu().double(), d64[0], d64[1], fwd.top_ids.cpu(), d64[2], dtype)
  close(got, want, bound)


def test_label_logprobs_grad_against_differences(cuda):
  """Central differences of the float64 loss; h = 1e-4 leaves a truncation below 1e-7 and a cancellation below 1e-10."""
  rows, v, k = 4, 37, 3
  x = rnd(1, rows, v)
  labels = torch.tensor([0, 36, -1, 5], dtype=torch.int32)
  a, b, c = rnd(2, rows), rnd(3, rows), rnd(4, rows, k)
  allowed = torch.rand((rows, v), generator=torch.Generator().manual_seed(5)) < 0.8
  allowed[:, 0], allowed[:, 36], allowed[:, 5] = True, True, True
  x = x.float().double()
  ids = score64(x, labels, k, allowed)["top_ids"]

  def loss(y):
    r = score64(y, labels, k, allowed)
    top = (y - r["lse"][:, None]).gather(1, ids.long())
    return (r["logprob"] * a + r["entropy"] * b).sum() + (top * c).sum()

  h, want = 1e-4, torch.zeros_like(x)
  for r in range(rows):
    for j in range(v):
      if allowed[r, j]:
        d = torch.zeros_like(x)
        d[r, j] = h
        want[r, j] = (loss(x + d) - loss(x - d)) / (2 * h)
  dev = lambda t: t.float().to(cuda)
  fwd = ops.label_logprobs(dev(x), labels.to(cuda), top_k=k, allowed=allowed.to(cuda))
  got = ops.label_logprobs_grad(dev(x), labels.to(cuda), fwd.lse, d_logprob=dev(a), entropy=fwd.entropy, d_entropy=dev(b),
                                top_ids=fwd.top_ids, d_top=dev(c), allowed=allowed.to(cuda))
  assert (got.cpu().double() - want).abs().max() <= 1e-5        # 40 roundings of terms up to 5


@pytest.mark.parametrize("v", [2, 3, 20, 32])
@pytest.mark.parametrize("lead", [2.0, 6.0, 11.0, 30.0])
def test_decided_rows_keep_their_significant_bits(cuda, v, lead):
  """ln p of a class that has nearly everything is -(the rest): relative, not absolute, to 2^-24.  z = x - M is a few roundings
  relative to the exponent, 3 u |z| in a term; the sums and the logarithm add 40 u.  The gradient of the label likewise."""
  x = -rnd(v, 5, v).abs().float()
  x[:, 1] = lead
  labels = torch.ones(5, dtype=torch.int32)
  got = ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=1)
  z = x.double() - x.double()[:, 1:2]
  z[:, 1] = -math.inf
  rest = torch.exp(z).sum(1)
  logp = -torch.log1p(rest)
  rel = U * (3 * (lead + 5) + 40)
  close(got.logprob, logp, rel * logp.abs())
  close(got.top_logprobs[:, 0], logp, rel * logp.abs())
  entropy = -logp + (torch.exp(z) * torch.where(z > -math.inf, -z, torch.zeros_like(z))).sum(1) / (1 + rest)
  close(got.entropy, entropy, 2 * rel * entropy)
  g = torch.full((5,), -0.75)
  lse = got.lse.cpu().double()
  grad = ops.label_logprobs_grad(x.to(cuda), labels.to(cuda), got.lse, d_logprob=g.to(cuda))[:, 1]
  want = 0.75 * torch.expm1(x.double()[:, 1] - lse)
  close(grad, want, 16 * U * want.abs())


def test_label_logprobs_grad_names_that_coincide(cuda):
  """The label among the alternatives, and the same alternative named twice: their gradients add up."""
  x = rnd(1, 3, 50).float()
  labels = torch.tensor([4, 4, 9], dtype=torch.int32)
  ids = torch.tensor([[4, 4, 7], [1, 2, -1], [9, 9, 9]], dtype=torch.int32)
  d_lp, d_top = rnd(2, 3), rnd(3, 3, 3)
  ref = score64(x, labels, 3, None)
  got = ops.label_logprobs_grad(x.to(cuda), labels.to(cuda), ref["lse"].float().to(cuda), d_logprob=d_lp.float().to(cuda),
                                top_ids=ids.to(cuda), d_top=d_top.float().to(cuda))
  want, bound = grad64(ref, labels, ref["lse"].float().double(), None, d_lp.float().double(), None, ids, d_top.float().double(), F32)
  close(got, want, bound)


def test_label_logprobs_grad_layouts(cuda):
  base = rnd(1, 6, 4, 90).to(BF16).to(cuda)
  for view in (base[..., 3:60], base[:, 2], base.transpose(0, 1), base[..., ::3]):
    v = view.shape[-1]
    labels = labels_for(view[..., 0].numel(), v, 1).view(view.shape[:-1]).to(cuda)
    fwd = ops.label_logprobs(view, labels)
    one = torch.ones((), device=cuda).expand(view.shape[:-1])       # the gradient of a sum: a broadcast scalar
    got = ops.label_logprobs_grad(view, labels, fwd.lse, d_logprob=one)
    want = ops.label_logprobs_grad(view.contiguous(), labels.contiguous(), fwd.lse.contiguous(), d_logprob=one.contiguous())
    assert got.shape == view.shape and torch.equal(got, want)


# ---------------------------------------------------------------------------------------------- together

def chain(x, w, bias, labels, allowed, d_lp, d_h):
  logits = ops.linear_i8(x, w, bias=bias)
  fwd = ops.label_logprobs(logits, labels, top_k=5, allowed=allowed)
  grad = ops.label_logprobs_grad(logits, labels, fwd.lse, d_logprob=d_lp, entropy=fwd.entropy, d_entropy=d_h, allowed=allowed)
  return (logits,) + tuple(fwd) + (grad,)


def chain_inputs(cuda, m, k, v, seed, dtype=BF16):
  x = rnd(seed, m, k).to(dtype).to(cuda)
  w = ops.quantize_rows((rnd(seed + 1, v, k) * 0.1).float().to(cuda))
  allowed = (torch.arange(v) != 0).to(cuda)
  return [x, w, rnd(seed + 2, v).float().to(cuda), labels_for(m, v, seed).to(cuda), allowed, rnd(seed + 3, m).float().to(cuda),
          rnd(seed + 4, m).float().to(cuda)]


@pytest.mark.parametrize("m,k,v", [(1, 256, 40000), (130, 100, 20), (70, 512, 1000)])
def test_a_layer_its_scores_and_their_gradient(cuda, m, k, v):
  a = chain_inputs(cuda, m, k, v, 11)
  logits, lp, h, lse, ids, tops, grad = chain(*a)
  x, w, bias, labels, allowed, d_lp, d_h = [t.cpu() if torch.is_tensor(t) else t for t in a]
  q, s = quant64(x)
  check_product(logits, *product64(q, s, w.codes.cpu(), w.scale.cpu(), bias, "none", None), BF16)
  ref = score64(logits.cpu(), labels, 5, allowed.expand(m, v))
  check_score(ops.LabelLogprobs(lp, h, lse, ids, tops), ref, v, 5)
  want, bound = grad64(ref, labels, lse.cpu().double(), h.cpu().double(), d_lp.double(), d_h.double(), None, None, BF16)
  close(grad, want, bound)


@pytest.mark.parametrize("m,k,v", [(1, 256, 40000), (300, 100, 20)])
def test_captured_and_replayed(cuda, m, k, v):
  """Two graphs of the chain, replayed in turn with new inputs and eager calls between: every replay equals the eager result."""
  side = torch.cuda.Stream(cuda)
  static = [chain_inputs(cuda, m, k, v, 20), chain_inputs(cuda, m, k, v, 30)]
  chain(*static[0])
  torch.cuda.synchronize()
  graphs, outs = [], []
  for s in static:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
      outs.append(chain(*s))
    graphs.append(g)
  for it in range(4):
    for n in (0, 1):
      fresh = chain_inputs(cuda, m, k, v, 40 + 7 * it + n)
      for dst, src in zip(static[n], fresh):
        if torch.is_tensor(dst):
          dst.copy_(src)
        else:
          dst.data.copy_(src.data)
          dst.scale.copy_(src.scale)
    want = [chain(*s) for s in static]
    torch.cuda.synchronize()
    for g in graphs:
      g.replay()
    torch.cuda.synchronize()
    for n in (0, 1):
      for got, ref in zip(outs[n], want[n]):
        assert torch.equal(got, ref)


def test_two_streams_at_once(cuda):
  ins = [chain_inputs(cuda, 1, 256, 40000, 50), chain_inputs(cuda, 90, 256, 3001, 60)]
  want = [chain(*i) for i in ins]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream(cuda), torch.cuda.Stream(cuda)]
  got = [[], []]
  for _ in range(5):
    for n in (0, 1):
      with torch.cuda.stream(streams[n]):
        got[n].append(chain(*ins[n]))
  torch.cuda.synchronize()
  for n in (0, 1):
    for run in got[n]:
      assert all(torch.equal(a, b) for a, b in zip(run, want[n]))


def test_only_the_rows_are_written(cuda):
  """The C entry points write the outputs' rows and nothing beside them."""
  from pclsegmentation_amd import engine as E
  lib, stream = E.load_library(), E.stream_handle(cuda)
  for m, n, k in ((3, 21, 70), (70, 33, 130), (3000, 1030, 70), (700, 4000, 200)):
    w = ops.quantize_rows(rnd(1, n, k).float().to(cuda))
    x = ops.quantize_rows(rnd(2, m, k).float().to(cuda))
    y = torch.full((m + 2, n + 7), 5.0, device=cuda)
    E.check(lib.pclseg_op_matmul_i8(x.data.data_ptr(), x.scale.data_ptr(), w.data.data_ptr(), w.scale.data_ptr(), m, n, k, None, 0,
                                    None, 0, y.data_ptr(), n + 7, 0, stream))
    assert (y[m:] == 5).all() and (y[:, n:] == 5).all() and torch.equal(y[:m, :n], ops.matmul_i8(x, w))
    # the residual may be the output
    res = rnd(4, m, n).float().to(cuda)
    want, z = ops.matmul_i8(x, w, act="relu", residual=res), torch.full((m + 2, n + 7), 5.0, device=cuda)
    z[:m, :n] = res
    E.check(lib.pclseg_op_matmul_i8(x.data.data_ptr(), x.scale.data_ptr(), w.data.data_ptr(), w.scale.data_ptr(), m, n, k, None, 1,
                                    z.data_ptr(), n + 7, z.data_ptr(), n + 7, 0, stream))
    assert torch.equal(z[:m, :n], want) and (z[m:] == 5).all() and (z[:, n:] == 5).all()
  for m, v in ((5, 21), (3, 9001)):
    logits = rnd(3, m, v).float().to(cuda)
    labels = labels_for(m, v, 1).to(cuda)
    fwd = ops.label_logprobs(logits, labels)
    d = torch.ones(m, device=cuda)
    grad = torch.full((m + 1, v + 5), 5.0, device=cuda)
    E.check(lib.pclseg_op_label_logprobs_grad(logits.data_ptr(), 0, m, v, v, labels.data_ptr(), 4, None, 0, fwd.lse.data_ptr(), None,
                                              d.data_ptr(), None, None, None, 0, grad.data_ptr(), v + 5, stream))
    assert (grad[m:] == 5).all() and (grad[:, v:] == 5).all()
    assert torch.equal(grad[:m, :v], ops.label_logprobs_grad(logits, labels, fwd.lse, d_logprob=d))


def test_offsets_beyond_32_bits(cuda):
  """More than 2^31 elements in the logits, the gradient, and an output of the product: the last rows are the ones looked at."""
  rows, v = 65540, 32769
  x = torch.zeros((rows, v), dtype=BF16, device=cuda)
  x[-3:] = rnd(1, 3, v).to(BF16).to(cuda)
  labels = torch.full((rows,), 32768, dtype=torch.int32, device=cuda)
  got = ops.label_logprobs(x, labels, top_k=3)
  tail = ops.LabelLogprobs(*[t[-3:] for t in got])
  ref = score64(x[-3:].cpu(), labels[-3:].cpu(), 3, None)
  check_score(tail, ref, v, 3)
  assert (got.lse[:-3] - math.log(v)).abs().max() <= 64 * U * 11 and (got.top_ids[:-3] == torch.arange(3, device=cuda, dtype=torch.int32)).all()
  d = torch.ones(rows, device=cuda)
  grad = ops.label_logprobs_grad(x, labels, got.lse, d_logprob=d)
  want, bound = grad64(ref, labels[-3:].cpu(), got.lse[-3:].cpu().double(), None, d[-3:].cpu().double(), None, None, None, BF16)
  close(grad[-3:], want, bound)
  del x, grad, got
  m, n, k = 132000, 16385, 40
  a = torch.zeros((m, k), dtype=BF16, device=cuda)
  a[-3:] = rnd(2, 3, k).to(BF16).to(cuda)
  w = ops.quantize_rows(rnd(3, n, k).float().to(cuda))
  y = ops.linear_i8(a, w)
  q, s = quant64(a[-3:].cpu())
  check_product(y[-3:], *product64(q, s, w.codes.cpu(), w.scale.cpu(), None, "none", None), BF16)
  assert not y[:-3].any()


# ---------------------------------------------------------------------------------------------- in the evaluation

def test_label_likelihood_tracker(cuda):
  from pclsegmentation_amd import eval as ev
  n, h, w, nc, none = 2, 5, 9, 11, 10
  logits = (rnd(1, n, h, w, nc) * 3).float()
  label = torch.randint(-1, nc + 1, (n, h, w), generator=torch.Generator().manual_seed(2)).to(torch.int32)
  m = ev.LabelLikelihood(nc, none)
  assert m.result() == (0.0, 0.0)
  m.update_state(label[:1], logits[:1])                                     # accumulates; host tensors or device tensors
  m.update_state(label[1:].to(cuda), logits[1:].to(cuda))
  x, lab = logits.double().reshape(-1, nc)[:, :none], label.reshape(-1).long()
  keep = (lab >= 0) & (lab < none)
  logp = torch.log_softmax(x, -1)
  nll = -logp[keep].gather(1, lab[keep][:, None]).mean()
  entropy = -(logp.exp() * logp)[keep].sum(-1).mean()
  got = m.result()
  assert abs(got[0] - nll) <= 1e-5 and abs(got[1] - entropy) <= 1e-5      # about 100 roundings of values up to 10
  m.reset_state()
  assert m.result() == (0.0, 0.0)
  with pytest.raises(ValueError):
    m.update_state(label, logits[..., :5])


def test_evaluation_prints_the_likelihood(cuda, tmp_path, capsys):
  import numpy as np
  import os
  from pclsegmentation_amd import eval as ev
  from pclsegmentation_amd import load_model_config
  g = np.load(os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "model_ssv2_real_32x240.npz"))
  d = tmp_path / "data" / "val"
  d.mkdir(parents=True)
  samples = np.stack([np.concatenate([g["raw"][i], g["labels"][i][..., None].astype(np.float32)], -1) for i in range(2)])
  for i in range(2):
    np.save(str(d / ("s%d.npy" % i)), samples[i].astype(np.float64))
  args = ["-d", str(tmp_path / "data"), "-i", "val", "-m", "squeezesegv2", "-n", "squeezesegv2"]
  plain = ev.main(args)
  assert "NLL" not in capsys.readouterr().out
  with_nll = ev.main(args + ["--likelihood"])
  out = capsys.readouterr().out
  assert plain[3] == with_nll[3] and np.array_equal(plain[0], with_nll[0])      # the other metrics keep their values
  got = [float(v) for v in (out.split("NLL:")[1].split()[0], out.split("Entropy:")[1].split()[0])]
  mc, model = load_model_config("squeezesegv2", "squeezesegv2")
  model.init_weights(4321)
  preds, mask, logits = model.predict_raw(samples[..., :5], return_mask=True, return_logits=True)      # host arrays
  none = mc.CLASSES.index("None")
  lab = torch.from_numpy(np.where(mask, g["labels"], none).astype(np.int64)).reshape(-1)
  x = torch.from_numpy(np.asarray(logits)).double().reshape(-1, mc.NUM_CLASS)
  x[:, none] = -math.inf
  logp = torch.log_softmax(x, -1)
  keep = (lab != none) & (lab >= 0) & (lab < mc.NUM_CLASS)
  p = torch.where(logp > -math.inf, logp.exp() * logp, torch.zeros_like(logp))
  want = [-logp[keep].gather(1, lab[keep][:, None]).mean().item(), -p[keep].sum(-1).mean().item()]
  assert all(abs(a - b) <= 1e-4 for a, b in zip(got, want))      # logits of two runs of the network agree to about 1e-5
  assert torch.equal(torch.from_numpy(np.asarray(preds)), torch.from_numpy(np.asarray(model.predict_raw(samples[..., :5]))))


@pytest.mark.parametrize("m", [1, 32, 33, 300])
def test_linear_i8_rows_side_by_side(cuda, m):
  """Input, residual and output as columns of one buffer share no element; a residual may be the output."""
  from pclsegmentation_amd import engine as E
  lib, stream = E.load_library(), E.stream_handle(cuda)
  k, n = 100, 40
  w = ops.quantize_rows(rnd(1, n, k).float().to(cuda))
  buf = rnd(2, m, k + 2 * n + 3).float().to(cuda)
  x, res = buf[:, :k].contiguous(), buf[:, k:k + n].contiguous()
  want = ops.linear_i8(x, w, residual=res)
  work = torch.empty(m * 132, dtype=torch.uint8, device=cuda)
  ld = buf.shape[1]
  call = lambda r, y: E.check(lib.pclseg_op_linear_i8(buf.data_ptr(), 0, ld, w.data.data_ptr(), w.scale.data_ptr(), m, n, k, None, 0,
                                                      r, ld, y, ld, 0, work.data_ptr(), work.numel(), stream))
  tail = buf[:, k + 2 * n:].clone()
  call(buf[:, k:].data_ptr(), buf[:, k + n:].data_ptr())
  assert torch.equal(buf[:, k + n:k + 2 * n], want)
  call(buf[:, k:].data_ptr(), buf[:, k:].data_ptr())
  assert torch.equal(buf[:, k:k + n], want) and torch.equal(buf[:, :k], x) and torch.equal(buf[:, k + 2 * n:], tail)


@pytest.mark.parametrize("rows,v", [(1, 20), (5, 21), (300, 20), (3, 9001)])
def test_label_logprobs_grad_beside_the_logits(cuda, rows, v):
  """The logits and their gradient as the two halves of one buffer's rows share no element."""
  from pclsegmentation_amd import engine as E
  buf = torch.full((rows, 2 * v + 3), 5.0, device=cuda)
  buf[:, 1:1 + v] = rnd(1, rows, v).float().to(cuda)
  logits, labels, d = buf[:, 1:1 + v].contiguous(), labels_for(rows, v, 1).to(cuda), torch.ones(rows, device=cuda)
  fwd = ops.label_logprobs(logits, labels)
  E.check(E.load_library().pclseg_op_label_logprobs_grad(
    buf[:, 1:].data_ptr(), 0, rows, v, 2 * v + 3, labels.data_ptr(), 4, None, 0, fwd.lse.data_ptr(), None, d.data_ptr(), None, None,
    None, 0, buf[:, 1 + v:].data_ptr(), 2 * v + 3, E.stream_handle(cuda)))
  assert torch.equal(buf[:, 1 + v:1 + 2 * v], ops.label_logprobs_grad(logits, labels, fwd.lse, d_logprob=d))
  assert torch.equal(buf[:, 1:1 + v], logits) and (buf[:, 0] == 5).all() and (buf[:, 1 + 2 * v:] == 5).all()


@pytest.mark.parametrize("rows,v", [(2100, 131072), (40, 1 << 20), (1, 1 << 20), (300, 40000)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_rows_of_like_terms(cuda, rows, v, dtype):
  """Terms that are all alike round the same way at every addition: the bound counts 32 of a lane's piece, 4 for the pieces
  however many they are, 6 + 6 of the lanes and blocks, and none in proportion to the row's length.  The first 512 classes give
  every lane an element above the others, whose terms are then no powers of two."""
  j = torch.arange(v, dtype=torch.float64)
  kinds = torch.stack([torch.where((j < 512) & (j % 4 == 0), 0.0, -5.0), torch.full((v,), 1.25, dtype=torch.float64),
                       torch.where(j % 2 == 0, -3.0, -3.5) + 5.0 * (j < 512) * (j % 4 == 0),
                       torch.where(j == 7, 4.0, -4.0)])
  kinds = kinds[:min(rows, 4)]
  ref = score64(kinds, None, 0, None)
  x = kinds.to(dtype).to(cuda).repeat((rows + len(kinds) - 1) // len(kinds), 1)[:rows]
  got = ops.label_logprobs(x)
  which = torch.arange(rows) % len(kinds)
  a, b, logs, m, lse, h = [ref[t].abs()[which] for t in ("a", "b", "logs", "m", "lse", "entropy")]
  rel_s = U * (48 + 4 + 4 * a)
  close(got.lse, ref["lse"][which], rel_s + 2 * U * logs + U * (m + lse))
  close(got.entropy, ref["entropy"][which], rel_s + 2 * U * logs + rel_s * a + U * (4 * b + (8 + 48) * a + h))


@pytest.mark.parametrize("rows,v", [(5, 32), (5, 33), (9, 200), (5, 513), (5, 1031), (5, 2048), (5, 2049), (1, 4099), (3, 30001), (40, 40001), (1, 131072),
                                    (2100, 2500)])
@pytest.mark.parametrize("lead", [2.0, 6.0, 11.0, 20.0, 30.0])
@pytest.mark.parametrize("top_k", [0, 2, 20])
def test_decided_rows_of_any_length(cuda, rows, v, lead, top_k):
  """What stands beside a decided row's maximum keeps its bits for every length of a row and every place of the maximum.  z is 3
  roundings relative to the exponent, the sums 64, the logarithm and what follows 40.  Rows with an excluded class behind
  their last agree as well: the classes of a row do not choose its precision."""
  x = -rnd(v, rows, v).abs().float()
  at = (torch.arange(rows) * 7919 + 1) % v
  at[0], at[-1] = v - 1, 0 if rows > 2 else v // 2
  x[torch.arange(rows), at] = lead
  labels = at.to(torch.int32)
  z = x.double() - lead
  z[torch.arange(rows), at] = -math.inf
  rest = torch.exp(z).sum(1)
  logp = -torch.log1p(rest)
  rel = U * (3 * (lead + 5) + 40 + 64)
  entropy = -logp + (torch.exp(z) * torch.where(z > -math.inf, -z, torch.zeros_like(z))).sum(1) / (1 + rest)
  wide = torch.full((rows, v + 1), 1e30)
  wide[:, :v] = x
  for got in (ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=top_k),
              ops.label_logprobs(wide.to(cuda), labels.to(cuda), top_k=top_k, allowed=(torch.arange(v + 1) < v).to(cuda))):
    close(got.logprob, logp, rel * logp.abs())
    close(got.entropy, entropy, 2 * rel * entropy)
    if top_k:
      assert torch.equal(got.top_ids[:, 0].cpu(), labels)
      close(got.top_logprobs[:, 0], logp, rel * logp.abs())


@pytest.mark.parametrize("v", [20, 300, 5000])
@pytest.mark.parametrize("dtype", TYPES)
def test_several_maxima(cuda, v, dtype):
  """Two and more equal maxima, next to each other, in different lanes, and at the two ends of a row."""
  x = torch.full((6, v), -12.0, dtype=torch.float64)
  for r, at in enumerate(([0, 1], [0, v - 1], [v // 2, v // 2 + 1, v - 1], [v - 2, v - 1], [3], list(range(0, v, 4)))):
    x[r, at] = 5.0
  labels = torch.tensor([1, 0, v - 1, 4, 3, 0], dtype=torch.int32)
  check_score(ops.label_logprobs(x.to(dtype).to(cuda), labels.to(cuda), top_k=3), score64(x, labels, 3, None), v, 3)


@pytest.mark.parametrize("rows,v", [(5, 2), (300, 20), (5, 33), (5, 1031), (3, 9001), (1, 131072)])
@pytest.mark.parametrize("lead", [2.0, 6.0, 11.3, 20.3, 30.0])
@pytest.mark.parametrize("masked", [False, True])
def test_gradient_of_decided_rows(cuda, rows, v, lead, masked):
  """Against the float64 gradient of the logits, not of the rounded lse: with the forward pass's log probabilities the gradient of
  a class that has nearly everything is right to its own bits, whether it is the label, an alternative, or only has
  an entropy to answer for.  rel bounds ln p as in test_decided_rows_of_any_length; the other classes' p = e^(x - lse) is right to the
  rounding of lse and of three products with the exponent."""
  x = -rnd(v + 1, rows, v).abs().float()
  at = (torch.arange(rows) * 7919 + 1) % v
  x[torch.arange(rows), at] = lead
  r = torch.arange(rows)
  allowed = torch.ones(rows, v, dtype=torch.bool)
  if masked:
    allowed[:, 0] = False
    at[at == 0] = v - 1
    x[r, at] = lead
    x[:, 0] = math.nan
  z = torch.where(allowed, x.double() - lead, -math.inf)
  z[r, at] = -math.inf
  rest = torch.exp(z).sum(1)
  logp = torch.where(allowed, torch.where(z > -math.inf, z, 0.0) - torch.log1p(rest)[:, None], -math.inf)
  p = torch.exp(logp)
  lp0 = torch.where(allowed, logp, 0.0)
  h = -(p * lp0).sum(1, keepdim=True)
  q = -torch.expm1(lp0[r, at])
  rel = U * (3 * (lead + 5) + 40 + 64)
  dev = lambda t: None if t is None else t.to(cuda)
  labels = at.to(torch.int32)
  other = torch.where(at == v - 1, v - 2, v - 1).to(torch.int32)          # a label beside the decided class
  got = ops.label_logprobs(dev(x), dev(labels), top_k=1, allowed=dev(allowed))
  beside = ops.label_logprobs(dev(x), dev(other), top_k=1, allowed=dev(allowed))
  g, ge = torch.full((rows,), -0.75), torch.full((rows,), 0.25)
  kept = dict(lse=got.lse, allowed=dev(allowed))
  # the rounding of p = e^(x - lse), relative, and what the label's p and z may be off
  rp = U * (got.lse.cpu().double().abs().nan_to_num(0, 0, 0)[:, None] + 5 * lp0.abs() + 12)
  named = torch.zeros_like(p)
  named[r, at] = 1.0
  own = q[:, None] * named

  def check(grad, want, bound):
    off = ~allowed
    close(grad, torch.where(off, 0.0, want), torch.where(off, 0.0, bound) + 2.0 ** -140)

  # the label, the alternative, and both (they add up)
  want = g.double()[:, None] * torch.where(named > 0, own, -p)
  bound = 0.75 * torch.where(named > 0, (rel + 24 * U) * own, p * rp)
  a = ops.label_logprobs_grad(dev(x), dev(labels), d_logprob=dev(g), logprob=got.logprob, **kept)
  check(a, want, bound)
  b = ops.label_logprobs_grad(dev(x), None, d_top=dev(g[:, None]), top_ids=got.top_ids, top_logprobs=got.top_logprobs, **kept)
  check(b, want, bound)
  both = ops.label_logprobs_grad(dev(x), dev(labels), d_logprob=dev(g), logprob=got.logprob, d_top=dev(g[:, None]),
                                 top_ids=got.top_ids, top_logprobs=got.top_logprobs, **kept)
  check(both, 2 * want, 2 * bound)
  # a row's gradient sums to 0: to the other classes' roundings
  total = a.cpu().double().sum(1)
  assert (total.abs() <= bound.sum(1) + 2.0 ** -140).all()
  # the entropy alone, the decided class named by the label or by the alternative
  eg = -0.25 * p * (lp0 + h)
  eb = 0.25 * p * ((lp0.abs() + h) * torch.where(named > 0, 3 * rel + 12 * U, rp + 3 * rel))
  for names in (dict(labels=dev(labels), logprob=got.logprob), dict(labels=None, top_ids=got.top_ids, top_logprobs=got.top_logprobs)):
    check(ops.label_logprobs_grad(dev(x), names.pop("labels"), entropy=got.entropy, d_entropy=dev(ge), **names, **kept), eg, eb)
  # a label beside the decided class: the decided class's own gradient is -p g, the label's g (1 - p)
  if v > 2 + masked:
    named = torch.zeros_like(p)
    named[r, other.long()] = 1.0
    want = -0.75 * torch.where(named > 0, 1 - p, -p)
    check(ops.label_logprobs_grad(dev(x), dev(other), d_logprob=dev(g), logprob=beside.logprob, **kept), want,
          0.75 * (p * rp + 24 * U * named))


@pytest.mark.parametrize("rows,v,top_k", [(300, 20, 3), (9, 33, 40), (5, 4099, 20), (1, 131072, 64), (9000, 129, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_with_log_probabilities(cuda, rows, v, top_k, dtype):
  """The log probabilities of the forward pass change a gradient by roundings only; labels that are not counted, excluded labels and
  rows with nothing, or with a NaN, as without them."""
  x = (rnd(v, rows, v) * 2).to(dtype)
  allowed = torch.rand((rows, v), generator=torch.Generator().manual_seed(v)) < 0.8
  if rows > 4:
    allowed[0] = False
    allowed[3] = True
    x[3, v // 2] = math.nan
  labels = labels_for(rows, v, 9)
  ref = score64(x, labels, top_k, allowed)
  dev = lambda t: t.to(cuda)
  fwd = ops.label_logprobs(dev(x), dev(labels), top_k=top_k, allowed=dev(allowed))
  d_lp, d_h, d_top = rnd(1, rows).float(), rnd(2, rows).float(), rnd(3, rows, top_k).float()
  got = ops.label_logprobs_grad(dev(x), dev(labels), fwd.lse, d_logprob=dev(d_lp), entropy=fwd.entropy, d_entropy=dev(d_h),
                                top_ids=fwd.top_ids, d_top=dev(d_top), allowed=dev(allowed), logprob=fwd.logprob,
                                top_logprobs=fwd.top_logprobs)
  want, bound = grad64(ref, labels, fwd.lse.cpu().double(), fwd.entropy.cpu().double(), d_lp.double(), d_h.double(), fwd.top_ids.cpu(),
                       d_top.double(), dtype)
  # a name's ln p is x - lse to the roundings of both: 4 u (|lse| + |ln p| + 16) times what its p and 1 - p weigh
  lse = fwd.lse.cpu().double().abs().nan_to_num(0, 0, 0)[:, None]
  weight = d_lp.abs()[:, None] + d_top.abs().sum(1, keepdim=True) + d_h.abs()[:, None] * (ref["entropy"].nan_to_num()[:, None] + 2)
  extra = 4 * U * (lse + 20) * weight.double()
  if rows > 4:
    assert torch.isnan(got[3][allowed[3]]).all() and not got[0].any()
    keep = torch.arange(rows) != 3
    close(got[keep.to(cuda)], want[keep], (bound + extra)[keep])
  else:
    close(got, want, bound + extra)


@pytest.mark.parametrize("cols", [1, 40, 300, 3000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows_at_the_small_end(cuda, cols, dtype):
  """Rows from 2^-149 to 2^-58: the scale is the float32 nearest to max / 127, a subnormal one too, and the codes belong to it."""
  rows = 1500
  g = torch.Generator().manual_seed(cols)
  e = torch.rand(rows, 1, generator=g, dtype=torch.float64) * 91 - 149
  x = (rnd(cols, rows, cols) * torch.exp2(e)).to(dtype)
  steps = torch.arange(1, rows // 3 + 1, dtype=torch.float64)[:, None]        # maxima of 1, 2, 3, ... and 127.5, ... smallest steps
  x[::3] = torch.round(steps * rnd(5, len(steps), cols).clamp(-1, 1)).to(dtype) * 2.0 ** -149 if dtype == F32 else x[::3]
  if dtype == F32:
    x[::3, 0] = (steps[:, 0] * 2.0 ** -149).to(dtype)
  q, scale = quant64(x)
  assert (scale == 0).sum() > (0 if dtype == BF16 else 20) and ((scale > 0) & (scale < 2.0 ** -126)).sum() > 100
  got = ops.quantize_rows(x.to(cuda))
  assert torch.equal(got.scale.cpu(), scale) and torch.equal(got.codes.cpu(), q)
  w = ops.quantize_rows((rnd(2, 20, cols) * 2.0 ** 60).float().to(cuda))
  for m in (8, 33):      # one launch and two, the same rows
    y = ops.linear_i8(x[:m].to(cuda), w, out_dtype=F32)
    assert torch.equal(y, ops.matmul_i8(ops.quantize_rows(x[:m].to(cuda)), w))
    check_product(y, *product64(q[:m], scale[:m], w.codes.cpu(), w.scale.cpu(), None, "none", None), F32)


@pytest.mark.parametrize("m,n,k", [(3, 21, 70), (40, 33, 130), (70, 400, 130), (3000, 1030, 70), (700, 4000, 200), (3000, 4100, 200), (20000, 64, 50)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_product_of_far_scales(cuda, m, n, k, dtype):
  """Scales whose product is ordinary: the sum times either of them alone can pass float32's range, or fall below it."""
  g = torch.Generator().manual_seed(m + n)
  qa = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
  qb = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
  qa[0], qb[0] = 127, 127
  e = torch.tensor([-110.0, 0.0, 64.0, 120.0])[torch.randint(0, 4, (m,), generator=g)]
  sb = (torch.rand(n, generator=g) + 0.5) * 2.0 ** -110
  bias, residual = rnd(1, n).float(), rnd(2, m, n).to(dtype)
  for sign in (1, -1):
    e[0] = 120.0
    sa = (torch.rand(m, generator=g) + 0.5) * torch.exp2(sign * e)
    st = sb if sign == 1 else 1 / sb
    a, b = ops.Int8Rows.from_codes(qa.to(cuda), sa.to(cuda)), ops.Int8Rows.from_codes(qb.to(cuda), st.to(cuda))
    want, bound = product64(qa, sa, qb, st, bias, "leaky", residual)
    assert want.abs().max() < 1e38 or sign == -1
    got = ops.matmul_i8(a, b, bias=bias.to(cuda), act="leaky", residual=residual.to(cuda), out_dtype=dtype)
    top = torch.finfo(dtype).max
    # a float32 holds the product before the activation: -1.5 max is an infinity, though leaky would bring it back to -0.15 max
    before = (qa.double() @ qb.double().t().contiguous()) * sa.double()[:, None] * st.double()[None, :]
    fin = (want.abs() < top * 0.99) & (before.abs() < torch.finfo(F32).max * 0.99)
    assert torch.isinf(got.cpu()[(want.abs() > top * 1.01) | (before.abs() > torch.finfo(F32).max * 1.01)]).all()
    check_product(got[fin.to(cuda)], want[fin], bound[fin] + 2.0 ** -148, dtype)


def test_linear_i8_of_rows_near_the_end_of_float32(cuda):
  """Rows of 1e36 and more with weights that bring them back: one launch, two launches, tiles."""
  k, n = 200, 300
  w = ops.quantize_rows((rnd(2, n, k) * 1e-30).float().to(cuda))
  for m in (2, 40, 3000):
    x = (rnd(m, m, k).clamp(-3, 3) * 1e38).float()
    x[1::2] *= 1e-35
    got = ops.linear_i8(x.to(cuda), w)
    q, s = quant64(x)
    check_product(got, *product64(q, s, w.codes.cpu(), w.scale.cpu(), None, "none", None), F32)


def test_stream_handle_of_the_current_stream(cuda):
  from pclsegmentation_amd import engine as E
  side = torch.cuda.Stream(cuda)
  with torch.cuda.stream(side):
    assert {E.stream_handle(d) for d in ("cuda:0", "cuda", 0, None, torch.device("cuda"), torch.device("cuda", 0))} == {side.cuda_stream}


def test_label_likelihood_of_any_number_type(cuda):
  """NumPy's own float64 logits and int64 labels; labels that only differ from a class above bit 31 are none."""
  from pclsegmentation_amd import eval as ev
  logits = (rnd(1, 40, 7) * 3).float()
  label = torch.randint(0, 7, (40,), generator=torch.Generator().manual_seed(3))
  far = torch.cat([label, label[:5] + 2 ** 32, label[:5] - 2 ** 40])
  want = ev.LabelLikelihood(7, 6)
  want.update_state(label, logits)
  for lab, x in ((label.numpy(), logits.double().numpy()), (label.double().numpy(), logits.double()), (label.to(torch.int16), logits),
                 (far, torch.cat([logits, logits[:10]])), (far.to(cuda), torch.cat([logits, logits[:10]]).double().to(cuda))):
    got = ev.LabelLikelihood(7, 6)
    got.update_state(lab, x)
    assert got.result() == want.result()


def test_a_call_that_drops_a_gradient_runs_and_warns(cuda):
  x = rnd(1, 5, 40).float().to(cuda).requires_grad_()
  w = ops.quantize_rows(rnd(2, 7, 40).float().to(cuda))
  with pytest.warns(UserWarning, match="outside of autograd"):
    y = ops.linear_i8(x, w)
  assert not y.requires_grad and torch.equal(y, ops.linear_i8(x.detach(), w))


@pytest.mark.parametrize("m,n,k", [(9001, 3001, 640), (9000, 3000, 640), (4090, 4091, 200), (8192, 2048, 384)])
@pytest.mark.parametrize("act", ["none", "relu", "leaky", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_tiles_with_their_epilogue(cuda, m, n, k, act, dtype):
  """256x256 tiles, inside and at both edges, with bias, activation and residual together (reference on the device in float64,
  whose products of integers are exact)."""
  g = torch.Generator(device=cuda).manual_seed(m + n)
  qa = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8, device=cuda)
  qb = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8, device=cuda)
  sa, sb = torch.rand(m, generator=g, device=cuda) * 1e-2 + 1e-4, torch.rand(n, generator=g, device=cuda) * 1e-2 / k ** 0.5 + 1e-6
  bias = torch.randn(n, generator=g, device=cuda)
  wide = torch.randn(m, n + 5, generator=g, device=cuda).to(dtype)
  residual = wide[:, 2:2 + n]
  got = ops.matmul_i8(ops.Int8Rows.from_codes(qa, sa), ops.Int8Rows.from_codes(qb, sb), bias=bias, act=act, residual=residual, out_dtype=dtype)
  p = (qa.double() @ qb.double().t().contiguous()) * sa.double()[:, None] * sb.double()[None, :]
  v = p + bias.double()
  want = ACT64[act](v) + residual.double()
  bound = 4 * U * p.abs() + 2 * U * v.abs() + (8 * U if act == "sigmoid" else 0.0) + U * want.abs()
  bound = bound + half_step(dtype) * (want.abs() + bound) + tiny(dtype)
  assert got.dtype == dtype and ((got.double() - want).abs() - bound).max() <= 0


@pytest.mark.parametrize("m,k,n", [(1, 1000, 8192), (1, 1000, 8193), (2, 4096, 20000), (3, 4096, 20000), (8, 4096, 4096), (8, 4096, 4097),
                                   (17, 500, 8192), (17, 500, 8200), (32, 1024, 4097), (32, 64, 30001)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_i8_few_rows_of_many_channels(cuda, m, k, n, dtype):
  """Both sides of the rule for one launch or two."""
  x, w = rnd(m, m, k).to(dtype), ops.quantize_rows((rnd(3, n, k) * 0.05).float().to(cuda))
  bias, residual = rnd(4, n).float(), rnd(5, m, n).to(dtype)
  got = ops.linear_i8(x.to(cuda), w, bias=bias.to(cuda), act="relu", residual=residual.to(cuda))
  assert torch.equal(got, ops.matmul_i8(ops.quantize_rows(x.to(cuda)), w, bias=bias.to(cuda), act="relu", residual=residual.to(cuda),
                                        out_dtype=dtype))
  q, s = quant64(x)
  check_product(got, *product64(q, s, w.codes.cpu(), w.scale.cpu(), bias, "relu", residual), dtype)


@pytest.mark.parametrize("v", [33, 40, 257, 500, 1031, 2048])
@pytest.mark.parametrize("top_k", [0, 1, 4])
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_odd_rows_and_masks_of_short_lists(cuda, v, top_k, dtype):
  """Short lists of rows of middle length: equal logits, the lowest value throughout, all -inf, outliers, NaN, +inf, rows with
  nothing, one or a few allowed, excluded classes that hold anything, rows behind a block's last."""
  lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
  j = torch.arange(v)
  rows = [torch.full((v,), 1.5), j * (8.0 / v), -j * (8.0 / v), torch.full((v,), lo), torch.full((v,), -math.inf), torch.zeros(v),
          torch.where(j == v // 2, 1e4, 0.0), torch.where(j == 1, lo, 0.5), torch.full((v,), hi), torch.where(j == v - 1, math.nan, 1.0),
          torch.where(j == 0, math.inf, 1.0), torch.where(j % 3 == 1, -math.inf, 2.0), torch.where(j == v - 1, 1.0, -math.inf)]
  x = torch.stack([r.double() for r in rows] + list(rnd(v, 28, v) * 2)).to(dtype)
  x[5, ::2] = -0.0
  labels = (torch.arange(len(x)) * 7 % v).to(torch.int32)
  got = ops.label_logprobs(x.to(cuda), labels.to(cuda), top_k=top_k)
  ref = score64(x, labels, max(top_k, 1), None)
  if not top_k:
    ref["top_ids"] = ref["top_logprobs"] = None
  check_score(got, ref, v, top_k)
  g = torch.Generator().manual_seed(v)
  allowed = torch.rand((len(x), v), generator=g) < 0.6
  allowed[13] = False
  allowed[14] = j == v - 1
  allowed[15] = j < 2
  allowed[16] = j == 0
  fill = torch.tensor([math.nan, math.inf, -math.inf, lo, hi])
  x = torch.where(allowed, x, fill[torch.randint(0, 5, x.shape, generator=g)].to(dtype))
  for mask in (allowed, allowed[20]):
    full = mask.expand(len(x), v)
    y = torch.where(full, x, fill[torch.randint(0, 5, x.shape, generator=g)].to(dtype)) if mask.dim() == 1 else x
    got = ops.label_logprobs(y.to(cuda), labels.to(cuda), top_k=top_k, allowed=mask.to(cuda))
    check_score(got, score64(y, labels, max(top_k, 1), full), v, top_k)


@pytest.mark.parametrize("m,v", [(1, 40000), (70, 1000), (300, 20)])
def test_gradient_with_log_probabilities_captured_and_replayed(cuda, m, v):
  """The pass and its gradient with the kept log probabilities in a graph on a stream of its own, with new logits for every replay."""
  def both(x, labels, d):
    f = ops.label_logprobs(x, labels, top_k=2)
    return tuple(f) + (ops.label_logprobs_grad(x, labels, f.lse, d_logprob=d, entropy=f.entropy, d_entropy=d, top_ids=f.top_ids,
                                               logprob=f.logprob, top_logprobs=f.top_logprobs),)
  x, labels, d = rnd(1, m, v).float().to(cuda), labels_for(m, v, 2).to(cuda), rnd(3, m).float().to(cuda)
  both(x, labels, d)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph, stream=torch.cuda.Stream(cuda)):
    out = both(x, labels, d)
  for it in range(4):
    x.copy_((rnd(10 + it, m, v) * 4).float())
    x[:, it] += 25.0 * (it % 2)
    want = both(x, labels, d)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
