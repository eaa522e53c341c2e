"""Layer norm, activations kept in 8 bits, microscaled 4-bit rows and their products, against float64 restatements
(oracle/csmri_blockscale.py).

Tolerances, with u = 2^-24 (half a step of fp32, relative) and s = finfo(dtype).eps / 2 of the output's type:
  * codes, scales and restored values: equal, a power-of-two scale divides exactly and there is one rounding;
  * a sum of n fp32 terms added in chains of at most L: L u sum|terms|;
  * products of bf16 or e2m1 numbers are exact in fp32, the matrix instruction adds 32 (bf16) or 128 (e2m1) of them before
    it rounds; it may truncate, so each of its additions counts 2 u;
  * every output: s relative to its value on top."""
import ctypes as C

import pytest
import torch

import csmri_blockscale as B

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]
IDS = ['f32', 'bf16']


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def pad8(c):
  return (c + 7) // 8 * 8


def pixels(n, c, dtype, seed, scale=1.0, offset=0.0, c_real=None):
  g = torch.Generator().manual_seed(seed)
  x = (torch.randn(n, c, generator=g) * torch.exp(torch.randn(c, generator=g)) * scale + offset)
  if c_real is not None:
    x[:, c_real:] = 0
  return x.to(dtype)


def close(got, ref, tol, what=''):
  got, ref, tol = got.double().cpu(), ref.double(), tol.double()
  bad = ~((got - ref).abs() <= tol)
  assert not bad.any(), '%s: %d of %d off, worst %.3g over its bound' % (
      what, int(bad.sum()), bad.numel(), float(((got - ref).abs() / tol.clamp(min=1e-300)).nan_to_num(1e9).max()))


# ---------------------------------------------------------------------------------------------------------------------
# without a GPU: the restatements themselves, the refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_restated_formats():
  x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -5.1, 7.9, -0.24] + [0.0] * 21])
  v = B.mx4(x)[0].tolist()
  assert v[:11] == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -6.0, 6.0, 0.0]
  g = torch.Generator().manual_seed(0)
  y = torch.randn(64, 32, generator=g)
  y[:, 0] = 1.0 + torch.rand(64, generator=g)          # block maximum in [1, 2) or above
  y = y.clamp(-1.999, 1.999)
  ref = (y * 128).to(torch.float8_e4m3fn).double() / 128
  assert torch.equal(B.act8(y), ref)
  assert torch.isnan(B.act8(torch.tensor([[float('inf')] + [1.0] * 39]))).sum() == 32
  q, s = B.mx4_pack(x.repeat(3, 5)[:, :136])
  assert q.shape == (3, 128) and s.shape == (3, 16)
  assert torch.equal(B.mx4_unpack(q, s, 136), B.mx4(x.repeat(3, 5)[:, :136]))


def test_layer_norm_restatement_against_differences():
  g = torch.Generator().manual_seed(1)
  x = torch.randn(5, 9, generator=g).double()
  ga, be, G = torch.rand(9, generator=g).double() + 0.5, torch.randn(9, generator=g).double(), torch.randn(5, 9, generator=g).double()
  z, h, _, r = B.layer_norm(x, ga, be, 1e-5, 0.1)
  gate = torch.where(z > 0, 1.0, 0.1).double()
  gx, dg, db = B.layer_norm_bwd(G, h, r, gate, ga)
  f = lambda x, ga, be: float((B.layer_norm(x, ga, be, 1e-5, 0.1)[0] * G).sum())
  e = 1e-6
  for _ in range(4):
    d = torch.randn(5, 9, generator=g).double()
    assert abs((f(x + e * d, ga, be) - f(x - e * d, ga, be)) / (2 * e) - float((gx * d).sum())) < 1e-6
    d = torch.randn(9, generator=g).double()
    assert abs((f(x, ga + e * d, be) - f(x, ga - e * d, be)) / (2 * e) - float((dg * d).sum())) < 1e-6
    assert abs((f(x, ga, be + e * d) - f(x, ga, be - e * d)) / (2 * e) - float((db * d).sum())) < 1e-6


def test_entry_points_refuse_bad_arguments():
  """Status codes of the C entry points; the pointers are never followed (every call is refused, or has nothing to do)."""
  import csmri_hip
  raw = csmri_hip.lib.raw
  p = 1 << 20                                     # an aligned address that is not used
  ARG, UNS, ALI = -1, -2, -3
  ln = raw('csmri_ln_fwd')
  ok = [0, p, 16, 2 * p, 16, 4, 16, 13, p, p, 1e-5, 1.0, None, None, None, None, None]

  def ln_with(**kw):
    a = list(ok)
    for k, v in kw.items():
      a[int(k[1:])] = v
    return ln(*a)

  assert ln_with(_5=0) == 0                       # no pixels: nothing to do
  assert ln_with(_0=2) == ARG and ln_with(_6=12, _2=16) == ARG and ln_with(_7=17) == ARG and ln_with(_7=0) == ARG
  assert ln_with(_2=8) == ARG and ln_with(_4=8) == ARG and ln_with(_8=None) == ARG and ln_with(_5=-1) == ARG
  assert ln_with(_3=p) == ARG                     # z is x
  assert ln_with(_14=p) == ARG and ln_with(_14=p, _15=p) == ARG       # codes without scales, without statistics
  assert ln_with(_1=p + 4) == ALI and ln_with(_2=18) == ALI and ln_with(_12=p + 4) == ALI
  assert ln_with(_6=8200, _2=8200, _4=8200) == UNS
  bw = raw('csmri_ln_bwd')
  okb = [0, p, 16, 2 * p, 16, None, None, None, None, 0, 3 * p, 16, 4, 16, 13, p, 1e-5, 1.0, p, p, p, 0, None]

  def bw_with(**kw):
    a = list(okb)
    for k, v in kw.items():
      a[int(k[1:])] = v
    return bw(*a)

  assert bw_with(_12=0, _19=None, _20=None) == 0
  assert bw_with(_3=None) == ARG and bw_with(_5=p, _6=p, _7=p) == ARG       # neither input, both inputs
  assert bw_with(_3=None, _5=p, _6=p) == ARG                                # kept input without statistics
  assert bw_with(_3=None, _5=p, _6=p, _7=p, _17=0.1) == ARG                 # ... and no sign
  assert bw_with(_18=None) == ARG and bw_with(_20=None) == ARG and bw_with(_15=None) == ARG
  assert bw_with(_10=p) == ARG and bw_with(_15=p + 4) == ALI
  sv, rs = raw('csmri_act8_save'), raw('csmri_act8_restore')
  assert sv(0, None, 16, 0, 16, None, None, None) == 0 and rs(None, None, 0, 16, 0, None, 16, None) == 0
  assert sv(0, p, 16, 4, 12, p, p, None) == ARG and sv(3, p, 16, 4, 16, p, p, None) == ARG and sv(0, p, 8, 4, 16, p, p, None) == ARG
  assert sv(0, None, 16, 4, 16, p, p, None) == ARG and sv(0, p + 8, 16, 4, 16, p, p, None) == ALI and sv(1, p, 20, 4, 16, p, p, None) == ALI
  assert rs(p, None, 4, 16, 0, p, 16, None) == ARG and rs(p + 4, p, 4, 16, 0, p, 16, None) == ALI
  wg = raw('csmri_act8_wgrad')
  assert wg(0, p, 16, p, p, 4, 16, 12, 16, 12, 1, None, p, None, 0, None) == ARG
  assert wg(0, p, 16, p, p, 4, 16, 16, 17, 16, 1, None, p, None, 0, None) == ARG
  assert wg(0, p, 16, p, p, 4, 16, 16, 16, 16, 2, None, p, None, 0, None) == ARG          # splits without a slab
  assert wg(0, p, 16, p, p, 4, 16, 16, 16, 16, 5, p, p, None, 0, None) == ARG             # more splits than pixels
  assert wg(0, p + 4, 16, p, p, 4, 16, 16, 16, 16, 1, None, p, None, 0, None) == ALI
  assert wg(1, p, 20, p, p, 4, 16, 16, 16, 16, 1, None, p, None, 0, None) == ALI
  assert raw('csmri_act8_wgrad_splits')(0, 0, 16, 16) == 1 and raw('csmri_act8_wgrad_splits')(1, 100, 16, 16) == 1
  assert raw('csmri_act8_wgrad_slab_bytes')(3, 5, 7) == 3 * 40 * 4 and raw('csmri_act8_wgrad_slab_bytes')(1, 5, 7) == 0
  assert [raw('csmri_mx4_code_bytes')(k) for k in (0, 8, 128, 136, 4096)] == [0, 64, 64, 128, 2048]
  assert [raw('csmri_mx4_scale_bytes')(k) for k in (0, 8, 512, 520, 4096)] == [0, 16, 16, 32, 128]
  qz, dq, li = raw('csmri_mx4_quantize'), raw('csmri_mx4_dequantize'), raw('csmri_mx4_linear')
  assert qz(0, None, 16, 0, 16, None, None, None) == 0
  assert qz(0, p, 16, 4, 12, p, p, None) == ARG and qz(0, p, 16, 4, 16, None, p, None) == ARG and qz(2, p, 16, 4, 16, p, p, None) == ARG
  assert qz(0, p, 16, 4, 16, p + 8, p, None) == ALI and dq(p, p + 8, 4, 16, 0, p, 16, None) == ALI
  okl = [1, p, 16, None, 4, 16, p, p, 24, None, 1.0, p, 1, 24, None, None]

  def li_with(**kw):
    a = list(okl)
    for k, v in kw.items():
      a[int(k[1:])] = v
    return li(*a)

  assert li_with(_4=0) == 0
  assert li_with(_5=12) == ARG and li_with(_8=0) == ARG and li_with(_13=16) == ARG and li_with(_12=2) == ARG and li_with(_6=None) == ARG
  assert li_with(_0=4) == ARG                                               # codes without scales
  assert li_with(_4=200) == ARG                                             # quantised x has nowhere to go
  assert li_with(_1=p + 2) == ALI and li_with(_7=p + 1) == ALI and li_with(_13=25, _12=1) == ALI
  assert raw('csmri_mx4_linear_work_bytes')(1, 200, 136, 24) == 200 * (128 + 16) and raw('csmri_mx4_linear_work_bytes')(4, 200, 136, 24) == 0


def test_weight_gradient_refuses_rows_beyond_32_bit_offsets():
  import csmri_hip
  wg = csmri_hip.lib.raw('csmri_act8_wgrad')
  p, wide = 1 << 20, 40000000                     # 64 rows of that many codes are more than 2^31 bytes
  assert wg(1, p, 16, p, p, 64, 16, wide, 16, wide, 1, None, p, None, 0, None) == -2
  assert wg(0, p, 1 << 25, p, p, 64, 16, 16, 16, 16, 1, None, p, None, 0, None) == -2


def test_4bit_rows_beyond_their_length_are_refused():
  import csmri_hip
  raw, p, k = csmri_hip.lib.raw, 1 << 20, (1 << 24) + 8
  assert raw('csmri_mx4_quantize')(1, p, k, 4, k, p, p, None) == -1
  assert raw('csmri_mx4_dequantize')(p, p, 4, k, 1, p, k, None) == -1
  assert raw('csmri_mx4_linear')(4, p, 0, p, 400, k, p, p, 24, None, 1.0, p, 1, 24, p, None) == -1


def test_layer_norm_backward_refuses_the_sign_of_z_under_a_negative_slope():
  import csmri_hip
  bw = csmri_hip.lib.raw('csmri_ln_bwd')
  p = 1 << 20
  kept = [0, p, 16, None, 0, p, p, p, 2 * p, 16, 3 * p, 16, 4, 16, 13, p, 1e-5, -0.5, p, p, p, 0, None]
  assert bw(*kept) == -1


def test_operators_refuse_host_tensors_and_shapes():
  import csmri_hip
  ops = csmri_hip.ops
  x = torch.zeros(4, 16)
  for f in (lambda: ops.layer_norm(x, torch.ones(16), torch.zeros(16)), lambda: ops.act8_save(x), lambda: ops.mx4_quantize(x)):
    with pytest.raises(RuntimeError):
      f()
  z = lambda *s: torch.zeros(*s, dtype=torch.uint8)
  ops.Mx4(z(3, 128), z(3, 16), 136)
  for args in ((z(3, 64), z(3, 16), 136), (z(3, 128), z(3, 8), 136), (z(3, 128), z(2, 16), 136), (z(3, 128).int(), z(3, 16), 136),
               (z(128, 3).t(), z(3, 16), 136), (z(3, 128), z(3, 16), 132)):
    with pytest.raises(ValueError):
      ops.Mx4(*args)


def test_kept_forms_refuse_what_does_not_fit_their_shape():
  import csmri_hip
  ops = csmri_hip.ops
  z = lambda *s: torch.zeros(*s, dtype=torch.uint8)
  ops.Act8(z(6, 40), z(6, 2), (2, 3, 40), torch.bfloat16)
  for q, s, shape in ((z(6, 40), z(6, 1), (6, 40)), (z(6, 40), z(5, 2), (6, 40)), (z(6, 40).int(), z(6, 2), (6, 40)),
                      (z(40, 6).t(), z(6, 2), (6, 40)), (z(6, 40), z(6, 2), (7, 40)), (z(6, 40), z(6, 2), (12, 20)), (z(6, 40), z(6, 2), ())):
    with pytest.raises(ValueError):
      ops.Act8(q, s, shape, torch.bfloat16)
  for shape in ((7, 136), (6, 64), (2, 136), ()):
    with pytest.raises(ValueError):
      ops.Mx4(z(6, 128), z(6, 16), 136, shape)
  for k in (0, -8):
    with pytest.raises(ValueError):
      ops.Mx4(z(6, 0), z(6, 0), k)


# ---------------------------------------------------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------------------------------------------------
@pytest.fixture(scope='module')
def ops():
  import csmri_hip
  assert torch.cuda.is_available()
  return csmri_hip.ops


def special(x):
  """Blocks of zeros, of tiny and of huge values, a negative maximum, ties."""
  n, c = x.shape
  f = x.float()
  f[0, :] = 0
  if n > 4:
    f[1] *= 2.0 ** -110
    f[2] *= 2.0 ** 100
    f[3, 0] = -float(f[3].abs().max()) * 1.5
    f[4] = (f[4] * 8).round() / 8
  return f.to(x.dtype)


FORMAT_SIZES = [(1, 8), (1, 4096), (7, 40), (33, 104), (5, 136), (257, 32), (64, 520), (3, 2056), (1000, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('n,c', FORMAT_SIZES)
def test_kept_values_and_4bit_rows(ops, n, c, dtype):
  x = special(pixels(n, c, dtype, 100 * n + c))
  a = ops.act8_save(x.cuda())
  v, code, e = B.block_round(x, B.E4M3, 7)
  assert torch.equal(a.q.cpu().long(), code[:, :c]) and torch.equal(a.s.cpu().long(), e.long() + 127)
  for dt in DTYPES:
    assert torch.equal(ops.act8_restore(a, dt).double().cpu(), v)
  m = ops.mx4_quantize(x.cuda())
  q, s = B.mx4_pack(x)
  assert torch.equal(m.codes.cpu(), q) and torch.equal(m.scales.cpu(), s)
  for dt in DTYPES:
    assert torch.equal(ops.mx4_dequantize(m, dt).double().cpu(), B.mx4(x))


@pytest.mark.gpu
def test_formats_of_nonfinite_values_slices_and_empty_tensors(ops):
  x = pixels(6, 72, torch.float32, 3)
  x[1, 5], x[2, 40], x[3, 71] = float('nan'), float('inf'), float('-inf')
  for f, back, ref in ((ops.act8_save, ops.act8_restore, B.act8), (ops.mx4_quantize, lambda m: ops.mx4_dequantize(m, torch.float32), B.mx4)):
    got = back(f(x.cuda())).double().cpu()
    assert int(torch.isnan(got).sum()) == 32 + 32 + 8
    assert torch.equal(torch.nan_to_num(got, nan=7e7), torch.nan_to_num(ref(x), nan=7e7))
    # channel slices of a wider buffer, permuted and broadcast pixels, a pointer off the 16-byte grid
    w = pixels(30, 96, torch.bfloat16, 4).view(2, 3, 5, 96).cuda()
    for t in (w[..., 32:], w[..., 8:48], w.permute(2, 0, 1, 3), w[:1].expand(4, 3, 5, 96), w[..., 4:44], w[:, 1:2, ::2], w[:0]):
      got = back(f(t))
      assert got.shape == t.shape
      assert torch.equal(got.double().cpu().reshape(-1, t.shape[-1]), ref(t.float().cpu().reshape(-1, t.shape[-1])).to(got.dtype).double())
  with pytest.raises(ValueError):
    ops.act8_save(torch.zeros(3, 12, device='cuda'))
  with pytest.raises(TypeError):
    ops.mx4_quantize(torch.zeros(3, 16, device='cuda', dtype=torch.float16))


def ln_bounds(x, gamma, eps):
  """(|error of h| bound, mean |x|): the mean's and the variance's sums run in chains of fewer than 60 additions."""
  x = x.double()
  _, h, mean, r = B.layer_norm(x, gamma, torch.zeros_like(gamma), eps, 1.0)
  dh = r * 64 * U * (x.abs() + x.abs().mean(1, keepdim=True)) + 64 * U * h.abs()
  return dh


LN_SIZES = [(1, 1), (64, 8), (97, 64), (129, 64), (8, 1024), (4, 2048), (5, 13), (70, 100), (33, 32), (9, 512), (6, 520), (17, 1024), (5, 2000), (3, 2056), (2, 8192), (3000, 24), (4, 4100)]


@pytest.mark.gpu
@pytest.mark.parametrize('keep8', [False, True], ids=['x', 'keep8'])
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('n,c', LN_SIZES)
def test_layer_norm(ops, n, c, dtype, keep8):
  cp, eps, slope = pad8(c), 1e-5, 0.1
  x = pixels(n, cp, dtype, n + c, 2.0, 0.5, c)
  gz = pixels(n, cp, dtype, n + c + 1, 0.01, 0.0, c)
  g = torch.Generator().manual_seed(9)
  gamma, beta = 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)
  z, sv = ops.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), eps, slope, keep8)
  xr, gr = x[:, :c], gz[:, :c]
  ref, h, mean, r = B.layer_norm(xr, gamma, beta, eps, slope)
  dh = ln_bounds(xr, gamma, eps)
  s = half_step(dtype)
  close(z[:, :c], ref, s * ref.abs() + gamma.abs() * dh + 4 * U * (h * gamma).abs() + 4 * U * beta.abs(), 'z')
  assert not z[:, c:].any()
  gx, dg, db = ops.layer_norm_bwd(gz.cuda(), sv, z)
  # the backward's own gate: the sign of the z that the forward returned
  gate = torch.where(z[:, :c].float().cpu() > 0, 1.0, slope).double()
  if keep8:
    h = (B.act8(x)[:, :c] - mean) * r
    assert torch.equal(ops.act8_restore(sv.kept).double().cpu(), B.act8(x))
  rgx, rdg, rdb = B.layer_norm_bwd(gr, h, r, gate, gamma)
  gg = (gr.double() * gate).abs()
  t = gg * gamma.abs().double()
  m1 = lambda v: v.mean(1, keepdim=True)
  tol = r * (64 * U * (t + m1(t) + 2 * h.abs() * m1(t * h.abs())) + dh * m1(t * h.abs()) + h.abs() * m1(t * dh)) + 64 * U * rgx.abs()
  close(gx[:, :c], rgx, s * rgx.abs() + tol, 'gx')
  assert not gx[:, c:].any()
  L = 64 + n / 1024
  close(dg, rdg, L * U * (gg * h.abs()).sum(0) + (gg * dh).sum(0), 'dgamma')
  close(db, rdb, L * U * gg.sum(0), 'dbeta')


@pytest.mark.gpu
def test_layer_norm_strides_accumulation_and_parts(ops):
  w = pixels(2 * 5 * 7, 96, torch.bfloat16, 11).view(2, 5, 7, 96).cuda()
  gamma, beta = torch.rand(40, device='cuda') + 0.5, torch.randn(40, device='cuda')
  dense = w[..., 16:56].contiguous()
  gz = pixels(70, 96, torch.bfloat16, 12).view(2, 5, 7, 96).cuda()[..., 56:]
  z0, s0 = ops.layer_norm(dense, gamma, beta, slope=0.2)
  want = ops.layer_norm_bwd(gz.contiguous(), s0)
  for t in (w[..., 16:56], w.permute(1, 0, 2, 3)[..., 16:56].permute(1, 0, 2, 3)):
    z, sv = ops.layer_norm(t, gamma, beta, slope=0.2)
    assert torch.equal(z, z0)
    for a, b in zip(ops.layer_norm_bwd(gz, sv), want):
      assert torch.equal(a, b)
  dg, db = torch.full((40,), 2.0, device='cuda'), torch.full((40,), -1.0, device='cuda')
  ops.layer_norm_bwd(gz, s0, dgamma=dg, dbeta=db, accumulate=True)
  assert torch.equal(dg, want[1] + 2) and torch.equal(db, want[2] - 1)
  gx, none, _ = ops.layer_norm_bwd(gz, s0, want_affine=False)
  assert none is None and torch.equal(gx, want[0])
  gx, dg, db = ops.layer_norm_bwd(gz, s0, want_x=False)
  assert gx is None and torch.equal(dg, want[1]) and torch.equal(db, want[2])
  e, se = ops.layer_norm(dense[:0], gamma, beta, keep8=True)
  assert e.shape == (0, 5, 7, 40)
  gx, dg, db = ops.layer_norm_bwd(gz[:0], se)
  assert gx.shape == (0, 5, 7, 40) and not dg.any() and not db.any()
  for bad in (lambda: ops.layer_norm(dense, gamma[:39], beta), lambda: ops.layer_norm(dense, gamma.double(), beta),
              lambda: ops.layer_norm_bwd(gz[:1], s0), lambda: ops.layer_norm_bwd(gz.float(), s0),
              lambda: ops.layer_norm_bwd(gz, ops.layer_norm(dense, gamma, beta, slope=0.2, keep8=True)[1])):
    with pytest.raises((ValueError, RuntimeError)):
      bad()


@pytest.mark.gpu
@pytest.mark.parametrize('keep8', [False, True], ids=['x', 'keep8'])
@pytest.mark.parametrize('n,c,c_real', [(5, 32, 13), (130, 64, 1), (7, 1040, 520), (3, 4104, 100), (9, 136, 128)])
def test_layer_norm_of_fewer_channels_than_the_pixels_hold(ops, n, c, c_real, keep8):
  """Whole vectors of pad channels: the results are those of the pixels cut to their real ones."""
  x, gz = pixels(n, c, torch.bfloat16, n + c, c_real=c_real), pixels(n, c, torch.bfloat16, n + c + 1, c_real=c_real)
  cut = pad8(c_real)
  gamma, beta = torch.rand(c_real, generator=torch.Generator().manual_seed(1)).cuda() + 0.5, torch.full((c_real,), 0.1).cuda()
  z, sv = ops.layer_norm(x.cuda(), gamma, beta, slope=0.2, keep8=keep8)
  gx, dg, db = ops.layer_norm_bwd(gz.cuda(), sv, z)
  assert not z[:, c_real:].any() and not gx[:, c_real:].any()
  ref, h, mean, r = B.layer_norm(x[:, :c_real], gamma.cpu(), beta.cpu(), 1e-5, 0.2)
  dh = ln_bounds(x[:, :c_real], gamma.cpu(), 1e-5)
  g64, s = gamma.cpu().double(), half_step(torch.bfloat16)
  close(z[:, :c_real], ref, s * ref.abs() + g64 * dh + 4 * U * (h * g64).abs() + 4 * U * 0.1, 'z')
  # the narrower pixels take other lanes, so their sums differ by roundings: both are within the bound of the exact sums
  z1, sv1 = ops.layer_norm(x[:, :cut].contiguous().cuda(), gamma, beta, slope=0.2, keep8=keep8)
  close(z1[:, :c_real], ref, s * ref.abs() + g64 * dh + 4 * U * (h * g64).abs() + 4 * U * 0.1, 'z of the cut pixels')
  if keep8:
    h = (B.act8(x)[:, :c_real] - mean) * r
  gate = torch.where(z[:, :c_real].float().cpu() > 0, 1.0, 0.2).double()
  rgx, rdg, rdb = B.layer_norm_bwd(gz[:, :c_real], h, r, gate, gamma.cpu())
  gg = (gz[:, :c_real].double() * gate).abs()
  t, m1 = gg * g64, lambda v: v.mean(1, keepdim=True)
  tol = r * (64 * U * (t + m1(t) + 2 * h.abs() * m1(t * h.abs())) + dh * m1(t * h.abs()) + h.abs() * m1(t * dh)) + 64 * U * rgx.abs()
  close(gx[:, :c_real], rgx, s * rgx.abs() + tol, 'gx')
  close(dg, rdg, 65 * U * (gg * h.abs()).sum(0) + (gg * dh).sum(0), 'dgamma')
  close(db, rdb, 65 * U * gg.sum(0), 'dbeta')


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 64, 128, 129])
def test_layer_norm_few_rows_accumulate(ops, n):
  """One workgroup writes the affine gradients itself, several through partial rows: either adds where asked to."""
  x, gz = pixels(n, 64, torch.float32, n).cuda(), pixels(n, 64, torch.float32, n + 1).cuda()
  _, saved = ops.layer_norm(x, torch.ones(64, device='cuda'), torch.zeros(64, device='cuda'))
  _, dg, db = ops.layer_norm_bwd(gz, saved)
  a, b = torch.full((64,), 3.0, device='cuda'), torch.full((64,), -2.0, device='cuda')
  for k in (1, 2):
    want_a, want_b = a + dg, b + db
    ops.layer_norm_bwd(gz, saved, dgamma=a, dbeta=b, accumulate=True)
    assert torch.equal(a, want_a) and torch.equal(b, want_b)
  ops.layer_norm_bwd(gz, saved, dgamma=a, dbeta=b)
  assert torch.equal(a, dg) and torch.equal(b, db)


@pytest.mark.gpu
def test_layer_norm_large_offset_and_nonfinite_rows(ops):
  """An offset of 1000 times the spread costs no more than its own rounding; a NaN stays in its row."""
  x = torch.randn(6, 64, generator=torch.Generator().manual_seed(2)) + 1000
  x[4, 3] = float('nan')
  one, zero = torch.ones(64), torch.zeros(64)
  z, _ = ops.layer_norm(x.cuda(), one.cuda(), zero.cuda(), 0.0)
  z = z.cpu()
  assert torch.isnan(z[4]).all() and not torch.isnan(z[[0, 1, 2, 3, 5]]).any()
  keep = [0, 1, 2, 3, 5]
  ref = B.layer_norm(x[keep], one, zero, 0.0, 1.0)[0]
  close(z[keep], ref, U * ref.abs() + ln_bounds(x[keep], one, 0.0), 'offset')


WGRAD_SIZES = [(1, 8, 8), (31, 8, 24), (33, 40, 1), (700, 72, 136), (2048, 64, 64), (5000, 16, 200), (300, 264, 129), (4099, 128, 72), (1030, 72, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('n,cin,cout', WGRAD_SIZES)
def test_weight_gradient_from_kept_activations(ops, n, cin, cout, dtype):
  x = special(pixels(n, cin, dtype, n + cin)).float()
  if n > 4:
    x[1:3] = 1.0                                   # (finite sums: no 2^100 rows here)
  x = x.to(dtype)
  cin_real = cin - 3
  gy = pixels(n, pad8(cout), dtype, n + cout, 0.1, 0.0, cout)
  a = ops.act8_save(x.cuda())
  xr = B.act8(x)[:, :cin_real]
  g = gy.double()[:, :cout]
  dw, db = ops.act8_wgrad(a, gy.cuda(), cout, cin_real)
  assert dw.shape == (cout, cin_real) and db.shape == (cout,)
  splits = ops.lib.raw('csmri_act8_wgrad_splits')(ops.dt_of(gy), n, pad8(cout), cin)
  parts = 3 if dtype == torch.float32 else 1
  L = 2 * parts * (n / splits / 32 + 1 + 32) + splits / 64 + 8
  close(dw, g.t() @ xr, (L + 1) * U * (g.abs().t() @ xr.abs()) + 1e-300, 'dw')
  close(db, g.sum(0), (L + 1) * U * g.abs().sum(0) + 1e-300, 'db')
  w0, b0 = torch.full_like(dw, 3.0), torch.full_like(db, -2.0)
  ops.act8_wgrad(a, gy.cuda(), cout, cin_real, dw=w0, db=b0, accumulate=True)
  assert torch.equal(w0, dw + 3) and torch.equal(b0, db - 2)
  w1, none = ops.act8_wgrad(a, gy.cuda(), cout, cin_real, want_bias=False)
  assert none is None and torch.equal(w1, dw)


@pytest.mark.gpu
def test_weight_gradient_of_many_pixels_and_wide_layers(ops):
  """Large tiles (256 a side), ragged in both directions and in pixels."""
  n, cin, cout = 147456 + 77, 504, 500
  x, gy = pixels(n, cin, torch.bfloat16, 5), pixels(n, pad8(cout), torch.bfloat16, 6, 0.1, 0.0, cout)
  a = ops.act8_save(x.cuda())
  dw, db = ops.act8_wgrad(a, gy.cuda(), cout, cin)
  xr, g = B.act8(x), gy.double()[:, :cout]
  splits = ops.lib.raw('csmri_act8_wgrad_splits')(ops.dt_of(gy), n, pad8(cout), cin)
  L = 2 * (n / splits / 32 + 1 + 32) + splits / 64 + 8
  close(dw, g.t() @ xr, (L + 1) * U * (g.abs().t() @ xr.abs()), 'dw')
  close(db, g.sum(0), (L + 1) * U * g.abs().sum(0), 'db')


@pytest.mark.gpu
def test_weight_gradient_edges(ops):
  a = ops.act8_save(torch.zeros(0, 16, device='cuda'))
  dw, db = ops.act8_wgrad(a, torch.zeros(0, 24, device='cuda'))
  assert dw.shape == (24, 16) and not dw.any() and not db.any()
  x = torch.ones(2, 3, 40, 48, device='cuda', dtype=torch.bfloat16)
  wide = torch.randn(2, 3, 40, 64, device='cuda').bfloat16()
  a = ops.act8_save(x)
  d0 = ops.act8_wgrad(a, wide[..., 24:56])
  d1 = ops.act8_wgrad(a, wide[..., 24:56].contiguous())
  assert torch.equal(d0[0], d1[0]) and torch.equal(d0[1], d1[1])
  x[0, 1, 3, 40] = float('nan')                    # its block is NaN, channels 32..47, nothing else
  dw, db = ops.act8_wgrad(ops.act8_save(x), wide)
  assert torch.isnan(dw[:, 32:]).all() and not torch.isnan(dw[:, :32]).any() and not torch.isnan(db).any()
  with pytest.raises(ValueError):
    ops.act8_wgrad(a, wide[:1])


LINEAR_SIZES = [(1, 8, 1), (1, 4096, 40), (16, 136, 24), (17, 512, 33), (40, 1032, 129), (64, 128, 8), (65, 264, 130), (300, 72, 256),
                (129, 640, 128), (1000, 328, 200)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,k,n', LINEAR_SIZES)
def test_4bit_product(ops, m, k, n, dtype):
  x = pixels(m, k, dtype, m + k)
  w = torch.randn(n, k, generator=torch.Generator().manual_seed(n)) / k ** 0.5
  bias = torch.randn(n, generator=torch.Generator().manual_seed(n + 1))
  xq, wq = B.mx4(x), B.mx4(w)
  wd = ops.mx4_quantize(w.cuda())
  ksteps = (k + 127) // 128
  for b, slope, odt, src in ((bias, 0.1, None, x.cuda()), (None, 1.0, torch.float32, x.cuda()), (bias, 0.0, dtype, ops.mx4_quantize(x.cuda()))):
    y = ops.mx4_linear(src, wd, None if b is None else b.cuda(), slope, odt)
    assert y.shape == (m, pad8(n)) and y.dtype == (odt or dtype) and not y[:, n:].any()
    v = xq @ wq.t() + (0 if b is None else b.double())
    ref = torch.where(v > 0, v, slope * v)
    tol = (2 * (ksteps + 8) + 8) * U * (xq.abs() @ wq.abs().t()) + 2 * U * v.abs() + half_step(y.dtype) * ref.abs()
    close(y[:, :n], ref, tol + 1e-300, 'y')


# beside the limits between the ways of multiplying: few rows with many outputs, splits of the channels, both tiles, bands
# of tiles that end early
LIMIT_SIZES = [(3, 264, 8200), (16, 136, 16400), (64, 1024, 4096), (64, 1024, 4104), (64, 4608, 264), (100, 4232, 512), (1100, 2056, 136),
               (2200, 264, 4100), (3300, 136, 4100), (66000, 72, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize('kept', [False, True], ids=['x', 'quantised'])
@pytest.mark.parametrize('m,k,n', LIMIT_SIZES)
def test_4bit_product_beside_the_limits(ops, m, k, n, kept):
  x = pixels(m, k, torch.bfloat16, m + k)
  w = torch.randn(n, k, generator=torch.Generator().manual_seed(n)) / k ** 0.5
  bias = torch.randn(n, generator=torch.Generator().manual_seed(n + 1))
  xq, wq = B.mx4(x), B.mx4(w)
  y = ops.mx4_linear(ops.mx4_quantize(x.cuda()) if kept else x.cuda(), ops.mx4_quantize(w.cuda()), bias.cuda(), 0.25, torch.float32)
  v = xq @ wq.t() + bias.double()
  ref = torch.where(v > 0, v, 0.25 * v)
  tol = (2 * ((k + 127) // 128 + 8) + 8) * U * (xq.abs() @ wq.abs().t()) + 2 * U * v.abs() + U * ref.abs()
  close(y[:, :n], ref, tol + 1e-300, 'y')
  assert not y[:, n:].any()


@pytest.mark.gpu
def test_4bit_product_of_every_code_pair_is_exact(ops):
  """Small multiples of 1/2 with unit scales: every product and sum is a short binary fraction, so the result is exact;
  pins the operand and scale lanes of the matrix instruction at every position of 512 channels."""
  g = torch.Generator().manual_seed(7)
  t = torch.tensor(B.E2M1)
  for m in (1, 16, 48, 200):
    x, w = [t[torch.randint(0, 8, (r, 512), generator=g)] * (1 - 2 * torch.randint(0, 2, (r, 512), generator=g)) for r in (m, 72)]
    x[:, ::32], w[:, ::32] = 6.0, 4.0              # every block holds its top binade: scale 1
    sx, sw = [torch.exp2(torch.randint(-3, 4, (r, 16), generator=g).float()).repeat_interleave(32, 1) for r in (m, 72)]
    y = ops.mx4_linear((x * sx).cuda(), ops.mx4_quantize((w * sw).cuda()))
    assert torch.equal(y.double().cpu(), (x * sx).double() @ (w * sw).double().t())


@pytest.mark.gpu
def test_4bit_product_edges(ops):
  w = ops.mx4_quantize(torch.randn(24, 64, device='cuda'))
  assert ops.mx4_linear(torch.zeros(2, 0, 64, device='cuda'), w).shape == (2, 0, 24)
  wide = torch.randn(3, 5, 7, 128, device='cuda').bfloat16()
  for rows in (wide, wide[:1, :2, :3]):
    assert torch.equal(ops.mx4_linear(rows[..., 64:], w), ops.mx4_linear(rows[..., 64:].contiguous(), w))
  for m in (4, 40, 90):
    x = torch.randn(m, 64, device='cuda')
    clean = ops.mx4_linear(x, w)
    x[2, 33] = float('inf')
    y = ops.mx4_linear(x, w)
    assert torch.isnan(y[2]).all() and torch.equal(y[3:], clean[3:]) and torch.equal(y[:2], clean[:2])
  for bad in (lambda: ops.mx4_linear(torch.zeros(3, 72, device='cuda'), w), lambda: ops.mx4_linear(x, w, torch.zeros(23, device='cuda')),
              lambda: ops.mx4_linear(x, w, torch.zeros(24, device='cuda', dtype=torch.bfloat16))):
    with pytest.raises(ValueError):
      bad()


# ---- in the framework's nodes ------------------------------------------------------------------------------------------
def conv_layer(ops, cout, cin, k, dtype, pads, seed, border='zero'):
  g = torch.Generator().manual_seed(seed)
  w = torch.nn.Parameter((torch.randn(cout, cin, k, k, generator=g) / (cin * k * k) ** 0.5).cuda())
  b = torch.nn.Parameter(torch.randn(cout, generator=g).cuda())
  return ops.ConvLayer(w, b, 1, pads, border, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('k', [1, 3])
def test_convolution_keeps_its_input_in_8_bits(ops, k):
  """ConvAct with layer.keep8: same output and data gradient, the weight gradient that of the kept input -- the kernel of
  the layer's own kind on the restored values (3 x 3), the one that reads the codes (1 x 1)."""
  dt = torch.bfloat16
  x = pixels(2 * 12 * 10, 40, dt, 5).view(2, 12, 10, 40).cuda().requires_grad_(True)
  gy = pixels(240, 24, dt, 6, 0.1).view(2, 12, 10, 24).cuda()
  pads = (0, 0, 0, 0) if k == 1 else (1, 1, 1, 1)
  outs = []
  for keep in (False, True):
    layer = conv_layer(ops, 24, 40, k, dt, pads, 3)
    layer.keep8 = keep
    x.grad = None
    y = ops.ConvAct.apply(x, None, layer.weight, layer.bias, layer, 0.1, None)
    y.backward(gy)
    outs.append((y.detach(), x.grad.clone(), layer.weight.grad.clone(), layer.bias.grad.clone(), layer))
  assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
  x8 = ops.act8_restore(ops.act8_save(x.detach()))
  g = ops.act_bwd(gy, outs[1][0], 0.1)
  if k == 3:
    ref = conv_layer(ops, 24, 40, k, dt, pads, 3)
    ops.conv_wgrad(ref, x8, None, g)
    assert torch.equal(ref.weight.grad, outs[1][2]) and torch.equal(ref.bias.grad, outs[1][3])
  else:
    gd, xd = g.double().cpu().view(-1, 24), x8.double().cpu().view(-1, 40)
    close(outs[1][2].view(24, 40), gd.t() @ xd, 100 * U * (gd.abs().t() @ xd.abs()), 'dw')
    close(outs[1][3], gd.sum(0), 100 * U * gd.abs().sum(0), 'db')
    # what the format costs: an e4m3 element is off by at most 2^-4 of its value, the smallest ones by half of their step,
    # 2^-10 of a scale that is at most 2^-7 of the block's maximum
    x = x.detach().double().cpu().view(-1, 40)
    off = 2.0 ** -4 * x.abs() + 2.0 ** -17 * x.abs().max()
    bound = gd.abs().t() @ off + 200 * U * (gd.abs().t() @ x.abs())
    close(outs[1][2].view(24, 40), outs[0][2].double().cpu().view(24, 40), bound, 'format')


@pytest.mark.gpu
def test_block_of_norm_and_4bit_product_trains(ops):
  """Layer norm -> 1 x 1 convolution on 4-bit operands with LeakyReLU, both inputs kept in 8 bits, against the formulas:
  rounding passes the gradient through, the data gradient multiplies by the bf16 weights."""
  dt, c, n = torch.bfloat16, 100, 60
  cp, npd = pad8(c), pad8(n)
  x = pixels(2 * 9 * 11, cp, dt, 21, 1.0, 0.3, c).view(2, 9, 11, cp).cuda().requires_grad_(True)
  gy = pixels(198, npd, dt, 22, 0.1, 0.0, n).view(2, 9, 11, npd).cuda()
  gamma = torch.nn.Parameter(1 + 0.1 * torch.randn(c, device='cuda'))
  beta = torch.nn.Parameter(0.1 * torch.randn(c, device='cuda'))
  layer = conv_layer(ops, n, c, 1, dt, (0, 0, 0, 0), 23)
  layer.mx4 = layer.keep8 = True

  def step():
    z = ops.LayerNormAct.apply(x, gamma, beta, 1e-5, 1.0, True)
    y = ops.ConvAct.apply(z, None, layer.weight, layer.bias, layer, 0.1, None)
    y.backward(gy)
    return z.detach(), y.detach()

  z, y = step()
  zd, yd = z.double().cpu().view(-1, cp), y.double().cpu().view(-1, npd)[:, :n]
  w = layer.weight.detach().cpu().view(n, c)
  wq = B.mx4(torch.nn.functional.pad(w, (0, cp - c)))
  zq = B.mx4(zd)
  v = zq @ wq.t() + layer.bias.detach().double().cpu()
  ref = torch.where(v > 0, v, 0.1 * v)
  close(yd, ref, half_step(dt) * ref.abs() + 40 * U * (zq.abs() @ wq.abs().t() + 1), 'y')
  gate = torch.where(yd > 0, 1.0, 0.1).double()
  g = (gy.double().cpu().view(-1, npd)[:, :n] * gate.float()).to(dt).double()
  z8 = B.act8(zd)[:, :c]
  close(layer.weight.grad.view(n, c), g.t() @ z8, 100 * U * (g.abs().t() @ z8.abs()), 'dw')
  gzr = g @ w.to(dt).double()
  # the data gradient is rounded to bf16 before the norm's backward reads it
  xd = x.detach().double().cpu().view(-1, cp)[:, :c]
  _, h, mean, r = B.layer_norm(xd, gamma.detach().cpu(), beta.detach().cpu(), 1e-5, 1.0)
  h8 = (B.act8(x.detach().double().cpu().view(-1, cp))[:, :c] - mean) * r
  gxr, dgr, dbr = B.layer_norm_bwd(gzr, h8, r, torch.ones_like(gzr), gamma.detach().cpu())
  eg = half_step(dt) * gzr.abs() + 100 * U * (g.abs() @ w.to(dt).double().abs())
  t, e = gzr.abs() * gamma.detach().double().cpu().abs(), eg * gamma.detach().double().cpu().abs()
  m1 = lambda q: q.mean(1, keepdim=True)
  tol = r * (e + m1(e) + h8.abs() * m1(e * h8.abs()) + 256 * U * (t + m1(t) + h8.abs() * m1(t * h8.abs())) * (1 + m1(h8.abs())))
  close(x.grad.view(-1, cp)[:, :c], gxr, half_step(dt) * gxr.abs() + 2 * tol, 'gx')
  close(gamma.grad, dgr, (eg * h8.abs()).sum(0) + 256 * U * (gzr.abs() * (h8.abs() + 1)).sum(0), 'dgamma')
  close(beta.grad, dbr, eg.sum(0) + 256 * U * gzr.abs().sum(0), 'dbeta')


@pytest.mark.gpu
def test_unet_with_kept_activations(ops):
  """set_keep8 / set_mx4_forward on a U-Net: the kept inputs change no output, no data gradient and no BatchNorm gradient;
  the forward pass leaves less memory behind.  The 4-bit product reaches the 1 x 1 head alone."""
  from models import unet, utils

  def build():
    torch.manual_seed(3)
    return unet.UNET(1, 1, 2, [32, 64], [32], 'none', kernel_size=3, upsampling_mode='nn-resize-conv', padding='reflection',
                     decoder_act_upsampling_only=True, compute_dtype='bf16').cuda().train()

  g = torch.Generator().manual_seed(4)
  x0, gy = torch.randn(2, 1, 64, 64, generator=g).cuda(), torch.randn(2, 1, 64, 64, generator=g).cuda()
  res = []
  for keep in (False, True):
    net = build()
    if keep:
      assert utils.set_keep8(net) == 8 and utils.set_keep8(net.cuda()) == 8
    x = x0.clone().requires_grad_(True)
    before = torch.cuda.memory_allocated()
    y = net(x)
    held = torch.cuda.memory_allocated() - before
    y.backward(gy)
    res.append((y.detach(), x.grad, held, {n: p.grad for n, p in net.named_parameters()}))
  assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
  assert res[1][2] < 0.9 * res[0][2], (res[0][2], res[1][2])
  for n, p in res[0][3].items():
    if p.dim() == 1 and 'head' not in n:
      assert torch.equal(p, res[1][3][n]), n
    else:
      assert torch.isfinite(res[1][3][n]).all() and res[1][3][n].any(), n
  net = build()
  assert utils.set_mx4_forward(net) == 1 and net.head['0'].layer.mx4
  y = net(x0)
  d = (y.detach() - res[0][0]).abs()
  assert d.any() and torch.isfinite(y).all()
  y.backward(gy)
  assert net.head['0'].weight.grad.any()
  utils.set_mx4_forward(net, False)
  assert torch.equal(build()(x0), res[0][0])


@pytest.mark.gpu
def test_captured_step_replays_like_the_eager_one(ops):
  dt = torch.bfloat16
  layer = conv_layer(ops, 64, 64, 1, dt, (0, 0, 0, 0), 31)
  layer.mx4 = layer.keep8 = True
  gamma, beta = torch.nn.Parameter(torch.ones(64, device='cuda')), torch.nn.Parameter(torch.zeros(64, device='cuda'))
  x = torch.zeros(2, 32, 32, 64, device='cuda', dtype=dt)
  gy = pixels(2048, 64, dt, 33, 0.1).view(2, 32, 32, 64).cuda()
  params = [gamma, beta, layer.weight, layer.bias]
  for p in params:
    p.grad = torch.zeros_like(p)

  def step():
    for p in params:
      p.grad.zero_()
    xi = x.detach().requires_grad_(True)
    z = ops.LayerNormAct.apply(xi, gamma, beta, 1e-5, 0.1, True)
    y = ops.ConvAct.apply(z, None, layer.weight, layer.bias, layer, 0.1, None)
    gx, = torch.autograd.grad(y, xi, gy)
    return y, gx

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(2):
      step()
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    y, gx = step()
  for i in range(4):
    x.copy_(pixels(2048, 64, dt, 40 + i).view(2, 32, 32, 64).cuda())
    graph.replay()
    got = [t.clone() for t in [y, gx] + [p.grad for p in params]]
    want = step()
    for a, b in zip(got, list(want) + [p.grad for p in params]):
      assert torch.equal(a, b), i
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_two_streams_at_once(ops):
  """The same operators on two streams, with workspaces of their own: each as if alone."""
  xs = [pixels(4096, 128, torch.bfloat16, 50 + i).cuda() for i in range(2)]
  w = ops.mx4_quantize(torch.randn(128, 128, device='cuda'))
  gamma, beta = torch.ones(128, device='cuda'), torch.zeros(128, device='cuda')

  def run(x):
    z, sv = ops.layer_norm(x, gamma, beta, keep8=True)
    y = ops.mx4_linear(z, w)
    return (y,) + ops.layer_norm_bwd(y, sv) + ops.act8_wgrad(ops.act8_save(z), y)

  want = [run(x) for x in xs]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in xs]
  for _ in range(5):
    got = [None, None]
    for i, s in enumerate(streams):
      with torch.cuda.stream(s):
        got[i] = run(xs[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
      assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_layer_norm_with_a_negative_slope(ops):
  """From x itself any slope has its gradient; from the kept form a negative one is refused."""
  x, gz = pixels(37, 24, torch.float32, 61), pixels(37, 24, torch.float32, 62)
  gamma, beta = torch.linspace(0.5, 1.5, 24), torch.linspace(-0.3, 0.3, 24)
  with pytest.raises(ValueError):
    ops.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), slope=-0.5, keep8=True)
  z, saved = ops.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), slope=-0.5)
  got = ops.layer_norm_bwd(gz.cuda(), saved)
  ref, h, mean, r = B.layer_norm(x, gamma, beta, 1e-5, -0.5)
  y = h * gamma.double() + beta.double()
  dh = ln_bounds(x, gamma, 1e-5)
  dy = gamma * dh + 4 * U * (h * gamma).abs() + 4 * U * beta.abs()
  assert (y.abs() > dy).all()                     # no output is so near to zero that rounding could turn its sign
  close(z, ref, U * ref.abs() + dy, 'z')
  gate = torch.where(y > 0, 1.0, -0.5).double()
  rgx, rdg, rdb = B.layer_norm_bwd(gz, h, r, gate, gamma)
  gg = (gz.double() * gate).abs()
  t, m1 = gg * gamma.double(), lambda v: v.mean(1, keepdim=True)
  tol = r * (64 * U * (t + m1(t) + 2 * h.abs() * m1(t * h.abs())) + dh * m1(t * h.abs()) + h.abs() * m1(t * dh)) + 64 * U * rgx.abs()
  close(got[0], rgx, U * rgx.abs() + tol, 'gx')
  close(got[1], rdg, 64 * U * (gg * h.abs()).sum(0) + (gg * dh).sum(0), 'dgamma')
  close(got[2], rdb, 64 * U * gg.sum(0), 'dbeta')


@pytest.mark.gpu
def test_gradient_buffers_that_do_not_fit_are_refused(ops):
  x = torch.randn(12, 24, device='cuda')
  f = lambda *s, **k: torch.zeros(*s, device='cuda', **k)
  kept = ops.act8_save(x)
  for kw in (dict(dw=f(24, 23)), dict(dw=f(24, 24).bfloat16()), dict(dw=f(24, 48)[:, ::2]), dict(dw=f(24, 24), db=f(23)),
             dict(dw=f(24, 24), db=f(24).double()), dict(db=f(24))):
    with pytest.raises(ValueError):
      ops.act8_wgrad(kept, x, **kw)
  z, saved = ops.layer_norm(x, f(24), f(24))
  for kw in (dict(dgamma=f(24)), dict(dbeta=f(24)), dict(dgamma=f(23), dbeta=f(24)), dict(dgamma=f(24), dbeta=f(48)[::2]),
             dict(dgamma=f(24).half(), dbeta=f(24))):
    with pytest.raises(ValueError):
      ops.layer_norm_bwd(x, saved, **kw)
  a, b = ops.act8_wgrad(kept, x, dw=f(24, 24, 1, 1), db=f(24)), ops.act8_wgrad(kept, x)
  assert torch.equal(a[0].view(24, 24), b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_layer_norm_node_refuses_computed_parameters(ops):
  """Its gradients go to gamma.grad: through a computed gamma they would not reach what it was computed from."""
  x = torch.randn(4, 16, device='cuda', requires_grad=True)
  w, b = torch.ones(16, device='cuda', requires_grad=True), torch.zeros(16, device='cuda', requires_grad=True)
  with pytest.raises(ValueError):
    ops.LayerNormAct.apply(x, w * 2, b)
  with pytest.raises(ValueError):
    ops.LayerNormAct.apply(x, w, b + 1)
  ops.LayerNormAct.apply(x, w, b.detach()).sum().backward()
  assert w.grad is not None and b.grad is None


@pytest.mark.gpu
def test_captured_forward_follows_loaded_weights(ops):
  """refresh_packs brings the 4-bit copies of replaced weights up to date in place: a captured graph reads them."""
  from models import unet, utils

  def build(seed):
    torch.manual_seed(seed)
    net = unet.UNET(1, 1, 2, [32, 64], [32], 'none', kernel_size=3, upsampling_mode='nn-resize-conv', padding='reflection',
                    decoder_act_upsampling_only=True, compute_dtype='bf16').cuda().eval()
    assert utils.set_mx4_forward(net) == 1
    return net

  net, other = build(5), build(6)
  x = torch.randn(2, 1, 64, 64, generator=torch.Generator().manual_seed(8)).cuda()
  with torch.no_grad():
    first, want = net(x), other(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      net(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      y = net(x)
    graph.replay()
    assert torch.equal(y, first) and not torch.equal(first, want)
    net.load_state_dict(other.state_dict())
    ops.bump_weight_epoch()
    utils.refresh_packs(net)
    for _ in range(2):
      graph.replay()
      assert torch.equal(y, want)
      torch.cuda.synchronize()


@pytest.mark.gpu
def test_tensors_beyond_32_bit_offsets(ops):
  """2^31 elements and more: the last rows come out as they do alone."""
  n, c, tail = 34000001, 64, 1000
  x = torch.empty(n, c, dtype=torch.bfloat16, device='cuda')
  for part in x.split(4000000):
    part.normal_()
  last = x[-tail:].clone()
  gamma, beta = torch.rand(c, device='cuda') + 0.5, torch.rand(c, device='cuda')
  z, sv = ops.layer_norm(x, gamma, beta, slope=0.2, keep8=True)
  z1, sv1 = ops.layer_norm(last, gamma, beta, slope=0.2, keep8=True)
  assert torch.equal(z[-tail:], z1)
  gz = torch.zeros_like(x)
  gz[-tail:] = last.flip(0)
  gx, dg, db = ops.layer_norm_bwd(gz, sv, z)
  gx1, dg1, db1 = ops.layer_norm_bwd(gz[-tail:], sv1, z1)
  assert torch.equal(gx[-tail:], gx1) and not gx[:1000].any()
  # the same terms in another order, and zeros
  h = ((last.double() - last.double().mean(1, keepdim=True)) / last.double().std(1, keepdim=True)).abs()
  for a, b, mag in ((dg, dg1, (gz[-tail:].double().abs() * h * 1.2).sum(0)), (db, db1, gz[-tail:].double().abs().sum(0))):
    assert ((a - b).double().abs() <= 2 * (64 + tail) * U * mag).all()
  del gx, z
  assert torch.equal(ops.act8_restore(sv.kept)[-tail:], ops.act8_restore(sv1.kept))
  dw, _ = ops.act8_wgrad(sv.kept, gz[:, :8])
  dw1, _ = ops.act8_wgrad(sv1.kept, gz[-tail:, :8].contiguous())
  mag = gz[-tail:, :8].double().abs().t() @ ops.act8_restore(sv1.kept).double().abs()
  assert ((dw - dw1).double().abs() <= 2 * (64 + tail) * 2 * U * mag).all()
  del sv, gz
  w = ops.mx4_quantize(torch.randn(16, c, device='cuda'))
  q = ops.mx4_quantize(x)
  assert torch.equal(ops.mx4_dequantize(q)[-tail:], ops.mx4_dequantize(ops.mx4_quantize(last)))
  assert torch.equal(ops.mx4_linear(q, w)[-tail:], ops.mx4_linear(last, w))
