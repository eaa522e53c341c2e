"""Layer norm, 8-bit kept activations and 4-bit products where layouts, devices and values leave the ordinary: broadcast
pixels, host tensors, buffers that meet, foreign codes, ends of the fp32 range.  The oracle is
oracle/csmri_blockscale.py, in float64; bounds count roundings like tests/test_block_scaled.py does (u = 2^-24, half a
step of fp32)."""
import pytest
import torch

import csmri_blockscale as B

U = 2.0 ** -24


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def close(got, ref, tol, what=''):
  got, ref, tol = got.double().cpu(), ref.double().cpu(), tol.double().cpu()
  bad = ~((got - ref).abs() <= tol)
  assert not bad.any(), '%s: %d of %d off, worst %.3g over its bound' % (
      what, int(bad.sum()), bad.numel(), float(((got - ref).abs() / tol.clamp(min=1e-300)).nan_to_num(1e9).max()))


@pytest.fixture
def host_ops(monkeypatch):
  """csmri_hip.ops for tests that stop short of a launch."""
  import csmri_hip
  return csmri_hip.ops


@pytest.fixture(scope='module')
def ops():
  import csmri_hip
  assert torch.cuda.is_available()
  return csmri_hip.ops


# ---- broadcast pixels --------------------------------------------------------------------------------------------------
def layouts(base):
  """(name, tensor [4, 8, 16, 32] or smaller) for a base [4, 8, 16, 32]: broadcast along every set of pixel axes, and views
  whose pixels do or do not lie at one stride."""
  for axes in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2), (0, 1, 2)):
    t = base
    for a in axes:
      t = t.narrow(a, 1, 1)
    yield 'broadcast %s' % (axes,), t.expand(base.shape)
    yield 'dense, broadcast %s' % (axes,), t.contiguous().expand(base.shape)
    yield 'batch of one, broadcast %s' % (axes,), t.contiguous().expand(base.shape)[:1]
  yield 'dense', base
  yield 'broadcast channels', base[..., :1].expand(base.shape)
  yield 'channels', base[..., 8:24]
  yield 'every other pixel', base[:, :, ::2]
  yield 'every other row', base[:, ::2]
  yield 'permuted', base.permute(2, 0, 1, 3)
  yield 'windows', base.flatten()[:512].as_strided((3, 32), (8, 1))
  yield 'strided channels', base[..., ::2]
  yield 'one pixel', base[:1, :1, :1]
  yield 'no pixel', base[:, :0]


def test_pixels_are_read_where_they_lie_or_copied(host_ops, monkeypatch):
  """What a kernel is given -- an address, a pixel count, a pixel stride -- names the tensor's own values, inside its
  storage, for any layout."""
  monkeypatch.setattr(host_ops, '_need_gpu', lambda t: None)
  base = torch.arange(4 * 8 * 16 * 32, dtype=torch.float32).view(4, 8, 16, 32)
  for name, t in layouts(base):
    r, n, c, ps = host_ops._pixels(t)
    assert n * c == t.numel() and c == t.shape[-1], name
    if n == 0:
      continue
    assert ps >= c and r.storage_offset() + (n - 1) * ps + c <= r.untyped_storage().nbytes() // 4, (name, tuple(t.stride()), ps)
    assert torch.equal(r.as_strided((n, c), (ps, 1)), t.reshape(n, c)), name


@pytest.mark.gpu
@pytest.mark.parametrize('keep8', [False, True], ids=['x', 'keep8'])
def test_layer_norm_behind_a_pooled_output(ops, keep8):
  """The gradient that sums over pixels send back is broadcast along the pixel axes."""
  x = torch.randn(4, 8, 16, 32, generator=torch.Generator().manual_seed(1))
  gamma, beta = torch.linspace(0.5, 1.5, 32), torch.linspace(-0.3, 0.3, 32)
  for dims in ((1, 2), (2,), (0, 1, 2)):
    xd = x.cuda().requires_grad_(True)
    ga, be = torch.nn.Parameter(gamma.cuda()), torch.nn.Parameter(beta.cuda())
    z = ops.LayerNormAct.apply(xd, ga, be, 1e-5, 1.0, keep8)
    s = z.sum(dim=dims)
    w = torch.randn(s.shape, generator=torch.Generator().manual_seed(2)).cuda()
    (s * w).sum().backward()
    g = w.view([1 if i in dims else x.shape[i] for i in range(4)]).expand(x.shape).contiguous()
    got = ops.layer_norm_bwd(g, ops.layer_norm(xd.detach(), ga.detach(), be.detach(), 1e-5, 1.0, keep8)[1])
    for a, b in zip((xd.grad, ga.grad, be.grad), got):
      assert torch.equal(a, b)


@pytest.mark.gpu
def test_broadcast_pixels_through_every_operator(ops):
  base = torch.randn(4, 8, 16, 32, generator=torch.Generator().manual_seed(3)).cuda()
  w = ops.mx4_quantize(torch.randn(24, 32, generator=torch.Generator().manual_seed(4)).cuda())
  kept = ops.act8_save(base)
  gamma, beta = torch.ones(32, device='cuda'), torch.zeros(32, device='cuda')
  for name, t in layouts(base):
    if t.shape != base.shape:
      continue
    d = t.clone(memory_format=torch.contiguous_format)
    assert torch.equal(ops.act8_restore(ops.act8_save(t)), ops.act8_restore(ops.act8_save(d))), name
    assert torch.equal(ops.mx4_linear(t, w), ops.mx4_linear(d, w)), name
    assert torch.equal(ops.layer_norm(t, gamma, beta)[0], ops.layer_norm(d, gamma, beta)[0]), name
    for a, b in zip(ops.act8_wgrad(kept, t), ops.act8_wgrad(kept, d)):
      assert torch.equal(a, b), name


# ---- tensors on the host -----------------------------------------------------------------------------------------------
def test_host_operands_reach_no_kernel(host_ops, monkeypatch):
  """Every operator refuses tensors on the host, whatever device is current."""
  def launched(name, *args):
    raise AssertionError('%s would have been launched' % name)
  monkeypatch.setattr(host_ops.lib, 'call', launched)
  monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda dev: 0, raising=False)
  monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: -1, raising=False)
  o = host_ops
  z = lambda *s: torch.zeros(*s, dtype=torch.uint8)
  kept = o.Act8(z(6, 40), z(6, 2), (6, 40), torch.bfloat16)
  rows, w = o.Mx4(z(6, 128), z(6, 16), 136), o.Mx4(z(24, 128), z(24, 16), 136)
  x = torch.zeros(6, 40)
  saved = o.LNSaved(x, None, torch.zeros(80), (6, 40), torch.float32, 40, 1e-5, 1.0)
  for f in (lambda: o.act8_save(x), lambda: o.act8_restore(kept), lambda: o.act8_restore(kept, torch.float32),
            lambda: o.act8_wgrad(kept, x), lambda: o.mx4_quantize(torch.zeros(6, 136)), lambda: o.mx4_dequantize(rows),
            lambda: o.mx4_linear(rows, w), lambda: o.mx4_linear(torch.zeros(6, 136), w),
            lambda: o.layer_norm(x, torch.ones(40), torch.zeros(40)), lambda: o.layer_norm_bwd(x, saved)):
    with pytest.raises(RuntimeError):
      f()


@pytest.mark.gpu
def test_host_operands_beside_device_tensors_are_refused(ops):
  z = lambda *s: torch.zeros(*s, dtype=torch.uint8)
  kept, rows = ops.Act8(z(6, 40), z(6, 2), (6, 40), torch.bfloat16), ops.Mx4(z(6, 128), z(6, 16), 136)
  x = torch.zeros(6, 40, device='cuda')
  for f in (lambda: ops.act8_restore(kept), lambda: ops.act8_wgrad(kept, x), lambda: ops.mx4_dequantize(rows),
            lambda: ops.mx4_linear(rows, rows), lambda: ops.mx4_linear(torch.zeros(6, 136, device='cuda'), rows),
            lambda: ops.mx4_quantize(torch.zeros(6, 136, device='cuda'), rows),
            lambda: ops.layer_norm(x, torch.ones(40), torch.zeros(40, device='cuda')),
            lambda: ops.act8_wgrad(ops.act8_save(x), x, dw=torch.zeros(40, 40))):
    with pytest.raises(RuntimeError):
      f()


# ---- a layer whose gradient comes from two kernels ----------------------------------------------------------------------
def pointwise_layer(ops, cout, cin, seed, dtype=torch.bfloat16):
  g = torch.Generator().manual_seed(seed)
  w = torch.nn.Parameter((torch.randn(cout, cin, 1, 1, generator=g) / cin ** 0.5).cuda())
  return ops.ConvLayer(w, torch.nn.Parameter(torch.randn(cout, generator=g).cuda()), 1, (0, 0, 0, 0), 'zero', dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('multi', ['0', '1', 'auto'])
@pytest.mark.parametrize('keeps', [(True, False), (False, True), (False, True, False), (True, False, True)],
                         ids=lambda k: ''.join('8' if v else '-' for v in k))
@pytest.mark.parametrize('fresh', [False, True], ids=['accumulate', 'fresh'])
def test_layer_used_with_kept_and_with_plain_inputs_in_one_backward(ops, monkeypatch, multi, keeps, fresh):
  """The reductions of plain weight gradients wait for the end of the backward pass: a kept one of the same layer comes
  after them.  ``fresh``: the gradients hold what a lazy zero left behind, to be overwritten."""
  monkeypatch.setattr(ops, 'WGRAD_FINISH_MULTI', multi)
  gen = torch.Generator().manual_seed(7)
  xs = [torch.randn(2, 24, 20, 40, generator=gen).bfloat16().cuda() for _ in keeps]
  gs = [(0.1 * torch.randn(2, 24, 20, 24, generator=gen)).bfloat16().cuda() for _ in keeps]
  layer = pointwise_layer(ops, 24, 40, 3)
  for p in (layer.weight, layer.bias):
    p.grad = torch.full_like(p, 7.0)
    p._grad_fresh = fresh
  ys = []
  for x, keep in zip(xs, keeps):
    layer.keep8 = keep
    ys.append(ops.ConvAct.apply(x, None, layer.weight, layer.bias, layer, 1.0, None))
  torch.autograd.backward(ys, gs)
  base = 0.0 if fresh else 7.0
  dw = torch.full((24, 40), base, dtype=torch.float64)
  db = torch.full((24,), base, dtype=torch.float64)
  mw, mb = dw.abs(), db.abs()
  for x, g, keep in zip(xs, gs, keeps):
    x, g = x.double().cpu().view(-1, 40), g.double().cpu().view(-1, 24)
    x = B.act8(x) if keep else x
    dw, db, mw, mb = dw + g.t() @ x, db + g.sum(0), mw + g.abs().t() @ x.abs(), mb + g.abs().sum(0)
  # 960 pixels in products that are exact in fp32: fewer than 100 additions in a chain, each at most 2 u
  close(layer.weight.grad.view(24, 40), dw, 200 * U * mw, 'dw')
  close(layer.bias.grad, db, 200 * U * mb, 'db')


# ---- layer norm of rows far from zero ------------------------------------------------------------------------------------
def ln_offset_bounds(x, eps):
  """Bounds of |error of h| for the two-step mean: m0 = mean + d0, |d0| <= 66 u mean|x| (chains of fewer than 64 additions,
  a division); d = x - m0, then mean(d) corrects both the deviations and the variance.  A deviation is off by
  u |d| + 67 u mean|d| + its own rounding, mean d^2 - mean(d)^2 by 70 u (var + 2 d0^2), 1 / sqrt by half of that relatively
  and 4 u."""
  x = x.double()
  mean = x.mean(1, keepdim=True)
  var = ((x - mean) ** 2).mean(1, keepdim=True)
  d0 = 66 * U * x.abs().mean(1, keepdim=True)
  dev = (x - mean).abs()
  r = 1 / torch.sqrt(var + eps)
  dnum = 70 * U * (dev + dev.mean(1, keepdim=True) + 2 * d0)
  drel = 35 * U * (var + 2 * d0 ** 2) / (var + eps) + 4 * U
  return r * dnum + (dev * r + r * dnum) * drel + 2 * U * dev * r


OFFSET_SIZES = [7, 13, 15, 64, 100, 520, 1000, 2056, 4100, 8190]


@pytest.mark.gpu
@pytest.mark.parametrize('offset', [1000.0, -10000.0])
@pytest.mark.parametrize('c', OFFSET_SIZES)
def test_layer_norm_of_constant_rows(ops, c, offset):
  """Every deviation is zero: z is beta, whatever the mean's sum rounds to."""
  cp = (c + 7) // 8 * 8
  for dtype in (torch.float32, torch.bfloat16):
    x = torch.zeros(5, cp, dtype=dtype)
    x[:, :c] = offset
    x[1, :c] = offset * 1.1
    gamma, beta = torch.linspace(0.5, 1.5, c), torch.linspace(-0.3, 0.3, c)
    z, saved = ops.layer_norm(x.cuda(), gamma.cuda(), beta.cuda())
    dh = ln_offset_bounds(x[:, :c], 1e-5)
    close(z[:, :c], beta.expand(5, c), half_step(dtype) * beta.abs().double() + gamma.double() * dh + 4 * U * beta.abs().double(), 'z')
    gz = torch.randn(5, cp, generator=torch.Generator().manual_seed(c)).to(dtype)
    gz[:, c:] = 0
    gx, dg, db = ops.layer_norm_bwd(gz.cuda(), saved)
    t = gz[:, :c].double() * gamma.double()
    ref, r = (t - t.mean(1, keepdim=True)) / 1e-5 ** 0.5, 1e-5 ** -0.5
    m1 = lambda v: v.mean(1, keepdim=True)
    close(gx[:, :c], ref, half_step(dtype) * ref.abs() + r * (70 * U * (t.abs() + m1(t.abs())) + dh * m1(t.abs() * dh)) + 64 * U * ref.abs(), 'gx')
    close(dg, torch.zeros(c), (gz[:, :c].double().abs() * dh).sum(0) + 1e-300, 'dgamma')


@pytest.mark.gpu
@pytest.mark.parametrize('spread', [1.0, 2.0 ** -6, 2.0 ** -10])
@pytest.mark.parametrize('c', OFFSET_SIZES)
def test_layer_norm_of_a_small_spread_around_a_large_offset(ops, c, spread):
  """fp32 rows around 1000 whose spread is a few of their own steps (2^-14) and more: what the statistics cost is relative
  to the spread, forward and backward."""
  cp, eps = (c + 7) // 8 * 8, 1e-5
  g = torch.Generator().manual_seed(c)
  x = torch.zeros(6, cp)
  x[:, :c] = 1000 + spread * torch.randn(6, c, generator=g)
  gz = torch.zeros(6, cp)
  gz[:, :c] = torch.randn(6, c, generator=g)
  gamma, beta = torch.linspace(0.5, 1.5, c), torch.linspace(-0.3, 0.3, c)
  z, saved = ops.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), eps)
  ref, h, mean, r = B.layer_norm(x[:, :c], gamma, beta, eps, 1.0)
  dh = ln_offset_bounds(x[:, :c], eps)
  g64, b64 = gamma.double(), beta.double()
  close(z[:, :c], ref, U * ref.abs() + g64 * dh + 4 * U * (h * g64).abs() + 4 * U * b64.abs(), 'z')
  gx, dg, db = ops.layer_norm_bwd(gz.cuda(), saved)
  rgx, rdg, rdb = B.layer_norm_bwd(gz[:, :c], h, r, torch.ones_like(h), gamma)
  t, m1 = gz[:, :c].double().abs() * g64, lambda v: v.mean(1, keepdim=True)
  h = h.abs()
  tol = r * (70 * U * (t + m1(t) + 2 * h * m1(t * h)) + dh * m1(t * h) + h * m1(t * dh) + dh * m1(t * dh))
  # r itself: 35 u (var + 2 d0^2) / (var + eps) + 4 u, at most 110 u with d0 <= 66 u 1000 against eps
  close(gx[:, :c], rgx, U * rgx.abs() + tol + 110 * U * r * (t + m1(t) + h * m1(t * h)), 'gx')
  close(dg, rdg, (gz[:, :c].double().abs() * (dh + 64 * U * h)).sum(0) + 1e-300, 'dgamma')


@pytest.mark.gpu
@pytest.mark.parametrize('c', [15, 100, 4100])
def test_kept_layer_norm_of_constant_rows(ops, c):
  """The kept form's statistics: the mean of a constant row is its value to one rounding, 1 / std that of eps."""
  cp = (c + 7) // 8 * 8
  x = torch.zeros(3, cp)
  x[:, :c] = torch.tensor([1000.0, -10000.0, 12345.678]).view(3, 1)
  _, saved = ops.layer_norm(x.cuda(), torch.ones(c).cuda(), torch.zeros(c).cuda(), keep8=True)
  mean, r = saved.aux[2 * cp:2 * cp + 3].double().cpu(), saved.aux[2 * cp + 3:].double().cpu()
  ref = x[:, 0].double()
  close(mean, ref, 2 * U * ref.abs(), 'mean')
  close(r, torch.full((3,), 1e-5 ** -0.5, dtype=torch.float64), torch.full((3,), 110 * U * 1e-5 ** -0.5, dtype=torch.float64), '1 / std')


# ---- the ends of the fp32 range in a gradient that is split into three bf16 parts ------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('n,cin,cout', [(40, 24, 16), (700, 72, 136)])
def test_weight_gradient_of_infinite_nan_and_largest_fp32_gradients(ops, n, cin, cout):
  """An infinity in dY stays one, with the sign of the activation it meets, NaN stays NaN, finite values beyond the largest
  bf16 number stay finite, and none of them leaves its output channel."""
  g = torch.Generator().manual_seed(n)
  x = (torch.rand(n, cin, generator=g) + 0.5) * (1 - 2 * torch.randint(0, 2, (1, cin), generator=g))   # one sign a channel
  x = x * 2.0 ** -10
  gy = 0.1 * torch.randn(n, cout, generator=g)
  top = torch.finfo(torch.float32).max
  gy[n - 1, 0], gy[3, 1], gy[5, 2] = float('inf'), -float('inf'), float('nan')
  gy[7, 3], gy[8, 4], gy[9, 5] = 3.4e38, -top, 3.396e38
  kept = ops.act8_save(x.cuda())
  xq = B.act8(x)
  dw, db = [t.double().cpu() for t in ops.act8_wgrad(kept, gy.cuda(), cout, cin)]
  for row, v in ((0, float('inf')), (1, -float('inf'))):
    assert torch.equal(dw[row], v * xq[0].sign()) and db[row] == v
  assert torch.isnan(dw[2]).all() and torch.isnan(db[2])
  rest = [i for i in range(cout) if i > 2]
  g64 = gy.double()[:, rest]
  # three parts of 8 bits each, of one sign: their products are exact, each of at most 6 (n / 32 + 33) additions 2 u
  L = 6 * (n / 32 + 33) + 8
  close(dw[rest], g64.t() @ xq, L * U * (g64.abs().t() @ xq.abs()), 'dw')
  close(db[rest], g64.sum(0), L * U * g64.abs().sum(0), 'db')


@pytest.mark.gpu
def test_weight_gradient_of_small_fp32_gradients(ops):
  """dY around 2^-100, whose third parts are the smallest that are still normal bf16 numbers: as exact as any other."""
  g = torch.Generator().manual_seed(5)
  x, gy = torch.randn(300, 40, generator=g), torch.randn(300, 24, generator=g) * 2.0 ** -98
  gy = torch.where(gy.abs() < 2.0 ** -103, torch.zeros(()), gy)
  dw, db = ops.act8_wgrad(ops.act8_save(x.cuda()), gy.cuda())
  xq, g64 = B.act8(x), gy.double()
  L = 6 * (300 / 32 + 33) + 8
  close(dw, g64.t() @ xq, L * U * (g64.abs().t() @ xq.abs()), 'dw')
  close(db, g64.sum(0), L * U * g64.abs().sum(0), 'db')


# ---- scale bytes that only codes from elsewhere hold ------------------------------------------------------------------------
@pytest.mark.gpu
def test_kept_codes_with_the_smallest_and_the_nan_scale(ops):
  """Scale byte 0 is 2^-127, 255 is NaN whatever the codes: where the values are restored, in the weight gradient and in
  the layer norm's backward."""
  g = torch.Generator().manual_seed(11)
  code = torch.randint(72, 120, (6, 64), generator=g).to(torch.uint8)      # e4m3 4 .. 240: with 2^-127 a normal number
  sign = torch.randint(0, 2, (6, 64), generator=g).to(torch.uint8) * 128
  code = code + sign
  scale = torch.tensor([0, 1, 254, 127, 0, 100], dtype=torch.uint8).view(6, 1).repeat(1, 2)
  value = torch.tensor(B.E4M3, dtype=torch.float64)[(code % 128).long()] * torch.where(sign > 0, -1.0, 1.0).double()
  value = value * torch.exp2(scale.double() - 127).repeat_interleave(32, 1)
  kept = lambda s: ops.Act8(code.cuda(), s.cuda(), (6, 64), torch.float32)
  got = ops.act8_restore(kept(scale)).double().cpu()
  ok = value.abs() < torch.finfo(torch.float32).max
  assert torch.equal(got[ok], value[ok]) and torch.isinf(got[~ok]).all()
  nan = scale.clone()
  nan[3, 1] = 255
  got = ops.act8_restore(kept(nan)).cpu()
  assert torch.isnan(got[3, 32:]).all() and int(torch.isnan(got).sum()) == 32
  assert torch.isnan(ops.act8_wgrad(kept(nan), torch.ones(6, 8, device='cuda'))[0][:, 32:]).all()
  # one pixel at a time, so that the large ones do not hide the small
  for p in (0, 1, 4, 5):
    gy = torch.full((1, 8), 2.0 ** 90)
    one = ops.Act8(code[p:p + 1].cuda(), scale[p:p + 1].cuda(), (1, 64), torch.float32)
    for dt in (torch.float32, torch.bfloat16):
      dw, _ = ops.act8_wgrad(one, gy.to(dt).cuda())
      assert torch.equal(dw.double().cpu(), value[p:p + 1].mul(2.0 ** 90).expand(8, 64)), (p, dt)
  x = torch.randn(6, 64, generator=g)
  z, saved = ops.layer_norm(x.cuda(), torch.ones(64).cuda(), torch.zeros(64).cuda(), keep8=True)
  saved.kept = kept(nan)
  gx = ops.layer_norm_bwd(torch.ones(6, 64, device='cuda'), saved, z)[0].cpu()
  assert torch.isnan(gx[3]).all()


# ---- outputs that meet ------------------------------------------------------------------------------------------------------
def test_gradients_that_share_memory_are_refused(host_ops, monkeypatch):
  """Two sums go to two places: threads that add to one would lose each other's."""
  raw, p = host_ops.lib.raw, 1 << 20
  bw, wg = raw('csmri_ln_bwd'), raw('csmri_act8_wgrad')
  ln = lambda dg, db: bw(0, p, 16, 2 * p, 16, None, None, None, None, 0, 3 * p, 16, 4, 16, 13, 4 * p, 1e-5, 1.0, 5 * p, dg, db, 1, None)
  for d in (0, 4, 48):
    assert ln(6 * p, 6 * p + d) == -1 and ln(6 * p + d, 6 * p) == -1
  act8 = lambda dw, db: wg(0, p, 16, 2 * p, 3 * p, 4, 16, 16, 13, 11, 1, None, dw, db, 1, None)
  for dw, db in ((6 * p, 6 * p), (6 * p, 6 * p + 4 * 142), (6 * p + 48, 6 * p)):
    assert act8(dw, db) == -1
  # npix == 0 writes too
  assert bw(0, None, 16, None, 16, None, None, None, None, 0, None, 16, 0, 16, 13, 4 * p, 1e-5, 1.0, 5 * p, 6 * p, 6 * p, 0, None) == -1
  monkeypatch.setattr(host_ops, '_need_gpu', lambda t: None)
  monkeypatch.setattr(host_ops.lib, 'call', lambda *a: pytest.fail('launched'))
  x, flat = torch.zeros(4, 24), torch.zeros(64)
  saved = host_ops.LNSaved(x, None, torch.zeros(48), (4, 24), torch.float32, 24, 1e-5, 1.0)
  for dg, db in ((flat[:24], flat[:24]), (flat[:24], flat[23:47])):
    with pytest.raises(ValueError):
      host_ops.layer_norm_bwd(x, saved, dgamma=dg, dbeta=db)
  kept = host_ops.Act8(torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), (4, 8), torch.float32)
  with pytest.raises(ValueError):
    host_ops.act8_wgrad(kept, x, 5, 8, dw=flat[:40], db=flat[39:44])
  p = torch.nn.Parameter(torch.ones(24))
  with pytest.raises(ValueError):
    host_ops.LayerNormAct.apply(x, p, p)


@pytest.mark.gpu
def test_gradients_side_by_side_are_written(ops):
  x = torch.randn(9, 24, generator=torch.Generator().manual_seed(12)).cuda()
  _, saved = ops.layer_norm(x, torch.ones(24, device='cuda'), torch.zeros(24, device='cuda'))
  want, flat = ops.layer_norm_bwd(x, saved), torch.zeros(24 * 24 + 24, device='cuda')
  ops.layer_norm_bwd(x, saved, dgamma=flat[24:48], dbeta=flat[:24])
  assert torch.equal(flat[24:48], want[1]) and torch.equal(flat[:24], want[2]) and not flat[48:].any()
  kept = ops.act8_save(x)
  want = ops.act8_wgrad(kept, x)
  ops.act8_wgrad(kept, x, dw=flat[:576], db=flat[576:])
  assert torch.equal(flat[:576].view(24, 24), want[0]) and torch.equal(flat[576:], want[1])


# ---- 4-bit copies of frozen layers -------------------------------------------------------------------------------------------
def small_unet(seed):
  from models import unet
  torch.manual_seed(seed)
  return unet.UNET(1, 1, 2, [32, 64], [32], 'none', kernel_size=3, upsampling_mode='nn-resize-conv', padding='reflection',
                   decoder_act_upsampling_only=True, compute_dtype='bf16').cuda()


@pytest.mark.gpu
def test_frozen_4bit_layers_follow_loaded_weights(ops):
  """refresh_packs reaches the 4-bit copies of frozen layers as it reaches their other packed ones, in place."""
  from models import utils
  x = torch.randn(2, 1, 64, 64, generator=torch.Generator().manual_seed(8)).cuda()
  net, other = small_unet(5).eval(), small_unet(6).eval()
  for m in (net, other):
    assert utils.set_mx4_forward(m) == 1
    utils.freeze(m)
  with torch.no_grad():
    first, want = net(x), other(x)
    layer = net.head['0'].layer
    assert layer._pack4 is not None and not torch.equal(first, want)
    buf = layer._pack4[1].addresses()
    net.load_state_dict(other.state_dict())
    ops.bump_weight_epoch()
    utils.refresh_packs(net)
    assert torch.equal(net(x), want)
    assert layer._pack4[1].addresses() == buf


# ---- inference with layers that keep their inputs --------------------------------------------------------------------------
@pytest.mark.gpu
def test_inputs_are_kept_only_where_a_backward_pass_can_follow(ops, monkeypatch):
  from models import utils
  calls = []
  save = ops.act8_save
  monkeypatch.setattr(ops, 'act8_save', lambda x: calls.append(x.shape) or save(x))
  net = small_unet(5)
  x = torch.randn(2, 1, 64, 64, generator=torch.Generator().manual_seed(8)).cuda()
  n = utils.set_keep8(net)
  with torch.no_grad():
    net.eval()(x)
    assert not calls
    y = net.train()(x)
    assert not calls
    with torch.enable_grad():
      z = net(x)
    assert len(calls) >= n
  assert torch.equal(y, z)
  z.sum().backward()
  assert all(p.grad is not None for p in net.parameters())
  del calls[:]
  for p in net.parameters():
    p.requires_grad_(False)
  net(x.requires_grad_(True))
  assert not calls


@pytest.mark.gpu
@pytest.mark.parametrize('slope', [1.0, 0.2])
def test_layer_norm_node_keeps_its_input_only_where_a_backward_pass_can_follow(ops, monkeypatch, slope):
  asked = []
  norm = ops.layer_norm
  monkeypatch.setattr(ops, 'layer_norm', lambda *a: asked.append(bool(a[5])) or norm(*a))
  x = torch.randn(33, 72, generator=torch.Generator().manual_seed(9)).cuda()
  ga, be = torch.nn.Parameter(torch.linspace(0.5, 1.5, 72).cuda()), torch.nn.Parameter(torch.linspace(-1, 1, 72).cuda())
  node = lambda x, ga, be: ops.LayerNormAct.apply(x, ga, be, 1e-5, slope, True)
  with torch.no_grad():
    a = node(x, ga, be)
    b = node(x.requires_grad_(True), ga, be)
  x = x.detach()
  c = node(x, ga.detach(), be.detach())
  assert asked == [False] * 3 and torch.equal(a, b) and torch.equal(a, c)
  z = node(x, ga, be)
  assert asked[3:] == [True] and torch.equal(z, a)
  z.sum().backward()
  assert ga.grad is not None and be.grad is not None


@pytest.mark.gpu
@pytest.mark.parametrize('multi', ['0', '1', 'auto'])
@pytest.mark.parametrize('defer', [0, 2])
def test_both_kinds_of_weight_gradient_on_the_side_stream(ops, monkeypatch, multi, defer):
  """The same with the weight gradients on their own stream, issued at once or held back."""
  backward = torch.autograd.backward

  def joined(*args):
    backward(*args)
    ops.join_wgrad_stream()
  monkeypatch.setattr(torch.autograd, 'backward', joined)
  monkeypatch.setattr(ops, 'WGRAD_DEFER', defer)
  ops.enable_wgrad_stream(True)
  try:
    for keeps in ((True, False), (False, True), (False, True, False)):
      for fresh in (False, True):
        test_layer_used_with_kept_and_with_plain_inputs_in_one_backward(ops, monkeypatch, multi, keeps, fresh)
  finally:
    ops.enable_wgrad_stream(False)
