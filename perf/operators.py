"""Layer norm, 8-bit kept activations and microscaled 4-bit products: the cases that are timed, and their plain forms.

Activations are pixel-major ([images, height, width, channels]) in bf16 or fp32, their channels padded with zeros to a
multiple of 8.  ``run`` computes one pass: with ``own`` by the framework's operators, otherwise by elementary torch
operations in fp32, rounded once at the end."""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
BLOCK = 32                   # channels that share a scale
MIN_EXP = -100               # a block's largest magnitude counts as at least 2^MIN_EXP
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def _pad8(c):
  return (c + 7) // 8 * 8


def _ops():
  pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'csmri-refinement_amd')
  if pkg not in sys.path:
    sys.path.insert(0, pkg)
  from csmri_hip import ops
  return ops


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------


def listed():
  return [
      # inference on one small map between two discriminator layers, ragged channels: a launch, little else
      {'name': 'norm_infer_8x8x100_fp32', 'op': 'norm', 'images': 1, 'height': 8, 'width': 8, 'channels': 100,
       'dtype': 'fp32', 'slope': 0.1},
      # a training pass over the U-Net's first level at the benchmark's batch: many pixels of few channels
      {'name': 'norm_train_8x256x256x32', 'op': 'norm_train', 'images': 8, 'height': 256, 'width': 256, 'channels': 32,
       'dtype': 'bf16', 'keep8': False},
      # a training pass over wide pixels with the input kept in 8 bits
      {'name': 'norm_train_8x64x64x1024_keep8', 'op': 'norm_train', 'images': 8, 'height': 64, 'width': 64,
       'channels': 1024, 'dtype': 'bf16', 'keep8': True},
      # a U-Net encoder map kept over the forward pass and restored in the backward
      {'name': 'keep_8x128x128x64', 'op': 'keep', 'images': 8, 'height': 128, 'width': 128, 'channels': 64,
       'dtype': 'bf16', 'sliced': False},
      # the same for the upper channels of a concatenated map of odd extents, fp32
      {'name': 'keep_3x65x33x104_fp32_sliced', 'op': 'keep', 'images': 3, 'height': 65, 'width': 33, 'channels': 104,
       'dtype': 'fp32', 'sliced': True},
      # weight gradient of a 1 x 1 layer of U-Net widths: a long sum, a small result
      {'name': 'wgrad_8x128x128_64to128', 'op': 'wgrad', 'images': 8, 'height': 128, 'width': 128, 'channels': 64,
       'outputs': 128, 'dtype': 'bf16'},
      # weight gradient of a wide layer: bound by the matrix units
      {'name': 'wgrad_16x32x32_2048to2048', 'op': 'wgrad', 'images': 16, 'height': 32, 'width': 32, 'channels': 2048,
       'outputs': 2048, 'dtype': 'bf16'},
      # a weight or activation matrix to 4 bits, read back as values
      {'name': 'quant_8x64x64x1024', 'op': 'quant', 'images': 8, 'height': 64, 'width': 64, 'channels': 1024,
       'dtype': 'bf16'},
      # a small ragged fp32 map to 4 bits
      {'name': 'quant_1x17x19x200_fp32', 'op': 'quant', 'images': 1, 'height': 17, 'width': 19, 'channels': 200,
       'dtype': 'fp32'},
      # one pixel through a wide layer: the weights are read once, latency counts
      {'name': 'linear_1x1x1_4096to4096', 'op': 'linear', 'images': 1, 'height': 1, 'width': 1, 'channels': 4096,
       'outputs': 4096, 'dtype': 'bf16', 'slope': 1.0},
      # the VGG stack's widths at eight images
      {'name': 'linear_8x32x32_512to512', 'op': 'linear', 'images': 8, 'height': 32, 'width': 32, 'channels': 512,
       'outputs': 512, 'dtype': 'bf16', 'slope': 0.0},
      # the largest: bound by the matrix units
      {'name': 'linear_16x32x32_4096to4096', 'op': 'linear', 'images': 16, 'height': 32, 'width': 32, 'channels': 4096,
       'outputs': 4096, 'dtype': 'bf16', 'slope': 1.0},
  ]


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(['norm', 'norm_train', 'norm_train', 'keep', 'wgrad', 'wgrad', 'quant', 'linear', 'linear', 'linear'])
  dtype = rng.choice(['bf16', 'bf16', 'fp32'])
  case = {'op': op, 'dtype': dtype}
  if op in ('wgrad', 'linear'):
    wide = 2048 if op == 'wgrad' else 4096
    case['channels'] = 8 * _log_int(rng, 1, wide // 8)
    case['outputs'] = _log_int(rng, 1, wide)
    top = 131072 if op == 'wgrad' else 16384
    # no more work than the largest listed case of the kind
    room = (16384 * 2048 * 2048 if op == 'wgrad' else 16384 * 4096 * 4096) // (case['channels'] * case['outputs'])
    pixels = _log_int(rng, 1, max(1, min(top, room)))
    if op == 'linear':
      case['slope'] = rng.choice([1.0, 0.1, 0.0])
  else:
    case['channels'] = _log_int(rng, 1 if op in ('norm', 'norm_train') else 8, 4096)
    if op in ('keep', 'quant'):
      case['channels'] = _pad8(case['channels'])
    room = (1 << 24) // _pad8(case['channels'])
    pixels = _log_int(rng, 1, min(room, 524288))
    if op == 'norm':
      case['slope'] = rng.choice([1.0, 0.1])
    if op == 'norm_train':
      case['keep8'] = rng.choice([True, False])
    if op == 'keep':
      case['sliced'] = rng.choice([True, False])
  case['images'] = rng.choice([i for i in (1, 2, 3, 8) if i <= pixels])
  case['height'] = max(1, int(math.sqrt(pixels // case['images'])))
  case['width'] = max(1, pixels // case['images'] // case['height'])
  return case


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------


def _pixels(case):
  return case['images'] * case['height'] * case['width']


def _activations(case, gen, channels, dtype, centred):
  """A feature map: channels of different spread, with an offset each where they come out of a convolution with a bias,
  cut to their positive side like behind a LeakyReLU where they do not."""
  cp = _pad8(channels)
  n = _pixels(case)
  spread = torch.exp(0.5 * torch.randn(cp, generator=gen, device='cuda'))
  x = torch.randn(n, cp, generator=gen, device='cuda')
  if centred:
    x = x * spread + 0.3 * torch.randn(cp, generator=gen, device='cuda')
  else:
    x = torch.where(x > 0, x, 0.1 * x) * spread
  x[:, channels:] = 0
  return x.to(dtype).view(case['images'], case['height'], case['width'], cp)


def prepare(case, seed):
  gen = torch.Generator(device='cuda')
  gen.manual_seed(int(seed))
  op, dtype, c = case['op'], DTYPES[case['dtype']], case['channels']
  st = {'case': case}
  if op in ('norm', 'norm_train'):
    st['x'] = _activations(case, gen, c, dtype, True)
    st['gamma'] = 1.0 + 0.1 * torch.randn(c, generator=gen, device='cuda')
    st['beta'] = 0.1 * torch.randn(c, generator=gen, device='cuda')
    if op == 'norm_train':
      g = 1e-2 * torch.randn(_pixels(case), _pad8(c), generator=gen, device='cuda')
      g[:, c:] = 0
      st['gz'] = g.to(dtype).view(st['x'].shape)
  elif op == 'keep':
    if case['sliced']:
      st['x'] = _activations(case, gen, 2 * c, dtype, False)[..., c:]
    else:
      st['x'] = _activations(case, gen, c, dtype, False)
  elif op == 'wgrad':
    st['x'] = _activations(case, gen, c, dtype, False)
    n = case['outputs']
    g = 1e-2 * torch.randn(_pixels(case), _pad8(n), generator=gen, device='cuda')
    g[:, n:] = 0
    st['gy'] = g.to(dtype).view(case['images'], case['height'], case['width'], _pad8(n))
  elif op == 'quant':
    st['x'] = _activations(case, gen, c, dtype, True)
  else:
    st['x'] = _activations(case, gen, c, dtype, True)
    n = case['outputs']
    w = torch.randn(n, c, generator=gen, device='cuda') / math.sqrt(c)
    st['w_codes'], st['w_scales'] = _pack_mx4(w)          # the weights as a 4-bit checkpoint holds them
    st['bias'] = 0.1 * torch.randn(n, generator=gen, device='cuda')
  return st


# ----------------------------------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------------------------------


def _pow2(e):
  """2^e for whole e in the range of normal fp32 numbers."""
  return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _blocks(x):
  """[rows, channels] -> [rows, blocks, 32] in fp32, zero padded."""
  rows, c = x.shape
  x = torch.nn.functional.pad(x.float(), (0, (-c) % BLOCK))
  return x.view(rows, -1, BLOCK)


def _block_exp(b):
  """floor(log2) of the largest magnitude of each block, at least MIN_EXP."""
  amax = b.abs().amax(dim=2, keepdim=True)
  e = torch.frexp(amax)[1] - 1
  return torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)


def _mx4_codes(b):
  """Blocks -> (codes 0..15, exponent of the scale)."""
  e = _block_exp(b) - 2
  y = b * _pow2(-e)
  m = y.abs()
  code = ((m > 0.25).to(torch.int32) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
  return code + 8 * (y < 0), e


def _mx4_values(x):
  """[rows, channels] -> what its 4-bit form stands for, fp32."""
  b = _blocks(x)
  code, e = _mx4_codes(b)
  mag = torch.tensor(E2M1, device=x.device)[code & 7]
  v = torch.where(code >= 8, -mag, mag) * _pow2(e)
  return v.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _pack_mx4(w):
  """[rows, k] -> codes uint8 [rows, 64 * ceil(k / 128)], two a byte, the even channel in the low half, and E8M0 scales
  uint8 [rows, 16 * ceil(k / 512)]; padding: code 0, scale 2^0."""
  rows, k = w.shape
  b = _blocks(w)
  code, e = _mx4_codes(b)
  code = torch.nn.functional.pad(code.view(rows, -1), (0, (-code.shape[1] * BLOCK) % 128)).to(torch.uint8)
  scale = torch.nn.functional.pad(e.view(rows, -1) + 127, (0, (-e.shape[1]) % 16), value=127).to(torch.uint8)
  return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scale.contiguous()


def _unpack_mx4(codes, scales, k):
  code = torch.stack([codes & 15, codes >> 4], dim=2).view(codes.shape[0], -1)[:, :k].long()
  mag = torch.tensor(E2M1, device=codes.device)[code & 7]
  v = torch.where(code >= 8, -mag, mag)
  s = _pow2(scales.to(torch.int32) - 127).repeat_interleave(BLOCK, dim=1)[:, :k]
  return v * s


def _keep8_values(x):
  """[rows, channels] -> what its 8-bit form stands for, fp32."""
  b = _blocks(x)
  e = _block_exp(b) - 7
  y = b * _pow2(-e)
  step = (torch.frexp(y)[1] - 1).clamp(min=-6) - 3
  v = torch.round(y * _pow2(-step)) * _pow2(step) * _pow2(e)
  return v.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _plain(st):
  case, op = st['case'], st['case']['op']
  x = st['x']
  c, cp = case['channels'], x.shape[-1]
  rows = x.reshape(-1, cp)
  if op in ('norm', 'norm_train'):
    xf = rows[:, :c].float()
    mean = xf.mean(dim=1, keepdim=True)
    d = xf - mean
    inv = torch.rsqrt((d * d).mean(dim=1, keepdim=True) + EPS)
    y = d * inv * st['gamma'] + st['beta']
    slope = case.get('slope', 1.0)
    if slope != 1.0:
      y = torch.where(y > 0, y, slope * y)
    z = torch.nn.functional.pad(y, (0, cp - c)).to(x.dtype).view(x.shape)
    if op == 'norm':
      return z
    if case['keep8']:
      d = _keep8_values(rows)[:, :c] - mean
    h = d * inv
    g = st['gz'].reshape(-1, cp)[:, :c].float()
    t = g * st['gamma']
    gx = inv * (t - t.mean(dim=1, keepdim=True) - h * (t * h).mean(dim=1, keepdim=True))
    gx = torch.nn.functional.pad(gx, (0, cp - c)).to(x.dtype).view(x.shape)
    return z, gx, (g * h).sum(dim=0), g.sum(dim=0)
  if op == 'keep':
    return _keep8_values(rows).to(x.dtype).view(x.shape)
  if op == 'wgrad':
    g = st['gy'].reshape(-1, st['gy'].shape[-1])[:, :case['outputs']].float()
    return torch.matmul(g.t(), _keep8_values(rows)), g.sum(dim=0)
  if op == 'quant':
    return _mx4_values(rows).to(x.dtype).view(x.shape)
  n = case['outputs']
  y = torch.matmul(_mx4_values(rows), _unpack_mx4(st['w_codes'], st['w_scales'], c).t()) + st['bias']
  if case['slope'] != 1.0:
    y = torch.where(y > 0, y, case['slope'] * y)
  return torch.nn.functional.pad(y, (0, _pad8(n) - n)).to(x.dtype).view(x.shape[:3] + (_pad8(n),))


def _own(st):
  ops, case = _ops(), st['case']
  op, x = case['op'], st['x']
  if op == 'norm':
    return ops.layer_norm(x, st['gamma'], st['beta'], EPS, case['slope'])[0]
  if op == 'norm_train':
    z, saved = ops.layer_norm(x, st['gamma'], st['beta'], EPS, keep8=case['keep8'])
    return (z,) + ops.layer_norm_bwd(st['gz'], saved)
  if op == 'keep':
    return ops.act8_restore(ops.act8_save(x))
  if op == 'wgrad':
    return ops.act8_wgrad(ops.act8_save(x), st['gy'], case['outputs'])
  if op == 'quant':
    return ops.mx4_dequantize(ops.mx4_quantize(x), x.dtype)
  return ops.mx4_linear(x, ops.Mx4(st['w_codes'], st['w_scales'], case['channels']), st['bias'], case['slope'])


def run(state):
  return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------------------------------------
# work and exact results
# ----------------------------------------------------------------------------------------------------------------------


def work(case):
  es = 2 if case['dtype'] == 'bf16' else 4
  p, c = _pixels(case), case['channels']
  t = p * _pad8(c) * es                                    # one activation tensor
  kept = p * (_pad8(c) + math.ceil(c / BLOCK))
  op = case['op']
  if op == 'norm':
    return {'bytes': 2 * t + 8 * c, 'flops': 8 * p * c}
  if op == 'norm_train':                                   # x, z, gz, gx (+ what is kept, written and read, for x)
    return {'bytes': 4 * t + (2 * kept if case['keep8'] else t) + 24 * c, 'flops': 20 * p * c}
  if op == 'keep':
    return {'bytes': 2 * t + 2 * kept, 'flops': 4 * p * c}
  if op == 'wgrad':
    n = case['outputs']
    return {'bytes': t + 2 * kept + p * _pad8(n) * es + 4 * n * (c + 1), 'flops': 2 * p * c * n}
  packed = lambda rows: rows * (64 * math.ceil(c / 128) + math.ceil(c / BLOCK))
  if op == 'quant':
    return {'bytes': 2 * t + 2 * packed(p), 'flops': 4 * p * c}
  n = case['outputs']
  return {'bytes': t + packed(n) + 4 * n + p * _pad8(n) * es, 'flops': 2 * p * c * n}


def _nearest(v, table):
  """float64 values -> nearest entry of the non-negative ``table`` with their sign, ties to the entry of even index,
  beyond the last entry: the last."""
  t = torch.tensor(table, dtype=torch.float64, device=v.device)
  mid = (t[1:] + t[:-1]) / 2
  a = v.abs().contiguous()
  i = torch.searchsorted(mid, a)
  tie = (i < mid.numel()) & (mid[i.clamp(max=mid.numel() - 1)] == a) & (i % 2 == 1)
  return torch.copysign(t[i + tie.long()], v)


def _exact_micro(x, table, top):
  """Exact block rounding: scale 2^(floor(log2 of the block's largest magnitude) - top)."""
  rows, c = x.shape
  v = torch.zeros(rows, (c + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64, device=x.device)
  v[:, :c] = x.double()
  v = v.view(rows, -1, BLOCK)
  e = torch.floor(torch.log2(v.abs().amax(dim=2, keepdim=True).clamp(min=2.0 ** MIN_EXP)))
  s = torch.exp2(e - top)
  return (_nearest(v / s, table) * s).view(rows, -1)[:, :c]


def _e4m3_table():
  sub = [i * 2.0 ** -9 for i in range(8)]
  return sub + [(8 + i % 8) * 2.0 ** (i // 8 - 9) for i in range(0, 14 * 8 + 7)]


def exact(case, seed):
  st = prepare(case, seed)
  op, x, c = case['op'], st['x'], case['channels']
  cp = x.shape[-1]
  rows = x.reshape(-1, cp)
  if op == 'keep':
    return _exact_micro(rows, _e4m3_table(), 7).view(x.shape)
  if op == 'quant':
    return _exact_micro(rows, E2M1, 2).view(x.shape)
  if op == 'wgrad':
    g = st['gy'].double().reshape(rows.shape[0], -1)[:, :case['outputs']]
    return torch.mm(g.t().contiguous(), _exact_micro(rows, _e4m3_table(), 7)), g.sum(dim=0)
  if op == 'linear':
    n = case['outputs']
    code = st['w_codes'].view(n, -1, 1).repeat(1, 1, 2)
    code[:, :, 0] %= 16
    code[:, :, 1] //= 16
    code = code.view(n, -1)[:, :c].long()
    w = torch.tensor(E2M1 + tuple(-m for m in E2M1), dtype=torch.float64, device=x.device)[code]
    w = w * torch.exp2(st['w_scales'].double() - 127).repeat_interleave(BLOCK, dim=1)[:, :c]
    y = torch.mm(_exact_micro(rows, E2M1, 2), w.t().contiguous()) + st['bias'].double()
    y = torch.maximum(y, case['slope'] * y)
    out = torch.zeros(rows.shape[0], _pad8(n), dtype=torch.float64, device=x.device)
    out[:, :n] = y
    return out.view(x.shape[:3] + (_pad8(n),))
  xd, gamma = rows[:, :c].double(), st['gamma'].double()
  mean = xd.mean(dim=1, keepdim=True)
  std = torch.sqrt(xd.var(dim=1, keepdim=True, unbiased=False) + EPS)
  y = (xd - mean) / std * gamma + st['beta'].double()
  slope = case.get('slope', 1.0)
  z = torch.zeros(rows.shape, dtype=torch.float64, device=x.device)
  z[:, :c] = torch.maximum(y, slope * y)
  if op == 'norm':
    return z.view(x.shape)
  if case['keep8']:
    xd = _exact_micro(rows, _e4m3_table(), 7)[:, :c]
  h = (xd - mean) / std
  g = st['gz'].double().reshape(rows.shape)[:, :c]
  t = g * gamma
  gx = torch.zeros(rows.shape, dtype=torch.float64, device=x.device)
  gx[:, :c] = (t - t.sum(dim=1, keepdim=True) / c - h * ((t * h).sum(dim=1, keepdim=True) / c)) / std
  return z.view(x.shape), gx.view(x.shape), torch.einsum('pc,pc->c', g, h), g.sum(dim=0)
