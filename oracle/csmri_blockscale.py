"""Plain restatements (CPU, float64) of the block-scaled formats, the layer norm and the products built on them: 32
consecutive channels of a pixel share a power-of-two scale taken from their largest magnitude."""
import torch

BLOCK = 32
MIN_EXP = -100
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [i * 2.0 ** -9 for i in range(8)] + [(8 + i % 8) * 2.0 ** (i // 8 - 9) for i in range(14 * 8 + 7)]


def nearest(v, table):
  """Nearest entry of a non-negative table with the sign of v, ties to the entry of even index, saturating."""
  t = torch.tensor(table, dtype=torch.float64)
  a = v.abs().unsqueeze(-1)
  d = (a - t).abs()
  best = d.min(dim=-1, keepdim=True).values
  hit = d == best
  idx = torch.arange(len(table))
  even = (hit & (idx % 2 == 0)).to(torch.int8).argmax(dim=-1)
  first = hit.to(torch.int8).argmax(dim=-1)
  i = torch.where((hit & (idx % 2 == 0)).any(dim=-1), even, first)
  return i, torch.copysign(t[i], v)


def blocks(x):
  rows, c = x.shape
  return torch.nn.functional.pad(x.double(), (0, (-c) % BLOCK)).view(rows, -(-c // BLOCK), BLOCK)


def block_round(x, table, top):
  """(values, codes, exponents): x [rows, C] rounded block by block with scales 2^(floor(log2 amax) - top); blocks with
  a non-finite value are NaN (code 0, exponent 128)."""
  b = blocks(x)
  amax = b.abs().amax(dim=2, keepdim=True)
  bad = ~torch.isfinite(b).all(dim=2, keepdim=True)
  amax = torch.where(bad, torch.ones_like(amax), amax)
  e = torch.where(amax > 0, torch.frexp(amax).exponent - 1, torch.full_like(amax, MIN_EXP, dtype=torch.int32)).clamp(min=MIN_EXP) - top
  s = torch.exp2(e.double())
  i, v = nearest(torch.where(bad, torch.zeros_like(b), b) / s, table)
  v = torch.where(bad, torch.full_like(v, float('nan')), v * s)
  code = i + (len(table) > 8 and 128 or 8) * torch.signbit(b).long()
  e = torch.where(bad, torch.full_like(e, 128), e)
  return v.flatten(1)[:, :x.shape[1]], code.flatten(1), e[:, :, 0]


def act8(x):
  return block_round(x, E4M3, 7)[0]


def mx4(x):
  return block_round(x, E2M1, 2)[0]


def mx4_pack(x):
  """(codes, scales) bytes of the rows of x, padding included."""
  _, code, e = block_round(x, E2M1, 2)
  code = torch.nn.functional.pad(code, (0, (-code.shape[1]) % 128))
  scale = torch.nn.functional.pad(e + 127, (0, (-e.shape[1]) % 16), value=127)
  code = torch.where(torch.nn.functional.pad(e, (0, code.shape[1] // BLOCK - e.shape[1])).repeat_interleave(BLOCK, 1) == 128,
                     torch.zeros_like(code), code)
  return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8), scale.to(torch.uint8)


def mx4_unpack(codes, scales, k):
  c = codes.long()
  v = torch.stack([c % 16, c // 16], dim=2).reshape(c.shape[0], -1)[:, :k]
  t = torch.tensor(E2M1, dtype=torch.float64)[v % 8]
  s = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)[:, :k]
  bad = (scales == 255).repeat_interleave(BLOCK, 1)[:, :k]
  return torch.where(bad, torch.full_like(t, float('nan')), torch.where(v >= 8, -t, t) * s)


def layer_norm(x, gamma, beta, eps, slope):
  """(z, h, mean, r) for rows x of real channels only."""
  x = x.double()
  mean = x.mean(1, keepdim=True)
  r = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
  h = (x - mean) * r
  y = h * gamma.double() + beta.double()
  return torch.where(y > 0, y, slope * y), h, mean, r


def layer_norm_bwd(gz, h, r, gate, gamma):
  """(gx, dgamma, dbeta); gate: 1 or slope."""
  g = gz.double() * gate
  t = g * gamma.double()
  gx = r * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
  return gx, (g * h).sum(0), g.sum(0)
