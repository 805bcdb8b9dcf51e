"""How near differential attention's bf16 gradients come to the formula in 64 bits where sums or maps cancel: lambda's gradient, which is one sum
over all rows of a head, and maps that have most of their result in common."""
import math

import pytest
import torch

from test_transformer_ops_gpu import BF16, DEV, F32, attn_inputs, attn_visible, ops, randn  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


def formula(q, k, v, dout, lam, keep, eps=1e-5):
  """Gradients in 64 bits, heads one by one, and for each head the root of the summed squares of the rows' terms of dlambda."""
  H, Hkv, d = q.shape[2], k.shape[2], q.shape[4]
  res = dict(dq=torch.zeros(q.shape, dtype=torch.float64, device=DEV), dk=torch.zeros(k.shape, dtype=torch.float64, device=DEV), dv=torch.zeros(v.shape, dtype=torch.float64, device=DEV),
             dw=torch.zeros(v.shape[-1], dtype=torch.float64, device=DEV), dlam=torch.zeros(H, dtype=torch.float64, device=DEV), root=torch.zeros(H, dtype=torch.float64, device=DEV))
  for h in range(H):
    g, L = h // (H // Hkv), float(lam[h if lam.numel() > 1 else 0])
    V, u = v[:, :, g].double(), dout[:, :, h].double()
    P = []
    for i in (0, 1):
      s = torch.matmul(q[:, :, h, i].double(), k[:, :, g, i].double().transpose(1, 2).contiguous()) * d ** -0.5
      P.append(torch.nan_to_num(torch.softmax(s.masked_fill(~keep, -math.inf), 2), nan=0.0))
    o = [torch.matmul(p, V) for p in P]
    O = o[0] - L * o[1]
    r = 1.0 / torch.sqrt(O.pow(2).mean(2, keepdim=True) + eps)
    dO = r * u - O * r ** 3 * (u * O).mean(2, keepdim=True)
    terms = (dO * o[1]).sum(2)
    res['dlam'][h], res['root'][h] = -terms.sum(), terms.norm()
    res['dw'] += (u * O * r).sum((0, 1))
    dP = torch.matmul(dO, V.transpose(1, 2).contiguous())
    for i, f in ((0, 1.0), (1, -L)):
      dS = f * P[i] * (dP - (dO * o[i]).sum(2, keepdim=True)) * d ** -0.5
      res['dq'][:, :, h, i] = torch.matmul(dS, k[:, :, g, i].double())
      res['dk'][:, :, g, i] += torch.matmul(dS.transpose(1, 2).contiguous(), q[:, :, h, i].double())
    res['dv'][:, :, g] += torch.matmul((P[0] - L * P[1]).transpose(1, 2).contiguous(), dO)
  return res


@pytest.mark.parametrize('shape', [(1, 300, 512, 2, 1, 64, 128), (1, 300, 512, 1, 1, 16, 32), (1, 260, 512, 1, 1, 128, 256), (1, 300, 512, 2, 2, 27, 54)], ids=str)
@pytest.mark.parametrize('lam', [0.8, 0.95, 1.0])
def test_diff_attention_gradients_of_maps_with_a_common_part(ops, shape, lam):
  """V has mean one, lambda is near one: O is several times smaller than O_1 and O_2, which may not bring their roundings into it.  Relative in the
  2-norm, with s = 2^-8 / sqrt(3) = 2.3e-3 the largest deviation of one rounding to bf16: dnorm_weight has O as saved (s), the roundings of P in it
  (sqrt(E V^2) s = 1.4 s: O consists of V's varying part alone) and its own, 2.0 s = 4.5e-3: 6e-3 allowed for, since it is the size of a few numbers.  dv has
  dO, P_1 - P_2 and its own rounding, and dO's error by O (1.7 s), 2.4 s = 5.4e-3: 6.5e-3.  dq and dk: dO, dS, their own, delta by O_2 (1.4 s twice) and dO's error
  by O (1.7 s), 3.2 s = 7.2e-3: 9e-3."""
  q, k, v, dout, _ = attn_inputs(*shape, BF16, seed=400)
  v = (v.float() + 1.0).to(BF16)
  lam = torch.full((shape[3],), lam, device=DEV)
  w = torch.ones(shape[6], device=DEV)
  want = formula(q, k, v, dout, lam, attn_visible(shape[0], shape[1], shape[2]))
  _, ctx = ops.diff_attn_fwd(q, k, v, lam, norm_weight=w, save=True)
  got = dict(zip(('dq', 'dk', 'dv', 'dlam', 'dw'), ops.diff_attn_bwd(dout, q, k, v, lam, ctx)))
  off = {n: float((got[n].double() - want[n]).norm() / want[n].norm()) for n in ('dq', 'dk', 'dv', 'dw')}
  assert off['dw'] <= 6e-3 and off['dv'] <= 6.5e-3 and off['dq'] <= 9e-3 and off['dk'] <= 9e-3, off


@pytest.mark.parametrize('B,T,causal,ragged', [(1, 230, False, False), (2, 333, True, False), (12, 16, True, True), (3, 200, False, True)])
@pytest.mark.parametrize('d', [9, 16, 27, 32, 64, 72, 128])
def test_diff_attention_lambda_gradient_is_free_of_first_order_roundings(ops, d, B, T, causal, ragged):
  """dlambda is a sum over all rows that cancels: the roundings of P and of the saved results may reach it in second order only, both where they stand
  beside dO and through O, which dO is made of.  A row's O is off by at most 2^-8 / sqrt(3) * sqrt(2 + 1) = 3.9e-3 relative (P of both maps, the saved value), a
  deviation; the second derivative of a row's term is at most a few times the term over |O|^2, so that the row is off by some 1e-4 of itself, and the rows'
  signs are independent: 2.5e-4 of the root of the terms' squares is allowed, which also is 2.5e-3 of dlambda wherever it is more than a tenth of that root.
  fp32 sums are 1e-6 of it."""
  for H, one in ((1, False), (2, False), (2, True)):
    for seed in range(20):
      q, k, v, dout, _ = attn_inputs(B, T, T, H, 1, d, 2 * d, BF16, seed=1000 + 10 * seed)
      lam = ops.diff_lambda(*[randn(1 if one else H, d, seed=2000 + 4 * seed + i, std=0.1) for i in range(4)], 0.3555)
      lens = torch.randint(1, T + 1, (B,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).to(DEV) if ragged else None
      _, ctx = ops.diff_attn_fwd(q, k, v, lam, causal=causal, kv_len=lens, out_scale=0.65, save=True)
      got = ops.diff_attn_bwd(dout, q, k, v, lam, ctx)[3].double()
      want = formula(q, k, v, 0.65 * dout.double(), lam, attn_visible(B, T, T, causal=causal, kv_len=lens))
      value, root = (want['dlam'].sum().view(1), want['root'].norm().view(1)) if one else (want['dlam'], want['root'])
      assert ((got - value).abs() <= 2.5e-4 * root).all(), (H, one, seed, ((got - value).abs() / root).tolist(), (value.abs() / root).tolist())
