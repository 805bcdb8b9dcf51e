"""GPU tests of the transformer-block operators (-m gpu) against plain implementations in 64 bits: gradient norm and clipping (ops.GradClip,
optim.clip_grad_norm_, Trainer's max_grad_norm), block norms (ops.block_norm_fwd / _bwd), differential attention (ops.diff_attn_fwd / _bwd).

Tolerances are componentwise: half a step of the output's type relative to the value, plus K fp32 roundings (2^-24 each) of the same
formula evaluated with absolute values -- a running error bound; K counts the roundings on the longest path of one output."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
F32, BF16 = torch.float32, torch.bfloat16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


@pytest.fixture(scope='module')
def ops():
  from carla_garage_amd import ops as m
  return m


def randn(*shape, dtype=F32, seed=0, std=1.0, mean=0.0):
  g = torch.Generator().manual_seed(1000 * seed + sum(shape) + len(shape))
  return (torch.randn(*shape, generator=g) * std + mean).to(dtype).to(DEV)


def within(name, got, want, tol):
  got, want = got.double(), want.double()
  tol = tol.double() if torch.is_tensor(tol) else torch.full_like(want, tol)
  assert got.shape == want.shape, (name, got.shape, want.shape)
  assert torch.isfinite(got).all(), f'{name}: not finite'
  over = (got - want).abs() - tol
  assert not (over > 0).any(), f'{name}: off by {float((got - want).abs().max()):.3e} where {float(tol.flatten()[over.argmax()]):.3e} is allowed'


# ------------------------------------------------------------------------------------------------ gradient norm and clipping
def clip_want(grads, max_norm, p, scale):
  flat = torch.cat([g.double().flatten() for g in grads] + [torch.zeros(1, dtype=torch.float64, device=DEV)]) * scale
  norm = flat.abs().max() if p == math.inf else (flat.abs().sum() if p == 1 else flat.pow(2).sum().sqrt())
  c = max_norm / (norm + 1e-6)
  return norm, torch.where(c > 1.0, torch.ones_like(c), c)


@pytest.mark.parametrize('p', [2.0, 1.0, math.inf])
@pytest.mark.parametrize('dtype,odtype', [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize('sizes', [(1,), (0, 3, 0), (7, 16384, 16385, 1, 50000), (3,) * 2500], ids=['one', 'empty', 'ragged', 'many'])
def test_clip_matches_64_bits(ops, sizes, dtype, odtype, p):
  grads = [randn(n, dtype=dtype, seed=i, std=10.0 ** (i % 5 - 2)) for i, n in enumerate(sizes)]
  keep = [g.clone() for g in grads]
  for max_norm, scale in ((0.5, 0.25), (1.0e9, 1.0)):
    out = [torch.full_like(g, 7.0, dtype=odtype) for g in grads]
    plan = ops.GradClip(grads, out=out)
    norm = plan.clip_(max_norm, norm_type=p, grad_scale=scale)
    want, c = clip_want(grads, max_norm, p, scale)
    # partials and sums are double: the norm is rounded once; coefficient: max_norm / (norm + 1e-6), two more fp32 roundings, then one per product
    within('norm', norm, want, 2 * U[F32] * want.abs())
    for g, k, o in zip(grads, keep, out):
      w = g.double() * scale * c
      within('out', o, w, (U[odtype] + 8 * U[F32]) * w.abs() + 2.0 ** -133)  # (2^-133: half a step of the smallest bf16)
      assert torch.equal(g, k)
    assert torch.equal(norm, plan.norm(norm_type=p, grad_scale=scale))
    n2, c2 = plan.coef(max_norm, norm_type=p, grad_scale=scale)
    assert torch.equal(n2, norm)
    within('coef', c2, c, 8 * U[F32])


def test_clip_in_place_views_layouts_and_neighbours(ops):
  """Odd offsets (no 16-byte alignment), channels-last weights, neighbours in the same buffer that are not in the list stay as they were."""
  flat = randn(1000, seed=1)
  guard = flat.clone()
  w = randn(8, 6, 3, 3, seed=2).to(memory_format=torch.channels_last)
  w0 = w.clone(memory_format=torch.preserve_format)
  t = randn(5, 7, seed=3).t()
  t0 = t.clone(memory_format=torch.preserve_format)
  views = [flat[1:18], flat[21:22], flat[23:991]]
  norm = ops.GradClip(views + [w, t]).clip_(0.5)
  want, c = clip_want([guard[1:18], guard[21:22], guard[23:991], w0, t0], 0.5, 2.0, 1.0)
  within('norm', norm, want, 2 * U[F32] * want)
  for got, old in ((flat[1:18], guard[1:18]), (flat[21:22], guard[21:22]), (flat[23:991], guard[23:991]), (w, w0), (t, t0)):
    within('clipped', got, old.double() * c, 8 * U[F32] * old.abs())
  hole = torch.ones(1000, dtype=torch.bool, device=DEV)
  for a, b in ((1, 18), (21, 22), (23, 991)):
    hole[a:b] = False
  assert torch.equal(flat[hole], guard[hole])


def test_clip_below_the_norm_leaves_every_bit(ops):
  g = [randn(70001, seed=4), randn(33, dtype=BF16, seed=5)]
  keep = [x.clone() for x in g]
  ops.GradClip(g).clip_(1.0e6)
  assert all(torch.equal(a, b) for a, b in zip(g, keep))


def test_clip_magnitudes_whose_squares_leave_fp32(ops):
  for mag in (1.0e-30, 1.0e30):
    g = [randn(5000, seed=6) * mag]
    want, c = clip_want(g, mag, 2.0, 1.0)
    got = ops.GradClip(g, out=[torch.empty_like(g[0])]).clip_(mag)
    within('norm', got, want, 2 * U[F32] * want)


@pytest.mark.parametrize('p', [2.0, 1.0, math.inf])
@pytest.mark.parametrize('bad', [math.nan, math.inf])
def test_clip_non_finite_as_torch(ops, p, bad):
  g = [randn(300, seed=7), randn(40000, seed=8)]
  g[1][39999] = bad
  ref = [torch.nn.Parameter(torch.zeros_like(x)) for x in g]
  for r, x in zip(ref, g):
    r.grad = x.clone()
  want = torch.nn.utils.clip_grad_norm_(ref, 1.0, norm_type=p, foreach=False)
  norm = ops.GradClip(g).clip_(1.0, norm_type=p)
  assert torch.equal(torch.isnan(norm), torch.isnan(want)) and torch.equal(torch.isinf(norm), torch.isinf(want))
  for r, x in zip(ref, g):
    np.testing.assert_array_equal(torch.isnan(x).cpu().numpy(), torch.isnan(r.grad).cpu().numpy())
    assert torch.equal(torch.nan_to_num(x) == 0, torch.nan_to_num(r.grad) == 0)


def test_clip_grad_norm_function(ops):
  from carla_garage_amd.optim import clip_grad_norm_
  ps = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (10, 3, 4000, 8)]
  for i, q in enumerate(ps[:3]):
    q.grad = randn(q.numel(), seed=10 + i)
  g0 = [q.grad.clone() for q in ps[:3]]
  want, c = clip_want(g0, 2.0, 2.0, 1.0)
  within('norm', clip_grad_norm_(iter(ps), 2.0, error_if_nonfinite=True), want, 2 * U[F32] * want)
  for q, g in zip(ps, g0):
    within('grad', q.grad, g.double() * c, 8 * U[F32] * g.abs())
  assert ps[3].grad is None
  ps[0].grad[3] = math.nan
  keep = ps[1].grad.clone()
  with pytest.raises(RuntimeError, match='non-finite'):
    clip_grad_norm_(ps, 2.0, error_if_nonfinite=True)
  assert torch.equal(ps[1].grad, keep)
  assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(2, device=DEV))], 1.0)) == 0.0


def test_clip_refusals(ops):
  x = randn(64)
  for bad in ([], [x.cpu()], [x.half()], [x[::2]], [x, x], [x[:40], x[30:]], [x.expand(2, 64)]):
    with pytest.raises((ValueError, TypeError)):
      ops.GradClip(bad)
  for out in ([], [torch.empty(63, device=DEV)], [x[1:].new_empty(64).half()], [torch.empty(8, 8, device=DEV)]):
    with pytest.raises((ValueError, TypeError)):
      ops.GradClip([x], out=out)
  y = randn(8, 8)
  with pytest.raises(ValueError):
    ops.GradClip([y], out=[torch.empty_like(y).t()])
  with pytest.raises(ValueError):
    ops.GradClip([x[:32], x[32:]], out=[x[32:], torch.empty(32, device=DEV)])
  with pytest.raises(ValueError):
    ops.GradClip([x]).clip_(1.0, norm_type=3)
  for m in (-1.0, math.nan):
    with pytest.raises(ValueError):
      ops.GradClip([x]).clip_(m)
  ops.GradClip([x, x], out=[torch.empty_like(x), torch.empty_like(x)]).clip_(1.0)  # (reading twice is fine)


def test_clip_captured_replays_and_two_graphs_share_nothing(ops):
  """Two captures of the same calls, replayed in turn and side by side on two streams with eager calls in between: every replay equals the eager result."""
  src = [randn(n, seed=20 + n) for n in (5, 70000, 333)]
  outs = [[torch.empty_like(x) for x in src] for _ in range(3)]
  plans = [ops.GradClip(src, out=o) for o in outs]
  graphs, norms = [], []
  side = torch.cuda.Stream()
  for k in (0, 1):
    plans[k].clip_(0.3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
      norms.append(plans[k].clip_(0.3))
    graphs.append(g)
  for step in range(4):
    for i, x in enumerate(src):
      x.copy_(randn(x.numel(), seed=40 + 7 * step + i))
    n2 = plans[2].clip_(0.3)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.current_stream()]
    for g, s in zip(graphs, streams):
      with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    for k in (0, 1):
      assert torch.equal(norms[k], n2)
      assert all(torch.equal(a, b) for a, b in zip(outs[k], outs[2]))


def test_adamw_takes_the_clipping_coefficient(ops):
  n = 5003
  g = randn(n, seed=50)
  res = []
  for fused in (False, True):
    p, m, v, vm = randn(n, seed=51), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    if fused:
      _, c = ops.GradClip([g]).coef(0.1, grad_scale=0.5)
      ops.adamw_amsgrad(p, g, m, v, vm, 1e-2, 0.9, 0.999, 1e-8, 0.01, 1, grad_scale=0.5, grad_coef=c)
    else:
      h = torch.empty_like(g)
      ops.GradClip([g], out=[h]).clip_(0.1, grad_scale=0.5)
      ops.adamw_amsgrad(p, h, m, v, vm, 1e-2, 0.9, 0.999, 1e-8, 0.01, 1)
    res.append((p, m, v))
  for a, b, k in zip(res[0], res[1], (8, 8, 16)):  # (the coefficient is rounded into the product in another place: a few roundings of each value)
    within('adamw', a, b.double(), k * U[F32] * b.abs() + (1e-2 * 16 * U[F32] if a is res[0][0] else 0.0))


# ------------------------------------------------------------------------------------------------ block norms
def norm_oracle(x, a, kind, o, gate, act, alpha, eps, dy=None, dh=None, mags=False):
  """fp64; with ``mags`` the same formulas over absolute values (running error magnitudes).  gate broadcast to x's shape by the caller."""
  A = torch.abs if mags else (lambda z: z)
  sub = (lambda p, q: p + q) if mags else (lambda p, q: p - q)
  mean_abs = lambda z: A(z).amax(-1, keepdim=True) if mags else z.mean(-1, keepdim=True)
  layer = kind == 'layer'

  def stats(z, true):
    zc = true - true.mean(-1, keepdim=True) if layer else true
    r = 1.0 / torch.sqrt(zc.pow(2).mean(-1, keepdim=True) + eps)
    n = zc * r
    return n, r, ((sub(A(z), mean_abs(z)) if layer else A(z)) * r if mags else n)

  g = None if gate is None else {0: lambda z: z, 2: torch.sigmoid, 4: torch.tanh}[act](gate)
  w = lambda k, none: torch.full((x.shape[-1],), none, dtype=torch.float64, device=DEV) if o.get(k) is None else o[k].double()
  sc, gg = w('scale', 1.0), (torch.ones_like(x) if g is None else g)
  res = {}
  if o.get('post', True):
    an, ar, am = stats(a, a)
    n, nm = an * w('post_weight', 1.0) + w('post_bias', 0.0), A(am) * A(w('post_weight', 1.0)) + A(w('post_bias', 0.0))
  else:
    an, ar, n, nm = a, None, a, A(a)
    am = A(a)
  y = alpha * x + sc * gg * n
  ym = A(alpha * x) + A(sc) * A(gg) * nm
  res['y'] = ym if mags else y
  if o.get('pre', True):
    yn, yr, yhm = stats(ym, y)
    res['h'] = (A(yhm) * A(w('pre_weight', 1.0)) + A(w('pre_bias', 0.0))) if mags else yn * w('pre_weight', 1.0) + w('pre_bias', 0.0)
  if dy is None and dh is None:
    return res
  d = torch.zeros_like(x) if dy is None else A(dy)

  def back(dz, zn, zm, r):
    zz = zm if mags else zn
    m1 = A(dz).mean(-1, keepdim=True) if layer else 0.0
    return r * sub(sub(A(dz), m1), A(zz) * (A(dz) * A(zz)).mean(-1, keepdim=True)) if mags else r * (dz - (dz.mean(-1, keepdim=True) if layer else 0.0) - zn * (dz * zn).mean(-1, keepdim=True))

  if dh is not None:
    d = d + back(dh * w('pre_weight', 1.0), yn, yhm, yr)
    res['pre_weight'] = (A(dh) * (A(yhm) if mags else yn)).flatten(0, -2).sum(0)
    res['pre_bias'] = A(dh).flatten(0, -2).sum(0)
  elif o.get('pre', True):
    res['pre_weight'] = res['pre_bias'] = torch.zeros(x.shape[-1], dtype=torch.float64, device=DEV)
  res['x'] = A(alpha * d)
  dn = d * A(sc) * A(gg)
  if g is not None:
    slope = {0: lambda z: torch.ones_like(z), 2: lambda z: z * (1 - z), 4: lambda z: (1 - z * z) if not mags else (1 + z * z)}[act](gg)
    res['gate'] = d * A(sc) * (nm if mags else n) * slope
  res['scale'] = (d * A(gg) * (nm if mags else n)).flatten(0, -2).sum(0)
  if o.get('post', True):
    res['a'] = back(dn * A(w('post_weight', 1.0)), an, am, ar)
    res['post_weight'], res['post_bias'] = (dn * (A(am) if mags else an)).flatten(0, -2).sum(0), dn.flatten(0, -2).sum(0)
  else:
    res['a'] = dn
  return res


# longest path of one output: row sums of <= 8 serial + 6 shuffle + 3 wave additions, twice in each of four norms (statistics, sums of the backward),
# the exponential of the gate (<= 16 roundings for |gate| < 8) and ~16 pointwise steps; column sums add their own serial length (below)
K_NORM = 4 * 2 * 17 + 16 + 16


def run_norm(ops, shape, dtype, kind, gate_kind, act=2, seed=0, alpha=1.0, strides=False, **o):
  C = shape[-1]
  wide = lambda *s, **k: randn(*s[:-1], s[-1] + 24, **k)[..., 8:8 + s[-1]] if strides else randn(*s, **k)
  x, a = wide(*shape, dtype=dtype, seed=seed + 1, std=2.0), wide(*shape, dtype=dtype, seed=seed + 2, std=0.5, mean=0.2)
  gate = None
  if gate_kind == 'token':
    gate = wide(*shape, dtype=dtype, seed=seed + 3)
  elif gate_kind == 'sample':
    gate = randn(shape[0], C, dtype=dtype, seed=seed + 3)
  dy, dh = wide(*shape, dtype=dtype, seed=seed + 4), wide(*shape, dtype=dtype, seed=seed + 5)
  y, h, ctx = ops.block_norm_fwd(x, a, kind=kind, gate=gate, gate_act=act if gate is not None else 0, alpha=alpha, **o)
  use_dh = dh if o.get('pre', True) else None
  into = {n: torch.ones(C, device=DEV) for n in ('scale', 'post_weight') if o.get(n) is not None}
  gr = ops.block_norm_bwd(dy, use_dh, ctx, into=into)
  full = None if gate is None else (gate.double().view(shape[0], *([1] * (len(shape) - 2)), C).expand(*shape) if gate_kind == 'sample' else gate.double())
  args = (kind, o, full, act if gate is not None else 0, alpha, 1e-5)
  dh64 = None if use_dh is None else dh.double()
  want = norm_oracle(x.double(), a.double(), *args, dy=dy.double(), dh=dh64)
  mag = norm_oracle(x.double(), a.double(), *args, dy=dy.double(), dh=dh64, mags=True)
  rows = x.numel() // C
  got = dict(gr, y=y, h=h)
  for n, g in got.items():
    if g is None or n not in want:
      assert g is None or n in ('gate',), n
      continue
    w, m = want[n], mag[n]
    if n == 'gate' and gate_kind == 'sample':
      w, m = (z.reshape(shape[0], -1, C).sum(1) for z in (w, m))
    k = K_NORM
    if n in ('scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias') or (n == 'gate' and gate_kind == 'sample'):
      k += min(rows, 4 + rows // 512 + 600)  # serial additions of one workgroup's rows and of one slice of the partials
    if n in into:
      w, m = w + 1.0, m + 1.0
    within(n, g, w.view(g.shape), (U[g.dtype] * w.abs() + k * U[F32] * m).view(g.shape))


def full_params(C, layer, seed=60):
  o = dict(scale=randn(C, seed=seed, std=0.3, mean=0.5), post_weight=randn(C, seed=seed + 1, std=0.2, mean=1.0), pre_weight=randn(C, seed=seed + 2, std=0.2, mean=1.0))
  if layer:
    o.update(post_bias=randn(C, seed=seed + 3, std=0.2), pre_bias=randn(C, seed=seed + 4, std=0.2))
  return o


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('kind', ['layer', 'rms'])
@pytest.mark.parametrize('gate', ['none', 'sample', 'token'])
@pytest.mark.parametrize('shape', [(1, 1, 8), (2, 3, 27), (3, 50, 72), (12, 20, 576), (2, 129, 1512), (1, 40, 2048), (2, 9, 4096), (1, 3, 4095)], ids=str)
def test_block_norm_forward_and_gradients(ops, shape, gate, kind, dtype):
  run_norm(ops, shape, dtype, kind, gate, **full_params(shape[-1], kind == 'layer'))


@pytest.mark.parametrize('o', [dict(post=False), dict(pre=False), dict(post=False, pre=False), dict()], ids=['no-post', 'no-pre', 'neither', 'no-parameters'])
@pytest.mark.parametrize('act', [0, 4])
def test_block_norm_parts(ops, o, act):
  run_norm(ops, (4, 33, 216), BF16, 'layer', 'token', act=act, alpha=0.7, **o)
  run_norm(ops, (4, 33, 216), F32, 'rms', 'sample', act=act, alpha=0.7, **o)


def test_block_norm_slices_of_wider_rows(ops):
  run_norm(ops, (3, 20, 64), BF16, 'layer', 'token', strides=True, **full_params(64, True))
  run_norm(ops, (3, 20, 61), F32, 'rms', 'none', strides=True, **full_params(61, False))


def test_block_norm_one_gradient_only(ops):
  """dh alone (the residual stream ends here) and dy alone equal the pair with zeros in the other place."""
  o = full_params(96, True)
  x, a, g = randn(2, 10, 96, dtype=BF16, seed=70), randn(2, 10, 96, dtype=BF16, seed=71), randn(2, 96, dtype=BF16, seed=72)
  _, _, ctx = ops.block_norm_fwd(x, a, gate=g, gate_act=2, **o)
  d, z = randn(2, 10, 96, dtype=BF16, seed=73), torch.zeros(2, 10, 96, dtype=BF16, device=DEV)
  for one, two in (((d, None), (d, z)), ((None, d), (z, d))):
    p, q = ops.block_norm_bwd(*one, ctx), ops.block_norm_bwd(*two, ctx)
    for n in p:
      assert (p[n] is None and q[n] is None) or torch.equal(p[n], q[n]), n


def test_block_norm_gradient_against_differences(ops):
  """Directional derivatives of the 64-bit forward by central differences (step 1e-5: truncation ~1e-10 of the third derivative)."""
  C = 48
  o = full_params(C, True)
  x, a, g = randn(2, 5, C, seed=80), randn(2, 5, C, seed=81), randn(2, 5, C, seed=82)
  dy, dh = randn(2, 5, C, seed=83).double(), randn(2, 5, C, seed=84).double()
  _, _, ctx = ops.block_norm_fwd(x, a, gate=g, gate_act=2, **o)
  gr = ops.block_norm_bwd(dy.float(), dh.float(), ctx)
  base = dict(x=x, a=a, gate=g, **o)

  def loss(v):
    r = norm_oracle(v['x'], v['a'], 'layer', {k: v[k] for k in o}, v['gate'], 2, 1.0, 1e-5)
    return (r['y'] * dy).sum() + (r['h'] * dh).sum()

  for n in base:
    direction = randn(*base[n].shape, seed=90).double()
    v = {k: t.double() for k, t in base.items()}
    e = 1e-5
    num = (loss({**v, n: v[n] + e * direction}) - loss({**v, n: v[n] - e * direction})) / (2 * e)
    want = (gr[n].double() * direction).sum()
    # each gradient element is within K_NORM fp32 roundings of magnitudes below ~50 here
    assert abs(float(num - want)) <= K_NORM * U[F32] * 50 * float(direction.abs().sum()) + 1e-6 * abs(float(num)), (n, float(num), float(want))


def test_block_norm_constant_rows_are_exact_zeros(ops):
  x = torch.zeros(1, 4, 64, device=DEV)
  y, h, ctx = ops.block_norm_fwd(x, torch.full_like(x, 3.0))
  assert not y.any() and not h.any()
  gr = ops.block_norm_bwd(torch.ones_like(x), torch.ones_like(x), ctx)
  assert all(torch.isfinite(t).all() for t in gr.values() if t is not None)


def test_block_norm_empty_and_refusals(ops):
  e = torch.empty(0, 5, 32, device=DEV)
  y, h, ctx = ops.block_norm_fwd(e, e, scale=torch.ones(32, device=DEV))
  assert y.shape == e.shape and not ops.block_norm_bwd(e, e, ctx)['scale'].any()
  x = randn(2, 3, 32)
  bad = [dict(x=x.half(), a=x.half()), dict(a=x.bfloat16()), dict(a=x[:, :2]), dict(x=x.cpu(), a=x.cpu()), dict(kind='batch'), dict(gate=x[0]), dict(gate=x, gate_act=1),
         dict(scale=torch.ones(31, device=DEV)), dict(scale=torch.ones(32, device=DEV, dtype=BF16)), dict(pre=False, pre_weight=torch.ones(32, device=DEV)),
         dict(x=randn(1, 4097), a=randn(1, 4097)), dict(x=randn(2, 32, 3).transpose(1, 2)), dict(x=randn(32).expand(2, 3, 32))]
  for kw in bad:
    kw = {'x': x, 'a': x, **kw}
    with pytest.raises((ValueError, TypeError)):
      ops.block_norm_fwd(kw.pop('x'), kw.pop('a'), **kw)
  _, _, ctx = ops.block_norm_fwd(x, x, pre=False)
  for args in ((None, None), (x, x), (x.bfloat16(), None), (x[:1], None)):
    with pytest.raises((ValueError, TypeError)):
      ops.block_norm_bwd(*args, ctx)
  with pytest.raises(ValueError):
    ops.block_norm_bwd(x, None, ctx, into=dict(scale=torch.zeros(32, device=DEV)))


def test_block_norm_captured(ops):
  o = full_params(576, True)
  x, a, g = (randn(2, 40, 576, dtype=BF16, seed=100 + i) for i in range(3))
  dy, dh = randn(2, 40, 576, dtype=BF16, seed=110), randn(2, 40, 576, dtype=BF16, seed=111)

  def step():
    y, h, ctx = ops.block_norm_fwd(x, a, gate=g, gate_act=2, **o)
    return [y, h] + [t for t in ops.block_norm_bwd(dy, dh, ctx).values() if t is not None]

  step()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    outs = step()
  for k in range(3):
    x.copy_(randn(2, 40, 576, dtype=BF16, seed=120 + k))
    want = step()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, want))


# ------------------------------------------------------------------------------------------------ differential attention
E32 = 2.0 ** -24


def attn_visible(B, Tq, Tk, causal=False, kv_len=None, key_mask=None, q_start=None):
  """[B, Tq, Tk] bool."""
  j = torch.arange(Tk, device=DEV)
  keep = torch.ones(B, Tq, Tk, dtype=torch.bool, device=DEV)
  if kv_len is not None:
    keep &= (j < kv_len[:, None])[:, None]
  if key_mask is not None:
    keep &= (key_mask != 0)[:, None]
  if causal:
    start = torch.full((B,), Tk - Tq, device=DEV) if q_start is None else (q_start if torch.is_tensor(q_start) else torch.full((B,), q_start, device=DEV))
    keep &= j <= (start[:, None] + torch.arange(Tq, device=DEV))[..., None]
  return keep


def attn_oracle(q, k, v, lam, keep, dout=None, scale=None, norm=True, w=None, eps=1e-5, c=1.0):
  """{name: (value, allowed error)} in 64 bits.  Errors: first-order propagation of every rounding of the kernels, worst case: U of the storage type for
  P, O_i, dO, dS, P_1 - lam P_2 and the result; 2^-24 times the length of a sum for fp32 accumulation; the scores' error enters P relatively."""
  u = U[q.dtype]
  ut = u if q.dtype == BF16 else 0.0  # fp32 operands are not rounded on their way into a product
  B, Tq, H, _, d = q.shape
  Tk, Hkv, dv = k.shape[1], k.shape[2], v.shape[3]
  scale = d ** -0.5 if scale is None else scale
  G = H // Hkv
  res = {n: torch.zeros(s, dtype=torch.float64, device=DEV) for n, s in
         (('out', (B, Tq, H, dv)), ('dq', q.shape), ('dk', k.shape), ('dv', v.shape), ('dlam', (H,)), ('dw', (dv,)))}
  err = {n: torch.zeros_like(t) for n, t in res.items()}
  W = torch.ones(dv, dtype=torch.float64, device=DEV) if w is None else w.double()
  for b in range(B):
    for h in range(H):
      g = h // G
      seen = keep[b].any(0)  # (values of keys that nobody sees may be anything)
      K = torch.where(seen[:, None, None], k[b, :, g].double(), 0.0)
      V = torch.where(seen[:, None], v[b, :, g].double(), 0.0)
      L = float(lam[h if lam.numel() > 1 else 0])
      P, eP, o, eo = [], [], [], []
      for i in (0, 1):
        Q = q[b, :, h, i].double()
        s = (Q @ K[:, i].T * scale).masked_fill(~keep[b], -math.inf)
        p = torch.nan_to_num(torch.softmax(s, 1), nan=0.0)
        mags = (Q.abs() @ K[:, i].abs().T * scale).masked_fill(~keep[b], 0.0).amax(1, keepdim=True)
        P.append(p)
        eP.append(2 * (d + 40) * E32 * mags + (Tk + 64) * E32)  # relative: both scores and maximum, the exponential, the sum
        o.append(p @ V)
        eo.append((eP[i] + ut + (Tk + 16) * E32) * (p @ V.abs()))
      O, eO = o[0] - L * o[1], eo[0] + abs(L) * eo[1] + 4 * E32 * (o[0].abs() + abs(L * o[1]))
      r = 1.0 / torch.sqrt(O.pow(2).mean(1, keepdim=True) + eps) if norm else torch.ones_like(O[:, :1])
      dr = lambda e: (r ** 3 * (O.abs() * e).mean(1, keepdim=True) + dv * E32 * r) if norm else 0.0 * r
      res['out'][b, :, h] = c * O * r * W
      err['out'][b, :, h] = abs(c) * W.abs() * (eO * r + O.abs() * dr(eO)) + (u + 8 * E32) * (c * O * r * W).abs()
      if dout is None:
        continue
      t = c * W * dout[b, :, h].double()
      eoS = [e + ut * x.abs() for e, x in zip(eo, o)]  # as stored
      eOS = eoS[0] + abs(L) * eoS[1] + 4 * E32 * (o[0].abs() + abs(L * o[1]))
      der, D = dr(eOS), dout[b, :, h].double().abs() * abs(c)
      if norm:
        m, ma = (t * O).mean(1, keepdim=True), (t * O).abs().mean(1, keepdim=True)
        dO = r * t - O * r ** 3 * m
        edO = der * t.abs() + r ** 3 * ma * eOS + 3 * r ** 2 * der * O.abs() * ma + O.abs() * r ** 3 * (t.abs() * eOS).mean(1, keepdim=True) + (dv + 32) * E32 * (r * t.abs() + O.abs() * r ** 3 * ma)
      else:
        dO, edO = t, 8 * E32 * t.abs()
      res['dw'] += (c * dout[b, :, h].double() * O * r).sum(0)
      err['dw'] += (D * (eOS * r + O.abs() * der)).sum(0) + (B * Tq * H + 16) * E32 * (D * O.abs() * r).sum(0)
      res['dlam'][h] -= (dO * o[1]).sum()
      err['dlam'][h] += (edO * o[1].abs() + dO.abs() * eoS[1]).sum() + (B * Tq + 300) * E32 * (dO * o[1]).abs().sum()
      edO = edO + ut * dO.abs()
      dP, edP = dO @ V.T, edO @ V.abs().T + (dv + 8) * E32 * (dO.abs() @ V.abs().T)
      for i, f in ((0, 1.0), (1, -L)):
        delta = (dO * o[i]).sum(1, keepdim=True)
        ed = (edO * o[i].abs() + dO.abs() * eoS[i]).sum(1, keepdim=True) + (dv + 8) * E32 * (dO * o[i]).abs().sum(1, keepdim=True)
        dS = f * P[i] * (dP - delta)
        eS = abs(f) * P[i] * (edP + ed) + (eP[i] + ut + 8 * E32) * dS.abs()
        res['dq'][b, :, h, i] = scale * (dS @ K[:, i])
        err['dq'][b, :, h, i] = scale * ((eS + (Tk + 8) * E32 * dS.abs()) @ K[:, i].abs())
        Qi = q[b, :, h, i].double()
        res['dk'][b, :, g, i] += scale * (dS.T @ Qi)
        err['dk'][b, :, g, i] += scale * ((eS + (G * Tq + 8) * E32 * dS.abs()).T @ Qi.abs())
      Pd = P[0] - L * P[1]
      ePd = eP[0] * P[0] + abs(L) * eP[1] * P[1] + (ut + 4 * E32) * Pd.abs()
      res['dv'][b, :, g] += Pd.T @ dO
      err['dv'][b, :, g] += ePd.T @ dO.abs() + Pd.abs().T @ (edO + (G * Tq + 8) * E32 * dO.abs())
  if lam.numel() == 1:
    res['dlam'], err['dlam'] = res['dlam'].sum().view(1), err['dlam'].sum().view(1)
  for n in ('dq', 'dk', 'dv'):
    err[n] += u * res[n].abs()
  if w is not None:
    err['dw'] += U[w.dtype] * res['dw'].abs()
  return {n: (res[n], err[n]) for n in res}


def attn_inputs(B, Tq, Tk, H, Hkv, d, dv, dtype, seed=0, lam_n=None):
  q, k = randn(B, Tq, H, 2, d, dtype=dtype, seed=seed + 1, std=1.5), randn(B, Tk, Hkv, 2, d, dtype=dtype, seed=seed + 2)
  v, dout = randn(B, Tk, Hkv, dv, dtype=dtype, seed=seed + 3), randn(B, Tq, H, dv, dtype=dtype, seed=seed + 4)
  lam = randn(H if lam_n is None else lam_n, seed=seed + 5, std=0.2, mean=0.5)
  return q, k, v, dout, lam


def attn_compare(ops, q, k, v, dout, lam, w=None, train=True, keep=None, outs=None, norm=True, c=0.65, **opt):
  B, Tq, Tk = q.shape[0], q.shape[1], k.shape[1]
  vis = attn_visible(B, Tq, Tk, **{n: opt[n] for n in ('causal', 'kv_len', 'key_mask', 'q_start') if n in opt})
  want = attn_oracle(q, k, v, lam, vis, dout=dout if train else None, scale=opt.get('scale'), norm=norm, w=w, c=c)
  out, ctx = ops.diff_attn_fwd(q, k, v, lam, norm=norm, norm_weight=w, out_scale=c, save=train, **opt)
  within('out', out, *want['out'])
  empty = ~vis.any(2)
  assert not out[empty].any()
  if not train:
    assert ctx is None
    return out
  plain, _ = ops.diff_attn_fwd(q, k, v, lam, norm=norm, norm_weight=w, out_scale=c, **opt)
  assert torch.equal(plain, out)
  got = dict(zip(('dq', 'dk', 'dv', 'dlam', 'dw'), ops.diff_attn_bwd(dout, q, k, v, lam, ctx, **(outs or {}))))
  for n, g in got.items():
    if g is None:
      assert n == 'dw' and w is None
      continue
    within(n, g, *want[n])
    if n in ('dq', 'dk', 'dv') and Tk >= 8:
      # five roundings at most lie on the way to an element (P, O_i, dO, dS, the result), each U relative: far below what a wrong term would make
      a, b = g.double(), want[n][0]
      assert float((a - b).norm()) <= 6 * max(U[q.dtype], 2.0 ** -16) * float(b.norm()) + 1e-6, (n, float((a - b).norm() / b.norm()))
  unseen = ~vis.any(1)
  assert not got['dk'][unseen].any() and not got['dv'][unseen].any() and not got['dq'][empty].any()
  again = ops.diff_attn_bwd(dout, q, k, v, lam, ctx)
  assert all(x is None or torch.equal(x, y) for x, y in zip(got.values(), again)), 'not reproducible'
  return out


SHAPES = [(1, 1, 1, 1, 1, 1, 1), (2, 3, 5, 2, 1, 9, 18), (1, 64, 64, 4, 2, 16, 32), (2, 65, 130, 2, 2, 27, 54), (3, 129, 200, 4, 1, 64, 128), (1, 320, 320, 4, 4, 72, 144),
          (1, 100, 77, 2, 1, 128, 256), (1, 33, 300, 3, 3, 80, 100), (8, 20, 70, 2, 2, 32, 64)]


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('mask', ['none', 'causal', 'len', 'keys', 'all'])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_diff_attention_forward_and_gradients(ops, shape, mask, dtype):
  B, Tq, Tk, H, Hkv, d, dv = shape
  q, k, v, dout, lam = attn_inputs(*shape, dtype)
  g = torch.Generator().manual_seed(sum(shape))
  lens = torch.randint(0, Tk + 1, (B,), generator=g, dtype=torch.int32)
  keys = torch.rand(B, Tk, generator=g) < 0.7
  keys[B - 1] = B > 1 and mask == 'all'  # (one sequence without any key)
  opt = {}
  if mask in ('causal', 'all'):
    opt['causal'] = True
  if mask in ('len', 'all'):
    opt['kv_len'] = lens.to(DEV)
  if mask in ('keys', 'all'):
    opt['key_mask'] = keys.to(DEV)
  if mask == 'all':
    opt['q_start'] = torch.randint(-Tq, Tk, (B,), generator=g, dtype=torch.int32).to(DEV)
  attn_compare(ops, q, k, v, dout, lam, w=randn(dv, dtype=dtype, seed=9, std=0.1, mean=1.0), **opt)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_diff_attention_options(ops, dtype):
  """Without the norm, without weights, fp32 weights beside bf16 heads, one lambda for all heads, negative and zero lambda, another scale, an int q_start."""
  q, k, v, dout, lam = attn_inputs(2, 40, 50, 4, 2, 24, 56, dtype, seed=20)
  attn_compare(ops, q, k, v, dout, lam, norm=False)
  attn_compare(ops, q, k, v, dout, lam)
  attn_compare(ops, q, k, v, dout, lam, w=randn(56, seed=21, mean=1.0, std=0.1))
  attn_compare(ops, q, k, v, dout, lam[:1].clone(), scale=0.3)
  attn_compare(ops, q, k, v, dout, -lam, causal=True, q_start=-7)
  attn_compare(ops, q, k, v, dout, torch.zeros_like(lam), causal=True, q_start=1000)
  attn_compare(ops, q, k, v, dout, lam, key_mask=(torch.arange(50, device=DEV) % 3 != 1).to(torch.uint8).repeat(2, 1))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('d,off', [(32, 0), (32, 1), (20, 0)])
def test_diff_attention_strides(ops, dtype, d, off):
  """Slices of one fused projection (aligned or not), caches in [B, H, T] order, gradients written into the fused gradient; its other columns stay."""
  B, T, H, Hkv, dv = 2, 70, 4, 2, 2 * d
  width = 2 * H * d + 2 * Hkv * d + Hkv * dv + 3
  fused = randn(B, T, width + off, dtype=dtype, seed=30)[..., off:]
  cut = lambda x: (x[..., :2 * H * d].unflatten(-1, (H, 2, d)), x[..., 2 * H * d:2 * (H + Hkv) * d].unflatten(-1, (Hkv, 2, d)), x[..., 2 * (H + Hkv) * d:-3].unflatten(-1, (Hkv, dv)))
  q, k, v = cut(fused)
  dfused = torch.full((B, T, width + off), 7.0, dtype=dtype, device=DEV)[..., off:]
  dq, dk, dv_ = cut(dfused)
  _, _, _, dout, lam = attn_inputs(B, T, T, H, Hkv, d, dv, dtype, seed=31)
  attn_compare(ops, q, k, v, dout.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), lam, outs=dict(dq=dq, dk=dk, dv=dv_), causal=True)
  assert (dfused[..., -3:] == 7.0).all()
  # [B, H, 2, T, d] storage
  q2, k2, v2 = q.permute(0, 2, 3, 1, 4).contiguous().permute(0, 3, 1, 2, 4), k.permute(0, 2, 3, 1, 4).contiguous().permute(0, 3, 1, 2, 4), v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
  buf = torch.full((B, H, T, dv + 5), 7.0, dtype=dtype, device=DEV)
  out, _ = ops.diff_attn_fwd(q2, k2, v2, lam, out=buf[..., :dv].permute(0, 2, 1, 3))
  assert (buf[..., dv:] == 7.0).all()
  ref, _ = ops.diff_attn_fwd(q.contiguous(), k.contiguous(), v.contiguous(), lam)
  within('order', out, ref.double(), 2 * U[dtype] * ref.abs() + 1e-5)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('d', [32, 27])
def test_diff_attention_left_out_keys_may_hold_anything(ops, dtype, d):
  q, k, v, dout, lam = attn_inputs(3, 35, 150, 2, 2, d, 2 * d, dtype, seed=40)
  lens = torch.tensor([150, 61, 0], dtype=torch.int32, device=DEV)
  mask = torch.ones(3, 150, dtype=torch.bool, device=DEV)
  mask[0, 3:40] = False
  mask[1, ::2] = False
  opt = dict(kv_len=lens, key_mask=mask)
  clean = ops.diff_attn_fwd(q, k, v, lam, save=True, **opt)
  cg = ops.diff_attn_bwd(dout, q, k, v, lam, clean[1])
  gone = ~(mask & (torch.arange(150, device=DEV) < lens[:, None]))
  for bad in (math.nan, math.inf, torch.finfo(dtype).min):
    k2, v2 = k.clone(), v.clone()
    k2[gone], v2[gone] = bad, bad
    out, ctx = ops.diff_attn_fwd(q, k2, v2, lam, save=True, **opt)
    assert torch.equal(out, clean[0])
    assert all(x is None or torch.equal(x, y) for x, y in zip(cg, ops.diff_attn_bwd(dout, q, k2, v2, lam, ctx)))


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_diff_attention_large_scores(ops, dtype):
  """Scores of several hundred, rising and falling along the keys: the running maximum moves often, nothing overflows."""
  q, k, v, dout, lam = attn_inputs(1, 64, 400, 2, 1, 64, 128, dtype, seed=50)
  ramp = torch.linspace(-6, 6, 400, device=DEV).view(1, 400, 1, 1, 1)
  for kk in ((k.float() * ramp).to(dtype), (k.float() * ramp.flip(1)).to(dtype)):
    attn_compare(ops, q, kk, v, dout, lam, w=randn(128, dtype=dtype, seed=51, mean=1.0, std=0.1))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('Tq', [1, 2, 5, 17])
@pytest.mark.parametrize('heads', [(4, 4, 72, 144), (8, 2, 64, 128), (16, 1, 32, 64), (2, 1, 128, 256), (3, 3, 9, 18)], ids=str)
def test_diff_attention_new_tokens_against_a_cache(ops, heads, Tq, dtype):
  H, Hkv, d, dv = heads
  for Tk, lens in ((40, [17, 33, 40]), (3000, [2999, 18, 1500]), (6000, [5000])):
    B = len(lens)
    q, k, v, dout, lam = attn_inputs(B, Tq, Tk, H, Hkv, d, dv, dtype, seed=60)
    kv_len = torch.tensor([max(n, Tq) for n in lens], dtype=torch.int32, device=DEV)
    stale = torch.arange(Tk, device=DEV) >= kv_len[:, None]
    k[stale], v[stale] = math.nan, math.nan
    cache = dict(k=k.permute(0, 2, 3, 1, 4).contiguous().permute(0, 3, 1, 2, 4), v=v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3))
    for kk, vv in ((k, v), (cache['k'], cache['v'])):
      attn_compare(ops, q, kk, vv, dout, lam, train=False, causal=True, kv_len=kv_len, q_start=kv_len - Tq, w=randn(dv, seed=61, mean=1.0, std=0.1))


def test_diff_attention_cache_of_length_zero_and_masks_with_one_token(ops):
  q, k, v, dout, lam = attn_inputs(4, 1, 2000, 4, 2, 64, 128, BF16, seed=70)
  lens = torch.tensor([0, 1, 2000, 1024], dtype=torch.int32, device=DEV)
  keys = torch.ones(4, 2000, dtype=torch.bool, device=DEV)
  keys[2, 100:1900] = False
  keys[3] = False
  out = attn_compare(ops, q, k, v, dout, lam, train=False, kv_len=lens, key_mask=keys)
  assert not out[0].any() and not out[3].any() and out[1].any()


def test_diff_attention_cache_behind_32_bit_offsets(ops):
  """A cache whose second sequence starts behind 2^31 elements, and whose tokens lie far apart."""
  B, Tk, Hkv, d, dv = 2, 300, 1, 64, 128
  ld = (1 << 31) // 300 + 64 - ((1 << 31) // 300) % 64
  store = torch.empty(2 * Tk * ld + 4096, dtype=BF16, device=DEV)
  k = store.as_strided((B, Tk, Hkv, 2, d), (Tk * ld, ld, 2 * d, d, 1))
  v = store.as_strided((B, Tk, Hkv, dv), (Tk * ld, ld, dv, 1), 512)
  q, k0, v0, dout, lam = attn_inputs(B, 3, Tk, 2, Hkv, d, dv, BF16, seed=80)
  k.copy_(k0)
  v.copy_(v0)
  attn_compare(ops, q, k, v, dout, lam, train=False)
  attn_compare(ops, q, k, v, dout, lam)


def test_diff_attention_gradient_against_differences(ops):
  """Directional derivatives of the 64-bit forward by central differences, lambda through its learned vectors."""
  B, T, H, Hkv, d, dv = 1, 12, 2, 1, 8, 16
  q, k, v, dout, _ = attn_inputs(B, T, T, H, Hkv, d, dv, F32, seed=90)
  vec = [randn(H, d, seed=95 + i, std=0.3) for i in range(4)]
  w = randn(dv, seed=99, mean=1.0, std=0.1)
  keep = attn_visible(B, T, T, causal=True)
  lam = ops.diff_lambda(*vec, 0.4)
  out, ctx = ops.diff_attn_fwd(q, k, v, lam, causal=True, norm_weight=w, out_scale=0.6, save=True)
  dq, dk, dvv, dlam, dw = ops.diff_attn_bwd(dout, q, k, v, lam, ctx)
  grads = dict(zip(('q', 'k', 'v', 'w', 0, 1, 2, 3), [dq, dk, dvv, dw] + list(ops.diff_lambda_bwd(dlam, *vec))))

  def loss(x):
    e = lambda i: torch.exp((x[i] * x[i + 1]).sum(1))
    L = e(0) - e(2) + 0.4
    r = 0.0
    for h in range(H):
      p = [torch.softmax((x['q'][0, :, h, i] @ x['k'][0, :, 0, i].T * d ** -0.5).masked_fill(~keep[0], -math.inf), 1) for i in (0, 1)]
      o = (p[0] - L[h] * p[1]) @ x['v'][0, :, 0]
      o = 0.6 * x['w'] * o / torch.sqrt(o.pow(2).mean(1, keepdim=True) + 1e-5)
      r = r + (o * dout[0, :, h].double()).sum()
    return r

  base = {'q': q.double(), 'k': k.double(), 'v': v.double(), 'w': w.double(), **{i: t.double() for i, t in enumerate(vec)}}
  for n, g in grads.items():
    direction = randn(*g.shape, seed=77).double()
    e = 1e-6
    num = float((loss({**base, n: base[n] + e * direction}) - loss({**base, n: base[n] - e * direction})) / (2 * e))
    # truncation e^2, rounding 1e-16 / e in the difference; fp32 kernels: well under 1e-5 of the gradient's own size (sums of <= 200 terms)
    assert abs(num - float((g.double() * direction).sum())) <= 2e-5 * float((g.double().abs() * direction.abs()).sum()) + 1e-7, n


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape', [(1, 1), (4, 9), (16, 128), (12,)], ids=str)
def test_diff_lambda_and_gradient(ops, shape, dtype):
  vec = [randn(*shape, dtype=dtype, seed=i, std=0.2) for i in range(4)]
  d = shape[-1]
  lam = ops.diff_lambda(*vec, 0.35)
  a = [t.double().view(-1, d) for t in vec]
  e = [torch.exp((a[0] * a[1]).sum(1)), torch.exp((a[2] * a[3]).sum(1))]
  tol = (d + 16) * E32 * (e[0] * (1 + (a[0] * a[1]).abs().sum(1)) + e[1] * (1 + (a[2] * a[3]).abs().sum(1)) + 0.35)
  within('lam', lam, e[0] - e[1] + 0.35, tol)
  dl = randn(lam.numel(), seed=9)
  want = [dl.double()[:, None] * s * x for s, x in ((e[0][:, None], a[1]), (e[0][:, None], a[0]), (-e[1][:, None], a[3]), (-e[1][:, None], a[2]))]
  for g, x in zip(ops.diff_lambda_bwd(dl, *vec), want):
    assert g.dtype == dtype and g.shape == vec[0].shape
    within('vector', g.view(-1, d), x, (U[dtype] + (2 * d + 32) * E32) * x.abs())


def test_diff_attention_empty_calls(ops):
  lam = torch.full((2,), 0.5, device=DEV)
  for B, Tq, Tk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
    q, k, v, dout, _ = attn_inputs(B, Tq, Tk, 2, 1, 16, 32, BF16)
    out, ctx = ops.diff_attn_fwd(q, k, v, lam, save=True)
    assert out.shape == (B, Tq, 2, 32) and not out.any()
    for g in ops.diff_attn_bwd(dout, q, k, v, lam, ctx)[:4]:
      assert not g.any()


def test_diff_attention_refusals(ops):
  q, k, v, dout, lam = attn_inputs(2, 6, 7, 4, 2, 16, 32, BF16)
  i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
  bad = [dict(q=q.half(), k=k.half(), v=v.half()), dict(k=k.float()), dict(q=q.cpu()), dict(q=q[:1]), dict(q=q[:, :, :3]), dict(k=k[:, :6]), dict(v=v[:, :, :1]),
         dict(q=q[..., :8]), dict(lam=lam[:2].clone()), dict(lam=lam.double()), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
         dict(norm_eps=0.0), dict(norm=False, norm_weight=torch.ones(32, device=DEV)), dict(norm_weight=torch.ones(31, device=DEV)),
         dict(norm_weight=torch.ones(32, device=DEV).half()), dict(kv_len=i32(1)), dict(kv_len=i32(1, 2).long()), dict(kv_len=i32(1, 2).cpu()), dict(q_start=i32(1, 2, 3)),
         dict(q_start=1 << 30), dict(key_mask=torch.ones(2, 6, device=DEV, dtype=torch.bool)), dict(key_mask=torch.ones(2, 7, device=DEV)),
         dict(key_mask=torch.ones(7, 2, device=DEV, dtype=torch.bool).t()), dict(out=torch.empty(2, 6, 4, 32, device=DEV)), dict(out=torch.empty(1, 6, 4, 32, device=DEV, dtype=BF16).expand(2, 6, 4, 32)),
         dict(q=q.transpose(3, 4).contiguous().transpose(3, 4))]
  for kw in bad:
    kw = {'q': q, 'k': k, 'v': v, 'lam': lam, **kw}
    with pytest.raises((ValueError, TypeError)):
      ops.diff_attn_fwd(kw.pop('q'), kw.pop('k'), kw.pop('v'), kw.pop('lam'), **kw)
  wide = attn_inputs(1, 2, 2, 1, 1, 129, 64, BF16)
  with pytest.raises(ValueError):
    ops.diff_attn_fwd(*wide[:3], wide[4])
  wide = attn_inputs(1, 2, 2, 1, 1, 64, 257, BF16)
  with pytest.raises(ValueError):
    ops.diff_attn_fwd(*wide[:3], wide[4])
  _, ctx = ops.diff_attn_fwd(q, k, v, lam, save=True)
  for kw in (dict(dout=dout.float()), dict(dout=dout[:1]), dict(q=q[:1], k=k[:1], v=v[:1], dout=dout[:1]), dict(dk=torch.empty_like(v)), dict(dq=q[:, :1].expand_as(q))):
    kw = {'dout': dout, 'q': q, 'k': k, 'v': v, **kw}
    with pytest.raises((ValueError, TypeError)):
      ops.diff_attn_bwd(kw.pop('dout'), kw.pop('q'), kw.pop('k'), kw.pop('v'), lam, ctx, **kw)
  for vec in ([lam, lam, lam, lam.double()], [lam.double()] * 4, [lam, lam, lam, lam[:1]], [lam.cpu()] * 4):
    with pytest.raises((ValueError, TypeError)):
      ops.diff_lambda(*vec, 0.5)


@pytest.mark.parametrize('Tq,Tk', [(200, 200), (1, 5000)])
def test_diff_attention_captured_on_two_streams(ops, Tq, Tk):
  """Forward and backward captured twice, replayed side by side on two streams between eager calls: every replay equals the eager result."""
  q, k, v, dout, lam = attn_inputs(2, Tq, Tk, 4, 2, 64, 128, BF16, seed=100)

  def step():
    out, ctx = ops.diff_attn_fwd(q, k, v, lam, causal=True, save=True)
    serve, _ = ops.diff_attn_fwd(q, k, v, lam, causal=True)
    return [out, serve] + [t for t in ops.diff_attn_bwd(dout, q, k, v, lam, ctx) if t is not None]

  step()
  torch.cuda.synchronize()
  graphs = []
  for _ in range(2):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      graphs.append((g, step()))
  side = torch.cuda.Stream()
  for n in range(4):
    q.copy_(randn(*q.shape, dtype=BF16, seed=110 + n))
    v.copy_(randn(*v.shape, dtype=BF16, seed=120 + n))
    want = step()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
      graphs[0][0].replay()
    graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
      assert all(torch.equal(a, b) for a, b in zip(outs, want))
  with torch.cuda.stream(side):  # inputs made on one stream, used on another after an event
    e = torch.cuda.Event()
  e.record()
  side.wait_event(e)
  with torch.cuda.stream(side):
    got = step()
  torch.cuda.synchronize()
  assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape', [(1, 1100, 96, 2, 1, 32, 64), (1, 540, 70, 4, 1, 72, 144), (1, 2080, 33, 1, 1, 128, 256)], ids=str)
def test_diff_attention_gradients_with_the_queries_split(ops, shape, dtype):
  """Few keys and many tiles of queries: dK and dV are summed in parts and joined."""
  B, Tq, Tk, H, Hkv, d, dv = shape
  assert (H // Hkv) * ((Tq + 31) // 32) >= 64
  q, k, v, dout, lam = attn_inputs(*shape, dtype, seed=170)
  keys = torch.arange(Tk, device=DEV)[None] % 5 != 2
  attn_compare(ops, q, k, v, dout, lam, w=randn(dv, seed=171, mean=1.0, std=0.2), key_mask=keys)
  attn_compare(ops, q, k, v, dout, lam, causal=True, q_start=-Tq // 2)


def test_diff_attention_query_starts_at_the_ends_of_their_range(ops):
  q, k, v, dout, lam = attn_inputs(4, 40, 70, 2, 1, 32, 64, BF16, seed=180)
  top = 2 ** 31 - 1
  starts = torch.tensor([-top - 1, top, -(1 << 30), 1 << 30], dtype=torch.int32, device=DEV)
  lens = torch.tensor([top, 70, -top - 1, 10], dtype=torch.int32, device=DEV)
  out, ctx = ops.diff_attn_fwd(q, k, v, lam, causal=True, q_start=starts, kv_len=lens, save=True)
  grads = ops.diff_attn_bwd(dout, q, k, v, lam, ctx)
  want, wctx = ops.diff_attn_fwd(q[[1, 3]], k[[1, 3]], v[[1, 3]], lam, kv_len=torch.tensor([70, 10], dtype=torch.int32, device=DEV), save=True)
  wgrads = ops.diff_attn_bwd(dout[[1, 3]], q[[1, 3]], k[[1, 3]], v[[1, 3]], lam, wctx)
  assert not out[[0, 2]].any() and torch.equal(out[[1, 3]], want)
  for g, w in zip(grads[:3], wgrads):
    assert not g[[0, 2]].any() and torch.equal(g[[1, 3]], w)


def test_diff_attention_outputs_may_not_overlap(ops):
  B, T, H, d = 2, 9, 2, 16
  fused = randn(B, T, H, 8 * d, dtype=BF16, seed=190)
  q, k, v = fused[..., :2 * d].unflatten(3, (2, d)), fused[..., 2 * d:4 * d].unflatten(3, (2, d)), fused[..., 4 * d:6 * d]
  lam = torch.full((1,), 0.5, device=DEV)
  want, ctx = ops.diff_attn_fwd(q, k, v, lam, save=True)
  got, _ = ops.diff_attn_fwd(q, k, v, lam, out=fused[..., 6 * d:])  # the free quarter of the same rows
  assert torch.equal(got, want)
  for bad in (fused[..., 4 * d:6 * d], fused[..., 3 * d:5 * d], fused[..., 5 * d:7 * d]):
    with pytest.raises(ValueError):
      ops.diff_attn_fwd(q, k, v, lam, out=bad)
  g = torch.empty_like(fused)
  dq, dk, dv = g[..., :2 * d].unflatten(3, (2, d)), g[..., 2 * d:4 * d].unflatten(3, (2, d)), g[..., 4 * d:6 * d]
  dout = randn(B, T, H, 2 * d, dtype=BF16, seed=191)
  res, plain = ops.diff_attn_bwd(dout, q, k, v, lam, ctx, dq=dq, dk=dk, dv=dv), ops.diff_attn_bwd(dout, q, k, v, lam, ctx)
  assert all(torch.equal(a, b) for a, b in zip(res[:4], plain))
  for bad in (dict(dq=dq, dk=dq), dict(dq=q), dict(dv=v), dict(dk=dk, dv=g[..., 3 * d:5 * d]), dict(dv=dout)):
    with pytest.raises(ValueError):
      ops.diff_attn_bwd(dout, q, k, v, lam, ctx, **bad)
  one = torch.zeros(3 * 32, device=DEV)
  x = randn(2, 32)
  _, _, nctx = ops.block_norm_fwd(x, x, post_weight=one[:32].clone(), pre_weight=one[:32].clone())
  with pytest.raises(ValueError):
    ops.block_norm_bwd(x, x, nctx, into=dict(post_weight=one[:32], pre_weight=one[16:48]))


# ------------------------------------------------------------------------------------------------ the operators together
def block_params(C, H, Hkv, d, dv, dtype, seed):
  p = {'w_in': randn(C, H * 2 * d + Hkv * (2 * d + dv), dtype=dtype, seed=seed, std=C ** -0.5), 'w_out': randn(H * dv, C, dtype=dtype, seed=seed + 1, std=(H * dv) ** -0.5)}
  for i, n in enumerate(('lq1', 'lk1', 'lq2', 'lk2')):
    p[n] = randn(H, d, seed=seed + 2 + i, std=0.1)
  for i, n in enumerate(('pre1', 'pre2', 'post2', 'scale2', 'head')):
    p[n] = randn(dv if n == 'head' else C, seed=seed + 8 + i, std=0.1, mean=1.0)
  return p


def block_plain(p, x, r, gate, heads, key_mask):
  """r joins the stream, its norm is the attention's input, the result is normalised, gated per sample and joins the stream; 64 bits."""
  H, Hkv, d, dv = heads
  B, T, C = x.shape
  norm = lambda z, w, eps=1e-5: z / torch.sqrt(z.pow(2).mean(-1, keepdim=True) + eps) * w
  y = x + r
  z = norm(y, p['pre1']) @ p['w_in']
  q, k, v = z[..., :H * 2 * d].view(B, T, H, 2, d), z[..., H * 2 * d:-Hkv * dv].view(B, T, Hkv, 2, d), z[..., -Hkv * dv:].view(B, T, Hkv, dv)
  lam = torch.exp((p['lq1'] * p['lk1']).sum(1)) - torch.exp((p['lq2'] * p['lk2']).sum(1)) + 0.3
  k, v = k.repeat_interleave(H // Hkv, 2), v.repeat_interleave(H // Hkv, 2)
  keep = attn_visible(B, T, T, causal=True, key_mask=key_mask)[:, None]
  P = []
  for i in (0, 1):
    s = (q[:, :, :, i].transpose(1, 2) @ k[:, :, :, i].transpose(1, 2).transpose(2, 3)) * d ** -0.5
    e = torch.exp((s - s.masked_fill(~keep, -1e30).amax(-1, keepdim=True).detach()).masked_fill(~keep, -1e4))  # (hidden: zero, and no gradient)
    P.append(e / e.sum(-1, keepdim=True).clamp_min(1e-30))
  o = (P[0] - lam[None, :, None, None] * P[1]) @ v.transpose(1, 2)
  a = (0.7 * norm(o, p['head'])).transpose(1, 2).reshape(B, T, H * dv) @ p['w_out']
  y2 = y + p['scale2'] * torch.sigmoid(gate)[:, None] * norm(a, p['post2'])
  return y2, norm(y2, p['pre2'])


def block_own(ops, p, x, r, gate, heads, key_mask, dy, dh, clip, grads):
  H, Hkv, d, dv = heads
  B, T, C = x.shape
  y, h, c1 = ops.block_norm_fwd(x, r, kind='rms', post=False, pre_weight=p['pre1'])
  z = h.view(B * T, C) @ p['w_in']
  view = lambda t: (t[:, :H * 2 * d].view(B, T, H, 2, d), t[:, H * 2 * d:-Hkv * dv].view(B, T, Hkv, 2, d), t[:, -Hkv * dv:].view(B, T, Hkv, dv))
  vec = [p[n] for n in ('lq1', 'lk1', 'lq2', 'lk2')]
  lam = ops.diff_lambda(*vec, 0.3)
  o, ca = ops.diff_attn_fwd(*view(z), lam, causal=True, key_mask=key_mask, norm_weight=p['head'], out_scale=0.7, save=True)
  o = o.view(B * T, H * dv)
  a = (o @ p['w_out']).view(B, T, C)
  y2, h2, c2 = ops.block_norm_fwd(y, a, kind='rms', post_weight=p['post2'], pre_weight=p['pre2'], scale=p['scale2'], gate=gate, gate_act=ops.ACT_SIGMOID)

  for n in ('post2', 'pre2', 'scale2', 'pre1'):
    ops.zero_(grads[n])
  g2 = ops.block_norm_bwd(dy, dh, c2, into=dict(post_weight=grads['post2'], pre_weight=grads['pre2'], scale=grads['scale2']))
  da = g2['a'].view(B * T, C)
  torch.mm(o.t(), da, out=grads['w_out'])
  do = torch.mm(da, p['w_out'].t().contiguous()).view(B, T, H, dv)
  dz = torch.empty_like(z)
  dq, dk, dvv = view(dz)
  _, _, _, dlam, dhead = ops.diff_attn_bwd(do, *view(z), lam, ca, dq=dq, dk=dk, dv=dvv)
  grads['head'].copy_(dhead)
  for n, t in zip(('lq1', 'lk1', 'lq2', 'lk2'), ops.diff_lambda_bwd(dlam, *vec)):
    grads[n].copy_(t)
  torch.mm(h.view(B * T, C).t(), dz, out=grads['w_in'])
  g1 = ops.block_norm_bwd(g2['x'], torch.mm(dz, p['w_in'].t().contiguous()).view(B, T, C), c1, into=dict(pre_weight=grads['pre1']))
  norm = clip.clip_(0.5)
  return dict(y=y2, h=h2, x=g1['x'], r=g1['a'], gate=g2['gate'], norm=norm, **grads)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_transformer_block_step_eager_and_captured(ops, dtype):
  """Norms, attention, gradients and their clipping as one training step, against autograd of the plain block in 64 bits, then captured: replays equal
  the eager step.  Tolerance, relative in the 2-norm: at most 12 roundings in the storage type lie on a path through the block and its backward (bf16:
  12 * 2^-8), sums of at most 192 terms in fp32 at each of these 12 stages (12 * 192 * 2^-24 = 1.4e-4), times 8 for what the norms' and softmaxes'
  derivatives amplify at rows of unit variance; roundings are independent, so bf16 is held to sqrt(12) * 8 * 2^-8 = 0.108 and fp32 to 1.1e-3."""
  tol = 1.1e-3 if dtype == F32 else 0.108
  B, T, C, heads = 2, 70, 96, (4, 2, 24, 48)
  p = block_params(C, *heads, dtype, 200)
  x, r, gate = randn(B, T, C, dtype=dtype, seed=220), randn(B, T, C, dtype=dtype, seed=221), randn(B, C, dtype=dtype, seed=222)
  dy, dh = randn(B, T, C, dtype=dtype, seed=223), randn(B, T, C, dtype=dtype, seed=224)
  mask = torch.ones(B, T, dtype=torch.bool, device=DEV)
  mask[1, 50:] = False
  mask[1, 0] = False  # the first query of this sequence sees no key
  grads = {n: torch.zeros_like(t) for n, t in p.items()}
  clip = ops.GradClip(list(grads.values()))
  step = lambda: block_own(ops, p, x, r, gate, heads, mask, dy, dh, clip, grads)

  def check(got):
    leaves = {n: t.double().requires_grad_() for n, t in (*p.items(), ('x', x), ('r', r), ('gate', gate))}
    y, h = block_plain({n: leaves[n] for n in p}, leaves['x'], leaves['r'], leaves['gate'], heads, mask)
    want = dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [dy.double(), dh.double()])), y=y.detach(), h=h.detach())
    norm = torch.sqrt(sum(want[n].pow(2).sum() for n in p))
    assert abs(float(got['norm']) - float(norm)) <= tol * float(norm)
    coef = min(1.0, 0.5 / float(norm))
    for n, w in want.items():
      w = w * (coef if n in p else 1.0)
      err, size = float((got[n].double() - w).norm()), float(w.norm())
      assert err <= (2 * tol if n in p else tol) * size, (n, err / size)  # (clipped ones: the norm's error comes on top)

  keep = lambda res: {n: t.clone() for n, t in res.items()}
  check(keep(step()))
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    outs = step()
  for i in range(3):
    x.copy_(randn(B, T, C, dtype=dtype, seed=230 + i))
    want = keep(step())
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for n, t in want.items():
      assert torch.equal(outs[n], t), n
  check(want)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_answers_token_by_token_equal_the_whole_sequence(ops, dtype):
  """A sequence written into a cache token by token, each through the norm and the attention over what the cache holds, equals the causal pass over the
  whole sequence.  Both sides are within the bound of the 64-bit formula, so they are within twice that of each other."""
  B, T, C, (H, Hkv, d, dv) = 2, 45, 64, (4, 2, 32, 64)
  q, k, v, _, lam = attn_inputs(B, T, T, H, Hkv, d, dv, dtype, seed=240)
  x, a, w = randn(B, T, C, dtype=dtype, seed=250), randn(B, T, C, dtype=dtype, seed=251), randn(C, seed=252)
  whole, _ = ops.diff_attn_fwd(q, k, v, lam, causal=True, out_scale=0.65)
  _, err = attn_oracle(q, k, v, lam, attn_visible(B, T, T, causal=True), c=0.65)['out']
  y, h, _ = ops.block_norm_fwd(x, a, kind='rms', pre_weight=w, save=False)
  kc, vc = torch.full((B, 64, Hkv, 2, d), math.nan, device=DEV, dtype=dtype), torch.full((B, 64, Hkv, dv), math.nan, device=DEV, dtype=dtype)
  lens = torch.zeros(B, dtype=torch.int32, device=DEV)
  for t in range(T):
    kc[:, t], vc[:, t] = k[:, t], v[:, t]
    lens += 1
    out, _ = ops.diff_attn_fwd(q[:, t:t + 1], kc, vc, lam, kv_len=lens, out_scale=0.65)
    within(f'token {t}', out[:, 0], whole[:, t].double(), 2 * err[:, t])
    yt, ht, _ = ops.block_norm_fwd(x[:, t], a[:, t], kind='rms', pre_weight=w, save=False)
    assert torch.equal(yt, y[:, t]) and torch.equal(ht, h[:, t])


def test_trainer_clips_the_averaged_gradients(ops):
  """Trainer(max_grad_norm): the reported norm is that of the arena, the moments are those of the clipped gradient -- eager and replayed -- and a bound
  above the norm changes no bit of the update."""
  from carla_garage_amd.config import GlobalConfig
  from carla_garage_amd.graph import GraphedTrainStep
  from carla_garage_amd.model import LidarCenterNet
  from carla_garage_amd.trainer import Trainer
  from oracle import tfpp_port as P
  m = LidarCenterNet(GlobalConfig(tfpp_dtype='bf16'))
  m.load_state_dict(P.make_state_dict(), strict=True)
  m.cuda().train()
  batch = {k: v.cuda() for k, v in P.make_labels(2).items()}
  for k, v in zip(('rgb', 'lidar_bev', 'target_point', 'ego_vel', 'command'), P.make_inputs(2)):
    batch[k] = v.cuda()
  tr = Trainer(m, lr=1e-5, max_grad_norm=0.25)

  def check(run, bound):
    tr.max_grad_norm = bound
    tr.apply_observed_layout()  # (the next eager step would move the arenas)
    m0, v0 = tr.exp_avg.clone(), tr.exp_avg_sq.clone()
    run()
    g = tr.eng.flat_grad.double()
    norm = g.norm()
    within('norm', tr.grad_norm, norm, 2 * U[F32] * norm)
    assert float(norm) > 0.25
    c = min(1.0, bound / (float(norm) + 1e-6))
    # three roundings of the coefficient, one of its product with g, three (five for the square) of the moment's update
    for got, old, b, x, k in ((tr.exp_avg, m0, 0.9, c * g, 8), (tr.exp_avg_sq, v0, 0.999, (c * g) ** 2, 14)):
      b32 = float(torch.tensor(b, dtype=F32))
      new, mag = b32 * old.double() + (1 - b32) * x, b32 * old.double().abs() + (1 - b32) * x.abs()
      within('moment', got, new, k * U[F32] * mag + 1e-37 + 2e-8 * x.abs())  # (1 - beta is rounded in fp32: 2^-24 absolute, squared gradients below 2^-126 vanish)

  check(lambda: tr.train_step(batch), 0.25)
  check(lambda: tr.train_step(batch), 0.25)
  step = GraphedTrainStep(tr, batch, warmup=1)
  for bound in (0.25, 0.01, 1e9):
    check(step, bound)


@pytest.mark.parametrize('seed', range(6))
@pytest.mark.parametrize('heads', [(1, 1, 9, 18), (1, 1, 72, 144), (2, 1, 64, 128)], ids=str)
def test_diff_attention_lambda_gradient_of_few_heads(ops, heads, seed):
  """dlambda of one or two heads is one number, often small beside the terms it is the sum of: the roundings of P and of the saved O_2 to bf16 may not be
  in it directly.  They remain in O, which dO(O) is made of.  With f(O) = sum of dO(O) . O_2 and g its derivative by O (O_2 held), independent roundings of
  at most 2^-8 relative, standard deviation 2^-8 / sqrt(3) at most, of O_1 and O_2 as stored and of each P give dlambda the deviation 2^-8 / sqrt(3) times
  the root of sum g^2 (O_1^2 + lam^2 O_2^2 + (P_1^2 + lam^2 P_2^2) V^2): four of these are allowed, and fp32 sums (1e-4 of the terms' root)."""
  H, Hkv, d, dv = heads
  B, T = 2, 333
  q, k, v, dout, lam = attn_inputs(B, T, T, H, Hkv, d, dv, BF16, seed=300 + 10 * seed)
  _, ctx = ops.diff_attn_fwd(q, k, v, lam, causal=True, save=True)
  got = ops.diff_attn_bwd(dout, q, k, v, lam, ctx)[3]
  keep = attn_visible(B, T, T, causal=True)
  want = attn_oracle(q, k, v, lam, keep, dout=dout)['dlam'][0]
  for h in range(H):
    L, terms, dev = float(lam[h]), 0.0, 0.0
    for b in range(B):
      V, P = v[b, :, h // (H // Hkv)].double(), []
      for i in (0, 1):
        P.append(torch.softmax((q[b, :, h, i].double() @ k[b, :, h // (H // Hkv), i].double().T * d ** -0.5).masked_fill(~keep[b], -math.inf), 1))
      o = [p @ V for p in P]
      O, u = (o[0] - L * o[1]).requires_grad_(), dout[b, :, h].double()
      r = 1.0 / torch.sqrt(O.pow(2).mean(1, keepdim=True) + 1e-5)
      each = (r * u - O * r ** 3 * (u * O).mean(1, keepdim=True)) * o[1]
      g, = torch.autograd.grad(each.sum(), O)
      dev += float((g.pow(2) * (o[0].pow(2) + L ** 2 * o[1].pow(2) + (P[0].pow(2) + L ** 2 * P[1].pow(2)) @ V.pow(2))).sum())
      terms += float(each.detach().pow(2).sum())
    tol = 4 * 2.0 ** -8 / math.sqrt(3) * math.sqrt(dev) + 1e-4 * math.sqrt(terms)
    assert abs(float(got[h] - want[h])) <= tol, (float(got[h]), float(want[h]), tol, math.sqrt(terms))
