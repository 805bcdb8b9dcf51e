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
