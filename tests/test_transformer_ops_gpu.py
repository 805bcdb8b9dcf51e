"""GPU tests of the transformer-block operators (-m gpu) against plain implementations in 64 bits: gradient norm and clipping (ops.GradClip,
optim.clip_grad_norm_, Trainer's max_grad_norm).

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
