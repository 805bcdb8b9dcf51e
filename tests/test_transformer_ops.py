"""What the transformer-block operators refuse, without a GPU: tensors in host memory, layouts, and the C entries' own checks (tfpp.h), which
return before anything is launched."""
import ctypes

import pytest
import torch

from carla_garage_amd import ops
from carla_garage_amd._lib import lib, BlockNormParams, DiffAttnParams, BF16, EINVAL, F32

FAKE = 0x10000  # an aligned, never dereferenced "device pointer"


@pytest.fixture(scope='module')
def L():
  lib.load()
  return lib


def test_host_tensors_are_refused():
  x = torch.zeros(2, 3, 8)
  q, v, lam = torch.zeros(1, 2, 2, 2, 8), torch.zeros(1, 2, 2, 16), torch.zeros(1)
  for call in (lambda: ops.GradClip([x]), lambda: ops.block_norm_fwd(x, x), lambda: ops.diff_attn_fwd(q, q, v, lam), lambda: ops.diff_lambda(lam, lam, lam, lam, 0.5),
               lambda: ops.diff_lambda_bwd(lam, lam, lam, lam, lam)):
    with pytest.raises(ValueError, match='device'):
      call()
  with pytest.raises(ValueError):
    ops.GradClip([])
  with pytest.raises(ValueError):
    ops.GradClip([x], out=[])


def test_clip_grad_norm_without_gradients():
  from carla_garage_amd.optim import clip_grad_norm_
  assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0
  assert float(clip_grad_norm_([], 1.0)) == 0.0


def test_row_views():
  x = torch.zeros(3, 4, 10)
  assert ops._row_view(x, x.shape, 'x') == 10
  assert ops._row_view(x[..., 2:6], (3, 4, 4), 'x') == 10           # columns of wider rows
  assert ops._row_view(x[:, 1:2], (3, 1, 10), 'x') == 40            # one row of each sample
  assert ops._row_view(x[:1, :1], (1, 1, 10), 'x') == 10
  for bad in (x[:, :3], x.transpose(1, 2), x[:1, :1].expand(3, 4, 10), x[..., ::2]):  # two strides, channels apart, the same row for all
    with pytest.raises(ValueError):
      ops._row_view(bad, bad.shape, 'x')
  with pytest.raises(ValueError):
    ops._row_view(x, (3, 4, 9), 'x')


def test_dense_tensors():
  x = torch.zeros(3, 4, 5)
  assert ops.is_dense(x) and ops.is_dense(x.permute(2, 0, 1)) and ops.is_dense(x[:, :1, :1][:1]) and ops.is_dense(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last))
  assert not ops.is_dense(x[:, :2]) and not ops.is_dense(x[..., ::2]) and not ops.is_dense(x[:, :1].expand(3, 4, 5))


def test_outputs_with_elements_in_common():
  x = torch.zeros(4, 6)
  ops._disjoint(x.t(), 'x')
  ops._disjoint(x[:, 2:4], 'x')
  ops._disjoint(x.view(-1)[:10].as_strided((2, 5), (5, 1)), 'x')
  for bad in (x[:1].expand(4, 6), x.as_strided((4, 6), (3, 1)), x.as_strided((3, 3), (1, 1))):
    with pytest.raises(ValueError):
      ops._disjoint(bad, 'x')


def test_outputs_apart_from_the_inputs():
  f = torch.zeros(2, 5, 3, 40)
  part = lambda a, b: f[..., a:b]
  for a, b in ((part(0, 10), part(10, 20)), (part(30, 40), part(0, 30)), (f[:, :2], f[:, 2:]), (f[0], f[1]), (f[:, :, 0], f[:, :, 1:]), (part(0, 10)[:, :2], part(10, 20)[:, 3:]),
               (part(0, 10).transpose(1, 2), part(10, 20)), (f, torch.zeros(3)), (f[:0], f)):
    ops._apart(a, 'a', [('b', b)])
    ops._apart(b, 'b', [('a', a)])
  for a, b in ((f[:], f), (f, f.view(-1)), (part(0, 11), part(10, 20)), (part(5, 6), part(0, 10)), (f[:, :3], f[:, 2:]), (f.view(-1)[1:], f.view(-1)[:-1]), (part(0, 4), f.view(torch.bfloat16)[..., 6:9])):
    with pytest.raises(ValueError):
      ops._apart(a, 'a', [('b', b)])
    with pytest.raises(ValueError):
      ops._apart(b, 'b', [('a', a)])
  with pytest.raises(ValueError):
    ops._apart(f, 'a', [('f', f)])


def norm_params(**kw):
  p = BlockNormParams()
  p.x = p.a = p.y = p.h = p.stat = p.dx = p.da = p.partial = p.dy = FAKE
  p.B, p.T, p.C, p.post, p.pre, p.layer, p.alpha, p.eps = 2, 3, 64, 1, 1, 1, 1.0, 1e-5
  for n, v in kw.items():
    setattr(p, n, v)
  return p


@pytest.mark.parametrize('kw', [dict(C=0), dict(C=4097), dict(B=0), dict(T=0), dict(x=None), dict(a=None), dict(y=None), dict(h=None), dict(gate_mode=3, gate=FAKE), dict(gate_mode=1),
                                dict(gate_mode=1, gate=FAKE, gate_act=1), dict(B=1 << 20, T=1 << 20)], ids=str)
def test_block_norm_entry_refuses(L, kw):
  assert L.raw('tfpp_block_norm_fwd')(ctypes.byref(norm_params(**kw)), BF16, None) == EINVAL


@pytest.mark.parametrize('kw', [dict(C=4097), dict(dx=None), dict(stat=None), dict(stat=FAKE + 4), dict(partial=None), dict(dy=None), dict(dh=FAKE, pre=0), dict(gate_mode=1, gate=FAKE),
                                dict(B=65531)], ids=str)
def test_block_norm_backward_entry_refuses(L, kw):
  assert L.raw('tfpp_block_norm_bwd')(ctypes.byref(norm_params(**kw)), F32, None) == EINVAL


def attn_params(**kw):
  p = DiffAttnParams()
  for n in ('q', 'k', 'v', 'lam', 'out', 'o1', 'o2', 'lse', 'dout', 'd_o', 'delta', 'partial', 'dlam', 'dq_out', 'dk_out', 'dv_out'):
    setattr(p, n, FAKE)
  p.B, p.Tq, p.Tk, p.H, p.Hkv, p.d, p.dv, p.n_lam, p.norm, p.scale, p.out_scale, p.eps = 2, 5, 7, 4, 2, 32, 64, 4, 1, 0.1, 1.0, 1e-5
  for n, v in kw.items():
    setattr(p, n, v)
  return p


BAD_ATTN = [dict(B=0), dict(Tq=0), dict(Tk=0), dict(Tq=1 << 29), dict(H=3), dict(Hkv=0), dict(d=0), dict(d=129), dict(dv=257), dict(n_lam=2), dict(scale=0.0), dict(scale=float('inf')),
            dict(scale=float('nan')), dict(eps=0.0), dict(q=None), dict(lam=None), dict(B=1 << 23)]


@pytest.mark.parametrize('kw', BAD_ATTN + [dict(out=None), dict(o2=None), dict(B=1, H=1, Hkv=1, n_lam=1, Tq=1, Tk=5000, partial=None)], ids=str)
def test_diff_attention_entry_refuses(L, kw):
  assert L.raw('tfpp_diff_attn_fwd')(ctypes.byref(attn_params(**kw)), BF16, None) == EINVAL
  assert L.raw('tfpp_diff_attn_fwd')(ctypes.byref(attn_params()), 7, None) == EINVAL
  assert L.raw('tfpp_diff_attn_fwd')(None, BF16, None) == EINVAL


@pytest.mark.parametrize('kw', BAD_ATTN + [dict(o1=None), dict(lse=None), dict(d_o=None), dict(delta=None), dict(partial=None), dict(dlam=None), dict(dk_out=None), dict(norm_w=FAKE),
                                           dict(o1=FAKE + 8), dict(B=1, H=65536, Hkv=1, n_lam=1)], ids=str)
def test_diff_attention_backward_entry_refuses(L, kw):
  assert L.raw('tfpp_diff_attn_bwd')(ctypes.byref(attn_params(**kw)), F32, None) == EINVAL


def test_other_entries_refuse(L):
  clip = L.raw('tfpp_grad_clip')
  good = [FAKE, 3, FAKE, 1.0, 2, 1.0, FAKE, 1, None]
  for i, v in ((0, None), (1, -1), (2, None), (3, -1.0), (3, float('nan')), (4, 3), (6, None)):
    assert clip(*[v if j == i else x for j, x in enumerate(good)]) == EINVAL, (i, v)
  assert L.raw('tfpp_diff_lambda')(FAKE, FAKE, FAKE, FAKE, 0.5, FAKE, 0, 4, F32, None) == EINVAL
  assert L.raw('tfpp_diff_lambda')(FAKE, FAKE, FAKE, FAKE, 0.5, FAKE, 1, 4, 5, None) == EINVAL
  assert L.raw('tfpp_adamw_amsgrad_clipped')(*[FAKE] * 5, 4, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, None, None) == EINVAL


def test_scratch_grows_with_the_splits_and_covers_every_width(L):
  """Scratch of the split passes: a multiple of the parts, wide enough for the padded heads the kernels write."""
  n = ctypes.c_int64()
  for d, dv, pad in ((8, 16, 1), (20, 40, 2), (33, 66, 5), (72, 144, 5), (81, 162, 8), (128, 256, 8), (16, 256, 8)):
    p = attn_params(B=1, H=2, Hkv=1, Tq=1, Tk=40000, d=d, dv=dv, n_lam=1)
    assert L.raw('tfpp_diff_attn_fwd_partial_floats')(ctypes.byref(p), ctypes.addressof(n)) == 0
    row = 2 * (pad * 32 + 2)
    assert n.value % (2 * row) == 0 and 1 < n.value // (2 * row) <= 64
    p = attn_params(B=1, H=2, Hkv=1, Tq=4000, Tk=100, d=d, dv=dv, n_lam=1)
    assert L.raw('tfpp_diff_attn_bwd_partial_floats')(ctypes.byref(p), ctypes.addressof(n)) == 0
    assert n.value >= 100 * (2 * ((pad + 1) // 2) + pad) * 32
  p = attn_params(Tk=100)
  assert L.raw('tfpp_diff_attn_fwd_partial_floats')(ctypes.byref(p), ctypes.addressof(n)) == 0 and n.value == 0
