"""Calls of differential attention that the documentation allows at the edges of its inputs: slots of a cache that no query sees yet, rows that share
memory, tiny eps with rows that see nothing, many sequences of single tokens, threads."""
import math

import pytest
import torch

from test_transformer_ops_gpu import BF16, DEV, F32, attn_compare, attn_inputs, attn_oracle, attn_visible, ops, randn, within  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('Tq,d', [(1, 64), (5, 27), (70, 32), (70, 72), (200, 64)])
def test_causal_calls_do_not_see_what_lies_behind_their_last_query(ops, Tq, d, dtype):
  """New tokens in the middle of a cache, without kv_len: what the slots behind them hold reaches neither the result nor a gradient."""
  B, Tk, H, Hkv = 3, 400, 4, 2
  q, k, v, dout, lam = attn_inputs(B, Tq, Tk, H, Hkv, d, 2 * d, dtype, seed=500)
  start = torch.tensor([0, 101, 400 - Tq - 1], dtype=torch.int32, device=DEV)
  behind = torch.arange(Tk, device=DEV) >= start[:, None] + Tq
  for opt in (dict(q_start=start), dict(q_start=37)):
    gone = behind if torch.is_tensor(opt['q_start']) else (torch.arange(Tk, device=DEV) >= 37 + Tq).expand(B, Tk)
    k0, v0 = k.clone(), v.clone()
    k0[gone], v0[gone] = 0.0, 0.0
    want, wctx = ops.diff_attn_fwd(q, k0, v0, lam, causal=True, save=True, **opt)
    wgrads = ops.diff_attn_bwd(dout, q, k0, v0, lam, wctx)
    for bad in (math.nan, math.inf, torch.finfo(dtype).min):
      k0[gone], v0[gone] = bad, bad
      got, ctx = ops.diff_attn_fwd(q, k0, v0, lam, causal=True, save=True, **opt)
      assert torch.equal(got, want)
      assert torch.equal(ops.diff_attn_fwd(q, k0, v0, lam, causal=True, **opt)[0], want)
      grads = ops.diff_attn_bwd(dout, q, k0, v0, lam, ctx)
      assert all(x is None or torch.equal(x, y) for x, y in zip(grads, wgrads))
      assert not grads[1][gone].any() and not grads[2][gone].any()


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('what', ['q', 'k', 'v', 'all', 'windows'])
@pytest.mark.parametrize('d', [32, 64, 72])
def test_tokens_that_share_memory(ops, what, d, dtype):
  """One query, key or value expanded over all tokens, or windows of a longer row.  The scores are large, so that a row that does not exist would not go
  unnoticed."""
  B, Tq, Tk, H, Hkv = 2, 41, 75, 2, 1
  q, k, v, dout, lam = attn_inputs(B, Tq, Tk, H, Hkv, d, 2 * d, dtype, seed=510)
  q, k = q * 6, k * 6
  if what == 'windows':  # token t has the channels 8 t ..
    base = randn(4 * 2 * d * (Tk + 8), dtype=dtype, seed=511)
    q = (base * 6).as_strided(q.shape, (Tq * 8 + 4 * d, 8, 2 * d, d, 1))
    v = base.as_strided(v.shape, (Tk * 8 + 4 * d, 8, 2 * d, 1), 16)
  else:
    q, k, v = (t[:, :1].expand_as(t) if what in (n, 'all') else t for n, t in (('q', q), ('k', k), ('v', v)))
  for opt in (dict(), dict(causal=True), dict(kv_len=torch.tensor([75, 33], dtype=torch.int32, device=DEV))):
    out, ctx = ops.diff_attn_fwd(q, k, v, lam, norm_eps=1e-5, save=True, **opt)
    grads = ops.diff_attn_bwd(dout, q, k, v, lam, ctx)
    assert torch.isfinite(out).all() and all(torch.isfinite(g).all() for g in grads if g is not None)
    want = attn_oracle(q, k, v, lam, attn_visible(B, Tq, Tk, **opt), dout=dout)
    # a probability below 2^-126 is zero in 32 bits: 1.2e-38 times |dP - delta| <= 1e4, |K| or |Q| <= 1e2 and 75 tokens, 1e-30 at most, whatever the value
    for n, g in zip(('out', 'dq', 'dk', 'dv', 'dlam'), (out, *grads)):
      within(n, g, want[n][0], want[n][1] + 1e-30)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_single_tokens_with_any_stride(ops, dtype):
  q, k, v, dout, lam = attn_inputs(2, 1, 1, 2, 1, 32, 64, dtype, seed=520)
  odd = lambda t: torch.cat([t.flatten(), t.new_zeros(64)]).as_strided(t.shape, (t.stride(0), 3, *t.stride()[2:]))
  attn_compare(ops, odd(q), odd(k), odd(v), dout, lam)


def test_outputs_may_not_lie_in_the_small_arguments(ops):
  """lambda, the norm's weights, lengths, starts and the mask are read while results are written: an output in their memory is refused."""
  B, T, H, d = 2, 9, 2, 16
  q, k, v, dout, _ = attn_inputs(B, T, T, H, H, d, 2 * d, F32, seed=530)
  arena = torch.zeros(q.numel() + 64, device=DEV)
  out, dq = arena[:dout.numel()].view(dout.shape), arena[:q.numel()].view(q.shape)
  ints = arena.view(torch.int32)
  small = dict(lam=arena[4:4 + H], norm_weight=arena[8:8 + 2 * d], kv_len=ints[2:2 + B], q_start=ints[2:2 + B], key_mask=arena.view(torch.uint8)[:B * T].view(B, T))
  for n, t in small.items():
    kw = {'lam': torch.full((H,), 0.5, device=DEV), **{n: t}}
    lam = kw.pop('lam')
    with pytest.raises(ValueError, match=n):
      ops.diff_attn_fwd(q, k, v, lam, causal=True, out=out, **kw)
    _, ctx = ops.diff_attn_fwd(q, k, v, lam, causal=True, save=True, **kw)
    for g in (dict(dq=dq), dict(dk=dq), dict(dv=out)):
      with pytest.raises(ValueError, match=n):
        ops.diff_attn_bwd(dout, q, k, v, lam, ctx, **g)
  far = {n: t.clone() for n, t in small.items() if n != 'q_start'}
  lam = far.pop('lam')
  ops.diff_attn_fwd(q, k, v, lam, out=arena[64:64 + dout.numel()].view(dout.shape), **far)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('heads', [(16, 4, 64, 128), (8, 2, 32, 64), (8, 8, 27, 54), (4, 2, 128, 256)], ids=str)
@pytest.mark.parametrize('Tq', [1, 2, 5])
def test_answers_do_not_depend_on_how_many_sequences_there_are(ops, Tq, heads, dtype):
  """New tokens of 512 and 1024 batch x heads take the kernel that a few sequences take: the same bits (a cache this short is not split)."""
  H, Hkv, d, dv = heads
  for total in (512, 1024):
    B, Tk = total // H, 320
    q, k, v, dout, lam = attn_inputs(B, Tq, Tk, H, Hkv, d, dv, dtype, seed=540)
    lens = torch.randint(Tq, Tk + 1, (B,), generator=torch.Generator().manual_seed(total), dtype=torch.int32).to(DEV)
    opt = dict(causal=True, norm_weight=randn(dv, seed=541, mean=1.0, std=0.1))
    out, _ = ops.diff_attn_fwd(q, k, v, lam, kv_len=lens, q_start=lens - Tq, **opt)
    for b in range(0, B, 16):
      s = slice(b, b + 16)
      part, _ = ops.diff_attn_fwd(q[s], k[s], v[s], lam, kv_len=lens[s].clone(), q_start=(lens - Tq)[s].clone(), **opt)
      assert torch.equal(out[s], part)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('Tk', [1, 50, 700])
@pytest.mark.parametrize('heads', [(8, 2, 64, 128), (8, 8, 16, 32)], ids=str)
def test_single_tokens_of_many_sequences(ops, heads, Tk, dtype):
  H, Hkv, d, dv = heads
  for B in (64, 128):
    q, k, v, dout, lam = attn_inputs(B, 1, Tk, H, Hkv, d, dv, dtype, seed=550)
    lens = torch.randint(0, Tk + 1, (B,), generator=torch.Generator().manual_seed(B), dtype=torch.int32).to(DEV)
    attn_compare(ops, q, k, v, dout, lam, train=B == 64, kv_len=lens)


def test_calls_of_several_threads(ops):
  """Threads with streams of their own, released together: their first calls of the wide kernels and later ones give what one thread gives."""
  import threading
  cases = [(2, 90, 150, 2, 1, d, 2 * d) for d in (128, 96, 72, 64)]
  start, got, errors = threading.Barrier(4), [None] * 4, []
  data = [attn_inputs(*c, BF16, seed=560) for c in cases]
  torch.cuda.synchronize()

  def step(i):
    q, k, v, dout, lam = data[i]
    out, ctx = ops.diff_attn_fwd(q, k, v, lam, causal=True, save=True)
    return [out, *ops.diff_attn_bwd(dout, q, k, v, lam, ctx)[:4]]

  def work(i):
    try:
      with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        for n in range(8):
          got[i] = step((i + n) % 4)
        torch.cuda.current_stream().synchronize()
    except Exception as e:  # noqa: BLE001
      errors.append(e)

  threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  assert not errors, errors
  for i in range(4):
    assert all(torch.equal(a, b) for a, b in zip(got[i], step((i + 7) % 4)))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('eps', [1e-30, 1e-5, 0.5])
def test_tiny_and_large_eps_with_queries_that_see_nothing(ops, eps, dtype):
  """r = 1 / sqrt(mean(O^2) + eps) is 1e15 for a query without keys: its powers leave 32 bits, its gradients are zeros all the same."""
  q, k, v, dout, lam = attn_inputs(2, 9, 40, 2, 1, 32, 64, dtype, seed=570)
  lens = torch.tensor([0, 33], dtype=torch.int32, device=DEV)
  w = randn(64, seed=571, mean=1.0, std=0.1)
  want = attn_oracle(q, k, v, lam, attn_visible(2, 9, 40, kv_len=lens), dout=dout, w=w, eps=eps)
  out, ctx = ops.diff_attn_fwd(q, k, v, lam, kv_len=lens, norm_weight=w, norm_eps=eps, save=True)
  for n, g in zip(('out', 'dq', 'dk', 'dv', 'dlam', 'dw'), (out, *ops.diff_attn_bwd(dout, q, k, v, lam, ctx))):
    within(n, g, *want[n])


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('d,pd', [(27, 32), (9, 16)])
def test_heads_padded_with_zeros(ops, d, pd, dtype):
  """Channels of zeros up to a multiple of 16 bytes, the scale of the narrow heads, weights and eps for the wider mean: the narrow heads' numbers."""
  B, Tq, Tk, H, Hkv, dv = 2, 45, 83, 2, 1, 2 * d
  pv = (dv + 7) // 8 * 8
  q, k, v, dout, lam = attn_inputs(B, Tq, Tk, H, Hkv, d, dv, dtype, seed=580)
  w = randn(dv, seed=581, mean=1.0, std=0.1)
  wide = lambda t, n: torch.nn.functional.pad(t, (0, n - t.shape[-1]))
  want = attn_oracle(q, k, v, lam, attn_visible(B, Tq, Tk, causal=True), dout=dout, w=w, eps=1e-5)
  out, ctx = ops.diff_attn_fwd(wide(q, pd), wide(k, pd), wide(v, pv), lam, causal=True, scale=d ** -0.5, norm_weight=wide(w, pv) * math.sqrt(dv / pv), norm_eps=1e-5 * dv / pv, save=True)
  dq, dk, dvv, dlam, dw = ops.diff_attn_bwd(wide(dout, pv), wide(q, pd), wide(k, pd), wide(v, pv), lam, ctx)
  for n, g, m in (('out', out, dv), ('dq', dq, d), ('dk', dk, d), ('dv', dvv, dv)):
    value, err = want[n]
    # (the weights' square root and product round three times in 32 bits: 2^-22 of a value)
    within(n, g[..., :m], value, err + 2.0 ** -22 * value.abs())
    assert n == 'dq' or n == 'dk' or not g[..., m:].any()
  within('dlam', dlam, want['dlam'][0], want['dlam'][1] * (1 + 2.0 ** -22))
  within('dw', dw[:dv] * math.sqrt(dv / pv), want['dw'][0], want['dw'][1] + 2.0 ** -22 * want['dw'][0].abs())
