"""Calls of differential attention that the documentation allows at the edges of its inputs: slots of a cache that no query sees yet, rows that share
memory, tiny eps with rows that see nothing, many sequences of single tokens, threads."""
import math

import pytest
import torch

from test_transformer_ops_gpu import BF16, DEV, F32, attn_compare, attn_inputs, ops, randn  # noqa: F401  (ops: the fixture)

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
