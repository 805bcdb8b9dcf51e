"""C entries of the transformer-block operators store saved rows, statistics and scratch 8 or 16 bytes at a time: pointers that are not aligned for it
are refused before anything is launched (no GPU needed)."""
import ctypes

import pytest

from carla_garage_amd._lib import BF16, EINVAL, F32
from test_transformer_ops import FAKE, L, attn_params, norm_params  # noqa: F401  (L: the fixture)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('kw', [dict(o1=FAKE + 8), dict(o2=FAKE + 4), dict(partial=FAKE + 8)], ids=str)
def test_diff_attention_forward_refuses(L, kw, dtype):
  assert L.raw('tfpp_diff_attn_fwd')(ctypes.byref(attn_params(**kw)), dtype, None) == EINVAL


@pytest.mark.parametrize('kw', [dict(o2=FAKE + 8), dict(d_o=FAKE + 8), dict(slope=FAKE + 8), dict(slope=None), dict(partial=FAKE + 4)], ids=str)
def test_diff_attention_backward_refuses(L, kw):
  assert L.raw('tfpp_diff_attn_bwd')(ctypes.byref(attn_params(**{'slope': FAKE, **kw})), BF16, None) == EINVAL


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_block_norm_forward_refuses(L, dtype):
  for off in (4, 8):
    assert L.raw('tfpp_block_norm_fwd')(ctypes.byref(norm_params(stat=FAKE + off)), dtype, None) == EINVAL
