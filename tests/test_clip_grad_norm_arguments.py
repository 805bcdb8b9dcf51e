"""optim.clip_grad_norm_ takes the arguments of torch.nn.utils.clip_grad_norm_ (no GPU needed: parameters without gradients)."""
import inspect

import pytest
import torch

from carla_garage_amd.optim import clip_grad_norm_


def test_the_arguments_are_those_of_torch():
  mine, torchs = (list(inspect.signature(f).parameters.values()) for f in (clip_grad_norm_, torch.nn.utils.clip_grad_norm_))
  assert [(p.name, p.default) for p in mine] == [(p.name, p.default) for p in torchs]


@pytest.mark.parametrize('foreach', [None, True, False])
def test_foreach_is_taken(foreach):
  p = torch.nn.Parameter(torch.zeros(3))
  assert float(clip_grad_norm_(p, 1.0, foreach=foreach)) == 0.0
  assert float(clip_grad_norm_((q for q in [p]), 1.0, 2.0, True, foreach)) == 0.0
