"""The optimizer operators where their surroundings change: parameters that move, default types, options between steps, states
from elsewhere."""
import numpy as np
import pytest
import torch

from tests.test_gpu_adamw import TYPES, _params

pytestmark = pytest.mark.gpu


def _snapshot(opt, ps):
  return [p.detach().clone() for p in ps] + [t.view(torch.uint8).clone() for held in opt.buffers.values() for t in held.values()]


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("clip", [None, 1.0])
def test_a_parameter_that_changes_the_order_of_its_elements_is_refused(typ, clip):
  """Moments lie in the order their parameter had: the same values in another order of memory would meet others' moments.  The
  same order elsewhere in memory is served."""
  from oi_vae_amd import optim
  for first in (lambda x: x, lambda x: x.t().contiguous().t()):
    x = first(torch.randn(24, 40, generator=torch.Generator().manual_seed(0)).to(TYPES[typ]).cuda())
    p = x.clone().requires_grad_()
    p.grad = torch.ones_like(x)
    opt = optim.AdamW([p], lr=0.1, max_grad_norm=clip)
    opt.step()
    p.data = p.data.clone()
    opt.step()
    was = _snapshot(opt, [p])
    p.data = p.data.t().contiguous().t() if p.is_contiguous() else p.data.contiguous()
    p.grad = p.grad.clone()
    with pytest.raises(ValueError, match="order of its elements"):
      opt.step()
    with pytest.raises(ValueError, match="order of its elements"):
      opt.sync_master()
    assert opt.steps() == [2] and all(torch.equal(a, b) for a, b in zip(was, _snapshot(opt, [p])))
    p.data = torch.empty_like(x).copy_(p.data)
    opt.step()
    assert opt.steps() == [3] and not torch.equal(was[0], p)
