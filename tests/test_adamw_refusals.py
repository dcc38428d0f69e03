"""What the optimizer operators refuse before anything reaches a GPU, beyond test_adamw_host.py."""
import ctypes

import numpy as np
import pytest
import torch


def test_watched_gradients_are_for_the_norm_alone():
  """OIVAE_F32_WATCHED names no parameter's or gradient's type: AdamW and clipping refuse it; the norm checks its alignment."""
  from oi_vae_amd import _lib, optim
  L = _lib.load()
  g = np.zeros(1, optim._GRAD)
  g["g"], g["n"], g["index"], g["type"] = 4096, 10, -1, _lib.F32_WATCHED
  need = L.oivae_grad_norm_workspace_bytes(1)
  assert L.oivae_clip_grad_norm(g.ctypes.data, 1, 1.0, 1 << 20, 2 << 20, need, None) == 1 and b"unknown gradient" in L.oivae_last_error()
  norm = lambda: L.oivae_grad_norm(g.ctypes.data, 1, 1, 1.0, 1.0, 1 << 20, None, 0.9, 0.999, 2 << 20, need, None)
  g["g"] = 4098
  assert norm() == 1 and b"aligned" in L.oivae_last_error()
  g["g"], g["type"] = 4096, _lib.F32_WATCHED + 1
  assert norm() == 1 and b"unknown gradient" in L.oivae_last_error()
  r, grp = np.zeros(1, optim._TENSOR), np.zeros(1, optim._GROUP)
  st = _lib.AdamwState(1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, None)
  for field in ("p_type", "g_type"):
    r["p"], r["g"], r["n"], r["step"], r["p_type"], r["g_type"] = 4096, 8192, 10, 1, 0, 0
    r[field] = _lib.F32_WATCHED
    assert L.oivae_adamw_f32(r.ctypes.data, 1, grp.ctypes.data, 1, ctypes.byref(st), 0.9, 0.999, 1e-8, 1.0, None, None) == 1


def test_sgd_prox_clip_refuses_what_sgd_prox_does():
  from oi_vae_amd import _lib
  L = _lib.load()
  for args in ((None, 4096, 1, 8), (4096, None, 1, 8), (4096, 8192, -1, 8), (4096, 8192, 1, 0), (4096, 8192, 1, (1 << 20) + 1), (4096, 8192, 1 << 40, 8)):
    rc = L.oivae_sgd_prox_f32(*args, 0.1, 1.0, 1, None, None, None)
    assert rc in (1, 2) and L.oivae_sgd_prox_clip_f32(*args, 0.1, 1.0, 1, None, None, None, None) == rc
    assert b"oivae_sgd_prox_clip_f32" in L.oivae_last_error()


def _script(name):
  import importlib.util
  import os
  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scripts", name + ".py")
  spec = importlib.util.spec_from_file_location(name, path)
  mod = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(mod)
  return mod


@pytest.mark.parametrize("kw", [dict(max_grad_norm=1.0), dict(state_bits=8), dict(weight_decay=0.01, native_optimizers=False),
                                dict(weight_decay=0.01, max_grad_norm=1.0, native_optimizers=False),
                                dict(max_grad_norm=1.0, native_optimizers=False)])
def test_an_experiment_refuses_options_it_would_drop(kw):
  from oi_vae_amd.experiments import Experiment
  with pytest.raises(ValueError, match="AdamW's"):
    Experiment(dim_x=8, dim_z=4, group_dims=[4, 4], group_input_dim=2, **kw)


@pytest.mark.parametrize("argv", [["--max-grad-norm", "1"], ["--state-bits", "8"], ["--state-bits", "8", "--max-grad-norm", "1"]])
def test_the_meg_driver_refuses_options_it_would_drop(argv, capsys):
  with pytest.raises(SystemExit) as e:
    _script("meg_oi_vae").main(argv)
  assert e.value.code == 2 and "--weight-decay" in capsys.readouterr().err


@pytest.mark.parametrize("argv", [["--max-grad-norm", "1"], ["--state-bits", "8"], ["--weight-decay", "0.1"], ["--optimizer", "adam", "--weight-decay", "0.1"]])
def test_the_autoencoder_driver_refuses_options_it_would_drop(argv, capsys):
  with pytest.raises(SystemExit) as e:
    _script("data_vs_test_loss_autoencoder").main(argv)
  assert e.value.code == 2 and "--optimizer adamw" in capsys.readouterr().err


def test_order_of_elements():
  """Row by row is 0, whatever the strides of dimensions of one element; other orders differ from it and from each other."""
  from oi_vae_amd import _tensor_lists
  order, x = _tensor_lists.order, torch.zeros(4, 6, 5)
  assert order(x) == 0 == order(x.view(24, 5)) == order(x.new_zeros(0, 3)) == order(x.new_zeros(())) == order(x.new_zeros(7, 1).t())
  others = [x.permute(2, 0, 1), x.permute(2, 1, 0), x.permute(1, 0, 2), x.new_zeros(24, 5).t(), x.new_zeros(5, 24).t()]
  codes = [order(t) for t in others]
  assert 0 not in codes and len(set(codes)) == len(codes)
  assert codes == [order(torch.empty_like(t)) for t in others] == [order(t[None]) for t in others]
  with pytest.raises(TypeError):
    order(3)


@pytest.mark.parametrize("limit", [1e-50, 1e-46, 0.0, -1.0, float("nan"), -float("inf")])
def test_limits_that_float32_does_not_hold_are_refused(limit):
  """The kernels take the limit as a float32, where 0 means no clipping."""
  from oi_vae_amd import optim
  p = torch.zeros(3, requires_grad=True)
  with pytest.raises(ValueError, match="max_norm must be positive"):
    optim.clip_grad_norm_([p], limit)
  with pytest.raises(ValueError, match="max_grad_norm must be positive"):
    optim.AdamW([p], max_grad_norm=limit)
  for fine in (1e-44, 1, np.float32(0.5), torch.tensor(2.0), 1e300, float("inf")):
    optim.AdamW([p], max_grad_norm=fine)


def test_zero_grad_in_place():
  """Gradients that are views of a flat buffer, that have a graph of their own, and plain ones."""
  from oi_vae_amd import optim
  flat = torch.ones(10)
  p, q, r = (torch.ones(5, requires_grad=True) for _ in range(3))
  p.grad = flat[2:7]
  (q ** 3).sum().backward(create_graph=True)
  r.grad = torch.ones(5)
  opt = optim.AdamW([p, q, r])
  opt.zero_grad(set_to_none=False)
  assert flat.tolist() == [1.0] * 2 + [0.0] * 5 + [1.0] * 3 and p.grad.data_ptr() == flat[2:].data_ptr()
  assert all((t.grad == 0).all() and not t.grad.requires_grad for t in (p, q, r))


def test_what_is_no_list_of_leaves():
  """A tensor in place of a list (whose rows would be stepped without gradients, that is not at all), results of operations,
  names beside parameters."""
  from oi_vae_amd import optim
  w = torch.zeros(3, 4, requires_grad=True)
  for cls in (optim.AdamW, optim.Adam, optim.SGD):
    with pytest.raises(TypeError, match="one tensor"):
      cls(w)
    group = cls([{"params": w}]).param_groups[0]
    assert len(group["params"]) == 1 and group["params"][0] is w
  for bad in ([w * 2], [w[0]], [{"params": [w, w.t()]}]):
    with pytest.raises(ValueError, match="result of an operation"):
      optim.AdamW(bad)
  for bad in ([("w", w)], {"params": [w]}, [{"params": "w"}]):
    with pytest.raises(ValueError, match="must be tensors"):
      optim.AdamW(bad)
  kept = w * 2
  kept.retain_grad()
  optim.AdamW([kept, w])
