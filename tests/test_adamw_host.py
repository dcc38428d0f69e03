"""Host side of the optimizer operators over lists of tensors: what the C entry points and oi_vae_amd.optim refuse, before
anything reaches a GPU."""
import ctypes

import numpy as np
import pytest
import torch


def _lib():
  from oi_vae_amd import _lib
  return _lib, _lib.load()


def _records(count=3, **kw):
  from oi_vae_amd import optim
  r = np.zeros(count, optim._TENSOR)
  r["p"], r["g"], r["n"], r["step"], r["index"] = 4096, 8192, 100, 1, np.arange(count)
  r["at"] = 128 * np.arange(count)
  for k, v in kw.items():
    r[k][count - 1] = v
  return r


def test_record_sizes_are_those_of_the_header(tmp_path):
  import os
  import subprocess
  from oi_vae_amd import optim
  lib, _ = _lib()
  root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
  src = tmp_path / "sizes.c"
  src.write_text('#include "oivae_hip.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) { printf("%zu %zu %zu %zu %zu %zu %zu %d",'
                 'sizeof(oivae_grad_t), sizeof(oivae_adamw_tensor_t), sizeof(oivae_adamw_group_t), sizeof(oivae_adamw_state_t),'
                 'sizeof(oivae_clip_t), sizeof(oivae_step_t), offsetof(oivae_adamw_tensor_t, step), OIVAE_ADAMW_BLOCK); return 0; }\n')
  exe = tmp_path / "sizes"
  subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
  got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
  assert got == [optim._GRAD.itemsize, optim._TENSOR.itemsize, optim._GROUP.itemsize, ctypes.sizeof(lib.AdamwState), 32, 16,
                 optim._TENSOR.fields["step"][1], lib.ADAMW_BLOCK]


@pytest.mark.parametrize("kw,word", [
  (dict(n=-1), "negative size"), (dict(g=0), "null gradient"), (dict(p=0), "is null"), (dict(g=8193, g_type=1), "aligned"),
  (dict(g=8194), "aligned"), (dict(p=4098), "aligned"), (dict(p_type=3), "unknown type"), (dict(g_type=-1), "unknown gradient"),
  (dict(p_type=1), "master"), (dict(at=64), "multiple of 128"), (dict(at=128), "reaches into"), (dict(at=0), "reaches into"), (dict(at=-128), "multiple of 128"), (dict(group=1), "group"),
  (dict(group=-1), "group"), (dict(index=-1), "index"), (dict(step=0), "step"), (dict(n=(1 << 40) + 1), "elements")])
def test_entry_points_refuse_bad_tensors(kw, word):
  from oi_vae_amd import optim
  lib, L = _lib()
  r = _records(**kw)
  grp = np.zeros(1, optim._GROUP)
  for eight in (False, True):
    st = lib.AdamwState(1 << 20, 2 << 20, 3 << 20, 4 << 20, None, None)
    args = (r.ctypes.data, 3, grp.ctypes.data, 1, ctypes.byref(st), 0.9, 0.999, 1e-8, 1.0)
    rc = L.oivae_adamw_f8(*args, 0, None, None) if eight else L.oivae_adamw_f32(*args, None, None)
    assert rc in (1, 2) and word in L.oivae_last_error().decode(), L.oivae_last_error()


def test_entry_points_refuse_bad_calls():
  from oi_vae_amd import optim
  lib, L = _lib()
  r, grp = _records(), np.zeros(1, optim._GROUP)
  good = lib.AdamwState(1 << 20, 2 << 20, 3 << 20, 4 << 20, None, None)

  def call(st=good, count=3, b1=0.9, b2=0.999, eps=1e-8, eight=False, tensors=r.ctypes.data):
    args = (tensors, count, grp.ctypes.data, 1, ctypes.byref(st), b1, b2, eps, 1.0)
    return L.oivae_adamw_f8(*args, 0, None, None) if eight else L.oivae_adamw_f32(*args, None, None)
  assert call(count=0) == 0 and call(count=-1) == 1 and call(tensors=None) == 1
  for bad in (dict(b1=1.0), dict(b2=1.0), dict(b1=-0.1), dict(eps=-1.0), dict(b2=float("nan"))):
    assert call(**bad) == 1, bad
  assert call(st=lib.AdamwState(None, 2 << 20, None, None, None, None)) == 1
  assert call(st=lib.AdamwState(1 << 20, (2 << 20) + 8, None, None, None, None)) == 1
  assert call(st=lib.AdamwState(1 << 20, 2 << 20, None, None, None, None), eight=True) == 1     # no scales
  g = np.zeros(2, optim._GRAD)
  g["g"], g["n"], g["index"] = 4096, 10, [0, 1]
  need = L.oivae_grad_norm_workspace_bytes(2)
  norm = lambda clip=1 << 20, steps=None, b1=0.9, ws=2 << 20, nb=need, count=2, rec=g.ctypes.data: L.oivae_grad_norm(
    rec, count, 1, 1.0, 1.0, clip, steps, b1, 0.999, ws, nb, None)
  scale = lambda out=1 << 20, ws=2 << 20, nb=need, count=2, rec=g.ctypes.data: L.oivae_clip_grad_norm(rec, count, 1.0, out, ws, nb, None)
  assert norm(clip=None) == 1 and norm(steps=1 << 20, b1=1.0) == 1 and scale(out=None) == 1
  for call in (norm, scale):
    assert call(count=-1) == 1 and call(rec=None) == 1 and call(ws=None) == 4 and call(nb=need - 1) == 4 and call(ws=(2 << 20) + 4) == 4
  for field, bad in (("type", 7), ("type", -1), ("index", -2), ("index", 1 << 29), ("n", -1), ("g", 0), ("g", 4098)):
    keep, g[field][1] = g[field][1], bad
    assert norm() == 1 and scale() == 1, (field, bad)
    g[field][1] = keep
  g["index"] = 5
  assert norm() == 1 and b"twice" in L.oivae_last_error() and scale() == 1
  assert L.oivae_grad_norm_workspace_bytes(0) >= 8 and L.oivae_grad_norm_workspace_bytes(10000) > need


def test_options_are_checked_when_they_are_given():
  from oi_vae_amd import optim
  p, q = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True)
  for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-0.1),
             dict(state_bits=4), dict(state_bits=16), dict(max_grad_norm=0.0), dict(max_grad_norm=-1.0), dict(seed=-1), dict(seed=1 << 32)):
    with pytest.raises(ValueError):
      optim.AdamW([p, q], **kw)
  for params in ([], [p, p], [{"params": [p]}, {"params": [p, q]}], [{"params": [p], "momentum": 0.9}],
                 [{"params": [p], "betas": (0.8, 0.9)}, {"params": [q]}], [{"params": [p], "state_bits": 7}]):
    with pytest.raises(ValueError):
      optim.AdamW(params)
  for bad in (0.0, -1.0, float("nan")):
    with pytest.raises(ValueError):
      optim.clip_grad_norm_([p], bad)
  opt = optim.AdamW([{"params": [p], "lr": 0.1}, {"params": [q], "weight_decay": 0.0, "state_bits": 8}])
  p.grad = torch.ones(3)
  opt.zero_grad(set_to_none=False)
  assert p.grad is not None and (p.grad == 0).all()
  opt.zero_grad()
  assert p.grad is None


def test_dense_means_one_piece_of_memory():
  from oi_vae_amd import optim
  x = torch.zeros(4, 6, 5)
  assert all(optim._dense(t) for t in (x, x.permute(2, 0, 1), x[1:3], x.new_zeros(0, 3), x.new_zeros(()), x.new_zeros(1, 7)[:, None]))
  assert not any(optim._dense(t) for t in (x[:, ::2], x[..., :4], x.new_zeros(1).expand(3), x[:, 1:3]))


def test_native_reader_leaves_the_unusual_to_python():
  """csrc/tensor_lists.cpp serves device memory only: a CPU tensor, a list that is none and short records are not read."""
  from oi_vae_amd import _tensor_lists, optim
  p, q = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True)
  rec, grads = np.zeros(2, optim._TENSOR), np.zeros(2, optim._GRAD)
  rec["n"] = 3
  assert _tensor_lists.parameters([p, q], rec, 0, grads) == (-1, 2) and (rec["g"] == 0).all() and (grads["index"] == -1).all()
  q.grad = torch.ones(3)
  assert _tensor_lists.parameters([p, q], rec, 0, None) == (1, 1)
  assert _tensor_lists.parameters([3, q], rec, 0, None)[0] == 0
  assert _tensor_lists.gradients([p], grads, False)[:2] == (0, -1) and _tensor_lists.gradients([p, q], grads, False) is None
  assert q.grad._version == 0
  for bad in (lambda: _tensor_lists.parameters((p,), rec, 0, None), lambda: _tensor_lists.parameters([p], rec, 0), lambda: _tensor_lists.gradients([p])):
    with pytest.raises(TypeError):
      bad()
  with pytest.raises(ValueError, match="fewer records"):
    _tensor_lists.parameters([p, q, p], rec, 0, None)
  with pytest.raises(BufferError):
    _tensor_lists.gradients([p, q], bytes(48), False)
