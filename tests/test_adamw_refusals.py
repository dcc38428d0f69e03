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
