"""Steps that AdamW leaves out, inside OIVAE: nothing of the model may move, Ws and its zero set included."""
import ctypes

import numpy as np
import pytest
import torch

from tests.test_gpu_adamw import _check, _np, _state, _vae

pytestmark = pytest.mark.gpu


def _everything(vae, opt):
  eng = vae.engine
  out = [eng.flat_params, eng.zero_mask, eng.row_norms] + [t.view(torch.uint8) for held in opt.buffers.values() for t in held.values()]
  return [t.clone() for t in out]


def _make(order, lam=1.0, bits=32):
  from oi_vae_amd import optim

  def opts(groups, ws):
    pair = [optim.AdamW(groups, lr=1e-3, weight_decay=0.05, state_bits=bits, max_grad_norm=10.0), optim.SGD(ws, lr=1e-4)]
    return pair if order == "AdamW first" else pair[::-1]
  vae, pair = _vae(opts)
  vae.lam = lam
  return vae, pair[0] if order == "AdamW first" else pair[1]


def _batches(B):
  g = torch.Generator().manual_seed(1)
  X = [torch.rand(B, 24, generator=g).cuda() for _ in range(3)]
  return X, [torch.randn(1, B, 8, generator=g) for _ in range(3)]


@pytest.mark.parametrize("lam", [1.0, 0.0])
@pytest.mark.parametrize("order", ["AdamW first", "SGD first"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("B", [16, 20000])     # the one-launch step, and the entry points
def test_a_batch_with_a_nan_changes_nothing(B, bits, order, lam):
  """One bad batch between good ones: nothing moves in it, and the next step is the second one of the optimizer.  The one-launch
  step adds in a fixed order: there the run goes on as one that never saw the batch, bit for bit (the entry points add some gradients
  with atomics, two runs of one program differ in their last places)."""
  X, eps = _batches(B)
  bad = X[1].clone()
  bad[3, 5] = float("nan")
  runs = []
  for seen in (True, False):
    vae, opt = _make(order, lam, bits)
    vae.step(X[0], 1e-3, 1, eps=eps[0])
    if seen:
      was = _everything(vae, opt)
      vae.step(bad, 1e-3, 1, eps=eps[1])
      assert not np.isfinite(opt.grad_norm.item()) and opt.skipped.item() == 1 and opt.steps() == [1]
      assert all(torch.equal(a, b) for a, b in zip(was, _everything(vae, opt)))
    before = _state(opt)
    vae.step(X[2], 1e-3, 1, eps=eps[2])
    g = _np(vae.engine.flat_grads[:vae.engine.adam_numel])
    _check(opt, before, _state(opt), [g], 2, [1e-3], [0.05], scale=min(1.0, 10.0 / (np.sqrt((g * g).sum()) + 1e-6)), codes=False)
    assert opt.steps() == [2] and opt.skipped.item() == int(seen) and np.isfinite(opt.grad_norm.item())
    runs.append(_everything(vae, opt))
  assert B != 16 or all(torch.equal(a, b) for a, b in zip(*runs))
  assert torch.isfinite(runs[0][0]).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("B", [16, 20000])
def test_a_gradient_of_Ws_alone_that_is_not_finite(B, value):
  """Only dWs is bad: it does not enter the norm that clips, but the step is left out all the same."""
  X, eps = _batches(B)
  vae, opt = _make("AdamW first")
  eng = vae.engine
  vae.step(X[0], 1e-3, 1, eps=eps[0])
  was = _everything(vae, opt)
  name = "small_step" if B == 16 else "forward_backward"
  plain = getattr(eng, name)

  def spoiled(*a, **kw):
    out = plain(*a, **kw)
    eng.g["Ws"].view(-1)[-1] = value
    return out
  setattr(eng, name, spoiled)
  vae.step(X[1], 1e-3, 1, eps=eps[1])
  delattr(eng, name)
  assert np.isnan(opt.grad_norm.item()) and opt.skipped.item() == 1 and opt.steps() == [1]
  assert all(torch.equal(a, b) for a, b in zip(was, _everything(vae, opt)))
  vae.step(X[1], 1e-3, 1, eps=eps[1])
  assert opt.steps() == [2] and not torch.equal(was[0], eng.flat_params) and torch.isfinite(eng.flat_params).all()


@pytest.mark.parametrize("count", [100, 300])      # one launch that concludes the norm itself, two with one behind them
@pytest.mark.parametrize("n", [1, 5, 4096, 300001, 5000000])
def test_watched_gradients_leave_the_norm_alone(n, count):
  """oivae_grad_norm with a watched tensor behind others: the same norm, coefficient and counters to the bit."""
  from oi_vae_amd import _lib, optim
  L = _lib.init_device(0)
  g = torch.Generator(device="cuda").manual_seed(n)
  grads = [torch.randn(1 + k % 7 * 333, generator=g, device="cuda") for k in range(count)]
  w = 1e19 * torch.randn(n, generator=g, device="cuda")
  got = []
  for last in (None, 0.0, float("inf")):
    rec = np.zeros(len(grads) + (last is not None), optim._GRAD)
    rec["g"][:count], rec["n"][:count], rec["index"][:count] = [x.data_ptr() for x in grads], [x.numel() for x in grads], np.arange(count)
    if last is not None:
      w[-1] = last
      rec[count] = (w.data_ptr(), n, _lib.F32_WATCHED, -1)
    clip, steps = torch.zeros(8, device="cuda"), torch.zeros(count, 4, device="cuda")
    nbytes = L.oivae_grad_norm_workspace_bytes(len(rec))
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    _lib.check(L.oivae_grad_norm(rec.ctypes.data, len(rec), 1, 1.0, 1.0, clip.data_ptr(), steps.data_ptr(), 0.9, 0.999, ws.data_ptr(),
                                 nbytes, torch.cuda.current_stream().cuda_stream), "oivae_grad_norm")
    torch.cuda.synchronize()
    got.append((clip.clone(), steps.clone()))
  assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
  assert torch.isnan(got[2][0][0]) and got[2][0].view(torch.int32)[2:4].tolist() == [1, 1] and (got[2][1] == 0).all()


@pytest.mark.parametrize("H", [3, 8, 32, 64, 512])
def test_sgd_prox_heeds_the_verdict(H):
  """Every row kernel of oivae_sgd_prox_clip_f32: a verdict that leaves the step out leaves Ws, mask and norms; any other, or none,
  gives oivae_sgd_prox_f32's bits."""
  from oi_vae_amd import _lib
  L = _lib.init_device(0)
  for rows in (7, 530000) if H == 8 else (7, 3000):
    g = torch.Generator(device="cuda").manual_seed(H)
    W, dW = (torch.randn(rows, H, generator=g, device="cuda") for _ in range(2))
    st = torch.cuda.current_stream().cuda_stream
    out = []
    for skip in ("plain", None, 0, 1):
      w, mask, norms = W.clone(), torch.full((rows,), 9, dtype=torch.uint8, device="cuda"), torch.full((rows,), -1.0, device="cuda")
      args = (w.data_ptr(), dW.data_ptr(), rows, H, 0.1, 1.0, 1, mask.data_ptr(), norms.data_ptr())
      if skip == "plain":
        rc = L.oivae_sgd_prox_f32(*args, st)
      else:
        clip = torch.tensor([0, 0, skip or 0, 0, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
        rc = L.oivae_sgd_prox_clip_f32(*args, None if skip is None else clip.data_ptr(), st)
      assert rc == 0
      torch.cuda.synchronize()
      out.append((w, mask, norms))
    assert all(torch.equal(a, b) for o in out[1:3] for a, b in zip(out[0], o))
    assert torch.equal(out[3][0], W) and (out[3][1] == 9).all() and (out[3][2] == -1).all()
    assert not torch.equal(out[0][0], W) and (out[0][1] < 2).all()
