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


def _made(kinds, **kw):
  """An AdamW over groups of parameters given as [(type, size, row-major?), ...], one step taken."""
  from oi_vae_amd import optim
  g = torch.Generator(device="cuda").manual_seed(len(kinds))
  groups = []
  for k, members in enumerate(kinds):
    ps = []
    for typ, shape, rows in members:
      x = torch.randn(shape, generator=g, device="cuda").to(TYPES[typ])
      p = (x if rows else x.t().contiguous().t()).requires_grad_()
      p.grad = torch.ones_like(p)
      ps.append(p)
    groups.append({"params": ps, "weight_decay": 0.01 * k})
  opt = optim.AdamW(groups, lr=1e-2, **kw)
  opt.step()
  return opt, [p for q in groups for p in q["params"]]


A, B = ("f32", (128,), True), ("bf16", (128,), True)
M, T = ("f32", (8, 16), True), ("f32", (8, 16), False)


@pytest.mark.parametrize("clip", [None, 1.0])
@pytest.mark.parametrize("theirs,mine", [([[A, B]], [[B, A]]),                 # equal sizes, types changed places
                                         ([[B, B]], [[("f16", (128,), True), B]]),
                                         ([[M, M]], [[M, T]]),                 # another order in memory
                                         ([[A, A], [A]], [[A], [A, A]]),       # another group
                                         ([[A, B], [B]], [[A], [B, B]])])
def test_a_state_of_other_types_orders_or_groups_is_refused(theirs, mine, clip):
  state = _made(theirs, max_grad_norm=clip)[0].state_dict()
  opt, ps = _made(mine, max_grad_norm=clip)
  was, steps = _snapshot(opt, ps), opt.steps()
  with pytest.raises(ValueError, match="other parameters or groups"):
    opt.load_state_dict(state)
  assert steps == opt.steps() and all(torch.equal(a, b) for a, b in zip(was, _snapshot(opt, ps)))
  opt, ps = _made(theirs, max_grad_norm=clip)
  opt.step()
  opt.load_state_dict(state)
  assert opt.steps() == steps


def test_states_from_before_they_held_their_layout():
  """Taken where the sizes decide the layout, refused where they do not."""
  for kinds, taken in (([[A, M]], True), ([[B, B]], True), ([[A, B]], False), ([[A], [A]], True)):
    opt, ps = _made(kinds)
    state = opt.state_dict()
    for k in ("types", "orders", "group_of"):
      del state[k]
    opt.step()
    was = _snapshot(opt, ps)
    if taken:
      opt.load_state_dict(state)
      assert opt.steps() == [1] * len(ps)
    else:
      with pytest.raises(ValueError, match="unknown types"):
        opt.load_state_dict(state)
      assert all(torch.equal(a, b) for a, b in zip(was, _snapshot(opt, ps)))


@pytest.mark.parametrize("clip", [None, 1.0])
@pytest.mark.parametrize("change", [lambda s: s["groups"][1].update(initial_lr=1e-2), lambda s: s["groups"][0].pop("eps"),
                                    lambda s: s["groups"][0].update(lr=-1.0), lambda s: s["groups"][1].update(betas=(0.8, 0.9)),
                                    lambda s: s["groups"][0].update(lr=torch.zeros(2)), lambda s: s["groups"][0].update(weight_decay=float("nan")),
                                    lambda s: s["steps"].pop(), lambda s: s["steps"].append(1), lambda s: s.update(steps=[1, -1, 1]),
                                    lambda s: s.update(steps=[1, 1 << 40, 1]), lambda s: s.update(seed=1 << 32), lambda s: s.pop("seed"),
                                    lambda s: s.pop("steps"), lambda s: s.pop("buffers"), lambda s: s["buffers"][32].pop("exp_avg_sq")])
def test_a_state_is_taken_whole_or_not_at_all(change, clip):
  opt, ps = _made([[A, B], [B]], max_grad_norm=clip)
  state = opt.state_dict()
  change(state)
  opt.step()
  options = [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]
  was, steps, seed = _snapshot(opt, ps), opt.steps(), opt.seed
  with pytest.raises((ValueError, OverflowError)):
    opt.load_state_dict(state)
  assert steps == opt.steps() and seed == opt.seed and all(torch.equal(a, b) for a, b in zip(was, _snapshot(opt, ps)))
  assert options == [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]


@pytest.mark.parametrize("there,here", [(1e-3, None), (None, 1e-3), (None, None), ("0-dim", None), (None, "0-dim")])
def test_learning_rates_of_a_state(there, here):
  """A number or one float32 on the device (of any shape of one element) on either side; the one here stays in place."""
  def lr(what, value):
    return value if what is not None and what != "0-dim" else torch.full(() if what else (1,), value, device="cuda")
  opt, ps = _made([[A]], capturable=True)
  opt.param_groups[0]["lr"] = lr(there, 0.25)
  state = opt.state_dict()
  mine = opt.param_groups[0]["lr"] = lr(here, 0.5)
  opt.load_state_dict(state)
  assert float(opt.param_groups[0]["lr"]) == 0.25 and (opt.param_groups[0]["lr"] is mine or not torch.is_tensor(mine))


def test_steps_left_out_are_counted_on_after_resuming():
  opt, ps = _made([[A, B]], max_grad_norm=1.0)
  ps[0].grad[3] = float("nan")
  for _ in range(2):
    opt.step()
  state = opt.state_dict()
  assert state["skipped"] == 2 and state["steps"] == [1, 1]
  other, qs = _made([[A, B]], max_grad_norm=1.0)
  other.load_state_dict(state)
  assert other.skipped.item() == 2
  qs[1].grad[0] = float("inf")
  other.step()
  assert other.skipped.item() == 3 and other.steps() == [1, 1]
  for bad in (-1, 1 << 31):
    with pytest.raises(ValueError, match="left out"):
      other.load_state_dict({**state, "skipped": bad})
  del state["skipped"]          # a state from before they were held
  other.load_state_dict(state)
  assert other.skipped.item() == 0
  plain = _made([[A, B]])[0]
  assert plain.state_dict()["skipped"] == 0
  plain.load_state_dict({**state, "skipped": 5})


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_under_another_default_type(default):
  """torch.set_default_dtype changes nothing: the norm is a float32, the step the same."""
  from oi_vae_amd import optim

  def run(default):
    ps = _params([300, 5000], torch.float32, seed=3)
    torch.set_default_dtype(default)
    try:
      opt = optim.AdamW(ps, lr=1e-2, max_grad_norm=0.1)
      opt.step()
      norms = [optim.grad_norm(ps), opt.grad_norm, optim.clip_grad_norm_(ps, 0.1), optim.grad_norm([]), optim.clip_grad_norm_([], 1.0)]
    finally:
      torch.set_default_dtype(torch.float32)
    assert all(n.dtype == torch.float32 for n in norms)
    return [n.item() for n in norms], _snapshot(opt, ps) + [p.grad.clone() for p in ps]
  want, got = run(torch.float32), run(default)
  assert got[0] == want[0] and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


@pytest.mark.parametrize("kw", [dict(), dict(capturable=True), dict(max_grad_norm=1.0)])
def test_options_that_became_bad_are_refused_before_anything_is_queued(kw):
  """The counts on the device advance with the norm, ahead of the step: a refused step must not have moved them."""
  opt, ps = _made([[A, B], [B]], **kw)
  was = _snapshot(opt, ps)
  for key, bad in (("eps", -1e-8), ("eps", float("nan")), ("betas", (1.0, 0.999)), ("betas", (0.9, -0.5)), ("betas", (0.9, float("nan")))):
    keep = [g[key] for g in opt.param_groups]
    for g in opt.param_groups:
      g[key] = bad
    with pytest.raises(ValueError, match="eps must|betas must|one 'betas'|one 'eps'|to every param group"):
      opt.step()
    for g, k in zip(opt.param_groups, keep):
      g[key] = k
    assert opt.steps() == [1, 1, 1] and all(torch.equal(a, b) for a, b in zip(was, _snapshot(opt, ps)))
  opt.step()
  assert opt.steps() == [2, 2, 2]


def test_a_limit_changed_between_steps():
  """A later limit is used, or refused as the constructor refuses it -- not taken for none; None takes no norm."""
  opt, ps = _made([[A, B]], max_grad_norm=1.0)
  was = _snapshot(opt, ps)
  for bad in (0.0, -1.0, float("nan"), 1e-50):
    opt.max_grad_norm = bad
    with pytest.raises(ValueError, match="max_grad_norm must be positive"):
      opt.step()
  assert opt.steps() == [1, 1] and all(torch.equal(a, b) for a, b in zip(was, _snapshot(opt, ps)))
  norms = []
  for limit in (0.5, 1e9):
    for p in ps:
      p.grad.mul_(2.0)
    opt.max_grad_norm = limit
    opt.step()
    norms.append(opt.grad_norm.clone())        # (grad_norm itself is the optimizer's buffer: the last step's)
  assert norms[1].item() == 2 * norms[0].item() and opt.grad_norm.item() == norms[1].item()
  opt.max_grad_norm = None
  opt.step()
  assert opt.steps() == [4, 4]


def test_clipping_refuses_what_it_cannot_scale_before_it_scales_anything():
  """An expanded gradient, and gradients that share some memory, beside plain ones: nothing is written.  The norm alone reads them."""
  from oi_vae_amd import optim
  flat = torch.ones(100, device="cuda")
  for grads, error in (([torch.ones(1, device="cuda").expand(50)], RuntimeError),
                       ([torch.ones(1, 7, device="cuda").expand(5, 7)], RuntimeError),
                       ([flat[:60], flat[59:]], ValueError), ([flat, flat[10:20]], ValueError),
                       ([flat[:60], flat[10:20], flat[70:80]], ValueError)):
    ps = [torch.zeros(g.shape, device="cuda").requires_grad_() for g in [torch.ones(40)] + grads]
    for p, g in zip(ps, [torch.ones(40, device="cuda")] + grads):
      p.grad = g
    for order in (ps, ps[::-1]):
      with pytest.raises(error):
        optim.clip_grad_norm_(order, 1e-3)
      assert all((p.grad == 1).all() for p in ps)
      assert abs(optim.grad_norm(order).item() - np.sqrt(sum(p.numel() for p in ps))) <= 2.0 ** -23 * 20
  ps = [torch.zeros(g.shape, device="cuda").requires_grad_() for g in (flat[:60], flat[60:])]      # neighbours share nothing
  ps[0].grad, ps[1].grad = flat[:60], flat[60:]
  optim.clip_grad_norm_(ps, 1.0)
  assert ((flat - 0.1).abs() <= 2.0 ** -23).all()
  wide = torch.ones(100, device="cuda")                                                            # interleaved: neither
  q = [torch.zeros(50, device="cuda").requires_grad_() for _ in range(2)]
  q[0].grad, q[1].grad = wide[::2], wide[1::2]
  optim.clip_grad_norm_(q, 1.0)
  assert ((wide - 0.1).abs() <= 2.0 ** -23).all()


def test_moments_of_8_bits_follow_the_exact_ones_over_many_steps():
  """3000 steps of the kernel on Gaussian gradients whose scales spread over two decades in a block, against exact moments: the
  codes' expectation is exact, so the mean over 8192 elements is too, up to six of its standard deviations.  Second moments:
  0.53 of the moment an element (test_adamw_codes.py), 6 * 0.53 / sqrt(8192) = 0.036.  First moments, in units of the gradients'
  sigma: a step moves m by (1 - b1) (g - m), 0.083 in the mean; a spacing is m / 8 at most, 0.023 in the mean (m's own sigma is
  0.23), and 2^-16 of the block's largest, 0.003, for the smallest; 1 / (1 - b1^2) steps: a variance of at most 5.3 * 0.083 *
  0.026 = 0.0114, 0.107 an element, 6 * 0.107 / sqrt(8192) = 0.0071."""
  from oi_vae_amd import optim
  n, b1, b2 = 8192, 0.9, 0.999
  gen = torch.Generator(device="cuda").manual_seed(5)
  sigma = 10 ** (-3 + 2 * torch.rand(n, generator=gen, device="cuda"))
  p = torch.zeros(n, device="cuda").requires_grad_()
  p.grad = torch.empty(n, device="cuda")
  opt = optim.AdamW([p], lr=1e-4, betas=(b1, b2), state_bits=8)
  m = v = torch.zeros(n, dtype=torch.float64, device="cuda")
  for _ in range(3000):
    torch.mul(sigma, torch.randn(n, generator=gen, device="cuda"), out=p.grad)
    opt.step()
    m = b1 * m + (1 - b1) * p.grad.double()
    v = b2 * v + (1 - b2) * p.grad.double() ** 2
  held = opt.buffers[8]
  got = {k: held[k].double() * held[k + "_scale"].double().repeat_interleave(128) for k in ("exp_avg", "exp_avg_sq")}
  assert abs((got["exp_avg_sq"] / v).mean().item() - 1.0) <= 0.036
  assert abs(((got["exp_avg"] - m) / sigma).mean().item()) <= 0.0071
  assert opt.steps() == [3000] and torch.isfinite(p).all()


@pytest.mark.parametrize("b1,b2", [(0.9, 0.999), (0.9, 0.95), (0.0, 0.9999999), (0.999, 0.0)])
def test_bias_corrections_on_the_device(b1, b2):
  """1 / (1 - b1^t) and 1 / sqrt(1 - b2^t) of steps that count on the device: formed in float64 and rounded once to float32, which
  is at most 2^-24 of the value; the float64 roundings before it are below a thousandth of that."""
  from oi_vae_amd import optim
  p = torch.ones(3, device="cuda").requires_grad_()
  p.grad = torch.ones(3, device="cuda")
  opt = optim.AdamW([p], lr=0.0, betas=(b1, b2), capturable=True)
  u = 2.0 ** -24
  for t in list(range(1, 20)) + [50, 100, 333, 1000, 4321, 10 ** 4, 10 ** 5, 10 ** 6, 2 * 10 ** 9]:
    opt.set_steps(t - 1)
    opt.step()
    c1, c2 = opt._steps_dev[0].view(torch.float32)[1:3].double().tolist()
    e1 = 1.0 if b1 == 0 else -np.expm1(t * np.log(b1))
    e2 = 1.0 if b2 == 0 else -np.expm1(t * np.log(b2))
    assert abs(c1 * e1 - 1.0) <= 1.001 * u and abs(c2 * np.sqrt(e2) - 1.0) <= 1.001 * u, (t, (c1 * e1 - 1) / u, (c2 * np.sqrt(e2) - 1) / u)


@pytest.mark.parametrize("bits", [32, 8])
def test_counts_on_the_device_and_on_the_host_give_one_step(bits):
  """The corrections are the same wherever the steps are counted, and so are the bits of the step."""
  from oi_vae_amd import optim
  for t in (1, 2, 3, 10, 77, 1000, 12345, 10 ** 6):
    runs = []
    for capturable in (False, True):
      ps = _params([300, 5000, 1], torch.bfloat16, seed=t)
      opt = optim.AdamW(ps, lr=1e-2, state_bits=bits, capturable=capturable)
      opt.set_steps(t - 1)
      opt.step()
      runs.append(_snapshot(opt, ps))
    assert all(torch.equal(a, b) for a, b in zip(*runs)), t


def test_keys_that_a_schedule_added_to_the_groups():
  """Where the state has them too they are taken over; where it has not, the ones here stay."""
  opt, _ = _made([[A], [B]])
  state = opt.state_dict()
  for k, g in enumerate(opt.param_groups):
    g["initial_lr"] = 0.5 + k
  opt.load_state_dict(state)
  assert [g["initial_lr"] for g in opt.param_groups] == [0.5, 1.5]
  state = opt.state_dict()
  for g in opt.param_groups:
    g["initial_lr"] = 7.0
  opt.load_state_dict(state)
  assert [g["initial_lr"] for g in opt.param_groups] == [0.5, 1.5]


@pytest.mark.parametrize("kw", [dict(), dict(capturable=True), dict(max_grad_norm=1.0)])
@pytest.mark.parametrize("odd", [False, True])      # a gradient in another order sends the list the way round the native reader
def test_parameters_without_elements_count_their_steps(odd, kw):
  from oi_vae_amd import optim
  ps = _params([0, 5, 3], torch.float32, seed=1) + [torch.zeros(0, 4, device="cuda", requires_grad=True)]
  ps[3].grad = torch.zeros(0, 4, device="cuda")
  if odd:
    ps.append(torch.zeros(6, 7, device="cuda", requires_grad=True))
    ps[4].grad = torch.ones(7, 6, device="cuda").t()
  opt = optim.AdamW(ps, lr=1e-2, **kw)
  opt.step()
  ps[1].grad = None
  opt.step()
  assert opt.steps() == [2, 1, 2, 2] + [2] * odd
  for p in ps[2:3] + ps[4:]:
    p.grad = None
  opt.step()                    # those without elements alone
  assert opt.steps() == [3, 1, 2, 3] + [2] * odd
