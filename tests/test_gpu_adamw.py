"""AdamW over lists of tensors (csrc/adamw.hip through oi_vae_amd.optim.AdamW), the gradient norm and clipping, against
float64 and -- the 8-bit moment codes -- bit for bit against float32 numpy.  Tolerances: _adamw_reference.py."""
import ctypes

import numpy as np
import pytest
import torch

from tests._adamw_reference import U, adamw64, decode, encode, moments32, random_bits

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
B1, B2, EPS = 0.9, 0.999, 1e-8
# one element, odd counts, a block of moments and its neighbours, a workgroup's 4096 and its neighbours, several workgroups
SIZES = {"one": [1], "few": [7, 0, 130, 1], "blocks": [127, 128, 129, 4095, 4096, 4097], "long": [70001, 3, 8192],
         "many": [1 + 37 * k % 301 for k in range(170)]}


def _params(sizes, typ, seed, offset=0):
  """Parameters with gradients, `offset` elements into their allocations."""
  g = torch.Generator(device="cuda").manual_seed(seed)
  out = []
  for n in sizes:
    p = (0.1 * torch.randn(n + offset, generator=g, device="cuda")).to(typ)[offset:].requires_grad_()
    p.grad = (1e-2 * torch.randn(n + offset, generator=g, device="cuda")).to(typ)[offset:]
    out.append(p)
  return out


def _np(t):
  return t.detach().double().cpu().numpy().reshape(-1)


def _opt(groups, t, seed=0, **kw):
  """An AdamW in the middle of a run: moments as after many steps, counts at t - 1."""
  from oi_vae_amd import optim
  opt = optim.AdamW(groups, betas=(B1, B2), eps=EPS, **kw)
  rng = np.random.default_rng(seed)
  opt.buffers
  for k in opt._kinds:
    bits, mine, rec = k.bits, k.mine, k.rec
    held = opt.buffers[bits]
    for r in rec:
      a, n = int(r["at"]), int(r["n"])
      m = (1e-3 * rng.standard_normal(n)).astype(np.float32)
      v = (1e-5 * rng.random(n)).astype(np.float32)
      if t == 1:
        m, v = 0 * m, 0 * v
      if bits == 8:
        b = slice(a // 128, (a + n + 127) // 128)
        for name, x, digits in (("exp_avg", m, 3), ("exp_avg_sq", v, 2)):
          c, s = encode(x, digits, np.full(n, 0.5))
          held[name].view(torch.uint8)[a:a + n] = torch.from_numpy(c).cuda()
          held[name + "_scale"].view(torch.uint8)[b] = torch.from_numpy(s).cuda()
      else:
        held["exp_avg"][a:a + n] = torch.from_numpy(m).cuda()
        held["exp_avg_sq"][a:a + n] = torch.from_numpy(v).cuda()
  opt.set_steps(t - 1)
  return opt


def _state(opt):
  """Per parameter: (w, m, v) as float64 arrays in the flat order, and the codes and scale bytes of 8-bit moments."""
  out = {}
  opt.buffers
  for k in opt._kinds:
    bits, mine, rec = k.bits, k.mine, k.rec
    held = opt.buffers[bits]
    for i, r in zip(mine, rec):
      a, n = int(r["at"]), int(r["n"])
      p = opt._leaves[i]
      w = held["master"][a:a + n] if r["p_type"] else torch.as_strided(p.detach(), (n,), (1,))
      s = {"w": _np(w), "p": _np(torch.as_strided(p.detach(), (n,), (1,))), "bits": bits}
      for name, digits in (("exp_avg", 3), ("exp_avg_sq", 2)):
        if bits == 8:
          c = held[name].view(torch.uint8)[a:a + n].cpu().numpy()
          b = held[name + "_scale"].view(torch.uint8)[a // 128:(a + n + 127) // 128].cpu().numpy()
          s[name + "_code"], s[name + "_byte"] = c, b
          s[name] = decode(c, b, digits)
        else:
          s[name] = _np(held[name][a:a + n])
      out[i] = s
  return out


def _check(opt, before, after, grads, t, lrs, wds, scale=1.0, seed=0, codes=True):
  for i, s in before.items():
    e = after[i]
    if len(s["w"]) == 0:
      continue
    w, m, v, tw, tm, tv = adamw64(s["w"], grads[i] * scale, s["exp_avg"], s["exp_avg_sq"], t, lrs[i], B1, B2, EPS, wds[i])
    assert np.all(np.abs(e["w"] - w) <= tw), ("w", i, np.max(np.abs(e["w"] - w) / tw))
    typ = opt._leaves[i].dtype
    assert np.all(np.abs(e["p"] - w) <= torch.finfo(typ).eps / 2 * np.abs(w) + tw + 2.0 ** -25), ("p", i)
    if s["bits"] == 32:
      assert np.all(np.abs(e["exp_avg"] - m) <= tm), ("m", i, np.max(np.abs(e["exp_avg"] - m) / tm))
      assert np.all(np.abs(e["exp_avg_sq"] - v) <= tv), ("v", i, np.max(np.abs(e["exp_avg_sq"] - v) / tv))
    elif codes:   # bit for bit: separately rounded float32 products and sums, then exact scalings and integer arithmetic
      m32, v32 = moments32((grads[i].astype(np.float32) * np.float32(scale)), s["exp_avg"], s["exp_avg_sq"], B1, B2)
      x = random_bits(seed, t, i, len(m32))
      for name, val, digits, noise in (("exp_avg", m32, 3, (x >> 12) / 2.0 ** 20), ("exp_avg_sq", v32, 2, (x & 0x1FFFFF) / 2.0 ** 21)):
        c, b = encode(val, digits, noise)
        assert np.array_equal(e[name + "_byte"], b), (name, i)
        assert np.array_equal(e[name + "_code"], c), (name, i)
    else:         # either neighbour: less than one spacing, 2^-3 or 2^-2 of the value, or the subnormals'
      for name, val, tol, digits, low in (("exp_avg", m, tm, 3, -9), ("exp_avg_sq", v, tv, 2, -16)):
        unit = np.repeat(2.0 ** (e[name + "_byte"].astype(np.float64) - 127 + low), 128)[:len(val)]
        assert np.all(np.abs(e[name] - val) <= 2.0 ** -digits * (np.abs(val) + tol) + unit + tol), (name, i)


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes,t", [(s, t) for s in SIZES for t in ((1, 1000) if s in ("many", "long") else (1, 2, 1000, 200000))])
def test_step_against_float64(sizes, bits, typ, t):
  ps = _params(SIZES[sizes], TYPES[typ], seed=t)
  opt = _opt(ps, t, lr=1e-3, weight_decay=0.1, state_bits=bits)
  before = _state(opt)
  grads = [_np(p.grad) for p in ps]
  opt.step()
  n = len(ps)
  _check(opt, before, _state(opt), grads, t, [1e-3] * n, [0.1] * n)
  assert opt.steps() == [t] * n
  assert all(np.array_equal(_np(p.grad), g) for p, g in zip(ps, grads))     # gradients stay as they are


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_start_anywhere(bits, typ):
  for offset in (1, 2, 3, 5):
    ps = _params([1, 33, 1000, 4099], TYPES[typ], seed=offset, offset=offset)
    opt = _opt(ps, 5, lr=1e-2, weight_decay=0.0, state_bits=bits)
    before = _state(opt)
    grads = [_np(p.grad) for p in ps]
    guard = [p.detach().untyped_storage().nbytes() for p in ps]
    opt.step()
    _check(opt, before, _state(opt), grads, 5, [1e-2] * 4, [0.0] * 4)
    assert guard == [p.detach().untyped_storage().nbytes() for p in ps]


def test_neighbours_of_a_tensor_stay_as_they_are():
  from oi_vae_amd import optim
  for typ in TYPES.values():
    flat = torch.full((10000,), 2.0, device="cuda", dtype=typ)
    gflat = torch.full((10000,), 3.0, device="cuda", dtype=typ)
    spans = [(1, 4), (9, 9), (21, 129), (200, 4097), (5000, 4095)]
    ps = []
    for a, n in spans:
      p = flat[a:a + n].detach().requires_grad_()
      p.grad = gflat[a:a + n]
      ps.append(p)
    inside = torch.zeros(10000, dtype=torch.bool, device="cuda")
    for a, n in spans:
      inside[a:a + n] = True
    for bits in (32, 8):
      optim.AdamW(ps, lr=0.5, state_bits=bits).step()
      assert (flat[~inside] == 2.0).all() and (flat[inside] != 2.0).all()
      flat.fill_(2.0)
    optim.clip_grad_norm_(ps, 1.0)
    assert (gflat[~inside] == 3.0).all() and (gflat[inside] < 1.0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_orders_of_dimensions(bits):
  """Parameters and gradients in other orders than row-major, and in orders that differ from each other."""
  from oi_vae_amd import optim
  g = torch.Generator(device="cuda").manual_seed(0)
  rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
  p = [rand(24, 40).t().detach().requires_grad_(), rand(3, 5, 7, 11).to(memory_format=torch.channels_last).requires_grad_(),
       rand(40, 24).requires_grad_(), rand(24, 40).t().detach().requires_grad_()]
  grads = [rand(40, 24), rand(3, 5, 7, 11), rand(24, 40).t(), rand(24, 40).t()]
  for q, d in zip(p, grads):
    q.grad = d
  ref = [q.detach().clone().contiguous().requires_grad_() for q in p]
  for q, d in zip(ref, grads):
    q.grad = d.contiguous()
  # moments of zero: the step is lr * sign(g) up to eps in either storage order, and 8-bit codes round m' and v' only after it
  for ps in (p, ref):
    optim.AdamW(ps, lr=0.1, weight_decay=0.1, state_bits=bits).step()
  for a, b in zip(p, ref):
    assert torch.equal(a, b)
  # ... and the moments lie in the parameter's order
  opt = optim.AdamW(p, lr=0.1, state_bits=32)
  opt.step()
  for q, flat in opt._views("exp_avg"):
    want = q.grad * np.float32(1 - B1)
    assert torch.equal(flat.as_strided(q.shape, q.stride()), want)


def test_groups_with_options_of_their_own():
  """More groups than one launch holds, 8- and 32-bit ones mixed, three types."""
  ps = [q for k in range(7) for q in _params([5 + k, 300 * k + 1], list(TYPES.values())[k % 3], seed=k)]
  groups = [{"params": [p], "lr": 1e-3 * (k + 1), "weight_decay": 0.01 * k, "state_bits": 8 if k % 3 else 32} for k, p in enumerate(ps)]
  assert len(groups) > 8
  opt = _opt(groups, 7)
  before = _state(opt)
  grads = [_np(p.grad) for p in ps]
  opt.step()
  _check(opt, before, _state(opt), grads, 7, [1e-3 * (k + 1) for k in range(len(ps))], [0.01 * k for k in range(len(ps))])


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_another_type_than_their_parameter(bits):
  """float32 gradients of 16-bit parameters (accumulated there) and the reverse, in one list, with clipping behind it."""
  from oi_vae_amd import optim
  ps = _params([300, 4097], torch.bfloat16, seed=3) + _params([129, 7], torch.float32, seed=4) + _params([1000], torch.float16, seed=5)
  for p, typ in zip(ps, (torch.float32, torch.float16, torch.bfloat16, torch.float16, torch.float32)):
    g = p.grad.to(typ)
    p.grad = None
    p.grad_dtype = typ
    p.grad = g
  opt = _opt(ps, 6, lr=1e-3, weight_decay=0.1, state_bits=bits)
  before, grads = _state(opt), [_np(p.grad) for p in ps]
  opt.step()
  _check(opt, before, _state(opt), grads, 6, [1e-3] * 5, [0.1] * 5)
  norm = np.sqrt(sum((g * g).sum() for g in grads))
  assert abs(optim.clip_grad_norm_(ps, norm / 3).item() - norm) <= 2 * U * norm
  for p, g in zip(ps, grads):
    eps = torch.finfo(p.grad.dtype).eps / 2
    assert np.all(np.abs(_np(p.grad) - g / 3) <= (eps + 8 * U) * np.abs(g / 3) + 1e-6 / norm * np.abs(g) + 2.0 ** -25)


@pytest.mark.parametrize("on_device", [False, True])
def test_parameters_without_a_gradient_wait(on_device):
  ps = _params([50, 60, 70], torch.float32, seed=1)
  opt = _opt(ps, 1, lr=1e-2, weight_decay=0.1, capturable=on_device)
  opt.step()
  ps[1].grad, keep = None, ps[1].detach().clone()
  before = _state(opt)
  opt.step()
  assert torch.equal(ps[1], keep) and np.array_equal(before[1]["exp_avg"], _state(opt)[1]["exp_avg"])
  assert opt.steps() == [2, 1, 2]
  ps[1].grad = torch.ones(60, device="cuda")
  before = _state(opt)
  opt.step()
  after = _state(opt)
  w, m, v, tw, tm, tv = adamw64(before[1]["w"], np.ones(60), before[1]["exp_avg"], before[1]["exp_avg_sq"], 2, 1e-2, B1, B2, EPS, 0.1)
  assert np.all(np.abs(after[1]["w"] - w) <= tw) and opt.steps() == [3, 2, 3]     # its own second step
  for p in ps:
    p.grad = None
  opt.step()
  assert opt.steps() == [3, 2, 3]


def test_codes_over_the_whole_range():
  """Blocks of zeros, of one value, of magnitudes from 1e-30 to 1e15, of signs and of alternating sizes."""
  rng = np.random.default_rng(5)
  blocks = [np.zeros(128), np.full(128, 1e-3), np.full(128, -3.0), rng.standard_normal(128) * 1e-30, rng.standard_normal(128) * 1e15,
            rng.standard_normal(128) * 10.0 ** rng.uniform(-9, 0, 128), np.where(np.arange(128) % 2, 1e-7, 10.0), np.eye(1, 128, 5)[0],
            -np.eye(1, 128, 77)[0] * 1e-20, 2.0 ** rng.integers(-30, 3, 128), rng.standard_normal(77)]
  g = torch.from_numpy(np.concatenate(blocks).astype(np.float32)).cuda()
  p = torch.zeros_like(g).requires_grad_()
  p.grad = g
  opt = _opt([p], 1, lr=1e-3, weight_decay=0.0, state_bits=8)
  for t in (1, 2, 3):
    before = _state(opt)
    opt.step()
    after = _state(opt)
    _check(opt, before, after, [_np(g)], t, [1e-3], [0.0])
    live = after[0]["exp_avg_sq"] > 0
    assert np.array_equal(live, (before[0]["exp_avg_sq"] > 0) | (np.float32(1e-3) * _np(g).astype(np.float32) ** 2 > 0))


def test_stochastic_rounding_has_no_bias():
  """The same value in 2^17 elements: the mean of its codes' values is the value, to five standard deviations of a mean of
  independent roundings (at most half a spacing each); and the rounding of m says nothing about that of v."""
  n = 1 << 17
  for value in (0.3, 1.1, 7.77):
    g = torch.full((n,), value, device="cuda")
    g[::128] = 100.0           # the block's scale, the same everywhere
    p = torch.zeros(n, device="cuda").requires_grad_()
    p.grad = g
    opt = _opt([p], 1, lr=0.0, weight_decay=0.0, state_bits=8)
    opt.step()
    s = _state(opt)[0]
    pick = np.arange(n) % 128 != 0
    m, v = s["exp_avg"][pick], s["exp_avg_sq"][pick]
    for got, want, digits in ((m, np.float32(1 - B1) * np.float32(value), 3), (v, np.float32(value) ** 2 * np.float32(1 - B2), 2)):
      lo, hi = got.min(), got.max()
      assert lo <= want <= hi and (hi - lo) <= 2.0 ** -digits * want * 1.0001
      assert abs(got.mean() - want) <= 5 * 0.5 * (hi - lo) / np.sqrt(len(got)) + 1e-6 * want
    if m.std() > 0 and v.std() > 0:
      assert abs(np.corrcoef(m, v)[0, 1]) <= 5 / np.sqrt(len(m))


def test_what_is_not_finite_stays_visible():
  """Without clipping a NaN or an infinity reaches the parameter and its block of 8-bit moments, and no other block."""
  minus_nan = torch.tensor([-4194304], dtype=torch.int32, device="cuda").view(torch.float32)[0]     # 0xFFC00000
  for bad in (float("nan"), minus_nan, float("inf"), -float("inf")):
    for bits in (32, 8):
      p = _params([512], torch.float32, seed=2)[0]
      p.grad[200] = bad
      opt = _opt([p], 3, lr=1e-3, state_bits=bits)
      opt.step()
      s = _state(opt)[0]
      hit = np.zeros(512, bool)
      hit[200] = True
      assert np.array_equal(np.isnan(s["w"]), hit)
      if bits == 8:
        hit[128:256] = True
        assert np.array_equal(np.isnan(s["exp_avg"]), hit) and np.array_equal(np.isnan(s["exp_avg_sq"]), hit)
      else:
        assert not np.isfinite(s["exp_avg"][200]) and not np.isfinite(s["exp_avg_sq"][200])
        assert np.isfinite(np.delete(s["exp_avg"], 200)).all()


# ---- norm and clipping -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("sizes", list(SIZES))
def test_norm_and_clipping(sizes, typ, offset):
  from oi_vae_amd import optim
  ps = _params(SIZES[sizes], TYPES[typ], seed=11, offset=offset)
  g = [_np(p.grad) for p in ps]
  norm = np.sqrt(sum((x * x).sum() for x in g))
  got = optim.grad_norm(ps)
  assert got.dim() == 0 and got.dtype == torch.float32
  assert abs(got.item() - norm) <= 2 * U * norm            # fp64 sums, one rounding to fp32
  assert all(torch.equal(got, optim.grad_norm(ps)) for _ in range(3))
  keep = [p.grad.clone() for p in ps]
  assert torch.equal(optim.clip_grad_norm_(ps, 2 * norm + 1), got)
  assert all(torch.equal(p.grad, k) for p, k in zip(ps, keep))      # a norm below the limit changes nothing
  limit = 0.25 * norm
  assert torch.equal(optim.clip_grad_norm_(iter(ps), limit), got)
  coef = limit / (norm + 1e-6)
  eps = torch.finfo(TYPES[typ]).eps / 2
  for p, x in zip(ps, g):       # the coefficient's roundings (norm, sum, quotient, limit: 5 U), the product's and the type's
    low = 2.0 ** -25 if typ == "f16" else 0.0
    assert np.all(np.abs(_np(p.grad) - coef * x) <= (eps + 6 * U) * np.abs(coef * x) + low + 2.0 ** -149)


def test_norm_of_extreme_and_odd_gradients():
  from oi_vae_amd import optim
  p = torch.zeros(1000, device="cuda").requires_grad_()
  p.grad = torch.full((1000,), 1e25, device="cuda")        # squares leave float32
  assert abs(optim.grad_norm(p).item() / (1e25 * np.sqrt(1000)) - 1) <= 1e-6
  p.grad.fill_(1e-25)
  assert abs(optim.grad_norm([p]).item() / (1e-25 * np.sqrt(1000)) - 1) <= 1e-6
  p.grad.fill_(0.0)
  assert optim.clip_grad_norm_([p], 1.0).item() == 0.0 and (p.grad == 0).all()
  assert optim.grad_norm([torch.zeros(3, device="cuda", requires_grad=True)]).item() == 0.0      # no gradient at all
  assert optim.clip_grad_norm_([], 1.0).item() == 0.0
  # transposed and strided gradients (the latter are not one piece of memory), beside one that waits without any
  q = torch.zeros(30, 20, device="cuda").requires_grad_()
  r = torch.zeros(50, device="cuda").requires_grad_()
  base = torch.randn(20, 30, device="cuda")
  wide = torch.randn(100, device="cuda")
  q.grad, r.grad = base.t(), wide[::2]
  want = float(torch.sqrt((base.double() ** 2).sum() + (wide[::2].double() ** 2).sum()))
  odd = wide[1::2].clone()
  qc, rc = base.clone(), wide[::2].clone()
  got = optim.clip_grad_norm_([q, p, r], 1.0)
  assert abs(got.item() - want) <= 2 * U * want
  for x, c in ((base, qc), (wide[::2], rc)):
    assert torch.allclose(x.double(), c.double() / (want + 1e-6), rtol=8 * U, atol=0)
  assert torch.equal(wide[1::2], odd)
  # NaN and infinity, as torch.nn.utils.clip_grad_norm_ leaves them
  for bad in (float("nan"), float("inf")):
    p.grad = torch.ones(1000, device="cuda")
    p.grad[3] = bad
    s = torch.zeros(1000, device="cuda").requires_grad_()
    s.grad = p.grad.clone()
    a, b = optim.clip_grad_norm_([p], 1.0), torch.nn.utils.clip_grad_norm_([s], 1.0)
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
    assert torch.equal(torch.isnan(p.grad), torch.isnan(s.grad)) and torch.equal(torch.nan_to_num(p.grad), torch.nan_to_num(s.grad))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("sizes", ["blocks", "many", "long", "several thousand blocks"])
def test_clipped_step(sizes, typ, bits):
  sizes = SIZES.get(sizes, [9000000, 5])     # one launch, two, more partial sums than one launch concludes, more than its blocks
  ps = _params(sizes, TYPES[typ], seed=4)
  opt = _opt(ps, 9, lr=1e-3, weight_decay=0.1, state_bits=bits, max_grad_norm=0.05)
  before = _state(opt)
  grads = [_np(p.grad) for p in ps]
  norm = 0.5 * np.sqrt(sum((x * x).sum() for x in grads))
  opt.step(grad_scale=0.5)
  assert abs(opt.grad_norm.item() - norm) <= 2 * U * norm and norm > 0.05
  _check(opt, before, _state(opt), grads, 9, [1e-3] * len(ps), [0.1] * len(ps), scale=0.5 * 0.05 / (norm + 1e-6), codes=False)
  assert all(np.array_equal(_np(p.grad), g) for p, g in zip(ps, grads))
  assert opt.steps() == [9] * len(ps) and opt.skipped.item() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_whose_norm_is_not_finite_is_left_out(bits):
  for bad in (float("nan"), float("inf")):
    ps = _params([100, 5000], torch.bfloat16, seed=6)
    opt = _opt(ps, 4, lr=1e-3, state_bits=bits, max_grad_norm=1.0)
    keep = {k: {n: t.view(torch.uint8).clone() for n, t in held.items()} for k, held in opt.buffers.items()}
    was = [p.detach().clone() for p in ps]
    ps[1].grad[17] = bad
    opt.step()
    assert not np.isfinite(opt.grad_norm.item()) and opt.skipped.item() == 1 and opt.steps() == [3, 3]
    assert all(torch.equal(p, w) for p, w in zip(ps, was))
    assert all(torch.equal(opt.buffers[k][n].view(torch.uint8), t) for k, held in keep.items() for n, t in held.items())
    ps[1].grad[17] = 0.0
    opt.step()
    assert opt.skipped.item() == 1 and opt.steps() == [4, 4] and not torch.equal(ps[0], was[0])


def test_tiny_and_zero_eps():
  """eps below what the hardware's root can hold, and none: gradients down to float32's subnormal squares."""
  from oi_vae_amd import optim
  g = torch.tensor(10.0 ** np.linspace(-21, 3, 1000), dtype=torch.float32, device="cuda")
  for eps in (0.0, 1e-18, 1e-12):
    for bits in (32, 8):
      p = torch.zeros(1000, device="cuda").requires_grad_()
      p.grad = g.clone()
      optim.AdamW([p], lr=1e-3, eps=eps, weight_decay=0.0, state_bits=bits).step()
      x = _np(g)
      v = (np.float32(1 - B2) * g.cpu().numpy() ** 2).astype(np.float64)      # as far as float32 holds it
      live = v > 2.0 ** -126
      want = -1e-3 * x / (np.sqrt(x * x) + eps)
      assert np.all(np.abs(_np(p) - want)[live] <= 64 * U * np.abs(want)[live]), (eps, bits)
  # nothing at all: 0 / 0 without eps, as the formula says; zero with it
  for eps, same in ((0.0, False), (1e-8, True)):
    for bits in (32, 8):
      p = torch.ones(5, device="cuda").requires_grad_()
      p.grad = torch.zeros(5, device="cuda")
      optim.AdamW([p], lr=1e-3, eps=eps, weight_decay=0.0, state_bits=bits).step()
      assert bool((p == 1).all()) == same and bool(torch.isnan(p).all()) != same


@pytest.mark.parametrize("b1,b2", [(0.0, 0.999), (0.9, 0.0), (0.0, 0.0), (0.5, 0.9999999)])
def test_other_betas(b1, b2):
  from oi_vae_amd import optim
  for kw in (dict(), dict(capturable=True)):
    for bits in (32, 8):
      p = _params([300], torch.float32, seed=3)[0]
      w, g = _np(p), _np(p.grad)
      optim.AdamW([p], lr=1e-2, betas=(b1, b2), eps=EPS, weight_decay=0.1, state_bits=bits, **kw).step()
      want = w * (1 - 1e-3) - 1e-2 * g / (np.abs(g) + EPS)        # the first step, whatever the betas
      assert np.all(np.abs(_np(p) - want) <= 4 * U * np.abs(w) + 64 * U * 1e-2 + 2 * U * np.abs(want)), (kw, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_2_to_the_32_elements(bits):
  """Offsets past 32 bits in the tensor, its moments and its random bits (bfloat16; about 60 GB with moments in 32 bits)."""
  from oi_vae_amd import optim
  n = (1 << 32) + 5003
  if torch.cuda.mem_get_info()[0] < 80 << 30:
    pytest.skip("needs 80 GB")
  p = torch.zeros(n, dtype=torch.bfloat16, device="cuda").requires_grad_()
  p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
  opt = optim.AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits, max_grad_norm=1e9)
  spots = [(0, 4096), ((1 << 31) - 2048, 4096), ((1 << 32) - 2048, 4096), (n - 1000, 1000)]
  g = torch.Generator(device="cuda").manual_seed(0)
  for a, k in spots:
    p.grad[a:a + k] = torch.randn(k, generator=g, device="cuda").bfloat16()
  norm = np.sqrt(sum((_np(p.grad[a:a + k]) ** 2).sum() for a, k in spots))
  opt.step()
  assert abs(opt.grad_norm.item() - norm) <= 2 * U * norm
  held = opt.buffers[bits]
  for a, k in spots:
    x = _np(p.grad[a:a + k])
    want = -1e-2 * x / (np.abs(x) + EPS)
    assert np.all(np.abs(_np(held["master"][a:a + k]) - want) <= 64 * U * 1e-2)
    lo = a // 128 * 128
    if bits == 8:
      full = np.zeros(a + k - lo)
      full[a - lo:] = x
      m32, v32 = moments32(full, 0 * full, 0 * full, B1, B2)
      noise = random_bits(0, 1, 0, len(full), first=lo)
      for name, val, digits, r in (("exp_avg", m32, 3, (noise >> 12) / 2.0 ** 20), ("exp_avg_sq", v32, 2, (noise & 0x1FFFFF) / 2.0 ** 21)):
        c, b = encode(val, digits, r)
        assert np.array_equal(held[name].view(torch.uint8)[lo:a + k].cpu().numpy(), c), (name, a)
    else:
      m = 0.1 * x
      assert np.all(np.abs(_np(held["exp_avg"][a:a + k]) - m) <= 4 * U * np.abs(m))
  assert (p[5000:1 << 20] == 0).all()
  got = optim.clip_grad_norm_(p, norm / 2)
  assert abs(got.item() - norm) <= 2 * U * norm
  a, k = spots[-1]
  assert abs(_np(p.grad[a:a + k])).max() > 0 and abs(optim.grad_norm(p).item() - norm / 2) <= 2.0 ** -8 * norm
  del p, opt, held
  torch.cuda.empty_cache()


def test_autograd_hears_of_the_step():
  """A graph that saved a weight refuses to run backward after the step, as behind torch.optim."""
  from oi_vae_amd import optim
  for shape in ((4, 4), (4, 8)):
    w = torch.randn(8, 8, device="cuda")[:, :shape[1]].t().contiguous().t().requires_grad_()
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    loss = ((x @ w) ** 2).sum()
    loss.backward(retain_graph=True)
    optim.AdamW([w], lr=0.1).step()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
      loss.backward()


# ---- streams, graphs, resuming ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.05])
def test_a_captured_step_advances(bits, clip):
  """Four replays, with eager work and synchronisation between, equal four eager steps bit for bit; lr from the device."""
  from oi_vae_amd import optim

  def make():
    ps = _params([300, 1, 5000] + [40] * 100, torch.bfloat16, seed=8)
    lr = torch.full((1,), 1e-2, device="cuda")
    opt = optim.AdamW(ps, lr=lr, state_bits=bits, max_grad_norm=clip, capturable=True)
    opt.buffers
    return ps, lr, opt
  ps, lr, opt = make()
  es, elr, eopt = make()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    opt.step()
  assert opt.steps() == [0] * len(ps)
  g = torch.Generator(device="cuda").manual_seed(1)
  for k in range(4):
    for p, e in zip(ps, es):
      x = 1e-2 * torch.randn(p.shape, generator=g, device="cuda")
      p.grad.copy_(x)
      e.grad.copy_(x)
    lr.fill_(1e-2 / (k + 1))
    elr.fill_(1e-2 / (k + 1))
    graph.replay()
    eopt.step()
    torch.cuda.synchronize()
    junk = torch.randn(1000, 1000, device="cuda").sum()      # the program's own work between the replays
    assert torch.isfinite(junk).item()
    assert opt.steps() == [k + 1] * len(ps) == eopt.steps()
    assert all(torch.equal(p, e) for p, e in zip(ps, es))
    for n in opt.buffers[bits]:
      assert torch.equal(opt.buffers[bits][n].view(torch.uint8), eopt.buffers[bits][n].view(torch.uint8)), n


def test_what_capture_cannot_hold_is_refused():
  from oi_vae_amd import optim
  ps = _params([300], torch.float32, seed=8)
  plain, fresh = optim.AdamW(ps), optim.AdamW(ps, capturable=True)
  plain.buffers
  for opt, what in ((plain, "capturable"), (fresh, "before capturing")):
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match=what):
      with torch.cuda.graph(graph):
        opt.step()
    torch.cuda.synchronize()


def test_clipping_captured_and_replayed():
  from oi_vae_amd import optim
  ps = _params([300, 5000], torch.float32, seed=9)
  src = [p.grad.clone() for p in ps]
  optim.clip_grad_norm_(ps, 1.0)      # the library is loaded before the capture
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    norm = optim.clip_grad_norm_(ps, 0.01)
  for k in range(1, 4):
    for p, s in zip(ps, src):
      p.grad.copy_(s * k)
    graph.replay()
    torch.cuda.synchronize()
    want = [(s * k).clone() for s in src]
    es = [torch.zeros_like(w).requires_grad_() for w in want]
    for e, w in zip(es, want):
      e.grad = w
    assert torch.equal(optim.clip_grad_norm_(es, 0.01), norm)
    assert all(torch.equal(p.grad, e.grad) for p, e in zip(ps, es))


def test_another_stream_and_resuming():
  from oi_vae_amd import optim
  for bits in (32, 8):
    runs = []
    for how in ("through", "resumed", "side stream"):
      ps = _params([300, 129, 5000], torch.float16, seed=10)
      groups = [{"params": ps[:1], "weight_decay": 0.0}, {"params": ps[1:]}]
      opt = optim.AdamW(groups, lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=5)
      g = torch.Generator(device="cuda").manual_seed(3)
      side = torch.cuda.Stream()
      for k in range(4):
        for p in ps:
          p.grad = (1e-2 * torch.randn(p.shape, generator=g, device="cuda")).half()
        if how == "resumed" and k == 2:
          import io
          file = io.BytesIO()
          torch.save(opt.state_dict(), file)
          file.seek(0)
          state = torch.load(file, weights_only=True)
          opt = optim.AdamW(groups, lr=0.5, state_bits=bits, max_grad_norm=1.0)
          opt.load_state_dict(state)
          assert opt.steps() == [2, 2, 2] and opt.seed == 5
        if how == "side stream":
          side.wait_stream(torch.cuda.current_stream())
          with torch.cuda.stream(side):
            opt.step()
          torch.cuda.current_stream().wait_stream(side)
        else:
          opt.step()
      torch.cuda.synchronize()
      runs.append(([p.detach().clone() for p in ps], {n: t.view(torch.uint8).clone() for n, t in opt.buffers[bits].items()}))
    for other in runs[1:]:
      assert all(torch.equal(a, b) for a, b in zip(runs[0][0], other[0]))
      assert all(torch.equal(runs[0][1][n], other[1][n]) for n in runs[0][1])


def test_gradients_that_are_not_plain_memory():
  """Expanded and negated-view gradients are copied into the parameter's order; clipping refuses to write an expanded one."""
  from oi_vae_amd import optim
  z = torch.randn(300, device="cuda", dtype=torch.complex64, generator=torch.Generator(device="cuda").manual_seed(4))
  views = [torch.full((1,), 0.5, device="cuda").expand(300), torch.conj(z).imag]
  assert views[1].is_neg()
  for g in views:
    for clip in (None, 1.0):
      p, q = (torch.ones(300, device="cuda").requires_grad_() for _ in range(2))
      p.grad, q.grad = g, g.clone().resolve_neg().contiguous()
      op, oq = optim.AdamW([p], lr=0.1, max_grad_norm=clip), optim.AdamW([q], lr=0.1, max_grad_norm=clip)
      op.step()
      oq.step()
      assert torch.equal(p, q) and torch.equal(op.buffers[32]["exp_avg"], oq.buffers[32]["exp_avg"])
    assert torch.equal(optim.grad_norm(p), optim.grad_norm(q))
  optim.clip_grad_norm_(p, 0.1)
  optim.clip_grad_norm_(q, 0.1)
  assert torch.equal(p.grad.resolve_neg(), q.grad)
  p.grad = views[0]
  with pytest.raises(RuntimeError):
    optim.clip_grad_norm_(p, 0.1)


def test_master_weights_follow_the_parameter_on_request():
  from oi_vae_amd import optim
  p = _params([200], torch.bfloat16, seed=1)[0]
  opt = optim.AdamW([p], lr=1e-4, weight_decay=0.0)
  assert torch.equal(opt.buffers[32]["master"][:200], p.detach().float())
  for _ in range(5):          # steps below half a unit of bfloat16 add up in the master
    opt.step()
  assert not torch.equal(opt.buffers[32]["master"][:200], p.detach().float())
  assert torch.equal(opt.buffers[32]["master"][:200].bfloat16(), p.detach())
  with torch.no_grad():
    p.fill_(3.0)
  opt.sync_master()
  opt.step()
  assert (opt.buffers[32]["master"][:200] - 3.0).abs().max() <= 1.1e-4 and (p == 3.0).all()


def test_options_changed_between_steps():
  from oi_vae_amd import optim
  ps = _params([300, 40], torch.float32, seed=2)
  opt = optim.AdamW(ps, lr=1e-2, weight_decay=0.0)
  opt.step()
  was = [p.detach().clone() for p in ps]
  opt.param_groups[0]["lr"] = 0.0
  opt.step()
  assert all(torch.equal(p, w) for p, w in zip(ps, was)) and opt.steps() == [2, 2]
  opt.param_groups[0]["lr"] = torch.zeros(1, device="cuda", dtype=torch.float64)
  with pytest.raises(ValueError, match="lr tensor"):
    opt.step()
  opt.param_groups[0]["lr"] = 0.0
  opt.max_grad_norm = 1.0
  with pytest.raises(RuntimeError, match="constructor"):
    opt.step()
  assert opt.steps() == [2, 2]
  clip = optim.AdamW(ps, lr=1e-2, max_grad_norm=1.0)
  clip.max_grad_norm = None      # a later change of mind is fine: the norm is no longer taken
  clip.step()
  assert clip.steps() == [1, 1]


def test_refusals_at_the_first_step():
  from oi_vae_amd import _lib, optim
  cpu = torch.zeros(4).requires_grad_()
  cpu.grad = torch.zeros(4)
  with pytest.raises(_lib.OivaeError):
    optim.AdamW([cpu]).step()
  with pytest.raises(_lib.OivaeError):
    optim.clip_grad_norm_([cpu], 1.0)
  p = torch.zeros(4, device="cuda", dtype=torch.float64).requires_grad_()
  p.grad = torch.zeros_like(p)
  with pytest.raises(ValueError, match="float32"):
    optim.AdamW([p]).step()
  holes = torch.zeros(8, device="cuda")[::2].requires_grad_()
  holes.grad = torch.zeros(4, device="cuda")
  with pytest.raises(ValueError, match="fill its memory"):
    optim.AdamW([holes]).step()
  q = torch.zeros(8, device="cuda").requires_grad_()
  q.grad = torch.zeros(8, device="cuda")
  opt = optim.AdamW([q])
  opt.step()
  q.data = torch.zeros(16, device="cuda")
  q.grad = torch.zeros(16, device="cuda")
  with pytest.raises(ValueError, match="changed its size"):
    opt.step()
  with pytest.raises(ValueError, match="more than once"):
    optim.clip_grad_norm_([q, q], 1.0)
  flat = torch.zeros(100, device="cuda")
  with pytest.raises(ValueError, match="share memory"):
    optim.AdamW([flat[:50].detach().requires_grad_(), flat[49:].detach().requires_grad_()]).buffers
  optim.AdamW([flat[:50].detach().requires_grad_(), flat[50:].detach().requires_grad_()]).buffers
  with pytest.raises(RuntimeError, match="max_grad_norm"):
    opt.grad_norm
  make = lambda sizes, **kw: optim.AdamW([torch.zeros(n, device="cuda").requires_grad_() for n in sizes], **kw)
  state = make([9, 200]).state_dict()
  for other, what in ((make([9, 200], state_bits=8), "bits"), (make([9]), "exp_avg"), (make([8, 201]), "other parameters"),
                      (make([200, 9]), "other parameters")):
    keep = {b: {k: t.view(torch.uint8).clone() for k, t in held.items()} for b, held in other.buffers.items()}
    with pytest.raises(ValueError, match=what):
      other.load_state_dict(state)
    assert all(torch.equal(t.view(torch.uint8), keep[b][k]) for b, held in other.buffers.items() for k, t in held.items())
  make([9, 200]).load_state_dict(state)


# ---- together, and in the framework's own training step --------------------------------------------------------------------
def test_autoencoder_step_with_clipping_and_the_proximal_operator():
  """The autoencoder variant's loop -- autograd, clipped AdamW, proximal step -- against float64 AdamW on the same gradients."""
  import oi_vae_amd as oi
  from oi_vae_amd import optim
  for bits in (32, 8):
    torch.manual_seed(0)
    enc = torch.nn.Linear(64, 8, bias=False).cuda()
    dec = oi.FirstLayerSparseDecoder([torch.nn.Sequential(torch.nn.Linear(1, 8, bias=False), torch.nn.Tanh(), torch.nn.Linear(8, 8, bias=False))
                                      for _ in range(8)], [1] * 8, 8)
    dec.cuda()
    params = list(enc.parameters()) + list(dec.parameters())
    opt = optim.AdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=0.1, eps=EPS, betas=(B1, B2))
    X = torch.rand(32, 64, device="cuda")
    for t in range(1, 5):
      opt.zero_grad()
      ((dec(enc(X)) - X) ** 2).sum().backward()
      before, grads = _state(opt), [_np(p.grad) for p in params]
      norm = np.sqrt(sum((x * x).sum() for x in grads))
      opt.step()
      n = len(params)
      _check(opt, before, _state(opt), grads, t, [1e-2] * n, [1e-2] * n, scale=min(1.0, 0.1 / (norm + 1e-6)), codes=False)
      dec.proximal_step(1e-2 * 0.5)
    assert all(torch.isfinite(p).all() for p in params) and (dec.connectivity() == 0).any()


def _vae(optimizers):
  import oi_vae_amd as oi
  torch.manual_seed(0)
  inference_net = oi.NormalNet(mu_net=torch.nn.Sequential(torch.nn.Linear(24, 8)),
                               sigma_net=torch.nn.Sequential(torch.nn.Linear(24, 8), oi.Lambda(torch.exp), oi.Lambda(lambda x: x * 0.1 + 1e-3)))

  def gen():
    ls = torch.log(1e-2 * torch.ones(8)).requires_grad_(True)
    return oi.NormalNet(mu_net=torch.nn.Linear(2, 8),
                        sigma_net=oi.Lambda(lambda x, ls: torch.exp(ls.expand(x.size(0), -1)) + 1e-3, extra_args=(ls,)))
  model = oi.BayesianGroupLassoGenerator([gen() for _ in range(3)], group_input_dim=2, dim_z=8)
  groups = [{"params": inference_net.parameters()}, {"params": model.group_generators_parameters()},
            {"params": [g.sigma_net.extra_args[0] for g in model.group_generators]}]
  opts = optimizers(groups, [model.Ws])
  vae = oi.OIVAE(inference_net, model, oi.Normal(torch.zeros(1, 8), torch.ones(1, 8)), oi.NormalPriorTheta(1.0), 1.0, opts)
  return vae, opts


@pytest.mark.parametrize("bits,clip", [(32, None), (32, 10.0), (8, None), (8, 10.0)])
@pytest.mark.parametrize("B", [16, 20000])     # the one-launch step, and the entry points
def test_oivae_trains_with_adamw(bits, clip, B):
  """OIVAE.step with AdamW on the engine's flat buffers: every update of four steps against float64 on the step's gradients."""
  from oi_vae_amd import optim
  vae, (opt, _) = _vae(lambda groups, ws: [optim.AdamW(groups, lr=1e-3, weight_decay=0.05, state_bits=bits, max_grad_norm=clip),
                                            optim.SGD(ws, lr=1e-4)])
  eng = vae.engine
  assert eng.small_step_applies(B, 1) == (B == 16)
  X = torch.rand(B, 24, generator=torch.Generator().manual_seed(1)).cuda()
  for t in range(1, 5):
    opt.buffers
    before = _state(opt)
    ws = eng.p["Ws"].clone()
    info = vae.step(X, 1e-3, 1)
    assert torch.isfinite(info["loss"]).item() and not torch.equal(ws, eng.p["Ws"])
    g = _np(eng.flat_grads[:eng.adam_numel])
    norm = np.sqrt((g * g).sum())
    scale = min(1.0, clip / (norm + 1e-6)) if clip else 1.0
    _check(opt, before, _state(opt), [g], t, [1e-3], [0.05], scale=scale, codes=clip is None)
    if clip:
      assert abs(opt.grad_norm.item() - norm) <= 2 * U * norm


def test_oivae_steps_adamw_behind_the_gradient_reduction(monkeypatch):
  """The data-parallel order of OIVAE.step: AdamW runs once, after both buckets are reduced (here by a stand-in that doubles
  the gradients when they are waited for)."""
  from oi_vae_amd import optim, parallel

  class Sync:
    def __init__(self, holder, group=None):
      self.flat = holder.flat_grads

    def decoder_grads_ready(self):
      pass

    encoder_grads_ready = decoder_grads_ready

    def wait(self):
      self.flat.mul_(2.0)
  monkeypatch.setattr(parallel, "is_active", lambda group=None: True)
  monkeypatch.setattr(parallel, "BucketedGradSync", Sync)
  monkeypatch.setattr(parallel, "reduce_scalars_", lambda scalars, group=None: scalars)
  vae, (opt, _) = _vae(lambda groups, ws: [optim.AdamW(groups, lr=1e-3, weight_decay=0.05, max_grad_norm=1.0), optim.SGD(ws, lr=1e-4)])
  X = torch.rand(16, 24, generator=torch.Generator().manual_seed(1)).cuda()
  for t in (1, 2):
    before = _state(opt)
    vae.step(X, 1e-3, 1)
    g = _np(vae.engine.flat_grads[:vae.engine.adam_numel])
    norm = np.sqrt((g * g).sum())
    _check(opt, before, _state(opt), [g], t, [1e-3], [0.05], scale=min(1.0, 1.0 / (norm + 1e-6)))
    assert abs(opt.grad_norm.item() - norm) <= 2 * U * norm


def test_engine_adamw_is_one_option_set():
  from oi_vae_amd import optim
  with pytest.raises(ValueError, match="weight_decay"):
    _vae(lambda groups, ws: [optim.AdamW([dict(g, weight_decay=0.1 * k) for k, g in enumerate(groups)]), optim.SGD(ws, lr=1e-4)])


def test_steps_queued_behind_a_failed_decoder_change_nothing():
  """As the other update kernels (test_gpu_wait_timeout.py): behind a decoder whose bounded wait ran out neither weights nor
  moments nor step counters move, in 32 and in 8 bits, with clipping and without; afterwards the same calls work."""
  import os
  from oi_vae_amd import _lib, optim
  from tests.test_gpu_scale import _engine
  L = _lib.bind(os.path.join(os.path.dirname(_lib.LIB_PATH), "liboivae_hip_waittest.so"))
  assert L.oivae_init(0) == 0
  G, K, B = 4, 64, 4096
  eng = _engine(G, 64, K, 64, 64, seed=5)
  g = torch.Generator(device="cuda").manual_seed(2)
  X = torch.rand(B, G * 64, generator=g, device="cuda")
  z = torch.randn(B, K, generator=g, device="cuda")
  dz = torch.empty(K, B, device="cuda")
  eng._ws_key = None
  ws = eng._workspace(B, 1)
  st = eng._stream()
  dec = (ctypes.byref(eng._shape), ctypes.byref(eng._pt), ctypes.byref(eng._gt), X.data_ptr(), B, 1, z.data_ptr(),
         1e-3, dz.data_ptr(), ws.data_ptr(), eng._ws_bytes, st)
  for bits in (32, 8):
    for clip in (None, 1.0):
      p = _params([5000], torch.float32, seed=1)[0]
      opt = optim.AdamW([p], lr=1e-2, state_bits=bits, max_grad_norm=clip)
      opt.buffers
      opt._lib = L                     # its calls go to the test library
      torch.cuda.synchronize()
      before, zero = p.detach().clone(), [t.view(torch.uint8).clone() for t in opt.buffers[bits].values()]
      assert L.oivae_decoder_fwd_bwd_f32(*dec) == 0
      heard = False
      try:
        opt.step()                     # queued behind the failing launch, or told of it if the host was not ahead
      except _lib.OivaeError:
        heard = True
      assert L.oivae_check_errors(st) == 3 or heard
      torch.cuda.synchronize()
      assert torch.equal(p, before)
      assert all(torch.equal(t.view(torch.uint8), q) for t, q in zip(opt.buffers[bits].values(), zero))
      if clip:
        assert opt.steps() == [0]
      assert L.oivae_check_errors(st) == 0
      opt.step()
      torch.cuda.synchronize()
      assert not torch.equal(p, before)


def _script(name):
  import importlib.util
  import os
  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scripts", name + ".py")
  spec = importlib.util.spec_from_file_location(name, path)
  mod = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(mod)
  return mod


@pytest.mark.parametrize("bits", ["32", "8"])
def test_drivers_run_with_adamw(tmp_path, bits):
  common = ["--weight-decay", "0.01", "--state-bits", bits, "--max-grad-norm", "10"]
  res = _script("data_vs_test_loss_autoencoder").main(["--epochs", "30", "--train-sizes", "8", "--lams", "0.1", "--test-samples", "64",
                                                       "--optimizer", "adamw", "--out", str(tmp_path / "a.json")] + common)
  assert len(res) == 1 and np.all(np.isfinite(res[0]["test_loss"])) and len(set(res[0]["train_loss"])) == 30
  exp = _script("meg_oi_vae").main(["--labels", "12", "--frames", "10000", "--max-iterations", "8", "--log-every", "4",
                                    "--out", str(tmp_path / "meg")] + common)
  opt = exp.optimizer
  assert opt.steps() == [8] and opt.skipped.item() == 0 and np.isfinite(opt.grad_norm.item())
  assert list(opt.buffers) == [int(bits)] and torch.isfinite(exp.vae.engine.flat_params).all()


def test_pointers_are_read_at_every_call():
  """Gradients and parameters that move between steps (the same optimizer, other memory)."""
  from oi_vae_amd import optim
  a = _params([1000, 33], torch.float32, seed=12)
  b = _params([1000, 33], torch.float32, seed=12)
  oa, ob = optim.AdamW(a, lr=1e-2), optim.AdamW(b, lr=1e-2)
  keep = []
  for k in range(3):
    for p, q in zip(a, b):
      g = torch.randn(p.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k))
      p.grad = g
      q.grad.copy_(g)
      keep.append(p.data)
      p.data = p.data.clone()
    oa.step()
    ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
