"""The optimizer operators over lists of tensors, as a training program calls them: an AdamW step with moments in 32 bits,
an AdamW step with moments in 8 bits, and the global gradient norm with clipping -- each alone, and the norm together with
the step it bounds.  Cases, their inputs, their plain forms in elementary torch operations, and their values in 64 bits.

A program's tensors lie in one flat buffer, each on a region padded with zeros to a multiple of 128 elements (one block of
the 8-bit moments); zeros stay zeros under every operator here, so a plain form works on the whole buffer as [blocks, 128]
with one learning rate and one decay per block."""
import math

import torch

own = False

BLOCK = 128
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

# The tied-bars autoencoder of scripts/data_vs_test_loss_autoencoder.py: encoder 256 -> 8, sixteen latent-to-group maps
# 8 -> 1, sixteen generators 1 -> 16 -> 16 -> 16.
AUTOENCODER = "2048,16*8,16*16,32*256"
# The scale-up model of bench.py (1024 groups of 64 outputs, K = H = M = 64), one tensor per parameter array, matrices first.
SCALE_UP = "4*4194304,2*64,3*65536"
# A model like the MEG script's, unpacked: two encoder heads of 10 x 6601 and, for 44 labels, weights, biases and log sigmas
# of the label's odd number of vertices.
MEG = "2*66010,2*10," + ",".join("3*%d" % (40 + (37 * k * k + 11 * k) % 220) for k in range(44))


def listed():
  """12 cases.  `sizes`: elements of each tensor, "k*n" for k of n; `decay`: the weight decay of the first two thirds of the
  tensors (matrices; the rest, biases and scales, have none); `max_norm`: 0 for a step without clipping; `step`: the step
  being taken when the case begins."""
  adamw, clip = dict(lr=1e-4, beta2=0.999, decay=0.01, step=1000), dict(lr=0.0, beta2=0.0, decay=0.0, step=0, bits=0)
  llm = dict(lr=1e-4, beta2=0.95, decay=0.1, step=2000)
  return [
    # 65 tiny tensors, an epoch of the autoencoder driver: all latency
    dict(name="adamw32_autoencoder", op="adamw", bits=32, type="float32", sizes=AUTOENCODER, max_norm=0.0, **{**adamw, "lr": 1e-3, "step": 10}),
    # 136 tensors of odd sizes, 130 of them tiny, with clipping
    dict(name="adamw32_meg_clipped", op="adamw", bits=32, type="float32", sizes=MEG, max_norm=1.0, **{**adamw, "lr": 1e-3}),
    # the scale-up model's parameters
    dict(name="adamw32_scale_up", op="adamw", bits=32, type="float32", sizes=SCALE_UP, max_norm=0.0, **{**adamw, "lr": 1e-3}),
    # half-precision parameters with 32-bit master weights, a large model's matrices and norms
    dict(name="adamw32_bf16_large", op="adamw", bits=32, type="bfloat16", sizes="14*16777216,32*1048576,64*2048", max_norm=0.0, **llm),
    # a first step (moments of zero, the largest bias correction) of a handful of odd tensors
    dict(name="adamw8_first_step", op="adamw", bits=8, type="float32", sizes="3*20011,4*4097,5*1023,1,7", max_norm=0.0, **{**adamw, "step": 1}),
    # odd sizes of an ordinary model, 8-bit moments under 32-bit parameters
    dict(name="adamw8_odd", op="adamw", bits=8, type="float32", sizes="5*1500007,6*250013,24*4099,24*1025", max_norm=0.0, **adamw),
    # the large model again with moments of 8 bits
    dict(name="adamw8_bf16_large", op="adamw", bits=8, type="bfloat16", sizes="14*16777216,32*1048576,64*2048", max_norm=0.0, **llm),
    # float16 parameters and gradients, norm and step together
    dict(name="adamw8_fp16_clipped", op="adamw", bits=8, type="float16", sizes="40*1638400,80*1280,333", max_norm=1.0, **llm),
    # clipping alone: the autoencoder, odd half-precision tensors, large 32-bit ones
    dict(name="clip_autoencoder", op="clip", type="float32", sizes=AUTOENCODER, max_norm=0.5, **clip),
    dict(name="clip_fp16_odd", op="clip", type="float16", sizes="9*524309,30*33333,60*771", max_norm=1.0, **clip),
    dict(name="clip_bf16", op="clip", type="bfloat16", sizes="64*1048576,64*1024", max_norm=1.0, **clip),
    dict(name="clip_fp32_large", op="clip", type="float32", sizes="14*16777216,32*1048576,64*2048", max_norm=1.0, **clip),
  ]


def draw(rng):
  """Lists of 1 to 160 tensors, a thousand to a hundred million elements in all, any parity."""
  total = int(10 ** rng.uniform(3, 8))
  count = int(round(10 ** rng.uniform(0, 2.2)))
  weights = [10 ** rng.uniform(-1.5, 1.0) for _ in range(count)]
  left = [max(1, int(total * w / sum(weights))) for w in weights]
  sizes = ",".join(str(n if rng.random() < 0.5 else max(1, n & ~63)) for n in sorted(left, reverse=True))
  op = rng.choice(("adamw", "adamw", "adamw", "clip"))
  typ = rng.choice(("float32", "bfloat16", "float16"))
  if op == "clip":
    return dict(op="clip", bits=0, type=typ, sizes=sizes, max_norm=round(10 ** rng.uniform(-1, 1), 3), lr=0.0, beta2=0.0, decay=0.0, step=0)
  return dict(op="adamw", bits=rng.choice((8, 32)), type=typ, sizes=sizes, max_norm=rng.choice((0.0, 0.0, 1.0)), lr=1e-4,
              beta2=rng.choice((0.95, 0.99, 0.999)), decay=rng.choice((0.0, 0.01, 0.1)), step=int(10 ** rng.uniform(0, 5)))


def _numels(case):
  got = []
  for word in case["sizes"].split(","):
    k, n = word.split("*") if "*" in word else ("1", word)
    got += [int(n)] * int(k)
  return got


BETA1, EPS, SEED = 0.9, 1e-8, 7


def work(case):
  """Each input read once and each output written once.  AdamW: weights and both moments both ways, gradients in, and the
  half-precision copy of the weights out; the norm adds nothing to the bytes.  Clipping: gradients both ways."""
  n = sum(_numels(case))
  half = 2 if case["type"] != "float32" else 0
  grad = half or 4
  if case["op"] == "clip":
    return {"bytes": 2 * grad * n, "flops": 3 * n}
  moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
  return {"bytes": (8 + half + grad + moments) * n, "flops": (14 + (10 if case["bits"] == 8 else 0) + (2 if case["max_norm"] else 0)) * n}


def _blocks(case):
  """Per block of 128: its tensor, its first element's index in that tensor, its number of elements."""
  numels = torch.tensor(_numels(case), dtype=torch.int64)
  per = (numels + BLOCK - 1) // BLOCK
  tensor = torch.repeat_interleave(torch.arange(len(numels)), per)
  first = (torch.arange(len(tensor)) - (per.cumsum(0) - per)[tensor]) * BLOCK
  return numels, per, tensor, first, (numels[tensor] - first).clamp(max=BLOCK)


def prepare(case, seed):
  gen = torch.Generator(device="cuda").manual_seed(seed)
  numels, per, tensor, first, count = _blocks(case)
  nb = len(tensor)
  tensor, first, count = (t.cuda() for t in (tensor, first, count))
  keep = torch.arange(BLOCK, device="cuda") < count[:, None]

  def rand(*shape, normal=True):
    return (torch.randn if normal else torch.rand)(*shape, generator=gen, device="cuda")

  # gradients of one scale per tensor, 0.0001 to 0.03, with tails, and one block in fifty that nothing reaches (a dead unit,
  # a row that the batch does not touch)
  scale = (10 ** (-4 + 2.5 * rand(len(numels), normal=False)))[tensor][:, None]
  g = scale * rand(nb, BLOCK) * torch.exp(0.5 * rand(nb, BLOCK)) * (rand(nb, 1, normal=False) > 0.02) * keep
  typ = TYPES[case["type"]]
  s = {"case": case, "g": g.to(typ), "step": case["step"], "tensor": tensor, "first": first}
  del g
  if case["op"] == "adamw":
    decayed = (2 * len(numels) + 2) // 3
    s["w"] = 0.05 * rand(nb, BLOCK) * keep
    if typ != torch.float32:
      s["p"] = s["w"].to(typ)
    begun = case["step"] > 1
    m = 0.3 * scale * rand(nb, BLOCK) * keep * begun
    v = scale * scale * (0.2 + rand(nb, BLOCK, normal=False)) * keep * begun
    if case["bits"] == 8:
      half = torch.zeros((), dtype=torch.int32, device="cuda")
      s["m"], s["m_scale"] = _to_e4m3(m, half + (1 << 19))
      s["v"], s["v_scale"] = _to_e5m2(v, half + (1 << 20))
    else:
      s["m"], s["v"] = m, v
    del m, v
    s["decay"] = torch.where(tensor < decayed, case["decay"], 0.0)[:, None]
  if own:
    starts = ((per.cumsum(0) - per) * BLOCK).tolist()
    leaf = s["p" if "p" in s else "w" if "w" in s else "g"].view(-1)
    flat = s["g"].view(-1)
    params = []
    for a, n in zip(starts, numels.tolist()):
      x = (leaf[a:a + n].detach() if case["op"] == "adamw" else torch.empty_like(flat[a:a + n])).requires_grad_()
      x.grad = flat[a:a + n]
      params.append(x)
    s["params"] = params
    if case["op"] == "adamw":
      from oi_vae_amd import optim
      groups = [{"params": params[:decayed], "weight_decay": case["decay"]}]
      if decayed < len(params):
        groups.append({"params": params[decayed:], "weight_decay": 0.0})
      opt = optim.AdamW(groups, lr=case["lr"], betas=(BETA1, case["beta2"]), eps=EPS, state_bits=case["bits"],
                        max_grad_norm=case["max_norm"] or None, seed=SEED)
      held = opt.buffers[case["bits"]]
      held["exp_avg"].copy_(s["m"].view(-1))
      held["exp_avg_sq"].copy_(s["v"].view(-1))
      if case["bits"] == 8:
        held["exp_avg_scale"].copy_(s["m_scale"])
        held["exp_avg_sq_scale"].copy_(s["v_scale"])
      if "p" in s:
        held["master"].copy_(s["w"].view(-1))
        s["w"] = held["master"].view(nb, BLOCK)
      opt.set_steps(case["step"] - 1)
      s.update(opt=opt, m=held["exp_avg"].view(nb, BLOCK), v=held["exp_avg_sq"].view(nb, BLOCK))
      if case["bits"] == 8:
        s.update(m_scale=held["exp_avg_scale"], v_scale=held["exp_avg_sq_scale"])
  return s


def run(s):
  case = s["case"]
  if own:
    if case["op"] == "clip":
      from oi_vae_amd import optim
      return {"norm": optim.clip_grad_norm_(s["params"], case["max_norm"]), "g": s["g"]}
    s["opt"].step()
    out = {k: s[k] for k in ("w", "p", "m", "v", "m_scale", "v_scale") if k in s}
    if case["max_norm"]:
      out["norm"] = s["opt"].grad_norm
    return out
  out = {}
  if case["max_norm"]:
    norm = torch.sum(s["g"].float() ** 2, dtype=torch.float64).sqrt().float()
    coef = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    out["norm"] = norm
  if case["op"] == "clip":
    s["g"] = (s["g"].float() * coef).to(s["g"].dtype)
    out["g"] = s["g"]
    return out
  g = s["g"].float()
  if case["max_norm"]:
    g = g * coef
  b1, b2, t, lr = BETA1, case["beta2"], s["step"], case["lr"]
  m, v = s["m"], s["v"]
  if case["bits"] == 8:
    m, v = m.float() * s["m_scale"].float()[:, None], v.float() * s["v_scale"].float()[:, None]
  m = m * b1 + g * (1 - b1)
  v = v * b2 + g * g * (1 - b2)
  s["step"] += 1
  s["w"] = s["w"] * (1 - lr * s["decay"]) - (lr / (1 - b1 ** t)) * (m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + EPS))
  if "p" in s:
    s["p"] = s["w"].to(s["p"].dtype)
  if case["bits"] == 8:
    x = _random_bits(s["tensor"], s["first"], t)
    s["m"], s["m_scale"] = _to_e4m3(m, (x >> 12) & 0xFFFFF)
    s["v"], s["v_scale"] = _to_e5m2(v, x & 0x1FFFFF)
  else:
    s["m"], s["v"] = m, v
  out.update({k: s[k] for k in ("w", "p", "m", "v", "m_scale", "v_scale") if k in s})
  return out


# ---- moments of 8 bits ---------------------------------------------------------------------------------------------------
# A block of 128 values shares one power of two, 2^(scale byte - 127).  First moments are held as e4m3 codes, second moments
# as e5m2 codes, rounded stochastically: a code is the value's distance from zero in units of its binade's spacing, plus
# random bits below that spacing, cut off.  The random bits are inputs: a fixed function of seed, step, tensor and element.

def _signed(c):
  return c - (1 << 32) if c >= 1 << 31 else c


C1, C2, C3, C4 = (_signed(c) for c in (0x9E3779B1, 0x6A09E667, 0xBB67AE85, 0x3C6EF373))


def _right(x, k):
  return (x >> k) & ((1 << (32 - k)) - 1)   # a 32-bit shift that brings in zeros


def _random_bits(tensor, first, step):
  k = (tensor * C4 + (SEED * C1 + step * C3)).to(torch.int32)
  k = (k ^ _right(k, 16)) * C2
  k = (k ^ _right(k, 15)) * C3
  k = k ^ _right(k, 16)
  base = (first * C1 + (first >> 32) * C4).to(torch.int32) + k
  x = base[:, None] + (torch.arange(BLOCK, device=first.device) * C1).to(torch.int32)
  x = (x ^ _right(x, 14)) * C2
  return x ^ _right(x, 14)


def _scale_byte(x, low, shift):
  e = x.abs().amax(dim=1).view(torch.int32) >> 23
  return torch.where(e == 255, 255, e.clamp(min=low) - shift)


def _to_e4m3(m, r):
  b = _scale_byte(m, 8, 7)
  z = (m * ((254 - b) << 23).view(torch.float32)[:, None]) * 2.0 ** -120   # the codes' smallest spacing on that of float32
  q = ((z.abs().view(torch.int32) + r) >> 20) + (z.view(torch.int32) < 0) * 128
  return q.to(torch.uint8).view(torch.float8_e4m3fn), b.to(torch.uint8).view(torch.float8_e8m0fnu)


def _to_e5m2(v, r):
  b = _scale_byte(v, 15, 14)
  z = (v * ((254 - b) << 23).view(torch.float32)[:, None]) * 2.0 ** -112
  q = torch.maximum((z.view(torch.int32) + r) >> 21, (v > 0).to(torch.int32))   # what is not zero stays above it
  return q.to(torch.uint8).view(torch.float8_e5m2), b.to(torch.uint8).view(torch.float8_e8m0fnu)


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
  s = prepare(case, seed)
  g = s["g"].to(torch.float64)
  out = {}
  if case["max_norm"]:
    total = math.sqrt(float(torch.dot(g.view(-1), g.view(-1))))
    g *= min(1.0, case["max_norm"] / (total + 1e-6))
    out["norm"] = torch.tensor(total, dtype=torch.float64)
  if case["op"] == "clip":
    return {**out, "g": g}
  m, v, t = s["m"].to(torch.float64), s["v"].to(torch.float64), case["step"]
  if case["bits"] == 8:
    m *= s["m_scale"].to(torch.float64)[:, None]
    v *= s["v_scale"].to(torch.float64)[:, None]
  m += (1.0 - BETA1) * (g - m)
  v += (1.0 - case["beta2"]) * (g * g - v)
  m_hat, v_hat = m / (1.0 - BETA1 ** t), v / (1.0 - case["beta2"] ** t)
  w = s["w"].to(torch.float64)
  w = w - case["lr"] * s["decay"].to(torch.float64) * w - case["lr"] * m_hat / (v_hat.sqrt() + EPS)
  del m_hat, v_hat
  out["w"] = w
  if "p" in s:
    out["p"] = w
  if case["bits"] == 32:
    return {**out, "m": m, "v": v}
  mask = 0xFFFFFFFF
  key = (SEED * 0x9E3779B1 + t * 0xBB67AE85 + s["tensor"] * 0x3C6EF373) & mask
  for shift, factor in ((16, 0x6A09E667), (15, 0xBB67AE85), (16, 1)):
    key = ((key ^ (key >> shift)) * factor) & mask
  x = (s["first"][:, None] + torch.arange(BLOCK, device="cuda")) * 0x9E3779B1 + key[:, None] & mask
  x = ((x ^ (x >> 14)) * 0x6A09E667) & mask
  x ^= x >> 14

  def rounded(y, top, digits, least, noise):
    """Codes (as values) and scales: each block by the power of two that brings its largest value into [2^top, 2^(top + 1))."""
    most = y.abs().amax(dim=1)
    power = torch.where(most > 0, torch.frexp(most).exponent - 1 - top, -126).clamp(min=-126).to(torch.float64)
    y = y * torch.exp2(-power)[:, None]
    spacing = torch.exp2((torch.frexp(y).exponent - 1).clamp(min=least).to(torch.float64) - digits)
    return torch.sign(y) * torch.floor(y.abs() / spacing + noise) * spacing, torch.exp2(power)

  out["m"], out["m_scale"] = rounded(m, 7, 3, -6, (x >> 12).to(torch.float64) * 2.0 ** -20)
  out["v"], out["v_scale"] = rounded(v, 14, 2, -14, (x & 0x1FFFFF).to(torch.float64) * 2.0 ** -21)
  out["v"] = torch.where(v > 0, out["v"].clamp(min=2.0 ** -16), 0.0)
  return out
