"""Engine-native optimizers with torch.optim's constructor shape.

`Adam` and `SGD` take the same param-group lists the reference's scripts pass to
torch.optim (bars_data_oivae.py:233-244).  Once the parameters live in an
engine (after `OIVAE(...)` adopted the model) they update them with ONE fused
HIP kernel each over the engine's flat buffers instead of one launch per
tensor; `SGD` on `Ws` is fused with the proximal step that follows it.
torch.optim optimizers keep working too (the parameters are ordinary views).

`AdamW` also steps parameters that no engine holds (torch modules on the GPU, such as the
autoencoder variant's), all of them in a few launches, with moments in 32 or in 8 bits;
`clip_grad_norm_` and `grad_norm` are the gradient norm over such parameters.
"""
import ctypes

import numpy as np
import torch

from . import _lib


class _EngineOptimizer(object):
  def __init__(self, params, **defaults):
    if torch.is_tensor(params):
      raise TypeError("params must be an iterable of tensors or of groups, got one tensor (give [tensor])")
    groups = list(params)
    if groups and not isinstance(groups[0], dict):
      groups = [{"params": groups}]
    self.param_groups = []
    for g in groups:
      extra = sorted(k for k in g if k != "params" and k not in defaults)
      if extra:
        # one fused kernel with one set of options: anything it would silently ignore is refused
        raise ValueError("%s: unsupported per-group option(s) %s (supported: %s); use torch.optim for them"
                         % (type(self).__name__, ", ".join(extra), ", ".join(sorted(defaults))))
      d = dict(defaults)
      d.update({k: v for k, v in g.items() if k != "params"})
      members = g["params"]
      d["params"] = [members] if torch.is_tensor(members) else list(members)   # (list() of a tensor are its rows)
      self.param_groups.append(d)
    self._engine = None

  def _uniform(self, key, groups=None):
    """The one value of an option across all param groups (read at step time: schedulers may change it)."""
    vals = {(tuple(g[key]) if isinstance(g[key], (list, tuple)) else g[key]) for g in groups or self.param_groups}
    if len(vals) != 1:
      raise ValueError("engine-native optimizers apply one %r to every param group, got %s" % (key, sorted(vals)))
    return vals.pop()

  def zero_grad(self, set_to_none=True):
    """Attached to an engine: nothing to do -- every parameter's .grad is a view of the engine's flat gradient buffer,
    bound once, and each step overwrites that buffer completely (no loop over thousands of per-group tensors)."""
    if self._engine is not None:
      return
    for g in self.param_groups:
      for p in g["params"]:
        p.grad = None

  def _attach(self, engine):
    self._engine = engine

  def _lr(self):
    return self._uniform("lr")


class Adam(_EngineOptimizer):
  """torch.optim.Adam with default options over every non-Ws parameter."""

  def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, amsgrad=False):
    if weight_decay != 0 or amsgrad:
      raise ValueError("oi_vae_amd.optim.Adam is torch.optim.Adam with default options (weight_decay=0, "
                       "amsgrad=False): the fused kernel implements nothing else")
    super().__init__(params, lr=lr, betas=betas, eps=eps)

  def covers(self, engine):
    ptrs = {p.data_ptr() for g in self.param_groups for p in g["params"]}
    want = {t.data_ptr() for t, _ in engine.bound if t.data_ptr() != engine.p["Ws"].data_ptr()}
    return ptrs == want

  def step(self):
    if self._engine is None:
      raise RuntimeError("oi_vae_amd.optim.Adam steps engine parameters: pass it to OIVAE(optimizers=[...])")
    self._engine.adam_step(self._lr(), betas=self._uniform("betas"), eps=self._uniform("eps"))


class SGD(_EngineOptimizer):
  """Plain SGD (momentum 0) on Ws; OIVAE fuses it with the proximal step."""

  def __init__(self, params, lr=1e-3, momentum=0):
    if momentum != 0:
      raise ValueError("the reference uses momentum=0 on Ws (bars_data_oivae.py:243); nothing else is fused")
    super().__init__(params, lr=lr, momentum=0)
    self.fused_with_prox = False

  def covers(self, engine):
    ptrs = [p.data_ptr() for g in self.param_groups for p in g["params"]]
    return ptrs == [engine.p["Ws"].data_ptr()]

  def step(self):
    if self._engine is None:
      raise RuntimeError("oi_vae_amd.optim.SGD steps engine parameters: pass it to OIVAE(optimizers=[...])")
    if self.fused_with_prox:
      return  # OIVAE.step runs oivae_sgd_prox_f32 right after the optimizers
    self._engine.sgd_prox_step(self._lr(), 0.0, do_prox=False)


# ---- lists of tensors ------------------------------------------------------------------------------------------------------
_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_GRAD = np.dtype([("g", "u8"), ("n", "i8"), ("type", "i4"), ("index", "i4")])                     # oivae_grad_t
_TENSOR = np.dtype([("p", "u8"), ("g", "u8"), ("n", "i8"), ("at", "i8"), ("p_type", "i4"), ("g_type", "i4"),
                    ("group", "i4"), ("index", "i4"), ("step", "i4"), ("order", "i4")])           # oivae_adamw_tensor_t
_GROUP = np.dtype([("lr", "f4"), ("weight_decay", "f4"), ("lr_dev", "u8")])                       # oivae_adamw_group_t


def _dense(t):
  """Whether t's elements fill one piece of memory as they stand, in any order of its dimensions."""
  if t.layout != torch.strided or t.is_neg():
    return False
  expect = 1
  for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
    if stride != expect:
      return False
    expect *= size
  return True


def _check_types(tensors, what):
  device = None
  for t in tensors:
    if not torch.is_tensor(t) or t.layout != torch.strided:
      raise ValueError("%s must be dense tensors, got %s" % (what, getattr(t, "layout", type(t).__name__)))
    if t.dtype not in _TYPES:
      raise ValueError("%s must be float32, bfloat16 or float16, got %s" % (what, t.dtype))
    if not t.is_cuda:
      raise _lib.OivaeError("%s must be on the GPU, got %s: there is no CPU fallback" % (what, t.device))
    if device is not None and t.device != device:
      raise ValueError("%s must be on one device, got %s and %s" % (what, device, t.device))
    device = t.device
  return device


_ZERO = 2.0 ** -150     # half of float32's smallest: what is not above it is zero there


def _limit(max_norm, what="max_norm"):
  """Refuses a limit for which float32, in which the kernels compare, has no positive value."""
  if not float(max_norm) > _ZERO:
    raise ValueError("%s must be positive (and not below float32's range), got %r" % (what, max_norm))


def _lists():
  """The native reader of tensor lists (csrc/tensor_lists.cpp)."""
  global _lists_module
  if _lists_module is None:
    try:
      from . import _tensor_lists
    except ImportError as e:
      raise _lib.OivaeError("oi_vae_amd/_tensor_lists.so is not built (%s): run `make -C oi_vae_amd/csrc`" % e)
    _lists_module = _tensor_lists
  return _lists_module


_lists_module = None


def _stream(index):
  """Handle of the current stream of a device (torch.cuda.current_stream builds a Stream object first, for 1 us)."""
  return torch._C._cuda_getCurrentRawStream(index)


def _written(t):
  """Tells autograd that a kernel writes t."""
  if not t.is_inference():
    torch.autograd.graph.increment_version(t)


def _grads_of(parameters, write):
  """(records, their number and address, device index, gradients, their dense copies where they are not one piece of memory)
  of the gradients that are there; None without any."""
  ps = [parameters] if torch.is_tensor(parameters) else list(parameters)
  rec = np.zeros(len(ps), _GRAD)
  got = _lists().gradients(ps, rec, write)
  if got is not None:
    count, device, address = got
    return (rec, count, address, device, (), ()) if count else None
  grads = [p.grad for p in ps if p.grad is not None]
  device = _check_types(grads, "gradients")
  if len({g.data_ptr() for g in grads if g.numel()}) != sum(1 for g in grads if g.numel()):
    raise ValueError("the same gradient appears more than once")
  if write:   # what cannot be written is refused before the others are
    if any(st == 0 and size > 1 for g in grads for st, size in zip(g.stride(), g.shape)):
      raise RuntimeError("an expanded gradient (several elements in one place) cannot be scaled in place")
    spans = sorted((g.data_ptr(), g.data_ptr() + g.numel() * g.element_size()) for g in grads if g.numel() and _dense(g))
    if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
      raise ValueError("two gradients share memory")
  with torch.no_grad():
    packed = [g if _dense(g) else torch.empty(g.shape, dtype=g.dtype, device=device).copy_(g) for g in grads]
  rec = np.zeros(len(grads), _GRAD)
  rec["g"] = [g.data_ptr() for g in packed]
  rec["n"] = [g.numel() for g in packed]
  rec["type"] = [_TYPES[g.dtype] for g in packed]
  rec["index"] = -1
  return (rec, len(rec), rec.ctypes.data, device.index, grads, packed) if grads else None


def _clip(got, max_norm):
  _, count, address, device = got[:4]
  if torch.cuda.current_device() != device:
    with torch.cuda.device(device):
      return _clip(got, max_norm)
  L = _lib.init_device(device)
  nbytes = L.oivae_grad_norm_workspace_bytes(count)
  # norm and workspace of this call alone: calls on other streams and in captured graphs have their own
  norm, ws = torch.empty((), dtype=torch.float32, device="cuda"), torch.empty(nbytes, dtype=torch.uint8, device="cuda")
  _lib.check(L.oivae_clip_grad_norm(address, count, max_norm, norm.data_ptr(), ws.data_ptr(), nbytes,
                                    _stream(device)), "oivae_clip_grad_norm")
  return norm


def grad_norm(parameters):
  """2-norm of the gradients of `parameters` (a tensor or an iterable of tensors; those without a gradient are left out)
  taken as one vector: a 0-dim float32 tensor on their device (a zero on the CPU without any), with no synchronisation.  Squares and sums are formed in
  fp64, in an order that depends on the sizes alone."""
  got = _grads_of(parameters, False)
  if got is None:
    return torch.zeros((), dtype=torch.float32)
  return _clip(got, 0.0)


def clip_grad_norm_(parameters, max_norm):
  """torch.nn.utils.clip_grad_norm_ (2-norm): scales the gradients in place by min(1, max_norm / (norm + 1e-6)) and returns
  the norm they had, without synchronising.  A norm that is not finite reaches the gradients as it does there (NaN)."""
  max_norm = float(max_norm)
  if not max_norm > _ZERO:
    _limit(max_norm)
  got = _grads_of(parameters, True)
  if got is None:
    return torch.zeros((), dtype=torch.float32)
  norm = _clip(got, max_norm)
  if got[4]:
    with torch.no_grad():
      for g, c in zip(*got[4:]):
        if c is not g:
          g.copy_(c)
        else:
          _written(g)
  return norm


class AdamW(_EngineOptimizer):
  """torch.optim.AdamW (decoupled weight decay) over many tensors at once.

  Two uses: handed to `OIVAE(optimizers=[AdamW(...), SGD(...)])` it steps the engine's flat buffers in place of `Adam` (one
  lr, weight_decay and state_bits for all groups); by itself it steps the `.grad` of any float32, bfloat16 or float16
  tensors on one GPU.  Per group: `lr`, `weight_decay`, `state_bits` (the last fixed at first use, as the parameters are);
  `betas` and `eps` are one for all.

  state_bits=8 holds both moments in 8 bits: blocks of 128 elements of a tensor share a power of two; first moments are
  e4m3 codes, second moments e5m2 codes, rounded stochastically with bits drawn from (seed, step, tensor, element) -- two
  runs of one program agree bit for bit.  16-bit parameters are rounded copies of fp32 master weights, which the optimizer
  keeps; whoever writes such parameters behind its back calls `sync_master()`.

  max_grad_norm: clips by the norm of all gradients of this optimizer (`grad_norm` holds it after a step).  The gradients
  themselves stay as they are, and a step whose norm is not finite is left out on the device (`skipped` counts them).
  Handed to OIVAE, the norm is that of every gradient but Ws's, which SGD applies unclipped; a gradient of Ws that is not
  finite leaves the step out too (the norm is NaN then), and a step that is left out leaves Ws alone as well.
  capturable: keeps the step counts on the device, so that a step captured into a graph advances them (max_grad_norm
  implies it); `lr` may then be a one-element float32 tensor on the device, which replays read anew.  Every other number --
  weight_decay, grad_scale, max_grad_norm, seed -- and the gradients' addresses are those of the capture.  Touch `buffers` (or
  take a step) before capturing.  A step behind a failed decoder launch is left out on the device; counts on
  the device stay then, counts on the host have moved when the host hears of it (at its next call, with an OivaeError).
  Steps of one optimizer follow each other: they share its buffers.  It is no torch.optim.Optimizer: a schedule writes
  `param_groups[k]["lr"]`.  Nothing here synchronises but `steps` and `state_dict` of counts on the device."""

  def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_grad_norm=None,
               capturable=False, seed=0):
    super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits)
    if max_grad_norm is not None:
      _limit(max_grad_norm, "max_grad_norm")
    seed = self._checked_seed(seed)
    seen = set()
    for g in self.param_groups:
      if g["state_bits"] not in (8, 32):
        raise ValueError("state_bits must be 8 or 32, got %r" % (g["state_bits"],))
      for p in g["params"]:
        if not torch.is_tensor(p):
          raise ValueError("parameters must be tensors, got %s" % type(p).__name__)
        if not (p.is_leaf or p.retains_grad):
          raise ValueError("a parameter is the result of an operation: it has no .grad to step from")
        if id(p) in seen:
          raise ValueError("a parameter appears more than once")
        seen.add(id(p))
    if not seen:
      raise ValueError("AdamW got no parameters")
    self._options()
    self.max_grad_norm = max_grad_norm
    self.seed = seed
    self._on_device = bool(capturable) or max_grad_norm is not None
    self._buffers = None

  @staticmethod
  def _checked_seed(seed):
    if not 0 <= int(seed) < 1 << 32:
      raise ValueError("seed must be in [0, 2^32), got %r" % (seed,))
    return int(seed)

  def _options(self, groups=None):
    groups = groups or self.param_groups
    b1, b2 = self._uniform("betas", groups)
    eps = self._uniform("eps", groups)
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
      raise ValueError("betas must be in [0, 1), got %r" % ((b1, b2),))
    if not eps >= 0.0:
      raise ValueError("eps must not be negative, got %r" % (eps,))
    for g in groups:
      if not torch.is_tensor(g["lr"]) and not g["lr"] >= 0.0:
        raise ValueError("lr must not be negative, got %r" % (g["lr"],))
      if not g["weight_decay"] >= 0.0:
        raise ValueError("weight_decay must not be negative, got %r" % (g["weight_decay"],))
    return b1, b2, eps

  # ---- engine ---------------------------------------------------------------
  covers = Adam.covers

  def _attach(self, engine):
    for key in ("lr", "weight_decay", "state_bits"):
      self._uniform(key)
    if self._buffers is not None:
      raise RuntimeError("this AdamW has stepped parameters already: give OIVAE a new one")
    super()._attach(engine)

  def zero_grad(self, set_to_none=True):
    """Drops the gradients (or, with set_to_none=False, zeroes them in place); nothing to do on an engine."""
    if self._engine is not None:
      return
    for g in self.param_groups:
      for p in g["params"]:
        if set_to_none:
          p.grad = None
        elif p.grad is not None:
          if p.grad.grad_fn is not None:
            p.grad.detach_()
          else:
            p.grad.requires_grad_(False)     # (detach_ refuses views, such as parts of a flat buffer of gradients)
          p.grad.zero_()

  # ---- storage ---------------------------------------------------------------
  def _setup(self):
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
      raise RuntimeError("AdamW allocates its moments at its first use: touch .buffers or take a step before capturing")
    if self._engine is not None:
      eng = self._engine
      leaves, groups = [eng.flat_params[:eng.adam_numel]], [0]
    else:
      leaves = [p for g in self.param_groups for p in g["params"]]
      groups = [i for i, g in enumerate(self.param_groups) for _ in g["params"]]
    device = _check_types(leaves, "parameters")
    for p in leaves:
      if not _dense(p):
        raise ValueError("a parameter of strides %s and shape %s does not fill its memory" % (p.stride(), tuple(p.shape)))
    spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in leaves if p.numel())
    if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
      raise ValueError("two parameters share memory")
    self._leaves, self._group_of, self.device = leaves, groups, device
    self._lib = _lib.init_device(device.index)
    self._kinds = []
    self._steps_dev = torch.zeros(len(leaves), 4, dtype=torch.int32, device=device) if self._on_device else None
    bits_of = [self.param_groups[g]["state_bits"] for g in groups]
    for bits in (32, 8):
      # 16-bit parameters first: the master buffer need not reach further than they do
      mine = sorted((i for i in range(len(leaves)) if bits_of[i] == bits), key=lambda i: leaves[i].dtype == torch.float32)
      if mine:
        self._kinds.append(_Kind(self, bits, mine, groups))
    buffers = {k.bits: k.held for k in self._kinds}
    self._groups = np.zeros(len(self.param_groups), _GROUP)
    self._groups_at = self._groups.ctypes.data
    self._clip = torch.zeros(8, dtype=torch.int32, device=device) if self._on_device else None
    if self._on_device:
      # the gradients of all kinds, one behind the other; on an engine then that of Ws, which is not clipped but leaves the
      # step out as well when it is not finite
      watched = [] if self._engine is None else [self._engine.g["Ws"]]
      self._norm_rec = np.zeros(len(leaves) + len(watched), _GRAD)
      for r, g in zip(self._norm_rec[len(leaves):], watched):
        r["g"], r["n"], r["type"], r["index"] = g.data_ptr(), g.numel(), _lib.F32_WATCHED, -1
      self._norm_at = self._norm_rec.ctypes.data
      self._ws = torch.empty(self._lib.oivae_grad_norm_workspace_bytes(len(self._norm_rec)), dtype=torch.uint8, device=device)
      at = 0
      for k in self._kinds:
        k.grads = self._norm_rec[at:at + len(k.mine)]
        at += len(k.mine)
    self._buffers = buffers
    self._take_master()

  @property
  def buffers(self):
    """The optimizer's state by number of bits: {32: {"exp_avg", "exp_avg_sq"[, "master"]}, 8: {"exp_avg", "exp_avg_scale",
    "exp_avg_sq", "exp_avg_sq_scale"[, "master"]}}, flat tensors in which every parameter has a region of whole blocks of
    128 elements (16-bit parameters first, else in the order given).  Allocated at first use."""
    if self._buffers is None:
      self._setup()
    return self._buffers

  def _views(self, name):
    """(parameter, its part of the flat buffer `name`) of every parameter that has one, parameter by parameter."""
    for k in self._kinds:
      flat = k.held.get(name)
      for i, r in zip(k.mine, k.rec):
        if flat is not None and (name != "master" or r["p_type"] != _lib.F32):
          yield self._leaves[i], flat[int(r["at"]):int(r["at"] + r["n"])]

  @torch.no_grad()
  def sync_master(self):
    """Takes the master weights of 16-bit parameters from the parameters again."""
    self.buffers
    for k in self._kinds:
      for p, r in zip(k.leaves, k.rec):
        self._check_parameter(p, r)
    self._take_master()

  @torch.no_grad()
  def _take_master(self):
    for p, flat in self._views("master"):
      flat.as_strided(p.shape, p.stride()).copy_(p)

  def _check_parameter(self, p, r):
    """Refuses a parameter that is not what its moments were made for."""
    if p.numel() != r["n"] or _TYPES.get(p.dtype) != r["p_type"]:
      raise ValueError("a parameter changed its size or type since this optimizer's first step")
    if not _dense(p):
      raise ValueError("a parameter of strides %s and shape %s does not fill its memory" % (p.stride(), tuple(p.shape)))
    if _lists().order(p) != r["order"]:
      raise ValueError("a parameter changed the order of its elements since this optimizer's first step: its moments lie in that "
                       "one, now it has strides %s" % (p.stride(),))

  @property
  def grad_norm(self):
    """Norm of the last step's gradients (after grad_scale): a 0-dim tensor on the device, a view of the optimizer's buffer that
    the next step overwrites (clone it to keep it).  Needs max_grad_norm."""
    if self.max_grad_norm is None:
      raise RuntimeError("AdamW computes the gradient norm where max_grad_norm is given")
    self.buffers
    return self._clip.view(torch.float32)[0]

  def _verdict(self):
    """Address of the last step's verdict (oivae_clip_t), None where none is formed."""
    return self._clip.data_ptr() if self._on_device else None

  @property
  def skipped(self):
    """Number of steps left out because their gradient norm was not finite: a 0-dim int32 tensor on the device, a view of the
    optimizer's buffer."""
    if not self._on_device:
      raise RuntimeError("AdamW leaves steps out where max_grad_norm (or capturable) is given")
    self.buffers
    return self._clip[3]

  def steps(self):
    """Steps taken so far, parameter by parameter (a list; reads the device where the counts live there)."""
    self.buffers
    if self._on_device:
      return self._steps_dev[:, 0].tolist()
    counts = np.zeros(len(self._leaves), np.int32)
    for k in self._kinds:
      counts[k.mine] = k.rec["step"]
    return counts.tolist()

  def _counts(self, steps):
    counts = np.broadcast_to(np.asarray(steps, np.int32), (len(self._leaves),))
    if (counts < 0).any():
      raise ValueError("step counts must not be negative")
    return counts

  def set_steps(self, steps):
    """Sets the step counts: one number for all parameters or one for each."""
    self.buffers
    counts = self._counts(steps)
    for k in self._kinds:
      k.rec["step"] = counts[k.mine]
    if self._on_device:
      self._steps_dev[:, 0] = torch.from_numpy(counts.copy()).to(self.device)

  def state_dict(self):
    """Everything a resumed run needs: counts, options and copies of `buffers`."""
    self.buffers
    return {"steps": self.steps(), "seed": self.seed, "sizes": [p.numel() for p in self._leaves], **self._layout(),
            "skipped": int(self._clip[3]) if self._on_device else 0,
            "groups": [{k: v.clone() if torch.is_tensor(v) else v for k, v in g.items() if k != "params"} for g in self.param_groups],
            "buffers": {bits: {k: t.clone() for k, t in held.items()} for bits, held in self.buffers.items()}}

  def _layout(self):
    """What decides, beside the sizes, where in the buffers a parameter's state lies and which options it has."""
    types, orders = [None] * len(self._leaves), [None] * len(self._leaves)
    for k in self._kinds:
      for i, r in zip(k.mine, k.rec):
        types[i], orders[i] = ("float32", "bfloat16", "float16")[r["p_type"]], int(r["order"])
    return {"types": types, "orders": orders, "group_of": list(self._group_of)}

  @torch.no_grad()
  def load_state_dict(self, state):
    """Takes over a state_dict of an AdamW over parameters of the same sizes, types, orders in memory and groups; any other is
    refused before anything is changed."""
    held = self.buffers
    lacking = [k for k in ("steps", "seed", "sizes", "groups", "buffers") if k not in state]
    if lacking:
      raise ValueError("the state holds no %s" % ", ".join(lacking))
    for what, mine, theirs in [("bits", held, state["buffers"])] + [("buffers", held[b], state["buffers"].get(b, {})) for b in held]:
      if sorted(mine) != sorted(theirs):
        raise ValueError("the state holds %s %s, this optimizer %s" % (what, sorted(theirs), sorted(mine)))
    pairs = [(t, state["buffers"][b][k], k) for b in held for k, t in held[b].items()]
    for t, src, k in pairs:
      if src.shape != t.shape or src.dtype != t.dtype:
        raise ValueError("%s is %s %s in the state, %s %s here" % (k, tuple(src.shape), src.dtype, tuple(t.shape), t.dtype))
    if (list(state["sizes"]) != [p.numel() for p in self._leaves] or len(state["groups"]) != len(self.param_groups)
        or any(src["state_bits"] != g["state_bits"] for src, g in zip(state["groups"], self.param_groups))):
      raise ValueError("the state was made for other parameters or groups")
    layout = self._layout()
    if any(k in state for k in layout):
      for k, mine in layout.items():
        if list(state.get(k, ())) != mine:
          raise ValueError("the state was made for other parameters or groups: %s %s there, %s here" % (k, state.get(k), mine))
    elif len(self._kinds) != 1 or len({t == "float32" for t in layout["types"]}) != 1:
      # written before states held their layout: the sizes alone say where everything lies where the moments have one number of
      # bits and the parameters are all of 32 or all of 16
      raise ValueError("the state was made for parameters of unknown types and groups, which these do not tell")
    if len(state["steps"]) != len(self._leaves):
      raise ValueError("the state holds %d step counts for %d parameters" % (len(state["steps"]), len(self._leaves)))
    skipped = int(state.get("skipped", 0))
    if not 0 <= skipped < 1 << 31:
      raise ValueError("the state counts %r steps left out" % (skipped,))
    counts, seed, options = self._counts(state["steps"]), self._checked_seed(state["seed"]), self._options_from(state["groups"])
    for t, src, _ in pairs:
      t.view(torch.uint8).copy_(src.view(torch.uint8))
    self.set_steps(counts)
    self.seed = seed
    if self._on_device:
      self._clip[3] = skipped
    for g, src in zip(self.param_groups, options):
      for k, v in src.items():
        if torch.is_tensor(g[k]):
          g[k].fill_(v)     # an lr on the device stays where a captured graph reads it
        else:
          g[k] = v

  def _options_from(self, groups):
    """A state's options, as numbers, once they are known to be ones that this optimizer's groups could have been given."""
    out = []
    for g, src in zip(self.param_groups, groups):
      strange = set(src) - set(g) | {"lr", "betas", "eps", "weight_decay", "state_bits"} - set(src)
      if strange:
        raise ValueError("a group of the state has other options than here: %s" % ", ".join(sorted(strange)))
      for k, v in list(src.items()) + [(k, v) for k, v in g.items() if k != "params"]:
        if torch.is_tensor(v) and v.numel() != 1:
          raise ValueError("%s has %d values" % (k, v.numel()))
      out.append({k: v.item() if torch.is_tensor(v) else v for k, v in src.items()})
    self._options(out)
    if self._engine is not None:
      for key in ("lr", "weight_decay"):
        self._uniform(key, out)
    return out

  # ---- the step ---------------------------------------------------------------
  @torch.no_grad()
  def _read(self, kind, copies):
    """Addresses of a kind's parameters and gradients into its records, the way round (csrc/tensor_lists.cpp takes lists
    that are all as their records say): copies gradients into their parameter's order, says what cannot be stepped.
    Returns the number without a gradient; the copies, which have to live until the step is queued, go into `copies`."""
    missing = 0
    for j, i in enumerate(kind.mine):
      p, r = self._leaves[i], kind.rec[j]
      g = p.grad
      if g is None:
        r["g"], missing = 0, missing + 1
        if kind.grads is not None:
          kind.grads[j] = (0, 0, 0, -1)
        continue
      if g.layout != torch.strided:
        raise ValueError("gradients must be dense tensors, got %s" % g.layout)
      if g.dtype not in _TYPES or g.device != self.device or p.device != self.device:
        raise ValueError("parameter and gradient must be float32, bfloat16 or float16 on %s, got %s on %s with %s on %s"
                         % (self.device, p.dtype, p.device, g.dtype, g.device))
      self._check_parameter(p, r)
      if g.shape != p.shape:
        raise ValueError("a gradient of shape %s for a parameter of shape %s" % (tuple(g.shape), tuple(p.shape)))
      if g.is_neg() or (g.stride() != p.stride() and not (p.is_contiguous() and g.is_contiguous())):
        g = torch.empty_like(p, dtype=g.dtype).copy_(g)
        copies.append(g)
      _written(p)
      r["p"], r["g"], r["g_type"] = p.data_ptr(), g.data_ptr() or 16, _TYPES[g.dtype]     # (0: no gradient)
      if kind.grads is not None:
        kind.grads[j] = (g.data_ptr(), g.numel(), _TYPES[g.dtype], r["index"])
    return missing

  def step(self, grad_scale=1.0):
    """One step from the parameters' gradients, times grad_scale (1 / loss scale).  Parameters without a gradient stay as
    they are and keep their count, as in torch.optim."""
    if self._buffers is None:
      self._setup()
    if torch.cuda.current_device() == self.device.index:
      self._step(float(grad_scale))
    else:
      with torch.cuda.device(self.device):
        self._step(float(grad_scale))

  def _step(self, grad_scale):
    first, L, index = self.param_groups[0], self._lib, self.device.index
    (b1, b2), eps = first["betas"], first["eps"]
    groups = self._groups
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0):
      self._options()      # says which; before the norm's launch, which advances the counts on the device
    for q, g in enumerate(self.param_groups):
      if g is not first and (g["eps"] != eps or tuple(g["betas"]) != (b1, b2)):
        raise ValueError("AdamW applies one 'betas' and one 'eps' to every param group")
      lr = g["lr"]
      groups[q] = self._lr_on_device(lr, g) if torch.is_tensor(lr) else (lr, g["weight_decay"], 0)
    limit = 0.0
    if self.max_grad_norm is not None:
      limit = float(self.max_grad_norm)
      if not limit > _ZERO:
        _limit(limit, "max_grad_norm")
      if not self._on_device:
        raise RuntimeError("max_grad_norm has to be given to the constructor (it may be changed or set to None later)")
    if not self._on_device and torch.cuda.is_current_stream_capturing():
      raise RuntimeError("a captured step would repeat its step count at every replay: use AdamW(capturable=True)")
    todo, partial, copies = [], False, []
    for k in self._kinds:
      if self._engine is not None:
        self._uniform("lr"), self._uniform("weight_decay")   # one for the flat buffer, whatever a schedule does
        k.rec["p"], k.rec["g"] = self._leaves[0].data_ptr(), self._engine.flat_grads.data_ptr()
        if k.grads is not None:
          k.grads[0] = (k.rec["g"][0], k.rec["n"][0], _lib.F32, 0)
        missing = 0
      else:
        unusual, missing = _lists().parameters(k.leaves, k.rec, index, k.grads)
        if unusual >= 0:
          missing = self._read(k, copies)
      rec = k.rec
      if missing:
        partial, rec = True, rec[rec["g"] != 0]
      todo.append((k, rec))
    if partial and not any(len(rec) for _, rec in todo):
      return
    stream = _stream(index)
    clip = None
    if self._on_device:
      clip = self._clip.data_ptr()
      _lib.check(L.oivae_grad_norm(self._norm_at, len(self._norm_rec), limit > 0.0, grad_scale, limit, clip, self._steps_dev.data_ptr(), b1, b2,
                                   self._ws.data_ptr(), self._ws.numel(), stream), "oivae_grad_norm")
    for k, rec in todo:
      if not len(rec):
        continue
      counts = k.rec["step"]
      if not self._on_device:
        counts += 1
        if rec is not k.rec:
          counts[k.rec["g"] == 0] -= 1
          rec["step"] += 1
      args = (k.rec_at if rec is k.rec else rec.ctypes.data, len(rec), self._groups_at, len(groups), k.state_ref, b1, b2, eps, grad_scale)
      if k.bits == 32:
        rc = L.oivae_adamw_f32(*args, clip, stream)
      else:
        rc = L.oivae_adamw_f8(*args, self.seed, clip, stream)
      if rc:
        if not self._on_device:
          counts[k.rec["g"] != 0] -= 1
        _lib.check(rc, "oivae_adamw_f%d" % k.bits)

  def _lr_on_device(self, lr, group):
    if lr.numel() != 1 or lr.dtype != torch.float32 or lr.device != self.device:
      raise ValueError("an lr tensor must be one float32 on %s" % self.device)
    return 0.0, group["weight_decay"], lr.data_ptr()


class _Kind(object):
  """The parameters of one AdamW whose moments have one number of bits: their records and flat buffers."""

  def __init__(self, opt, bits, mine, groups):
    leaves, device = opt._leaves, opt.device
    self.bits, self.mine, self.leaves, self.grads = bits, mine, [leaves[i] for i in mine], None
    self.rec = rec = np.zeros(len(mine), _TENSOR)
    rec["n"] = [p.numel() for p in self.leaves]
    whole = (rec["n"] + _lib.ADAMW_BLOCK - 1) // _lib.ADAMW_BLOCK * _lib.ADAMW_BLOCK
    rec["at"] = np.cumsum(whole) - whole
    rec["p_type"] = [_TYPES[p.dtype] for p in self.leaves]
    rec["group"] = [groups[i] for i in mine]
    rec["index"] = mine
    rec["order"] = [_lists().order(p) for p in self.leaves]
    self.rec_at = rec.ctypes.data
    total, half = max(int(whole.sum()), _lib.ADAMW_BLOCK), int(whole[rec["p_type"] != _lib.F32].sum())
    self.held = held = {}
    if bits == 32:
      for name in ("exp_avg", "exp_avg_sq"):
        held[name] = torch.zeros(total, dtype=torch.float32, device=device)
    else:
      for name, typ in (("exp_avg", torch.float8_e4m3fn), ("exp_avg_sq", torch.float8_e5m2)):
        held[name] = torch.zeros(total, dtype=torch.uint8, device=device).view(typ)
        held[name + "_scale"] = torch.zeros(total // _lib.ADAMW_BLOCK, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    if half:
      held["master"] = torch.zeros(half, dtype=torch.float32, device=device)
    ptr = lambda k: held[k].data_ptr() if k in held and held[k].numel() else None
    self.state = _lib.AdamwState(ptr("exp_avg"), ptr("exp_avg_sq"), ptr("exp_avg_scale"), ptr("exp_avg_sq_scale"), ptr("master"),
                                 opt._steps_dev.data_ptr() if opt._on_device else None)
    self.state_ref = ctypes.byref(self.state)
