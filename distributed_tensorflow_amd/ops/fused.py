"""Device-dispatching entry points of the fused element-wise ops.

On a GPU these call the hand-written HIP kernels of the in-tree extension
(`ops/native.py`); on the CPU (tests, gloo runs) the same arithmetic is a few
torch ops.  A GPU tensor with the extension missing raises - there is no silent
library fallback on the device path.
"""
from __future__ import annotations

import itertools
from typing import Dict, Optional, Sequence

import torch
from torch.autograd import forward_ad

__all__ = ["sgd_momentum_l2", "clipped_sgd_momentum_l2", "TensorTable", "global_norm", "clip_by_global_norm",
           "residual_norm", "residual_norm_grad"]


def sgd_momentum_l2(params: torch.Tensor, grads: torch.Tensor, velocity: torch.Tensor,
                    l2x2: torch.Tensor, lr: float, momentum: float, grad_scale: float = 1.0,
                    skip=None):
  """Keras-form SGD step on flat fp32 buffers, in place.

      g  = grads * grad_scale + l2x2 * params      (l2x2 = 2*lambda per element)
      v <- momentum * v - lr * g
      w <- w + v
  """
  if params.device.type == "cuda":
    from . import native  # pylint: disable=import-outside-toplevel
    native.sgd_momentum_l2(params, grads, velocity, l2x2, lr, momentum, grad_scale, skip)
    return
  if skip is not None:
    raise ValueError("a device-side skip flag needs the native optimizer kernel")
  with torch.no_grad():
    g = grads * grad_scale if grad_scale != 1.0 else grads
    g = torch.addcmul(g, l2x2, params)
    if momentum:
      velocity.mul_(momentum).add_(g, alpha=-lr)
      params.add_(velocity)
    else:
      params.add_(g, alpha=-lr)

# ---- the seam between two residual blocks ----------------------------------------------------------

MAX_CHANNELS = 8192      # of the native kernels


_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_FP32 = torch.float32


def _row_pitch(name: str, t: torch.Tensor, channels: int) -> int:
  """Elements from one row of `t` to the next; rows are everything but the last dimension."""
  if t.is_contiguous():
    return channels
  if channels > 1 and t.stride(-1) != 1:
    raise ValueError("%s: the channels of a row have to lie next to each other" % name)
  if t.dim() == 1:
    return channels
  last = t.dim() - 2
  while last > 0 and t.shape[last] == 1:      # a dimension of one row has no distance of its own
    last -= 1
  pitch = t.stride(last)
  for d in range(last):
    if t.shape[d] > 1 and t.stride(d) != pitch * t.shape[d + 1:-1].numel():
      raise ValueError("%s: its rows lie at different distances" % name)
  return pitch


def _pitch(name: str, t: torch.Tensor, channels: int, shape, dtype, device: int) -> int:
  if t.shape != shape or t.dtype is not dtype or t.get_device() != device:
    raise ValueError("%s: %s %s on %s, but the rows are %s %s on device %d" % (
        name, tuple(t.shape), t.dtype, t.device, tuple(shape), dtype, device))
  return _row_pitch(name, t, channels)


def _seam(like, y, post_gamma, post_beta, gate, gate_act, pre_gamma, pre_beta, norm, eps):
  """Checks what `residual_norm` and `residual_norm_grad` have in common; (rows, channels, rows that share a gate row
  or 0, gate pitch, sigmoid, layer).  (Written for its own speed: it runs before every launch.)"""
  shape, dtype, device = like.shape, like.dtype, like.get_device()
  if not shape or shape[-1] < 1:
    raise ValueError("rows of at least one channel, got %s" % (tuple(shape),))
  if dtype not in _TYPES:
    raise ValueError("element type %s (bfloat16, float16 and float32 are built)" % dtype)
  c = shape[-1]
  rows = like.numel() // c
  layer = norm == "layer"
  if not layer:
    if norm != "rms":
      raise ValueError("norm is 'rms' or 'layer', not %r" % (norm,))
    if post_beta is not None or pre_beta is not None:
      raise ValueError("norm='rms' has no beta")
  if not eps > 0:
    raise ValueError("eps has to be positive")
  sigmoid = gate_act == "sigmoid"
  if not sigmoid and gate_act != "none":
    raise ValueError("gate_act is 'none' or 'sigmoid', not %r" % (gate_act,))
  if y is None and (post_gamma is not None or gate is not None):
    raise ValueError("post_gamma and gate belong to y")
  if (post_beta is not None and post_gamma is None) or (pre_beta is not None and pre_gamma is None):
    raise ValueError("a beta goes with its gamma")
  for name, t in (("post_gamma", post_gamma), ("post_beta", post_beta), ("pre_gamma", pre_gamma),
                  ("pre_beta", pre_beta)):
    if t is not None and (t.dim() != 1 or t.numel() != c or t.dtype is not _FP32 or t.get_device() != device
                          or not t.is_contiguous()):
      raise ValueError("%s: %d contiguous float32 values on the rows' device" % (name, c))
  group_rows, gate_pitch = 0, c
  if gate is not None:
    if gate.dtype is dtype and gate.shape == shape:
      gate_pitch = _pitch("gate", gate, c, shape, dtype, device)
    elif gate.dtype is _FP32 and gate.get_device() == device and gate.dim() in (1, 2) and gate.shape[-1] == c:
      groups = gate.numel() // c
      if groups < 1 or rows % groups:
        raise ValueError("gate: %d rows of it do not divide %d rows" % (groups, rows))
      group_rows = rows // groups
      gate_pitch = _row_pitch("gate", gate, c)
    else:
      raise ValueError("gate: one value per element in the rows' type, or float32 [groups, %d] with groups that "
                       "divide the rows; got %s %s on %s" % (c, tuple(gate.shape), gate.dtype, gate.device))
  return rows, c, group_rows, gate_pitch, sigmoid, layer


def _no_graph(*tensors):
  """These entry points compute values; a gradient that autograd would have to record is refused, not lost."""
  if torch.is_grad_enabled():
    for t in tensors:
      if t is not None and t.requires_grad:
        raise ValueError("an argument requires a gradient: it is computed by residual_norm_grad, call under "
                         "torch.no_grad()")
  _no_tangent(tensors)


def _no_tangent(*lists):
  """A forward-mode derivative that an argument carries is refused, not lost (whether or not gradients are recorded)."""
  if forward_ad._current_level < 0:      # outside of forward_ad.dual_level() and torch.func.jvp
    return
  for t in itertools.chain(*lists):
    if t is not None and forward_ad.unpack_dual(t).tangent is not None:
      raise ValueError("an argument carries a forward-mode derivative, which is not computed here")


def _normalised(v: torch.Tensor, layer: bool, eps: float):
  if layer:
    v = v - v.mean(-1, keepdim=True)
  r = torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
  return v * r, r


def _normalised_grad(d, hat, r, layer):
  d_mean = d.mean(-1, keepdim=True) if layer else 0.0
  return r * (d - d_mean - hat * (d * hat).mean(-1, keepdim=True))


def _gate_factor(gate, rows, channels, group_rows, sigmoid):
  """The gate's factor per row and its derivative, in float32."""
  g = gate.float().reshape(-1, channels)
  g = g.repeat_interleave(group_rows, 0) if group_rows else g[:rows]
  if not sigmoid:
    return g, 1.0
  # (a * (1 - a) of a rounded a loses its digits where the gate is open)
  e = torch.exp(-g.abs())
  d = 1 / (1 + e)
  return torch.where(g < 0, e * d, d), e * d * d


def residual_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None, *, post_gamma=None, post_beta=None, gate=None,
                  gate_act: str = "none", residual_scale: float = 1.0, pre_gamma=None, pre_beta=None,
                  norm: str = "rms", eps: float = 1e-6):
  """What lies between two residual blocks, in one pass over the rows.

      n = N(y) * post_gamma + post_beta             the norm after the block (n = y without post_gamma)
      h = x + residual_scale * act(gate) * n        the residual stream (h is x without y)
      z = N(h) * pre_gamma + pre_beta               the norm before the next block (None without pre_gamma)

  returns (h, z).  `x`, `y` and the results are [..., channels] in bfloat16, float16 or float32, 1 to 8192
  channels (pixels of an NHWC activation, tokens); rows may lie at any one distance, their channels next to each other.
  N is v / sqrt(mean(v^2) + eps) with norm="rms", (v - mean) / sqrt(var + eps) with norm="layer".  gammas and
  betas are float32 [channels], betas only with "layer".  `gate` is a value per element in the type of x, or float32
  [groups, channels] (or [channels]) whose rows hold for rows / groups consecutive rows each: a learnt scale per channel,
  a gate per image.  gate_act is "none" or "sigmoid".  Arithmetic is float32, z comes from the unrounded h.  Squares
  are summed in float32: where their sum over a row passes 3.4e38 (all values at 1.8e19 / sqrt(channels): 2.9e17 of 4096)
  the row counts as infinitely large, and N of it is zero.
  No graph is recorded; `residual_norm_grad` is the gradient.
  """
  rows, c, group_rows, ldgate, sigmoid, layer = _seam(x, y, post_gamma, post_beta, gate, gate_act, pre_gamma, pre_beta,
                                                      norm, eps)
  _no_graph(x, y, post_gamma, post_beta, gate, pre_gamma, pre_beta)
  ldx = _row_pitch("x", x, c)
  ldy = c if y is None else _pitch("y", y, c, x.shape, x.dtype, x.get_device())
  if x.is_cuda:
    if c > MAX_CHANNELS:
      raise ValueError("at most %d channels, got %d" % (MAX_CHANNELS, c))
    from . import native  # pylint: disable=import-outside-toplevel
    return native.residual_norm(x, ldx, y, ldy, rows, c, gate, ldgate, group_rows, sigmoid, layer, residual_scale, eps,
                                post_gamma, post_beta, pre_gamma, pre_beta)
  h, z = x.float().reshape(-1, c), None
  out = x
  if y is not None:
    n = y.float().reshape(-1, c)
    if post_gamma is not None:
      n = _normalised(n, layer, eps)[0] * post_gamma
      n = n if post_beta is None else n + post_beta
    if gate is not None:
      n = n * _gate_factor(gate, rows, c, group_rows, sigmoid)[0]
    h = h + residual_scale * n
    out = h.to(x.dtype).view(x.shape)
  if pre_gamma is not None:
    z = _normalised(h, layer, eps)[0] * pre_gamma
    z = (z if pre_beta is None else z + pre_beta).to(x.dtype).view(x.shape)
  return out, z


def residual_norm_grad(dh: Optional[torch.Tensor], dz: Optional[torch.Tensor], h: torch.Tensor,
                       y: Optional[torch.Tensor] = None, *, post_gamma=None, post_beta=None, gate=None,
                       gate_act: str = "none", residual_scale: float = 1.0, pre_gamma=None, pre_beta=None,
                       norm: str = "rms", eps: float = 1e-6) -> Dict[str, Optional[torch.Tensor]]:
  """Gradient of `residual_norm` at its result h and its input y (x is not needed).

  `dh`: gradient of h from its other uses (None: there are none), `dz`: gradient of z (given exactly when pre_gamma
  is).  Returns a dict of dx, dy (the type of h), dgate (the type and shape of gate; a row of a [groups, channels] gate sums
  over its rows), dpost_gamma, dpost_beta, dpre_gamma, dpre_beta (float32 [channels]), None for what was not
  given.  The norms' statistics are taken from h and y again, so nothing has to be kept from the forward call.
  Sums over rows run in a fixed order, float32 within the few rows that one place on the grid adds up and 64 bits
  beyond: the same call gives the same bits.
  """
  rows, c, group_rows, ldgate, sigmoid, layer = _seam(h, y, post_gamma, post_beta, gate, gate_act, pre_gamma, pre_beta,
                                                      norm, eps)
  _no_graph(dh, dz, h, y, post_gamma, post_beta, gate, pre_gamma, pre_beta)
  if (dz is None) != (pre_gamma is None):
    raise ValueError("dz goes with pre_gamma")
  if dz is None and dh is None:
    raise ValueError("neither dh nor dz")
  shape, dtype, device = h.shape, h.dtype, h.get_device()
  ldh = _row_pitch("h", h, c)
  lddh = c if dh is None else _pitch("dh", dh, c, shape, dtype, device)
  lddz = c if dz is None else _pitch("dz", dz, c, shape, dtype, device)
  ldy = c if y is None else _pitch("y", y, c, shape, dtype, device)
  if h.is_cuda:
    if c > MAX_CHANNELS:
      raise ValueError("at most %d channels, got %d" % (MAX_CHANNELS, c))
    from . import native  # pylint: disable=import-outside-toplevel
    return native.residual_norm_grad(dh, lddh, dz, lddz, h, ldh, y, ldy, rows, c, gate, ldgate, group_rows, sigmoid,
                                     layer, residual_scale, eps, post_gamma, post_beta, pre_gamma, pre_beta)
  out: Dict[str, Optional[torch.Tensor]] = dict.fromkeys(
      ("dx", "dy", "dgate", "dpost_gamma", "dpost_beta", "dpre_gamma", "dpre_beta"))
  up = dh.float().reshape(-1, c) if dh is not None else torch.zeros(rows, c)
  if dz is not None:
    d = dz.float().reshape(-1, c)
    hat, r = _normalised(h.float().reshape(-1, c), layer, eps)
    out["dpre_gamma"] = (d * hat).sum(0)
    if pre_beta is not None:
      out["dpre_beta"] = d.sum(0)
    up = up + _normalised_grad(d * pre_gamma, hat, r, layer)
  out["dx"] = up.to(h.dtype).view(h.shape)
  if y is None:
    return out
  up = residual_scale * up
  n = y.float().reshape(-1, c)
  if post_gamma is not None:
    hat, r = _normalised(n, layer, eps)
    n = hat * post_gamma
    n = n if post_beta is None else n + post_beta
  if gate is not None:
    a, slope = _gate_factor(gate, rows, c, group_rows, sigmoid)
    dg = up * n * slope
    if group_rows or not rows:
      dg = dg.view(gate.numel() // c, -1, c).sum(1) if rows else torch.zeros(gate.shape)
    out["dgate"] = dg.to(gate.dtype).view(gate.shape)
    up = up * a
  if post_gamma is not None:
    out["dpost_gamma"] = (up * hat).sum(0)
    if post_beta is not None:
      out["dpost_beta"] = up.sum(0)
    up = _normalised_grad(up * post_gamma, hat, r, layer)
  out["dy"] = up.to(h.dtype).view(h.shape)
  return out


# ---- the norm over all gradients -------------------------------------------------------------------

def _overlaps(spans) -> bool:
  spans = sorted(s for s in spans if s[0] != s[1])
  return any(a[1] > b[0] for a, b in zip(spans, spans[1:]))


def _span(t: torch.Tensor):
  return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class TensorTable:
  """A list of tensors as `global_norm` and `clip_by_global_norm` walk it, built once for gradients that live in the
  same buffers step after step (a plan, like the launch plan of a training step).

  `out`: where clipped tensors go, a list of the same shapes and types (the tensors themselves: in place); without
  it they are clipped in place.  The table keeps the tensors alive and follows them: one whose storage, length, type or
  layout was exchanged since is looked up again, and checked again, by the next call.  Keep the table itself for as long
  as a graph that was captured with it.  Contiguous bfloat16, float16 or float32 tensors of one device; outputs may not
  overlap each other, nor any input but their own.
  """

  def __init__(self, tensors: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None, *, _kept=True):
    self._kept = _kept
    self.tensors = list(tensors)
    self.out = self.tensors if out is None else list(out)
    if not self.tensors:
      raise ValueError("an empty list of tensors")
    if len(self.out) != len(self.tensors):
      raise ValueError("%d outputs for %d tensors" % (len(self.out), len(self.tensors)))
    self.device = self.tensors[0].device
    self.held = []          # device tables that a captured graph reads, now and after an exchange of storages
    self._build(self._kept)

  def _build(self, upload):
    for i, (t, o) in enumerate(zip(self.tensors, self.out)):
      if t.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("tensor %d: element type %s (bfloat16, float16 and float32 are built)" % (i, t.dtype))
      if t.device != self.device or o.device != self.device:
        raise ValueError("tensor %d: the list lives on %s" % (i, self.device))
      if not t.is_contiguous() or not o.is_contiguous():
        raise ValueError("tensor %d is not contiguous" % i)
      if o.shape != t.shape or o.dtype != t.dtype:
        raise ValueError("output %d: %s %s for %s %s" % (i, tuple(o.shape), o.dtype, tuple(t.shape), t.dtype))
    at = [t.data_ptr() for t in self.tensors]
    to = at if self.out is self.tensors else [o.data_ptr() for o in self.out]
    # refused by clip_by_global_norm alone: a norm may count a tensor twice
    outs = self._out_spans = [_span(o) for o in self.out]
    apart = [_span(t) for t, o in zip(self.tensors, self.out) if t.data_ptr() != o.data_ptr()]
    self._clash = _overlaps(outs) or (bool(apart) and _overlaps_two(outs, apart))
    # native: the launches, the doubles they need, their table in device memory and the stream it was written on
    self.list, self.workspace, self.resident, self.stream = None, 0, None, 0
    self._upload_due = False
    if self.device.type == "cuda":
      from . import native  # pylint: disable=import-outside-toplevel
      native.clip_list_build(self, at, to)
      self._upload_due = self._kept and self.list.pieces > 1
      if upload:
        self._upload()
    # last: a build that raises leaves the table as changed as it found it
    self._keys = [self._keys_of(ts) for ts in self._lists()] if self._kept else None

  def _lists(self):
    return (self.tensors,) if self.out is self.tensors else (self.tensors, self.out)

  def _keys_of(self, tensors):
    """What the launches depend on of every tensor: address, length, type, order of its elements."""
    if self.device.type == "cuda":
      from . import native  # pylint: disable=import-outside-toplevel
      keys = native.ext().tensor_keys(tensors)
      if keys is not None:
        return keys
    return _Keys(tensors)

  def _upload(self):
    from . import native  # pylint: disable=import-outside-toplevel
    self._upload_due = self._upload_due and not native.clip_list_upload(self)

  def _current(self) -> "TensorTable":
    # a list that changed is walked from launch arguments; its table goes to the device once a call finds it unchanged,
    # so that storages that are exchanged at every step neither pile up tables nor wait for their upload
    if not all(k.same(ts) for k, ts in zip(self._keys, self._lists())):
      self._build(upload=False)
    elif self._upload_due:
      self._upload()
    return self


class _Keys:
  """Keys of a list of tensors by their attributes (`TensorKeys` of the native extension is the fast form)."""

  def __init__(self, tensors):
    self._keys = self._read(tensors)

  @staticmethod
  def _read(tensors):
    return [(t.data_ptr(), t.numel(), t.dtype, t.is_contiguous()) for t in tensors]

  def same(self, tensors) -> bool:
    return self._keys == self._read(tensors)


def _overlaps_two(a, b) -> bool:
  """Whether a span of `a` overlaps one of `b` (the spans of each list apart from one another, or not)."""
  events = sorted([(s[0], s[1], 0) for s in a if s[0] != s[1]] + [(s[0], s[1], 1) for s in b if s[0] != s[1]])
  ends = [0, 0]
  for lo, hi, which in events:
    if ends[1 - which] > lo:
      return True
    ends[which] = max(ends[which], hi)
  return False


def _table(tensors) -> TensorTable:
  if isinstance(tensors, TensorTable):
    return tensors._current()
  if isinstance(tensors, torch.Tensor):
    raise ValueError("a list of tensors (or a TensorTable), not a tensor")
  return TensorTable(tensors, _kept=False)


def _squares(tensors) -> torch.Tensor:
  return torch.stack([t.detach().double().square().sum() for t in tensors]).sum()


def global_norm(tensors) -> torch.Tensor:
  """sqrt of the sum of squares over all tensors of a list or `TensorTable`: a float32 scalar on their device.

  Squares are summed in 64 bits in a fixed order; nothing is read back to the host, and no graph is recorded.
  """
  t = _table(tensors)
  _no_tangent(t.tensors)
  if t.device.type != "cuda":
    return _squares(t.tensors).sqrt().float()
  from . import native  # pylint: disable=import-outside-toplevel
  return native.clip_list_norm(t)


def clip_by_global_norm(tensors, clip_norm: float, use_norm: Optional[torch.Tensor] = None, out=None):
  """Scales all tensors by min(1, clip_norm / norm) of their global norm, as tf.clip_by_global_norm does; returns
  (list of clipped tensors, norm).

  `tensors`: a list, clipped into new tensors or into `out` (a list of the same shapes and types; the list itself:
  in place), or a `TensorTable`, which brings its own.  `use_norm`: a float32 scalar on the device that takes the
  place of the norm (of a model whose gradients are spread over processes).  A norm that is infinite or NaN makes
  every result NaN; a norm of zero changes nothing.  Nothing is read back to the host, and no graph is recorded.
  """
  clip_norm = float(clip_norm)
  if not clip_norm > 0:
    raise ValueError("clip_norm has to be positive, got %r" % clip_norm)
  if isinstance(tensors, TensorTable):
    if out is not None:
      raise ValueError("a TensorTable brings its own outputs")
    t = tensors._current()
  else:
    tensors = list(tensors)
    t = TensorTable(tensors, [torch.empty_like(x, memory_format=torch.contiguous_format) for x in tensors]
                    if out is None else out, _kept=False)
  _no_tangent(t.tensors, t.out, (use_norm,))
  if t._clash:
    raise ValueError("outputs overlap each other, or another tensor's input")
  if use_norm is not None and (use_norm.dtype != torch.float32 or use_norm.numel() != 1
                               or use_norm.device != t.device):
    raise ValueError("use_norm: a float32 scalar on %s" % t.device)
  if use_norm is not None and any(lo <= use_norm.data_ptr() < hi for lo, hi in t._out_spans):
    raise ValueError("use_norm lies in an output: it is read while outputs are written")
  if t.device.type == "cuda":
    from . import native  # pylint: disable=import-outside-toplevel
    return list(t.out), native.clip_list_scale(t, clip_norm, use_norm)
  with torch.no_grad():
    norm = _squares(t.tensors).sqrt() if use_norm is None else use_norm.double().reshape(())
    factor = torch.clamp(clip_norm / norm, max=1.0) if bool(torch.isfinite(norm)) else norm * float("nan")
    for x, o in zip(t.tensors, t.out):
      o.copy_(x.float() * factor.float())
  return list(t.out), norm.float() if use_norm is None else use_norm


def clipped_sgd_momentum_l2(params: torch.Tensor, grads: torch.Tensor, velocity: torch.Tensor, l2x2: torch.Tensor,
                            lr: float, momentum: float, clip_norm: float, grad_scale: float = 1.0,
                            skip=None) -> torch.Tensor:
  """`sgd_momentum_l2` with the gradient clipped to `clip_norm` by its global norm, in place; returns that norm (a
  float32 scalar on the device, before clipping).

      g  = grads * grad_scale + l2x2 * params
      g <- g * min(1, clip_norm / |g|)
      v <- momentum * v - lr * g
      w <- w + v

  The norm is that of the whole gradient, the regulariser's part included.  `skip` as in `sgd_momentum_l2`: with a
  flag that is set nothing is updated.  A norm that is not finite, without `skip`, makes parameters and velocity NaN.
  """
  _no_tangent((params, grads, velocity, l2x2))
  n = params.numel()
  for name, t in (("params", params), ("grads", grads), ("velocity", velocity), ("l2x2", l2x2)):
    if t.dtype != torch.float32 or not t.is_contiguous() or t.device != params.device:
      raise ValueError("clipped_sgd_momentum_l2 wants contiguous fp32 tensors on one device (%s)" % name)
    if t.numel() != n and (name != "velocity" or momentum):
      raise ValueError("clipped_sgd_momentum_l2: buffer sizes differ")
  if n == 0:
    raise ValueError("clipped_sgd_momentum_l2: no parameters")
  if not clip_norm > 0:
    raise ValueError("clip_norm has to be positive, got %r" % clip_norm)
  at = sorted([params.data_ptr(), grads.data_ptr(), l2x2.data_ptr()] + ([velocity.data_ptr()] if momentum else []))
  if min(b - a for a, b in zip(at, at[1:])) < 4 * n:
    raise ValueError("clipped_sgd_momentum_l2: buffers overlap")
  if skip is not None and (skip.dtype != torch.float32 or skip.numel() < 2 or skip.device != params.device
                           or not skip.is_contiguous()):
    raise ValueError("skip: two contiguous float32 values on %s" % params.device)
  if skip is not None and any(lo - 8 < skip.data_ptr() < lo + 4 * n
                              for lo in [params.data_ptr()] + ([velocity.data_ptr()] if momentum else [])):
    raise ValueError("skip lies in a buffer that is updated: it is read while that is written")
  if params.device.type == "cuda":
    from . import native  # pylint: disable=import-outside-toplevel
    return native.clipped_sgd_momentum_l2(params, grads, velocity, l2x2, lr, momentum, clip_norm, grad_scale, skip)
  if skip is not None:
    raise ValueError("a device-side skip flag needs the native optimizer kernel")
  with torch.no_grad():
    g = torch.addcmul(grads * grad_scale, l2x2, params)
    norm = g.double().square().sum().sqrt()
    factor = float(torch.clamp(clip_norm / norm, max=1.0)) if bool(torch.isfinite(norm)) else float("nan")
    if momentum:
      velocity.mul_(momentum).add_(g, alpha=-lr * factor)
      params.add_(velocity)
    else:
      params.add_(g, alpha=-lr * factor)
  return norm.float()
