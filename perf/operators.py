"""Operators next to the training step, as cases that can be timed and compared.

Four operators in two pairs:

* `residual_norm` / `residual_norm_grad`: the seam between two residual blocks.  The block's output is
  normalised, gated, scaled and added to the residual stream, and the sum is normalised for the next block;
  the gradient of the same.  Rows are pixels of an NHWC activation or tokens, columns are channels.
* `clip_by_global_norm` / `clipped_sgd_momentum_l2`: the norm over all gradients of a model and what is done
  with it - gradients scaled down to it, or the momentum update with the scaled gradients.

`run` computes a case with elementary torch operations in 32 bits (64 for long sums) or, where `own` is set,
through `distributed_tensorflow_amd.ops.fused`.  `exact` is the definition in 64 bits.
"""
import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
LR, MOMENTUM = 0.1, 0.9


def listed():
  return [
      # one token through the seam of a served model: a gate of its own per channel, nothing but latency
      dict(name="norm_one_token", op="norm", rows=1, channels=4096, dtype="bf16", norm="rms", post=True, pre=True,
           groups=-1, act="sigmoid", scale=1.0),
      # last stage of ResNet-50 at batch 256 (7x7 pixels): per-pixel LayerNorm and a learnt scale per channel
      dict(name="norm_stage5_layer", op="norm", rows=12544, channels=2048, dtype="bf16", norm="layer", post=False,
           pre=True, groups=1, act="none", scale=1.0),
      # as many channels as the ImageNet head has classes, a prime number of rows: nothing divides or aligns
      dict(name="norm_odd", op="norm", rows=4099, channels=1001, dtype="fp16", norm="rms", post=True, pre=True,
           groups=-1, act="none", scale=0.5),
      # second stage of ResNet-50 at batch 256 (28x28 pixels): a gate per image (conditioning, dropped paths)
      dict(name="norm_stage3_per_image", op="norm", rows=200704, channels=512, dtype="bf16", norm="rms", post=True,
           pre=True, groups=256, act="none", scale=0.7),
      # a batch of pooled features: a training step that is bound by launches
      dict(name="grad_small_fp32", op="norm_grad", rows=128, channels=1000, dtype="fp32", norm="layer", post=True,
           pre=True, groups=1, act="none", scale=1.0),
      # first stage of the CIFAR ResNets at batch 128: rows of 64 bytes
      dict(name="grad_cifar_narrow", op="norm_grad", rows=131072, channels=16, dtype="fp32", norm="layer", post=False,
           pre=True, groups=1, act="none", scale=1.0),
      # last stage of ResNet-50 at batch 256, a gate per image
      dict(name="grad_stage5_per_image", op="norm_grad", rows=12544, channels=2048, dtype="bf16", norm="rms",
           post=True, pre=True, groups=256, act="none", scale=0.7),
      # the largest: a sigmoid gate per element, all of whose gradient is written
      dict(name="grad_stage3_element", op="norm_grad", rows=200704, channels=512, dtype="bf16", norm="rms", post=True,
           pre=True, groups=-1, act="sigmoid", scale=1.0),
      # the gradients of ResNet-50: 161 variables
      dict(name="clip_resnet50", op="clip", tensors=161, elements=25_600_000, dtype="fp32", clip=1.0),
      # a large model with 16-bit weights whose norms and embeddings stay in 32 bits
      dict(name="clip_large_mixed", op="clip", tensors=384, elements=400_000_000, dtype="mixed", clip=1.0),
      # ResNet-20: the whole update is a few microseconds
      dict(name="update_resnet20", op="update", elements=272_474, clip=1.0, grad_scale=1.0),
      # ResNet-50, gradients summed over eight replicas
      dict(name="update_resnet50", op="update", elements=25_610_152, clip=1.0, grad_scale=0.125),
  ]


def _log(rng, lo, hi):
  return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
  op = rng.choice(["norm", "norm_grad", "norm", "norm_grad", "clip", "update"])
  if op == "clip":
    return dict(op=op, tensors=rng.randint(1, 400), elements=_log(rng, 1000, 300_000_000),
                dtype=rng.choice(["fp32", "bf16", "fp16", "mixed"]), clip=rng.choice([0.01, 1.0, 1e6]))
  if op == "update":
    return dict(op=op, elements=_log(rng, 1000, 60_000_000), clip=rng.choice([0.01, 1.0, 1e6]),
                grad_scale=rng.choice([1.0, 0.125]))
  channels = _log(rng, 16, 8192)
  if rng.random() < 0.5:
    channels = max(16, channels // 8 * 8)
  rows = _log(rng, 1, min(200_704, 100_000_000 // channels))
  groups = rng.choice([-1, -1, 0, 1, 2])
  if groups == 2:
    per = max(1, min(rows, _log(rng, 4, 1024)))
    groups = max(1, rows // per)
    rows = groups * per
  return dict(op=op, rows=rows, channels=channels, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
              norm=rng.choice(["rms", "layer"]), post=rng.random() < 0.7, pre=rng.random() < 0.85, groups=groups,
              act=rng.choice(["none", "sigmoid"]) if groups else "none", scale=rng.choice([1.0, 0.22, 0.7]))


def _sizes(case):
  """Elements per tensor: a third are vectors (scales, offsets), the others spread over a factor of a thousand."""
  n, total = case["tensors"], case["elements"]
  r = np.random.RandomState(n * 7919 + total % 65537)
  share = np.exp(r.uniform(0, np.log(1000.0), n))
  vector = r.uniform(size=n) < 1 / 3
  sizes = np.maximum(1, (share / share.sum() * total)).astype(np.int64)
  sizes[vector] = np.minimum(sizes[vector], r.randint(1, 4097, n)[vector])
  sizes[n - 1] = max(1, total - int(sizes[:-1].sum()))
  small = (sizes <= 4096).tolist()
  kinds = [("fp32" if s else "bf16") if case["dtype"] == "mixed" else case["dtype"] for s in small]
  return sizes.tolist(), kinds


def _randn(gen, *shape):
  return torch.randn(*shape, generator=gen, device=gen.device)


def _device():
  return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _inputs(case, seed):
  gen = torch.Generator(device=_device())
  gen.manual_seed(int(seed))
  s = dict(case)
  if case["op"] in ("norm", "norm_grad"):
    rows, channels, dt = case["rows"], case["channels"], DTYPES[case["dtype"]]
    loud = 1.0 + 7.0 * (torch.rand(channels, generator=gen, device=gen.device) < 0.01)   # a few loud channels
    s["x"] = (_randn(gen, rows, channels) * loud).to(dt)
    s["y"] = (_randn(gen, rows, channels) * 0.8 + 0.1).to(dt)
    layer = case["norm"] == "layer"
    for side in ("post", "pre"):
      if case[side]:
        s[side + "_gamma"] = 1.0 + 0.2 * _randn(gen, channels)
        if layer:
          s[side + "_beta"] = 0.1 * _randn(gen, channels)
    if case["groups"] == -1:
      s["gate"] = _randn(gen, rows, channels).to(dt)
    elif case["groups"] > 0:
      s["gate"] = 0.5 + 0.3 * _randn(gen, case["groups"], channels)
    if case["op"] == "norm_grad":
      s["h"] = s.pop("x")
      s["dh"] = (_randn(gen, rows, channels) * 0.02).to(dt)
      if case["pre"]:
        s["dz"] = (_randn(gen, rows, channels) * 0.05).to(dt)
  elif case["op"] == "clip":
    sizes, kinds = _sizes(case)
    s["grads"] = [(_randn(gen, n) * 10.0 ** (-3 + 2 * (i % 7) / 6)).to(DTYPES[k])
                  for i, (n, k) in enumerate(zip(sizes, kinds))]
  else:
    n = case["elements"]
    s["params"] = _randn(gen, n) * 0.05
    s["grads"] = _randn(gen, n) * 0.01
    s["velocity"] = _randn(gen, n) * 0.001
    # weight decay on the matrices, none on the scales and offsets between them
    s["l2x2"] = 2e-4 * ((torch.arange(n, device=gen.device) // 256) % 16 != 0)
  return s


def prepare(case, seed):
  s = _inputs(case, seed)
  if case["op"] == "clip":
    # clipped gradients go to flat buffers, one per type, every tensor at a 16-byte boundary of its own
    s["flats"], s["out"] = {}, [None] * len(s["grads"])
    for dt in sorted({g.dtype for g in s["grads"]}, key=str):
      mine = [i for i, g in enumerate(s["grads"]) if g.dtype == dt]
      room = [-(-s["grads"][i].numel() // 8) * 8 for i in mine]
      flat = torch.zeros(sum(room), dtype=dt, device=_device())
      s["flats"][str(dt)] = flat
      at = 0
      for i, r in zip(mine, room):
        s["out"][i] = flat[at:at + s["grads"][i].numel()]
        at += r
    if own:
      from distributed_tensorflow_amd.ops import fused
      s["table"] = fused.TensorTable(s["grads"], out=s["out"])     # built once, like a launch plan
  return s


def _present(d):
  return {k: v for k, v in d.items() if v is not None}


_SEAM = ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")


def _grouped(s, v):
  """[rows, channels] as [groups, rows of a group, channels], in 32 bits."""
  groups = s["groups"] if s["groups"] > 0 else s["rows"] if s["groups"] == -1 else 1
  return v.float().view(groups, s["rows"] // groups, s["channels"])


def _hat(v, s):
  """The normalised rows and what they were multiplied with."""
  if s["norm"] == "layer":
    v = v - v.mean(-1, keepdim=True)
  r = 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
  return v * r, r


def _affine(v, gamma, beta):
  v = v * gamma
  return v if beta is None else v + beta


def _hat_back(d, hat, r, s):
  t = d - hat * (d * hat).mean(-1, keepdim=True)
  if s["norm"] == "layer":
    t = t - d.mean(-1, keepdim=True)
  return r * t


def _gate_value(s):
  """The gate's factor and its derivative, [groups, 1, channels]."""
  if "gate" not in s:
    return 1.0, 0.0
  g = s["gate"].float().unsqueeze(1)
  if s["act"] == "sigmoid":
    a = 1.0 / (1.0 + torch.exp(-g))
    return a, a * (1.0 - a)
  return g, 1.0


def _plain_norm(s):
  dt = s["x"].dtype
  n = _grouped(s, s["y"])
  if s["post"]:
    n = _affine(_hat(n, s)[0], s["post_gamma"], s.get("post_beta"))
  h = _grouped(s, s["x"]) + s["scale"] * (_gate_value(s)[0] * n)
  out = {"h": h.to(dt).view(s["rows"], -1)}
  if s["pre"]:
    out["z"] = _affine(_hat(h, s)[0], s["pre_gamma"], s.get("pre_beta")).to(dt).view(s["rows"], -1)
  return out


def _over_rows(v, dims):
  return v.sum(dims, dtype=torch.float64).float()


def _plain_norm_grad(s):
  dt, out = s["h"].dtype, {}
  up = _grouped(s, s["dh"])
  if s["pre"]:
    dz, (hat, r) = _grouped(s, s["dz"]), _hat(_grouped(s, s["h"]), s)
    out["dpre_gamma"] = _over_rows(dz * hat, (0, 1))
    if "pre_beta" in s:
      out["dpre_beta"] = _over_rows(dz, (0, 1))
    up = up + _hat_back(dz * s["pre_gamma"], hat, r, s)
  out["dx"] = up.to(dt).view(s["rows"], -1)
  up = s["scale"] * up
  n = _grouped(s, s["y"])
  if s["post"]:
    hat, r = _hat(n, s)
    n = _affine(hat, s["post_gamma"], s.get("post_beta"))
  a, slope = _gate_value(s)
  if s["groups"] == -1:
    out["dgate"] = (up * n * slope).to(dt).view(s["rows"], -1)
  elif s["groups"] > 0:
    out["dgate"] = (_over_rows(up * n, 1) * (slope if isinstance(slope, float) else slope.squeeze(1)))
  up = up * a
  if s["post"]:
    out["dpost_gamma"] = _over_rows(up * hat, (0, 1))
    if "post_beta" in s:
      out["dpost_beta"] = _over_rows(up, (0, 1))
    up = _hat_back(up * s["post_gamma"], hat, r, s)
  out["dy"] = up.to(dt).view(s["rows"], -1)
  return out


def _factor(squares, clip):
  norm = torch.sqrt(squares)
  return norm.float(), torch.clamp(clip / norm, max=1.0).float()


def _plain_clip(s):
  norm, f = _factor(torch.stack([g.double().square().sum() for g in s["grads"]]).sum(), s["clip"])
  _ = [o.copy_(g.float() * f) for o, g in zip(s["out"], s["grads"])]
  return [*s["flats"].values(), norm]


def _plain_update(s):
  g = s["grads"] * s["grad_scale"] + s["l2x2"] * s["params"]
  norm, f = _factor(g.double().square().sum(), s["clip"])
  s["velocity"].mul_(MOMENTUM).sub_(g * f * LR)
  s["params"].add_(s["velocity"])
  return [s["params"], s["velocity"], norm]


def run(state):
  s = state
  if not own:
    return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "clip": _plain_clip, "update": _plain_update}[s["op"]](s)
  from distributed_tensorflow_amd.ops import fused
  if s["op"] == "clip":
    _, norm = fused.clip_by_global_norm(s["table"], s["clip"])
    return [*s["flats"].values(), norm]
  if s["op"] == "update":
    norm = fused.clipped_sgd_momentum_l2(s["params"], s["grads"], s["velocity"], s["l2x2"], LR, MOMENTUM, s["clip"],
                                         grad_scale=s["grad_scale"])
    return [s["params"], s["velocity"], norm]
  seam = dict(norm=s["norm"], eps=EPS, gate_act=s["act"], residual_scale=s["scale"],
              **{k: s[k] for k in _SEAM if k in s})
  if s["op"] == "norm":
    h, z = fused.residual_norm(s["x"], s["y"], **seam)
    return _present(dict(h=h, z=z))
  return _present(fused.residual_norm_grad(s["dh"], s.get("dz"), s["h"], s["y"], **seam))


def work(case):
  if case["op"] == "clip":
    sizes, kinds = _sizes(case)
    size = sum(n * (4 if k == "fp32" else 2) for n, k in zip(sizes, kinds))
    return {"bytes": 2 * size, "flops": 3 * sum(sizes)}
  if case["op"] == "update":
    return {"bytes": 6 * 4 * case["elements"], "flops": 10 * case["elements"]}
  item, n = (4 if case["dtype"] == "fp32" else 2), case["rows"] * case["channels"]
  small = 4 * case["channels"]
  vectors = small * (case["post"] + case["pre"]) * (2 if case["norm"] == "layer" else 1) + small * max(case["groups"], 0)
  element = case["groups"] == -1
  if case["op"] == "norm":
    return {"bytes": n * item * (3 + case["pre"] + element) + vectors, "flops": n * (4 + 5 * (case["post"] + case["pre"]))}
  # read: dh, y and, where the sum was normalised, h and dz; written: dx, dy; the gate read and its gradient written
  return {"bytes": n * item * (4 + 2 * case["pre"] + 2 * element) + 2 * vectors,
          "flops": n * (6 + 12 * (case["post"] + case["pre"]))}


def _definition(s, x, y, p):
  """The seam as its definition has it, for 64-bit inputs (differentiable)."""
  def norm(v, gamma, beta):
    if s["norm"] == "layer":
      var, mean = torch.var_mean(v, dim=1, keepdim=True, correction=0)
    else:
      var, mean = v.pow(2).mean(1, keepdim=True), 0.0
    v = (v - mean) * (var + EPS).rsqrt() * gamma
    return v if beta is None else v + beta

  n = norm(y, p["post_gamma"], p.get("post_beta")) if s["post"] else y
  if "gate" in p:
    g = torch.sigmoid(p["gate"]) if s["act"] == "sigmoid" else p["gate"]
    n = n * g.repeat_interleave(s["rows"] // g.shape[0], 0)
  h = x + s["scale"] * n
  return h, norm(h, p["pre_gamma"], p.get("pre_beta")) if s["pre"] else None


def exact(case, seed):
  s = _inputs(case, seed)
  if case["op"] == "clip":
    norm = torch.linalg.vector_norm(torch.cat([g.double() for g in s["grads"]]))
    f = min(1.0, case["clip"] / float(norm))
    flats = {}
    for g in s["grads"]:
      flats.setdefault(str(g.dtype), []).append(torch.nn.functional.pad(g.double() * f, (0, -g.numel() % 8)))
    return [*(torch.cat(flats[k]) for k in sorted(flats)), norm]
  if case["op"] == "update":
    p, v = s["params"].double(), s["velocity"].double()
    g = s["grads"].double() * case["grad_scale"] + s["l2x2"].double() * p
    norm = torch.linalg.vector_norm(g)
    v = MOMENTUM * v - LR * g * min(1.0, case["clip"] / float(norm))
    return [p + v, v, norm]
  p = {k: s[k].double() for k in _SEAM if k in s}
  if case["op"] == "norm":
    h, z = _definition(s, s["x"].double(), s["y"].double(), p)
    return _present(dict(h=h, z=z))
  # the gradient by differentiating the definition at the x that gives this h
  y = s["y"].double()
  with torch.no_grad():
    x = s["h"].double() - _definition({**s, "pre": False}, 0.0, y, p)[0]
  for t in (x, y, *p.values()):
    t.requires_grad_(True)
  h, z = _definition(s, x, y, p)
  total = (h * s["dh"].double()).sum()
  if z is not None:
    total = total + (z * s["dz"].double()).sum()
  names = ["x", "y", *p]
  return {"d" + k: g for k, g in zip(names, torch.autograd.grad(total, [x, y, *p.values()]))}
