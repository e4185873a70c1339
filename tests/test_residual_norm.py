"""The seam between two residual blocks and its gradient against the definition in 64 bits.

Bounds.  U = 2^-24 is half a step of fp32, `half_step(t)` half a step of the result's type.  A result may be off by
half a step of its own type (its one rounding) plus A * U * M, where M bounds the magnitudes that are added up on the
way to it and A counts fp32 roundings: a sum over a row has at most 16 serial additions in a lane, 6 butterfly steps and 8
waves (30); a normalised value sees the mean's sum (30), half of the sum of squares' error (15), a square root, a division,
a centring and two products (5), and what its input carries (the h of the seam: 5 more, after y's own normalisation) - under
128 in all.  A gradient sees two such sums on top of each normalised value: under 256.  Errors of a first normalisation
that pass through a second one are carried along explicitly.
"""
import itertools

import pytest
import torch

from distributed_tensorflow_amd.ops import fused

U = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
VECTORS = ("post_gamma", "post_beta", "pre_gamma", "pre_beta")


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def make(dev, rows, channels, dtype, norm, post=True, pre=True, gate="none", groups=1, seed=0, offset=0.3):
  gen = torch.Generator().manual_seed(seed + rows * 131 + channels)
  r = lambda *s: torch.randn(*s, generator=gen)
  t = dict(x=(r(rows, channels) * 2 + offset).to(dtype), y=(r(rows, channels) + offset).to(dtype),
           dh=(r(rows, channels) * 0.1).to(dtype), dz=(r(rows, channels) * 0.1).to(dtype))
  kw = dict(norm=norm, eps=1e-5, residual_scale=0.7)
  for side, on in (("post", post), ("pre", pre)):
    if on:
      kw[side + "_gamma"] = 1 + 0.3 * r(channels)
      if norm == "layer":
        kw[side + "_beta"] = 0.2 * r(channels)
  if gate == "element":
    kw["gate"] = r(rows, channels).to(dtype)
  elif gate == "group":
    kw["gate"] = r(groups, channels)
  kw = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
  return {k: v.to(dev) for k, v in t.items()}, kw


def norm64(v, gamma, beta, norm, eps):
  mean = v.mean(-1, keepdim=True) if norm == "layer" else 0.0
  r = ((v - mean).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
  out = (v - mean) * r * gamma
  return (out if beta is None else out + beta), r


def seam64(x, y, kw):
  """(h, z) of the definition, in the type of its arguments (64 bits)."""
  n = y
  if n is not None:
    if "post_gamma" in kw:
      n = norm64(y, kw["post_gamma"], kw.get("post_beta"), kw["norm"], kw["eps"])[0]
    g = kw.get("gate")
    if g is not None:
      g = torch.sigmoid(g) if kw.get("gate_act") == "sigmoid" else g
      if g.dim() == 1:
        g = g[None]
      n = n * g.repeat_interleave(x.shape[0] // max(g.shape[0], 1), 0) if g.shape[0] else n * g
    x = x + kw["residual_scale"] * n
  z = norm64(x, kw["pre_gamma"], kw.get("pre_beta"), kw["norm"], kw["eps"])[0] if "pre_gamma" in kw else None
  return x, z


def to64(kw):
  return {k: v.double().cpu() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}


def row_max(v):
  return v.abs().amax(-1, keepdim=True) if v.numel() else v.abs()


def check_forward(t, kw, h, z):
  dtype = t["x"].dtype
  x, y, k = t["x"].double().cpu(), t["y"].double().cpu(), to64(kw)
  h64, z64 = seam64(x, y, k)
  n = y
  growth = 1.0
  if "post_gamma" in k:
    n, r = norm64(y, k["post_gamma"], k.get("post_beta"), k["norm"], k["eps"])
    growth = row_max(y) * r * k["post_gamma"].abs().max() + (k["post_beta"].abs().max() if "post_beta" in k else 0)
  g = k.get("gate")
  gmax = 1.0 if g is None or kw.get("gate_act") == "sigmoid" else g.abs().max()
  m_h = row_max(x) + k["residual_scale"] * gmax * (row_max(n) + growth)
  off_h = 128 * U * m_h
  diff = (h.double().cpu() - h64).abs()
  assert h.dtype == dtype and h.shape == t["x"].shape
  assert (diff <= half_step(dtype) * h64.abs() * (1 + 1e-6) + off_h + torch.finfo(dtype).tiny).all(), diff.max()
  assert (z is None) == ("pre_gamma" not in k)
  if z is not None:
    _, r = norm64(h64, k["pre_gamma"], None, k["norm"], k["eps"])
    gain = r * k["pre_gamma"].abs().max()
    # an error of h shifts the normalised value by itself, through the mean and through the mean square
    off = gain * (2 + (row_max(h64) * r) ** 2) * off_h + 128 * U * (gain * row_max(h64) + 1)
    diff = (z.double().cpu() - z64).abs()
    assert z.dtype == dtype and z.shape == t["x"].shape
    assert (diff <= half_step(dtype) * z64.abs() * (1 + 1e-6) + off + torch.finfo(dtype).tiny).all(), diff.max()


def grads64(h, y, dh, dz, kw):
  """Gradients of <h, dh> + <z, dz> by differentiating the definition in 64 bits."""
  k = to64(kw)
  h, y = h.double().cpu(), None if y is None else y.double().cpu()
  with torch.no_grad():
    x = h - seam64(torch.zeros_like(h), y, {a: b for a, b in k.items() if not a.startswith("pre_")})[0]
  leaves = dict(x=x, **({} if y is None else dict(y=y)), **{n: v for n, v in k.items() if isinstance(v, torch.Tensor)})
  for v in leaves.values():
    v.requires_grad_(True)
  k.update({n: leaves[n] for n in leaves if n in k})
  h2, z2 = seam64(leaves["x"], leaves.get("y"), k)
  total = 0.0
  if dh is not None:
    total = total + (h2 * dh.double().cpu()).sum()
  if dz is not None:
    total = total + (z2 * dz.double().cpu()).sum()
  got = torch.autograd.grad(total, list(leaves.values()), allow_unused=True)
  return {"d" + n: torch.zeros_like(v) if g is None else g for (n, v), g in zip(leaves.items(), got)}


def check_grad(t, kw, out, use_dh=True):
  dtype = t["x"].dtype
  h, y, k = t["x"].double().cpu(), t["y"].double().cpu(), to64(kw)
  dh = t["dh"] if use_dh else None
  dz = t["dz"] if "pre_gamma" in kw else None
  ref = grads64(t["x"], t["y"], dh, dz, kw)
  assert {n for n, v in out.items() if v is not None} == set(ref)
  rows = h.shape[0]
  m_up = row_max(dh.double().cpu()) if use_dh else 0.0
  hat_h = None
  if dz is not None:
    one = torch.ones(h.shape[-1], dtype=torch.float64)
    hat_h, r = norm64(h, one, None, k["norm"], k["eps"])
    m_hat = row_max(h) * r                              # before centring: what the fp32 sums run over
    d = dz.double().cpu()
    m_up = m_up + r * row_max(d) * k["pre_gamma"].abs().max() * (2 + m_hat ** 2)
  off_up = 256 * U * m_up
  bound = {"dx": off_up}
  s, g = k["residual_scale"], k.get("gate")
  sig = kw.get("gate_act") == "sigmoid"
  gmax = 1.0 if g is None or sig else g.abs().max()
  m_n, m_haty, r_y, gam = row_max(y), row_max(y), 1.0, 1.0
  if "post_gamma" in k:
    one = torch.ones(h.shape[-1], dtype=torch.float64)
    _, r_y = norm64(y, one, None, k["norm"], k["eps"])
    m_haty = row_max(y) * r_y
    gam = k["post_gamma"].abs().max()
    m_n = m_haty * gam + (k["post_beta"].abs().max() if "post_beta" in k else 0)
    bound["dy"] = r_y * gam * gmax * s * (2 + m_haty ** 2) * (off_up + 256 * U * m_up)
  else:
    bound["dy"] = gmax * s * (off_up + 8 * U * m_up)
  term_gate = s * m_n * (off_up + 256 * U * m_up)
  # sums over rows: the terms' own errors, and as many roundings of the running sum as rows meet in one place
  depth = (64 + rows / 256) * U
  total = lambda v: (v if isinstance(v, torch.Tensor) else torch.tensor(v)).expand(rows, 1).sum()
  if g is not None:
    if kw["gate"].shape == t["x"].shape and kw["gate"].dtype == dtype:
      bound["dgate"] = term_gate
    else:
      groups = g.numel() // g.shape[-1]
      per = (term_gate + depth * s * m_n * m_up).expand(rows, 1).reshape(groups, -1).sum(1)
      if rows // groups <= 4 * 128:                     # a slot may add up a whole small group by itself
        per = per + (rows // groups) * U * (s * m_n * m_up).expand(rows, 1).reshape(groups, -1).sum(1)
      bound["dgate"] = per[:, None].expand(groups, g.shape[-1]).reshape(g.shape)
  if "post_gamma" in k:
    bound["dpost_gamma"] = total(gmax * s * m_haty * (off_up + (256 * U + depth) * m_up)) + rows * U
    bound["dpost_beta"] = total(gmax * s * (off_up + (8 * U + depth) * m_up)) + rows * U
  if dz is not None:
    bound["dpre_gamma"] = total(m_hat * row_max(d) * (128 * U + depth))
    bound["dpre_beta"] = total(row_max(d) * depth)
  for n, want in ref.items():
    got = out[n]
    is_vector = n[1:] in VECTORS
    like = torch.float32 if is_vector else kw["gate"].dtype if n == "dgate" else dtype
    assert got.dtype == like, n
    assert got.shape == want.shape, n
    diff = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all(), n
    limit = half_step(like) * want.abs() * (1 + 1e-6) + bound[n] + torch.finfo(like).smallest_normal
    assert (diff <= limit).all(), (n, diff.max(), (diff - limit).max())


CHANNELS = [1, 2, 7, 8, 16, 17, 31, 64, 100, 129, 256, 511, 512, 513, 1000, 1001, 2048, 4095, 4097, 5001, 8191, 8192]
SHAPES = [(1, c) for c in CHANNELS] + [(3, 16), (129, 16), (257, 40), (1000, 8), (67, 1001), (130, 512), (33, 8192),
                                       (1500, 33), (2500, 64)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("rows,channels", SHAPES)
def test_forward_and_gradient_by_shape(dev, dtype, norm, rows, channels):
  """Every row length class, both norms, all types; a gate per element."""
  t, kw = make(dev, rows, channels, dtype, norm, gate="element")
  check_forward(t, kw, *fused.residual_norm(t["x"], t["y"], **kw))
  check_grad(t, kw, fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("norm,post,pre", list(itertools.product(["rms", "layer"], [True, False], [True, False])))
@pytest.mark.parametrize("gate,act", [("none", "none"), ("element", "sigmoid"), ("group", "none"), ("group", "sigmoid")])
@pytest.mark.parametrize("rows,channels", [(60, 24), (36, 777)])
def test_every_combination(dev, dtype, norm, post, pre, gate, act, rows, channels):
  t, kw = make(dev, rows, channels, dtype, norm, post, pre, gate, groups=6)
  kw["gate_act"] = act
  check_forward(t, kw, *fused.residual_norm(t["x"], t["y"], **kw))
  check_grad(t, kw, fused.residual_norm_grad(t["dh"], t["dz"] if pre else None, t["x"], t["y"], **kw))
  if pre:      # the stream ends here: z is all that is used
    check_grad(t, kw, fused.residual_norm_grad(None, t["dz"], t["x"], t["y"], **kw), use_dh=False)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("rows,groups,channels", [
    (12, 12, 40), (1, 1, 16), (2000, 2000, 16), (2100, 1050, 24), (2048, 8, 16), (2048, 1, 16), (4000, 40, 100),
    (1300, 1300, 520), (2600, 1300, 520), (96, 3, 600), (97, 1, 600), (1024, 2, 4104), (30, 10, 512), (5000, 5, 300)])
@pytest.mark.parametrize("act", ["none", "sigmoid"])
def test_gate_of_groups(dev, rows, groups, channels, act):
  """One gate row for a run of rows: as many groups as rows, more groups than blocks, one group for all."""
  t, kw = make(dev, rows, channels, torch.bfloat16, "rms", gate="group", groups=groups)
  kw["gate_act"] = act
  check_forward(t, kw, *fused.residual_norm(t["x"], t["y"], **kw))
  check_grad(t, kw, fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_first_norm_of_a_model(dev, norm):
  """Without y there is only the norm: h is x itself."""
  t, kw = make(dev, 50, 96, torch.bfloat16, norm, post=False)
  h, z = fused.residual_norm(t["x"], **kw)
  assert h is t["x"]
  check_forward(dict(t, y=torch.zeros_like(t["y"])), kw, h, z)
  out = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], **kw)
  assert out["dy"] is None and out["dgate"] is None
  ref = grads64(t["x"], None, t["dh"], t["dz"], kw)
  for n, want in ref.items():
    assert torch.allclose(out[n].double().cpu(), want, rtol=half_step(out[n].dtype) * 1.01, atol=2e-5), n


@pytest.mark.parametrize("dev", DEVICES)
def test_shapes_with_more_dimensions_and_strided_rows(dev):
  """[N, H, W, C] activations; rows cut out of wider ones, at an odd element offset, and broadcast from one."""
  t, kw = make(dev, 2 * 3 * 5, 50, torch.bfloat16, "layer", gate="group", groups=2)
  flat = fused.residual_norm(t["x"], t["y"], **kw)
  four = fused.residual_norm(t["x"].view(2, 3, 5, 50), t["y"].view(2, 3, 5, 50), **kw)
  for a, b in zip(flat, four):
    assert b.shape == (2, 3, 5, 50) and torch.equal(a, b.view(30, 50))
  wide = {n: torch.randn(30, 131, device=dev).to(torch.bfloat16) for n in ("x", "y", "dh", "dz")}
  for n in wide:
    wide[n][:, 3:53] = t[n]
  cut = {n: v[:, 3:53] for n, v in wide.items()}
  for a, b in zip(flat, fused.residual_norm(cut["x"], cut["y"], **kw)):
    assert torch.equal(a, b) and b.is_contiguous()
  for a, b in zip(flat, fused.residual_norm(wide["x"].view(5, 6, 131)[..., 3:53],
                                            wide["y"].view(5, 6, 131)[..., 3:53], **kw)):
    assert torch.equal(a, b.view(30, 50))
  g0 = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  g1 = fused.residual_norm_grad(cut["dh"], cut["dz"], cut["x"], cut["y"], **kw)
  for n, v in g0.items():
    assert v is None or torch.equal(v, g1[n]), n
  one = t["x"][:1].expand(30, 50)
  check_forward(dict(t, x=one), kw, *fused.residual_norm(one, t["y"], **kw))
  gates = torch.randn(2, 77, device=dev)
  gates[:, 5:55] = kw["gate"]
  for a, b in zip(flat, fused.residual_norm(t["x"], t["y"], **dict(kw, gate=gates[:, 5:55]))):
    assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("groups", [0, 3])
def test_no_rows(dev, groups):
  t, kw = make(dev, 0, 32, torch.bfloat16, "layer")
  if groups == 0:
    h, z = fused.residual_norm(t["x"], t["y"], **kw)
    assert h.shape == z.shape == (0, 32)
    out = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
    assert out["dx"].shape == out["dy"].shape == (0, 32)
  else:
    kw["gate"] = torch.ones(groups, 32, device=dev)
    out = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
    assert out["dgate"].shape == (3, 32) and not out["dgate"].any()
  for n in VECTORS:
    assert out["d" + n].shape == (32,) and not out["d" + n].any()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("channels", [24, 600])
def test_bad_values_stay_in_their_row(dev, channels):
  """An infinity or NaN spoils its own row, never another one (nor, through idle lanes, the sums over rows); a row of
  zeros and a row of one repeated value (variance zero) are ordinary rows."""
  t, kw = make(dev, 40, channels, torch.bfloat16, "layer")
  clean = fused.residual_norm(t["x"], t["y"], **kw)
  t["x"][3, 5] = float("inf")
  t["y"][17, 9] = float("nan")
  h, z = fused.residual_norm(t["x"], t["y"], **kw)
  good = [i for i in range(40) if i not in (3, 17)]
  for a, b in zip(clean, (h, z)):
    assert torch.equal(a[good], b[good])
  assert torch.isnan(z[17]).all() and not torch.isfinite(z[3]).any()
  t, kw = make(dev, 37, channels, torch.float32, "layer")
  t["x"][5], t["y"][5], t["x"][6], t["y"][6] = 0, 0, 3.0, -2.0
  check_forward(t, kw, *fused.residual_norm(t["x"], t["y"], **kw))
  t["x"][5:7] = torch.tensor([[0.0], [3.0]], device=dev)
  check_grad(t, kw, fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw))


@pytest.mark.parametrize("dev", DEVICES)
def test_layer_norm_far_from_zero(dev):
  """A mean a thousand times the spread: the variance comes from centred values, not from a difference of squares."""
  t, kw = make(dev, 64, 300, torch.float32, "layer", post=True, offset=0.0)
  t["y"] = t["y"] * 0.01 + 10.0
  check_forward(t, kw, *fused.residual_norm(t["x"], t["y"], **kw))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_gradient_against_differences(dev, norm):
  """Directional derivatives of the definition by central differences in 64 bits against the gradient."""
  t, kw = make(dev, 20, 36, torch.float32, norm, gate="group", groups=4)
  kw["gate_act"] = "sigmoid"
  h, _ = fused.residual_norm(t["x"], t["y"], **kw)
  out = fused.residual_norm_grad(t["dh"], t["dz"], h, t["y"], **kw)
  k = to64(kw)
  values = dict(x=t["x"].double().cpu(), y=t["y"].double().cpu(), **{n: v for n, v in k.items() if isinstance(v, torch.Tensor)})

  def loss(v):
    hh, zz = seam64(v["x"], v["y"], dict(k, **{n: v[n] for n in v if n in k}))
    return float((hh * t["dh"].double().cpu()).sum() + (zz * t["dz"].double().cpu()).sum())

  gen = torch.Generator().manual_seed(5)
  for n, v in values.items():
    step = torch.randn(v.shape, generator=gen, dtype=torch.float64)
    e = 1e-5
    diff = (loss(dict(values, **{n: v + e * step})) - loss(dict(values, **{n: v - e * step}))) / (2 * e)
    g = out["d" + n].double().cpu()
    # fp32 gradients: 2^-12 of the sum of the terms' magnitudes is 4096 roundings of each; the differences' own error
    # (e^2 and 2^-53 / e) is far below
    assert abs(float((g * step).sum()) - diff) <= 2.0 ** -12 * float((g * step).abs().sum()) + 1e-7, n


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
  t, kw = make(dev, 12, 32, torch.bfloat16, "layer", gate="group", groups=3)
  x, y = t["x"], t["y"]
  g = torch.ones(32, device=dev)
  bad = [
      (dict(norm="batch"), "norm"), (dict(eps=0.0), "eps"), (dict(gate_act="relu"), "gate_act"),
      (dict(norm="rms", post_gamma=g, post_beta=g), "rms"), (dict(pre_beta=g, norm="layer"), "gamma"),
      (dict(post_gamma=g[:31]), "post_gamma"), (dict(post_gamma=g.half()), "post_gamma"),
      (dict(post_gamma=torch.ones(64, device=dev)[::2]), "post_gamma"),
      (dict(gate=torch.ones(5, 32, device=dev)), "divide"), (dict(gate=torch.ones(0, 32, device=dev)), "divide"),
      (dict(gate=torch.ones(12, 31, device=dev)), "gate"), (dict(gate=torch.ones(3, 32, device=dev).half()), "gate"),
      (dict(gate=torch.ones(32, 3, device=dev).t()), "channels"),
  ]
  for more, what in bad:
    with pytest.raises(ValueError, match=what):
      fused.residual_norm(x, y, **more)
    with pytest.raises(ValueError, match=what):
      fused.residual_norm_grad(t["dh"], None, x, y, **more)
  with pytest.raises(ValueError, match="y"):
    fused.residual_norm(x, y[:11])
  with pytest.raises(ValueError, match="y"):
    fused.residual_norm(x, y.float())
  with pytest.raises(ValueError, match="belong to y"):
    fused.residual_norm(x, post_gamma=g)
  with pytest.raises(ValueError, match="belong to y"):
    fused.residual_norm(x, gate=g)
  with pytest.raises(ValueError, match="element type"):
    fused.residual_norm(x.double(), y.double())
  with pytest.raises(ValueError, match="channels"):
    fused.residual_norm(x.t(), y.t())
  with pytest.raises(ValueError, match="different distances"):
    fused.residual_norm(torch.zeros(4, 6, 32, device=dev, dtype=x.dtype)[:, ::2][:, :2],
                        torch.zeros(4, 2, 32, device=dev, dtype=x.dtype))
  with pytest.raises(ValueError, match="dz"):
    fused.residual_norm_grad(t["dh"], None, x, y, pre_gamma=g)
  with pytest.raises(ValueError, match="dz"):
    fused.residual_norm_grad(t["dh"], t["dz"], x, y)
  with pytest.raises(ValueError, match="neither"):
    fused.residual_norm_grad(None, None, x, y)
  with pytest.raises(ValueError, match="requires a gradient"):
    fused.residual_norm(x, y, post_gamma=g.clone().requires_grad_(True))
  with torch.no_grad():
    fused.residual_norm(x, y, post_gamma=g.clone().requires_grad_(True))


@pytest.mark.gpu
def test_gpu_refuses_wider_rows():
  x = torch.zeros(2, 8193, device="cuda")
  with pytest.raises(ValueError, match="8192"):
    fused.residual_norm(x, x)
  with pytest.raises(ValueError, match="8192"):
    fused.residual_norm_grad(x, None, x, x)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,channels,gate,groups", [(3000, 48, "group", 2), (700, 1001, "element", 1), (900, 256, "none", 1)])
def test_gpu_same_bits_every_time_and_nothing_behind_the_rows(rows, channels, gate, groups):
  """No atomics: two calls agree bit for bit, also when another stream runs the same call; results end at their end."""
  t, kw = make("cuda", rows, channels, torch.bfloat16, "layer", gate=gate, groups=groups)
  a = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    b = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  c = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  torch.cuda.synchronize()
  for n in a:
    if a[n] is not None:
      assert torch.equal(a[n], b[n]) and torch.equal(a[n], c[n]), n
  # through the op itself, into the front of buffers whose rest is marked
  from distributed_tensorflow_amd.ops import native
  n = rows * channels
  h, z = (torch.full((n + 64,), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
  args = dict(dt=0, P=rows, C=channels, layer=1, scale=0.7, eps=1e-5, x=t["x"].data_ptr(), y=t["y"].data_ptr(),
              h=h.data_ptr(), z=z.data_ptr(), **{v: kw[v].data_ptr() for v in VECTORS})
  if gate != "none":
    args.update(gate=kw["gate"].data_ptr(), group_rows=rows // groups if gate == "group" else 0)
  native.run_op("residual_norm_fwd", args)
  torch.cuda.synchronize()
  want = fused.residual_norm(t["x"], t["y"], **kw)
  for got, w in zip((h, z), want):
    assert torch.equal(got[:n].view(rows, channels), w) and (got[n:] == 7.0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("channels", [16, 24, 136, 512, 640, 1032, 4096])
@pytest.mark.parametrize("gate,act", [("none", "none"), ("element", "sigmoid"), ("group", "none")])
def test_infinities_and_nans_stay_in_their_row_of_whole_chunks(dev, channels, gate, act):
  """Rows of whole chunks read their last chunk again in the lanes behind it: bad values there reach no other row, and
  no sum over rows but their own channel's."""
  rows = 21
  t, kw = make(dev, rows, channels, torch.bfloat16, "layer", gate=gate, groups=7)
  kw["gate_act"] = act
  clean = fused.residual_norm(t["x"], t["y"], **kw)
  clean_g = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  for n in ("x", "y", "dh", "dz"):
    t[n][rows - 1, -1] = float("inf")
    t[n][rows - 2, -2] = float("nan")
  good = list(range(rows - 2))
  for a, b in zip(clean, fused.residual_norm(t["x"], t["y"], **kw)):
    assert torch.equal(a[good], b[good])
  g = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  for n in ("dx", "dy"):
    assert torch.equal(clean_g[n][good], g[n][good])
  if gate == "group":
    assert torch.equal(clean_g["dgate"][:6], g["dgate"][:6])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,channels", [(4_200_000, 512), (2_150_000, 1001), (265_000, 8192)])
def test_gpu_offsets_past_32_bits(rows, channels):
  """More than 2^31 elements a tensor: the last rows as a call on them alone gives them."""
  z = lambda: torch.zeros(rows, channels, dtype=torch.bfloat16, device="cuda")
  t, kw = make("cuda", 64, channels, torch.bfloat16, "rms", gate="group", groups=1)
  big = {n: z() for n in t}
  for n in t:
    big[n][-64:] = t[n]
  want = fused.residual_norm(t["x"], t["y"], **kw)
  got = fused.residual_norm(big["x"], big["y"], **kw)
  for a, b in zip(want, got):
    assert torch.equal(a, b[-64:]) and not b[:64].any()
  del got
  want = fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  got = fused.residual_norm_grad(big["dh"], big["dz"], big["x"], big["y"], **kw)
  for n, a in want.items():
    if a is not None and n in ("dx", "dy"):
      assert torch.equal(a, got[n][-64:]) and not got[n][:64].any()
    elif a is not None:      # the same 64 terms of a column in other places of the sum; a term is under 16 (|dz| + |dh|)
      terms = 16 * (t["dz"].float().abs().sum(0) + t["dh"].float().abs().sum(0))
      assert ((a - got[n]).abs() <= 64 * U * terms).all(), n


@pytest.mark.gpu
def test_gpu_captured_and_replayed():
  """Two captures of the same calls, replayed in turn with eager work between, new values in the same buffers."""
  t, kw = make("cuda", 500, 200, torch.bfloat16, "layer", gate="group", groups=5)
  graphs, outs = [], []
  fused.residual_norm(t["x"], t["y"], **kw)
  fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw)
  torch.cuda.synchronize()
  for _ in range(2):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      h, z = fused.residual_norm(t["x"], t["y"], **kw)
      d = fused.residual_norm_grad(t["dh"], t["dz"], h, t["y"], **kw)
    graphs.append(g)
    outs.append(dict(h=h, z=z, **d))
  for i in range(4):
    for n in t:
      t[n].copy_(torch.randn(t[n].shape, device="cuda") * (i + 1))
    graphs[i % 2].replay()
    torch.cuda.synchronize()
    h, z = fused.residual_norm(t["x"], t["y"], **kw)
    want = dict(h=h, z=z, **fused.residual_norm_grad(t["dh"], t["dz"], h, t["y"], **kw))
    torch.cuda.synchronize()
    for n, w in want.items():
      assert torch.equal(outs[i % 2][n], w), (i, n)


@pytest.mark.gpu
def test_gpu_as_entries_of_a_launch_plan():
  """Forward and backward recorded in a plan, run and replayed as a captured graph: the bits of the direct calls."""
  from distributed_tensorflow_amd.ops import native
  rows, c = 256, 640
  t, kw = make("cuda", rows, c, torch.bfloat16, "rms", gate="element")
  h, z, dx, dy, dg = (torch.zeros(rows, c, dtype=torch.bfloat16, device="cuda") for _ in range(5))
  v = torch.zeros(2, c, device="cuda")
  ws = torch.zeros(native.ext().residual_norm_workspace_floats(rows, c, 0, 0, 0), device="cuda")
  common = dict(dt=0, P=rows, C=c, scale=0.7, eps=1e-5, y=t["y"].data_ptr(), gate=kw["gate"].data_ptr(),
                post_gamma=kw["post_gamma"].data_ptr(), pre_gamma=kw["pre_gamma"].data_ptr())
  plan = native.Plan()
  plan.add("residual_norm_fwd", dict(common, x=t["x"].data_ptr(), h=h.data_ptr(), z=z.data_ptr()), "seam")
  plan.add("residual_norm_bwd", dict(common, h=h.data_ptr(), dh=t["dh"].data_ptr(), dz=t["dz"].data_ptr(),
                                     dx=dx.data_ptr(), dy=dy.data_ptr(), dgate=dg.data_ptr(), ws=ws.data_ptr(),
                                     dpost_gamma=v[0].data_ptr(), dpre_gamma=v[1].data_ptr()), "seam gradient")
  stream = torch.cuda.Stream()
  plan.run(0, 2, stream.cuda_stream)
  graph = plan.capture(0, 2, stream.cuda_stream)
  for i in range(3):
    stream.synchronize()
    t["x"].copy_(torch.randn(rows, c, device="cuda"))
    torch.cuda.synchronize()
    plan.replay(graph, stream.cuda_stream)
    stream.synchronize()
    wh, wz = fused.residual_norm(t["x"], t["y"], **kw)
    w = fused.residual_norm_grad(t["dh"], t["dz"], wh, t["y"], **kw)
    torch.cuda.synchronize()
    for got, want in ((h, wh), (z, wz), (dx, w["dx"]), (dy, w["dy"]), (dg, w["dgate"]), (v[0], w["dpost_gamma"]),
                      (v[1], w["dpre_gamma"])):
      assert torch.equal(got, want), i
  with pytest.raises(ValueError, match="ws"):
    native.run_op("residual_norm_bwd", dict(common, h=h.data_ptr(), dh=t["dh"].data_ptr(), dz=t["dz"].data_ptr(),
                                            dx=dx.data_ptr(), dy=dy.data_ptr(), dgate=dg.data_ptr(),
                                            dpost_gamma=v[0].data_ptr(), dpre_gamma=v[1].data_ptr()))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,channels,groups", [
    (50, 16, 0), (21, 1001, 0), (40, 16, 20), (1500, 16, 500), (6000, 16, 2), (2048, 64, 4), (300, 600, 3), (30, 520, 30),
    (9000, 48, 1), (12, 5001, 4)])
def test_gradient_of_open_and_closed_sigmoid_gates(dev, dtype, rows, channels, groups):
  """Gates far from zero, whose slope is as small as e^-|g|: gradients relative to their own size.

  Without norms up = dh, n = y and dgate = sum over the group's rows of 0.5 dh y times the slope; all terms positive.  The
  slope sees the exponential ((|g| + 8) U with the hardware's), a sum, a reciprocal and two products: (|g| + 16) U; dgate
  the terms' product, the last one and the sum's serial roundings besides.  A place adds at most 512 rows in turn, the joins
  behind it under 64, blocks of long groups rows / 256.  dy = 0.5 dh a: (|g| + 16) U.  Half a step for the result's type; what
  falls below the smallest normal of that type is off by one of its smallest steps."""
  gen = torch.Generator().manual_seed(rows + channels)
  dh = (1000 + 2000 * torch.rand(rows, channels, generator=gen)).to(dtype).to(dev)
  y = (10 + 20 * torch.rand(rows, channels, generator=gen)).to(dtype).to(dev)
  values = torch.tensor([8.0, -8.0, 12.0, -12.0, 16.0, -16.0, 18.0, -18.0, 0.0, 20.0, -30.0, 2.5])
  n = groups or rows
  gate = values[(torch.arange(n * channels) * 5) % 12].view(n, channels).to(torch.float32 if groups else dtype).to(dev)
  out = fused.residual_norm_grad(dh, None, y, y, gate=gate, gate_act="sigmoid", residual_scale=0.5)
  g = gate.double().cpu()
  slope = 1 / (2 + torch.exp(g) + torch.exp(-g))
  per = 0.5 * dh.double().cpu() * y.double().cpu()
  want = (per.view(groups, -1, channels).sum(1) if groups else per) * slope
  depth = 576 + rows / 256 if groups else 0
  limit = half_step(gate.dtype) * (1 + 1e-6) + (depth + 32 + g.abs()) * U
  f = torch.finfo(gate.dtype)
  assert out["dgate"].dtype == gate.dtype
  assert ((out["dgate"].double().cpu() - want).abs() <= limit * want + f.smallest_normal * f.eps).all()
  a = torch.sigmoid(g).repeat_interleave(rows // n, 0)
  want = 0.5 * dh.double().cpu() * a
  limit = half_step(dtype) * (1 + 1e-6) + (16 + g.abs().repeat_interleave(rows // n, 0)) * U
  f = torch.finfo(dtype)
  assert ((out["dy"].double().cpu() - want).abs() <= limit * want + f.smallest_normal * f.eps).all()


def test_few_groups_are_spread_over_the_grid():
  """Groups that do not fill the row slots of a block share the slots, and their parts several blocks; only many short
  ones go to a slot each.  (A block leaves five rows of partial sums.)"""
  from distributed_tensorflow_amd.ops import native
  if not native.available():
    pytest.skip("no native extension")
  blocks = lambda rows, c, group_rows: native.ext().residual_norm_workspace_floats(rows, c, group_rows, 0, 0) // (5 * c)
  for c in (16, 64, 200):                         # 128, 32 and 8 slots
    slots = {16: 128, 64: 32, 200: 8}[c]
    for groups in (1, 2, 7):
      for per in (4 * slots - 1, slots + 1, 40):
        assert blocks(groups * per, c, per) >= groups * min(-(-per // slots), 4), (c, groups, per)
    for groups, per in ((20_000, 1), (20_000, 2), (20_000, 16)):
      sets = -(-groups // slots)                  # 512 blocks fill the grid, 768 that of a sweep past the caches
      assert blocks(groups * per, c, per) in (min(sets, 512), min(sets, 768)), (c, groups, per)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,groups,channels", [
    (511, 1, 16), (510, 2, 16), (2555, 5, 16), (127, 1, 64), (254, 2, 64), (31, 1, 200), (93, 3, 200), (66, 2, 512),
    (20_000, 5000, 16), (16_000, 1000, 24), (32_000, 1000, 16), (33_000, 1000, 16), (4800, 300, 200)])
@pytest.mark.parametrize("norm,act", [("rms", "sigmoid"), ("layer", "none")])
def test_gate_of_few_long_and_many_short_groups(dev, dtype, rows, groups, channels, norm, act):
  """On either side of the rule that gives groups to slots."""
  t, kw = make(dev, rows, channels, dtype, norm, gate="group", groups=groups)
  kw["gate_act"] = act
  check_forward(t, kw, *fused.residual_norm(t["x"], t["y"], **kw))
  check_grad(t, kw, fused.residual_norm_grad(t["dh"], t["dz"], t["x"], t["y"], **kw))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(dev, grad):
  from torch.autograd import forward_ad
  t, kw = make(dev, 6, 16, torch.float32, "layer", gate="element")
  with forward_ad.dual_level(), torch.set_grad_enabled(grad):
    fused.residual_norm(t["x"], t["y"], **kw)                    # a level alone is nothing
    dual = lambda v: forward_ad.make_dual(v, torch.ones_like(v))
    for n in ("x", "y"):
      with pytest.raises(ValueError, match="forward-mode"):
        fused.residual_norm(**dict({a: t[a] for a in ("x", "y")}, **{n: dual(t[n])}), **kw)
    for n in VECTORS + ("gate",):
      with pytest.raises(ValueError, match="forward-mode"):
        fused.residual_norm(t["x"], t["y"], **dict(kw, **{n: dual(kw[n])}))
    for i in range(4):
      args = [t["dh"], t["dz"], t["x"], t["y"]]
      args[i] = dual(args[i])
      with pytest.raises(ValueError, match="forward-mode"):
        fused.residual_norm_grad(*args, **kw)
  with pytest.raises(ValueError, match="forward-mode"):
    torch.func.jvp(lambda v: fused.residual_norm(v, t["y"], **kw), (t["x"],), (t["x"],))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("channels", [64, 4096, 5000, 8192])
def test_the_largest_values_a_row_may_hold(dev, dtype, norm, channels):
  """Squares sum to float32's largest number, sqrt(2^128 / channels) a value: a tenth below, rows are right; above (an
  eighth, past the 2^-9 that bf16 may round down and what centring takes off) their normalised values are zero, as stated."""
  gen = torch.Generator().manual_seed(channels)
  limit = (2.0 ** 128 / channels) ** 0.5
  sign = (torch.rand(2, channels, generator=gen) < 0.5).float() * 2 - 1
  sign[:, channels // 2:] = -sign[:, :channels // 2]              # as many of either: a mean of zero
  gamma, dz = 1 + 0.3 * torch.randn(channels, generator=gen), torch.randn(2, channels, generator=gen).to(dtype)
  x = (sign * (limit * torch.tensor([[0.9], [1.125]]))).to(dtype)
  gamma, dz, x = gamma.to(dev), dz.to(dev), x.to(dev)
  h, z = fused.residual_norm(x, pre_gamma=gamma, norm=norm)
  assert h is x
  want = norm64(x[:1].double().cpu(), gamma.double().cpu(), None, norm, 1e-6)[0]
  limit_z = half_step(dtype) * want.abs() + 128 * U * (want.abs().max() + 1)
  assert ((z[:1].double().cpu() - want).abs() <= limit_z).all()
  assert (z[1] == 0).all()
  out = fused.residual_norm_grad(None, dz, x, pre_gamma=gamma, norm=norm)
  want = dz[0].double().cpu() * want[0] / gamma.double().cpu()       # the second row's share is nothing
  assert ((out["dpre_gamma"].double().cpu() - want).abs() <= 256 * U * (want.abs().max() + 1)).all()
  assert torch.isfinite(out["dx"].float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,channels", [(131_072, 16), (131_072, 24), (65_536, 64), (20_000, 200), (8192, 512), (16_384, 600)])
def test_gpu_sums_over_many_rows(rows, channels):
  """dpre_beta is the sum of dz itself.  With positive terms only the roundings on the way count: those of a slot's own rows,
  one for a block's partial sum and one for the result; the joins are in 64 bits.  Equal terms of these values would be
  rounded the same way again and again by joins in 32 (131072 of 16 channels: 8.7 U instead of 3)."""
  from distributed_tensorflow_amd.ops import native
  gen = torch.Generator().manual_seed(channels)
  dz = 1 + torch.rand(rows, channels, generator=gen)
  dz[:, ::2] = 1 + (5033592 + 144 * torch.arange(0, channels, 2)) / 2.0 ** 23
  ones = torch.ones(channels, device="cuda")
  h = torch.randn(rows, channels, generator=gen).cuda()
  out = fused.residual_norm_grad(None, dz.cuda(), h, pre_gamma=ones, pre_beta=ones, norm="layer")
  lanes = 2
  while lanes * 8 < channels:
    lanes *= 2
  slots = 256 // lanes if channels <= 512 else 1
  blocks = native.ext().residual_norm_workspace_floats(rows, channels, 0, 2, 1) // (5 * channels)
  own = -(-rows // (blocks * slots))
  want = dz.double().sum(0)
  assert ((out["dpre_beta"].double().cpu() - want).abs() <= (own - 1 + 2) * U * want * (1 + 1e-6)).all()
