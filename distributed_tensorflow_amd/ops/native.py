"""Loader and thin Python API of the in-tree HIP extension `_dtf_native`.

The extension is built ahead of time by `ops/build.py` (hipcc, gfx950) and lives next to
this file.  Importing this module on a machine with a GPU and no built extension raises: the
device path never falls back to library kernels silently.
"""
from __future__ import annotations

import contextlib
import struct
from typing import Dict, List, Optional, Sequence

import torch

try:
  from . import _dtf_native as _ext          # noqa: F401
except ImportError as e:                      # pragma: no cover - exercised only without a build
  _ext = None
  _import_error = e

__all__ = ["available", "ext", "run_op", "Plan", "stream_handle", "sgd_momentum_l2", "loss_scale_step",
           "clipped_sgd_momentum_l2", "clip_list_norm", "clip_list_scale",
           "residual_norm", "residual_norm_grad", "dtype_code", "pack_desc_bytes", "pack_blocks", "PACK_PER_BLOCK"]

PACK_PER_BLOCK = 256 * 8


def available() -> bool:
  return _ext is not None


def ext():
  if _ext is None:
    raise RuntimeError(
        "native extension _dtf_native is not built; run "
        "`python -m distributed_tensorflow_amd.ops.build` (%s)" % (_import_error,))
  return _ext


def stream_handle(device: Optional[torch.device] = None) -> int:
  """Raw hipStream_t of torch's current stream (kernels are ordered with torch ops)."""
  return int(torch.cuda.current_stream(device).cuda_stream)


def run_op(kind: str, args: Dict, stream: Optional[int] = None):
  ext().run_op(kind, args, stream_handle() if stream is None else stream)


def Plan():
  return ext().Plan()


def sgd_momentum_l2(params: torch.Tensor, grads: torch.Tensor, velocity: torch.Tensor,
                    l2x2: torch.Tensor, lr: float, momentum: float, grad_scale: float = 1.0,
                    skip: Optional[torch.Tensor] = None):
  """`skip`: two device floats [skip flag, extra gradient factor] of a device-side loss-scale
  state (`loss_scale_step`); flag != 0 leaves the update out."""
  for t in (params, grads, velocity, l2x2):
    if t.dtype != torch.float32 or not t.is_contiguous() or t.device != params.device:
      raise ValueError("sgd_momentum_l2 wants contiguous fp32 tensors on one device")
  n = params.numel()
  if grads.numel() != n or l2x2.numel() != n or (momentum and velocity.numel() != n):
    raise ValueError("sgd_momentum_l2: buffer sizes differ")
  run_op("sgd", dict(p=params.data_ptr(), g=grads.data_ptr(), v=velocity.data_ptr(),
                     l2x2=l2x2.data_ptr(), n=n, lr=float(lr), momentum=float(momentum),
                     grad_scale=float(grad_scale),
                     skip=skip.data_ptr() if skip is not None else None))


_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}     # DT_BF16 / DT_F16 / DT_F32 of common.h


def dtype_code(dtype: torch.dtype) -> int:
  try:
    return _DT[dtype]
  except KeyError:
    raise ValueError("element type %s (bfloat16, float16 and float32 are built)" % dtype) from None


@contextlib.contextmanager
def _on_device(device: torch.device):
  """The device's current stream; kernels of another device than the current one are launched from there."""
  if device.index is None or device.index == torch.cuda.current_device():
    yield stream_handle()
  else:
    with torch.cuda.device(device):
      yield stream_handle()


def clipped_sgd_momentum_l2(params: torch.Tensor, grads: torch.Tensor, velocity: torch.Tensor, l2x2: torch.Tensor,
                            lr: float, momentum: float, clip_norm: float, grad_scale: float = 1.0,
                            skip: Optional[torch.Tensor] = None) -> torch.Tensor:
  """Two launches: the norm's partial sums, the update (arguments checked by `fused`)."""
  n = params.numel()
  dev = params.device
  with _on_device(dev) as stream:
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(ext().clipped_sgd_blocks(n), dtype=torch.float64, device=dev)
    run_op("clipped_sgd", dict(p=params.data_ptr(), g=grads.data_ptr(), v=velocity.data_ptr(),
                               l2x2=l2x2.data_ptr(), n=n, lr=float(lr), momentum=float(momentum),
                               clip=float(clip_norm), grad_scale=float(grad_scale),
                               skip=skip.data_ptr() if skip is not None else None,
                               ws=ws.data_ptr(), norm=norm.data_ptr()), stream)
  return norm


def clip_list_norm(table) -> torch.Tensor:
  """Global norm of a `fused.TensorTable`.  The workspace is the call's own: tables are shared between streams."""
  lst, dev = table._list, table.device
  with _on_device(dev) as stream:
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(max(lst.workspace_doubles, 1), dtype=torch.float64, device=dev)
    lst.global_norm(ws.data_ptr(), norm.data_ptr(), stream)
  return norm


def clip_list_scale(table, clip_norm: float, use_norm: Optional[torch.Tensor]) -> torch.Tensor:
  """Clips a `fused.TensorTable` into its outputs; the norm."""
  lst, dev = table._list, table.device
  with _on_device(dev) as stream:
    if use_norm is not None:
      lst.clip(0, use_norm.data_ptr(), clip_norm, 0, stream)
      return use_norm
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(max(lst.workspace_doubles, 1), dtype=torch.float64, device=dev)
    lst.clip(ws.data_ptr(), 0, clip_norm, norm.data_ptr(), stream)
  return norm


def _vectors(args: Dict, post_gamma, post_beta, pre_gamma, pre_beta):
  if post_gamma is not None:
    args["post_gamma"] = post_gamma.data_ptr()
    if post_beta is not None:
      args["post_beta"] = post_beta.data_ptr()
  if pre_gamma is not None:
    args["pre_gamma"] = pre_gamma.data_ptr()
    if pre_beta is not None:
      args["pre_beta"] = pre_beta.data_ptr()


def residual_norm(x, y, rows: int, channels: int, pitch: Dict, gate, group_rows: int, sigmoid: bool, layer: bool,
                  scale: float, eps: float, post_gamma, post_beta, pre_gamma, pre_beta):
  """One launch (arguments checked by `fused`); `pitch`: elements from one row to the next."""
  dev = x.device
  with _on_device(dev) as stream:
    args = dict(dt=_DT[x.dtype], P=rows, C=channels, layer=int(layer), sigmoid=int(sigmoid), scale=scale, eps=eps,
                x=x.data_ptr(), ldx=pitch["x"])
    h, z = x, None
    if y is not None:
      h = torch.empty(x.shape, dtype=x.dtype, device=dev)
      args.update(y=y.data_ptr(), ldy=pitch["y"], h=h.data_ptr())
      if gate is not None:
        args.update(gate=gate.data_ptr(), ldgate=pitch["gate"], group_rows=group_rows)
    if pre_gamma is not None:
      z = torch.empty(x.shape, dtype=x.dtype, device=dev)
      args["z"] = z.data_ptr()
    _vectors(args, post_gamma, post_beta, pre_gamma, pre_beta)
    if rows and (h is not x or z is not None):
      run_op("residual_norm_fwd", args, stream)
  return h, z


def residual_norm_grad(dh, dz, h, y, rows: int, channels: int, pitch: Dict, gate, group_rows: int, sigmoid: bool,
                       layer: bool, scale: float, eps: float, post_gamma, post_beta, pre_gamma, pre_beta) -> Dict:
  """The sweep over the rows and, where sums over rows are asked for, one or two launches that finish them."""
  dev = h.device
  with _on_device(dev) as stream:
    def rows_like():
      return torch.empty(h.shape, dtype=h.dtype, device=dev)

    # the four vectors' gradients sit in one buffer
    names = [n for n, t in (("pre_gamma", pre_gamma), ("pre_beta", pre_beta), ("post_gamma", post_gamma),
                            ("post_beta", post_beta)) if t is not None]
    make = torch.empty if rows else torch.zeros
    vectors = make((max(len(names), 1), channels), dtype=torch.float32, device=dev)
    out = dict(dx=rows_like(), dy=None, dgate=None, dpost_gamma=None, dpost_beta=None, dpre_gamma=None,
               dpre_beta=None)
    for i, n in enumerate(names):
      out["d" + n] = vectors[i]
    if y is not None:
      out["dy"] = rows_like()
    if gate is not None:
      out["dgate"] = make(gate.shape, dtype=gate.dtype, device=dev)
    if rows:
      ws = torch.empty(ext().residual_norm_workspace_floats(rows, channels, group_rows), dtype=torch.float32, device=dev)
      args = dict(dt=_DT[h.dtype], P=rows, C=channels, layer=int(layer), sigmoid=int(sigmoid), scale=scale, eps=eps,
                  ws=ws.data_ptr())
      for n, t in (("dh", dh), ("dz", dz), ("h", h), ("y", y), ("gate", gate)):
        if t is not None:
          args[n] = t.data_ptr()
          args["ld" + n] = pitch[n]
      if gate is not None:
        args["group_rows"] = group_rows
      _vectors(args, post_gamma, post_beta, pre_gamma, pre_beta)
      for n, t in out.items():
        if t is not None:
          args[n] = t.data_ptr()
      run_op("residual_norm_bwd", args, stream)
  return out


def loss_scale_step(grads: torch.Tensor, state: torch.Tensor, flag: torch.Tensor,
                    loss_scale_dev: Optional[torch.Tensor], growth: int, multiplier: float):
  """Dynamic loss scaling without a host round trip: one pass over the flat gradients sets
  `flag` when any element is inf / nan, then a one-thread kernel advances
  state = [scale, clean steps, skipped steps, skip, 1 / scale used] and writes the next
  step's scale to `loss_scale_dev` (the executor's loss-gradient factor)."""
  if state.dtype != torch.float32 or state.numel() < 5 or flag.dtype != torch.int32:
    raise ValueError("loss_scale_step: state is 5 floats, flag one int32")
  run_op("nonfinite_flag", dict(g=grads.data_ptr(), n=grads.numel(), flag=flag.data_ptr()))
  run_op("loss_scale_update", dict(
      state=state.data_ptr(), flag=flag.data_ptr(),
      loss_scale_dev=loss_scale_dev.data_ptr() if loss_scale_dev is not None else None,
      growth=float(growth), multiplier=float(multiplier)))


def pack_blocks(d: Dict) -> int:
  """Thread blocks the weight-pack kernel spends on descriptor `d`: tiles of 32 input channels
  x 64 output channels per tap for the forward layout (mode 0, a transpose), 2048 elements
  per block for the data-gradient layout (mode 1, a strided copy)."""
  if d["mode"] == 0:
    return d["TI"] * d["TJpad"] * (-(-d["Cpad"] // 32)) * (-(-d["Cout"] // 64))
  return -(-d["count"] // PACK_PER_BLOCK)


def pack_desc_bytes(descs: Sequence[Dict]) -> bytes:
  """Serialises weight-pack descriptors to the C `PackDesc` layout (64 bytes each)."""
  out = bytearray()
  for d in descs:
    out += struct.pack("<qq8iqq", d["src_off"], d["dst_off"], d["TI"], d["TJ"], d["Cin"],
                       d["Cout"], d["TJpad"], d["Cpad"], d["CoutPad"], d["mode"], d["count"],
                       d["first_block"])
  if _ext is not None and descs and len(out) // len(descs) != _ext.pack_desc_size():
    raise RuntimeError("PackDesc layout mismatch between Python and C++")
  return bytes(out)
