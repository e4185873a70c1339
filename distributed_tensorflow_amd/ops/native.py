"""Loader and thin Python API of the in-tree HIP extension `_dtf_native`.

The extension is built ahead of time by `ops/build.py` (hipcc, gfx950) and lives next to
this file.  Importing this module on a machine with a GPU and no built extension raises: the
device path never falls back to library kernels silently.
"""
from __future__ import annotations

import struct
from typing import Dict, List, Optional, Sequence

import torch

try:
  from . import _dtf_native as _ext          # noqa: F401
except ImportError as e:                      # pragma: no cover - exercised only without a build
  _ext = None
  _import_error = e

__all__ = ["available", "ext", "run_op", "Plan", "stream_handle", "sgd_momentum_l2", "loss_scale_step",
           "clipped_sgd_momentum_l2", "clip_list_build", "clip_list_upload", "clip_list_norm", "clip_list_scale",
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


def _elsewhere(index: int) -> bool:
  """Whether device `index` is not the current one: its kernels are then launched from `torch.cuda.device(index)`."""
  return index != torch.cuda.current_device()


# Kernels write through addresses, which autograd does not see: without this a backward pass would use a tensor that it
# has saved and that was overwritten since, instead of refusing it.
_written = torch.autograd.graph.increment_version


# raw hipStream_t of a device's current stream, without a Stream object (0.1 instead of 2.8 us)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def clipped_sgd_momentum_l2(params: torch.Tensor, grads: torch.Tensor, velocity: torch.Tensor, l2x2: torch.Tensor,
                            lr: float, momentum: float, clip_norm: float, grad_scale: float = 1.0,
                            skip: Optional[torch.Tensor] = None) -> torch.Tensor:
  """Two launches: the norm's partial sums, the update (arguments checked by `fused`)."""
  index = params.get_device()
  if _elsewhere(index):
    with torch.cuda.device(index):
      return clipped_sgd_momentum_l2(params, grads, velocity, l2x2, lr, momentum, clip_norm, grad_scale, skip)
  n = params.numel()
  norm = params.new_empty(())
  ws = params.new_empty(ext().clipped_sgd_blocks(n), dtype=torch.float64)
  ext().clipped_sgd(params.data_ptr(), grads.data_ptr(), velocity.data_ptr(), l2x2.data_ptr(), n, lr, momentum,
                    grad_scale, clip_norm, skip.data_ptr() if skip is not None else 0, ws.data_ptr(),
                    norm.data_ptr(), _current_stream(index))
  _written([params, velocity] if momentum else [params])
  return norm


def clip_list_build(table, at: List[int], to: List[int]):
  """Native half of a `fused.TensorTable`."""
  ts = table.tensors
  table.list = ext().ClipList(at, to, [t.numel() for t in ts], [dtype_code(t.dtype) for t in ts])
  table.workspace = max(table.list.workspace_doubles, 1)


def clip_list_upload(table) -> bool:
  """Writes the list to device memory, where one launch walks any number of tensors; False while a graph is captured (the
  upload would become part of it)."""
  with torch.cuda.device(table.device):
    if torch.cuda.is_current_stream_capturing():
      return False
    # a blocking copy: complete for every stream when it returns
    table.resident = torch.frombuffer(bytearray(table.list.table()), dtype=torch.uint8).to(table.device)
    table.stream = _current_stream(table.device.index)
  return True


def _clip_list_launch(table, stream: int):
  """(address of the device table or 0, norm, workspace) of a call.  The workspace is the call's own: tables are shared
  between streams.  The device table is held back from reuse until a foreign stream is done with it, and for good once
  a graph has captured it."""
  dev = table.device
  resident = 0
  if table.resident is not None:
    resident = table.resident.data_ptr()
    if torch.cuda.is_current_stream_capturing():
      if not any(r is table.resident for r in table.held):
        table.held.append(table.resident)
    elif stream != table.stream:
      table.resident.record_stream(torch.cuda.current_stream(dev))
  return (resident, torch.empty((), dtype=torch.float32, device=dev),
          torch.empty(table.workspace, dtype=torch.float64, device=dev))


def clip_list_norm(table) -> torch.Tensor:
  """Global norm of a `fused.TensorTable`."""
  index = table.device.index
  if _elsewhere(index):
    with torch.cuda.device(index):
      return clip_list_norm(table)
  stream = _current_stream(index)
  resident, norm, ws = _clip_list_launch(table, stream)
  table.list.global_norm(resident, ws.data_ptr(), norm.data_ptr(), stream)
  return norm


def clip_list_scale(table, clip_norm: float, use_norm: Optional[torch.Tensor]) -> torch.Tensor:
  """Clips a `fused.TensorTable` into its outputs; the norm."""
  index = table.device.index
  if _elsewhere(index):
    with torch.cuda.device(index):
      return clip_list_scale(table, clip_norm, use_norm)
  stream = _current_stream(index)
  resident, norm, ws = _clip_list_launch(table, stream)
  if use_norm is not None:
    table.list.clip(resident, 0, use_norm.data_ptr(), clip_norm, 0, stream)
    norm = use_norm
  else:
    table.list.clip(resident, ws.data_ptr(), 0, clip_norm, norm.data_ptr(), stream)
  _written(table.out)
  return norm


def _ptr(t: Optional[torch.Tensor]) -> int:
  return 0 if t is None else t.data_ptr()


def residual_norm(x, ldx, y, ldy, rows, channels, gate, ldgate, group_rows, sigmoid, layer, scale, eps, post_gamma,
                  post_beta, pre_gamma, pre_beta):
  """One launch (arguments checked by `fused`); ld*: elements from one row to the next."""
  index = x.get_device()
  if _elsewhere(index):
    with torch.cuda.device(index):
      return residual_norm(x, ldx, y, ldy, rows, channels, gate, ldgate, group_rows, sigmoid, layer, scale, eps,
                           post_gamma, post_beta, pre_gamma, pre_beta)
  h = x if y is None else torch.empty_like(x, memory_format=torch.contiguous_format)
  z = None if pre_gamma is None else torch.empty_like(x, memory_format=torch.contiguous_format)
  if rows and (h is not x or z is not None):
    ext().residual_norm_fwd(_DT[x.dtype], rows, channels, layer, sigmoid, scale, eps, x.data_ptr(), ldx, _ptr(y), ldy,
                            _ptr(gate), ldgate, group_rows, _ptr(post_gamma), _ptr(post_beta), _ptr(pre_gamma),
                            _ptr(pre_beta), h.data_ptr(), _ptr(z), _current_stream(index))
  return h, z


def residual_norm_grad(dh, lddh, dz, lddz, h, ldh, y, ldy, rows, channels, gate, ldgate, group_rows, sigmoid, layer,
                       scale, eps, post_gamma, post_beta, pre_gamma, pre_beta) -> Dict:
  """The sweep over the rows and, where sums over rows are asked for, one launch that finishes them."""
  index = h.get_device()
  if _elsewhere(index):
    with torch.cuda.device(index):
      return residual_norm_grad(dh, lddh, dz, lddz, h, ldh, y, ldy, rows, channels, gate, ldgate, group_rows, sigmoid,
                                layer, scale, eps, post_gamma, post_beta, pre_gamma, pre_beta)
  # the gradients of the four vectors sit in one buffer
  names = [n for n, t in (("dpre_gamma", pre_gamma), ("dpre_beta", pre_beta), ("dpost_gamma", post_gamma),
                          ("dpost_beta", post_beta)) if t is not None]
  out = dict.fromkeys(("dx", "dy", "dgate", "dpost_gamma", "dpost_beta", "dpre_gamma", "dpre_beta"))
  vectors = None
  if names:
    vectors = (h.new_empty if rows else h.new_zeros)((len(names), channels), dtype=torch.float32)
    out.update(zip(names, vectors.unbind(0)))
  dx = out["dx"] = torch.empty_like(h, memory_format=torch.contiguous_format)
  dy = out["dy"] = None if y is None else torch.empty_like(h, memory_format=torch.contiguous_format)
  dgate = None
  if gate is not None:
    dgate = (torch.empty_like if rows else torch.zeros_like)(gate, memory_format=torch.contiguous_format)
    out["dgate"] = dgate
  if rows:
    e = ext()
    ws = h.new_empty(e.residual_norm_workspace_floats(rows, channels, group_rows, _DT[h.dtype], layer), dtype=torch.float32)
    e.residual_norm_bwd(_DT[h.dtype], rows, channels, layer, sigmoid, scale, eps, h.data_ptr(), ldh, _ptr(y), ldy,
                        _ptr(gate), ldgate, group_rows, _ptr(post_gamma), _ptr(post_beta), _ptr(pre_gamma),
                        _ptr(pre_beta), _ptr(dh), lddh, _ptr(dz), lddz, dx.data_ptr(), _ptr(dy), _ptr(dgate),
                        _ptr(vectors), ws.data_ptr(), _current_stream(index))
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
