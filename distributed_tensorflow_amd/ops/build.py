"""Builds the native extension `_dtf_native` for gfx950 with hipcc (of torch only the header of DLPack's C structures).

    python -m distributed_tensorflow_amd.ops.build [--force] [--jobs N]

Sources live in `ops/csrc`; objects go to `ops/csrc/build`, the shared object is written
next to this file so that it travels with the source tree.  hipcc cross-compiles for
gfx950 on a machine without a GPU.
"""
from __future__ import annotations

import argparse
import concurrent.futures
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "build")
ARCH = "gfx950"
# No packed fp32 arithmetic: -O3 pairs ordinary float operations into v_pk_add / mul / fma_f32 by itself, and some of
# their operand-select forms have lost elements on this hardware without any error (see conv_epilogue.h).  The host pass
# of hipcc warns that it does not know the feature.
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
SOURCES = ["conv_igemm.hip", "conv_pipe.hip", "conv_halo.hip", "conv_rows.hip", "conv_wgrad_rows.hip", "conv_wgrad.hip", "bn.hip", "pool.hip", "loss.hip", "optim.hip", "dense.hip", "residual_norm.hip",
           "residual_norm_bf16.hip", "residual_norm_f16.hip", "residual_norm_f32.hip",
           "grad_clip.hip",
           "rccl_comm.cpp", "bindings.cpp"]
HEADERS = ["common.h", "conv_params.h", "conv_epilogue.h", "elementwise.h", "rccl_comm.h"]
# headers of one kernel file and the bindings
_RESIDUAL_NORM = ["residual_norm.h", "residual_norm_kernels.h"]
OWN_HEADERS = {"residual_norm.hip": _RESIDUAL_NORM, "residual_norm_bf16.hip": _RESIDUAL_NORM,
               "residual_norm_f16.hip": _RESIDUAL_NORM, "residual_norm_f32.hip": _RESIDUAL_NORM,
               "grad_clip.hip": ["grad_clip.h"], "bindings.cpp": ["residual_norm.h", "grad_clip.h", "tensor_keys.h"]}


def so_path() -> str:
  return os.path.join(HERE, "_dtf_native" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))


def _includes():
  import pybind11  # pylint: disable=import-outside-toplevel
  torch = os.path.dirname(importlib.util.find_spec("torch").origin)
  return ["-I" + sysconfig.get_paths()["include"], "-I" + pybind11.get_include(), "-I" + CSRC,
          "-I" + os.path.join(torch, "include")]


def _stale(target, deps, cmd):
  """Whether `target` is missing, older than what it is made of, or was made by another command: objects of other
  flags are not linked with today's."""
  if not os.path.exists(target):
    return True
  t = os.path.getmtime(target)
  if any(os.path.getmtime(d) > t for d in deps):
    return True
  try:
    with open(_command_file(target)) as f:
      return f.read() != "\n".join(cmd)
  except OSError:
    return True


def _command_file(target):
  return os.path.join(OBJ, os.path.basename(target) + ".cmd")


def _run(cmd, target, what):
  r = subprocess.run(cmd, capture_output=True, text=True)
  if r.returncode != 0:
    raise RuntimeError("%s:\n%s\n%s" % (what, r.stdout, r.stderr))
  with open(_command_file(target), "w") as f:
    f.write("\n".join(cmd))


def _compile(src, force):
  obj = os.path.join(OBJ, os.path.splitext(src)[0] + ".o")
  deps = [os.path.join(CSRC, src)] + [os.path.join(CSRC, h) for h in HEADERS + OWN_HEADERS.get(src, [])]
  cmd = ["hipcc", "--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden"] + NO_PACKED_FP32 + [
      "-x", "hip", "-c", os.path.join(CSRC, src), "-o", obj] + _includes()
  if not force and not _stale(obj, deps, cmd):
    return obj, False
  _run(cmd, obj, "hipcc failed for " + src)
  return obj, True


def data_so_path() -> str:
  return os.path.join(HERE, "_dtf_data" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))


def build_data(force: bool = False, verbose: bool = True) -> str:
  """Host-only module `_dtf_data` (input pipeline): plain g++, no GPU code."""
  src = os.path.join(CSRC, "data_loader.cpp")
  target = data_so_path()
  cmd = ["g++", "-O3", "-std=c++17", "-shared", "-fPIC", "-pthread", "-fvisibility=hidden",
         src, "-o", target, "-ldl"] + _includes()
  os.makedirs(OBJ, exist_ok=True)
  if force or _stale(target, [src, os.path.join(CSRC, "jpeg_region.h")], cmd):
    _run(cmd, target, "g++ failed for data_loader.cpp")
    if verbose:
      print("built", target)
  elif verbose:
    print("up to date:", target)
  return target


def build(force: bool = False, jobs: int = 4, verbose: bool = True) -> str:
  os.makedirs(OBJ, exist_ok=True)
  build_data(force, verbose)
  with concurrent.futures.ThreadPoolExecutor(max_workers=max(1, jobs)) as ex:
    results = list(ex.map(lambda s: _compile(s, force), SOURCES))
  objs = [o for o, _ in results]
  target = so_path()
  cmd = ["hipcc", "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", target] + objs
  if force or any(c for _, c in results) or _stale(target, objs, cmd):
    _run(cmd, target, "link failed")
    if verbose:
      print("built", target)
  elif verbose:
    print("up to date:", target)
  return target


if __name__ == "__main__":
  ap = argparse.ArgumentParser()
  ap.add_argument("--force", action="store_true")
  ap.add_argument("--jobs", type=int, default=4)
  a = ap.parse_args()
  build(a.force, a.jobs)
