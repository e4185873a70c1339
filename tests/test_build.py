"""What the build of the native extension takes for up to date."""
import os
import types

import pytest

from distributed_tensorflow_amd.ops import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
  """The sources as empty files, a compiler that writes its target and says what it was asked for."""
  csrc, ran = tmp_path / "csrc", []
  csrc.mkdir()
  names = build.SOURCES + build.HEADERS + sum(build.OWN_HEADERS.values(), []) + ["data_loader.cpp", "jpeg_region.h"]
  for n in set(names):
    (csrc / n).write_text("")
    os.utime(csrc / n, (1e9, 1e9))
  monkeypatch.setattr(build, "HERE", str(tmp_path))
  monkeypatch.setattr(build, "CSRC", str(csrc))
  monkeypatch.setattr(build, "OBJ", str(csrc / "build"))

  def run(cmd, **_):
    target = cmd[cmd.index("-o") + 1]
    open(target, "w").close()
    ran.append(os.path.basename(target))
    return types.SimpleNamespace(returncode=0, stdout="", stderr="")

  monkeypatch.setattr(build.subprocess, "run", run)

  def built():
    ran.clear()
    build.build(jobs=4, verbose=False)
    return sorted(ran)

  return types.SimpleNamespace(csrc=csrc, built=built)


def test_other_flags_make_objects_stale(tree, monkeypatch):
  everything = tree.built()
  objects = [n for n in everything if n.endswith(".o")]
  assert len(objects) == len(build.SOURCES) and len(everything) == len(objects) + 2
  assert tree.built() == []
  monkeypatch.setattr(build, "NO_PACKED_FP32", [])
  assert [n for n in tree.built() if n.endswith(".o")] == objects
  assert tree.built() == []
  monkeypatch.setattr(build, "ARCH", "gfx942")
  assert len(tree.built()) == len(objects) + 1                       # and the link
  assert tree.built() == []


def test_objects_of_an_unknown_command_are_stale(tree):
  """A tree whose objects are from before commands were recorded."""
  everything = tree.built()
  for n in os.listdir(tree.csrc / "build"):
    if n.endswith(".cmd"):
      os.remove(tree.csrc / "build" / n)
  assert tree.built() == everything
  assert tree.built() == []


def test_a_newer_source_or_header_is_compiled_again(tree):
  tree.built()
  later = os.path.getmtime(tree.csrc / "build" / "bn.o") + 10
  os.utime(tree.csrc / "grad_clip.h", (later, later))
  assert [n for n in tree.built() if n.endswith(".o")] == ["bindings.o", "grad_clip.o"]


def test_a_failed_compilation_is_tried_again(tree, monkeypatch):
  run = build.subprocess.run
  monkeypatch.setattr(build.subprocess, "run",
                      lambda cmd, **_: types.SimpleNamespace(returncode=1, stdout="", stderr="no"))
  with pytest.raises(RuntimeError, match="no"):
    tree.built()
  monkeypatch.setattr(build.subprocess, "run", run)
  assert len(tree.built()) == len(build.SOURCES) + 2
