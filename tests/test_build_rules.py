"""The build's rules: what a change of the flags or of a header has to compile anew, and the probes' documented command."""
import glob
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "oi_vae_amd", "csrc")


@pytest.mark.parametrize("changed", [os.path.join(CSRC, "Makefile"), os.path.join(ROOT, "include", "oivae_hip.h"), os.path.join(CSRC, "common.h")])
def test_flags_and_headers_rebuild_every_object(changed):
  """The flags stand in the Makefile: objects of an earlier build, compiled with others, must not be linked again."""
  out = subprocess.run(["make", "-C", CSRC, "-n", "-W", changed, "all"], check=True, capture_output=True, text=True).stdout
  objects = re.search(r"^OBJS\s*:=(.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1).split()
  names = [os.path.basename(o) for o in objects] + ["mfma_decoder_waittest.o"]
  assert len(names) == 1 + len(glob.glob(os.path.join(CSRC, "*.hip")))
  for name in names:
    assert re.search(r"-c \S+ -o \S*/build/%s\b" % re.escape(name), out), name
  for target in ("liboivae_hip.so", "liboivae_hip_waittest.so", "c_host_prox"):
    assert re.search(r"-o \S*/%s\s" % re.escape(target), out + "\n"), target
  assert changed.endswith("common.h") or re.search(r"-o \S*/_tensor_lists\.so\b", out)


def _sources():
  return [f for pattern in ("oi_vae_amd/csrc/*", "tools/probe/*.hip", "examples/*") for f in glob.glob(os.path.join(ROOT, pattern)) if f.endswith((".hip", ".h", ".cpp"))]


def test_no_source_writes_packed_fp32_instructions():
  """The flags keep the compiler from forming them; by hand they do not assemble under these flags either."""
  assert len(_sources()) > 20
  for f in _sources():
    for line in open(f).read().split("\n"):
      assert not re.search(r'"[^"]*v_pk_(add|mul|fma)_f32', line), (f, line)


def test_loads_in_inline_assembly_wait_in_their_block():
  """The compiler takes an asm block's outputs as written where the block ends."""
  for f in _sources():
    for block in re.findall(r"\basm\s*(?:volatile)?\s*\((.*?)\)\s*;", open(f).read(), re.S):
      text = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', block))
      if re.search(r"\b(global_load|flat_load|buffer_load|ds_read|ds_load|s_load)\w*", text) and " lds" not in text:
        assert "s_waitcnt" in text, (f, block)


@pytest.mark.parametrize("probe", ["mfma_probe2", "mfma_probe3"])
def test_probes_build_with_the_documented_flags(probe, tmp_path):
  """The two that held packed instructions."""
  readme = open(os.path.join(ROOT, "tools", "probe", "README.md")).read()
  flags = re.search(r"`hipcc (.*?) tools/probe/X\.hip", readme).group(1).split()
  assert "-packed-fp32-ops" in flags and "--offload-arch=gfx950" in flags
  subprocess.run(["/opt/rocm/bin/hipcc"] + flags + ["--cuda-device-only", "-c", "tools/probe/%s.hip" % probe, "-o", str(tmp_path / "probe.o")],
                 check=True, cwd=ROOT, stderr=subprocess.DEVNULL)


def test_build_compiles_everything_every_time(monkeypatch):
  import __graft_entry__ as entry
  from oracle import prox_oracle
  calls = []
  monkeypatch.setattr(entry.subprocess, "check_call", lambda argv, **kw: calls.append(argv))
  monkeypatch.setattr(prox_oracle, "build", lambda force=False: calls.append(force))
  entry.build()
  assert calls[0][0] == "make" and "-B" in calls[0] and calls[1:] == [True]


def test_the_profile_stamp_covers_the_flags(tmp_path, monkeypatch):
  """A decoder built with other flags is another decoder: its profile's stamp differs; other lines of the Makefile do not matter."""
  import bench
  was = bench.decoder_source_digest()
  text = open(os.path.join(ROOT, bench.BUILD_FILE)).read()
  for change, same in ((lambda s: s.replace("COMMON := -O3", "COMMON := -O2"), False), (lambda s: s + "# more\n", True)):
    other = tmp_path / "Makefile"
    other.write_text(change(text))
    monkeypatch.setattr(bench, "BUILD_FILE", str(other))
    assert (bench.decoder_source_digest() == was) == same
