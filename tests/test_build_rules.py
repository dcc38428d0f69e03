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
