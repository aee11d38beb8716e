"""How the kernels are compiled (csrc/Makefile)."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "open_spiel-1_amd",
                    "csrc")


def test_every_unit_is_built_without_packed_float32_operations():
  """Some forms of gfx950's v_pk_{add,mul,fma}_f32 have given wrong results."""
  out = subprocess.run(["make", "-n", "-B", "-C", CSRC], check=True, capture_output=True, text=True)
  units = [line for line in out.stdout.splitlines() if " -c -o " in line]
  sources = [f for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp"))]
  assert len(units) == len(sources)
  for line in units:
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, line


def test_no_source_writes_packed_float32_operations():
  for name in os.listdir(CSRC):
    if name.endswith((".h", ".hip", ".cpp")):
      text = open(os.path.join(CSRC, name)).read()
      assert not any("v_pk_%s_f32" % op in text for op in ("add", "mul", "fma", "mov")), name


def test_a_counter_record_goes_stale_with_its_kernels_only(tmp_path, monkeypatch):
  """bench.kernel_source_hash: the sources and flags of the search kernels count,
  those of the host units and of the policy operators do not."""
  import shutil
  import sys
  sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
  import bench
  src = tmp_path / "open_spiel-1_amd" / "csrc"
  src.mkdir(parents=True)
  for name in os.listdir(CSRC):
    if os.path.isfile(os.path.join(CSRC, name)):
      shutil.copy(os.path.join(CSRC, name), src / name)
  assert bench.kernel_source_hash() == bench.kernel_source_hash()
  here = bench.kernel_source_hash()
  monkeypatch.setattr(bench, "ROOT", str(tmp_path))
  assert bench.kernel_source_hash() == here

  def changed(name, old="", new="// x\n"):
    text = (src / name).read_text()
    (src / name).write_text(text.replace(old, new, 1) if old else text + new)
    got = bench.kernel_source_hash() != here
    (src / name).write_text(text)
    return got
  for name in ("os_policy.h", "os_policy.hip", "os_policy_launch.h", "os_policy_f32.hip", "os_error.h",
               "os_engine.hip", "os_host.cpp", "os_host.h"):
    assert not changed(name), name
  assert not changed("Makefile", "POLICY := ", "POLICY := x ")
  for name in ("os_wave.h", "os_az.h", "os_kernels.h", "os_game_go.hip"):
    assert changed(name), name
  assert changed("Makefile", "-O3 -std", "-O2 -std")
  assert changed("Makefile", "-Xclang -packed-fp32-ops ", "")
