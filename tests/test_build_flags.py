"""Other builds of a kernel source (A/B variants, resource tables) use the flags and the objects of the library: no GPU, no compiler."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "timeautodiff_amd", "csrc")


def make(target):
    return subprocess.run(["make", "-s", "-C", CSRC, target], capture_output=True, text=True, check=True).stdout.split()


def test_variants_are_built_like_the_library():
    env = dict(os.environ, HIPCC="echo")              # the commands, not run
    out = subprocess.run(["bash", os.path.join(ROOT, "scripts", "build_variant.sh"), "x", "mm16.hip", "mm16", "-DY=1"], capture_output=True, text=True,
                         check=True, env=env).stdout.splitlines()
    compiled, linked = out[0].split(), out[1].split()
    assert "-packed-fp32-ops" in compiled and "-ffp-contract=off" in compiled and "-DY=1" in compiled
    objects = make("show-objects")
    assert {o[:-2] for o in objects} == {f.rsplit(".", 1)[0] for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp"))}
    assert [o for o in linked if o.endswith(".o") and "exp/" not in o] == [o for o in objects if o != "mm16.o"]


def test_every_kernel_is_compiled_without_packed_float32():
    flags = make("show-flags")
    at = flags.index("-packed-fp32-ops")
    assert flags[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"] and "--offload-arch=gfx950" in flags


def test_build_compiles_every_source_again(monkeypatch):
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "run", lambda cmd, **kw: calls.append(cmd))
    entry.build()
    monkeypatch.undo()
    assert len(calls) == 1
    plan = subprocess.run(calls[0] + ["-n"], capture_output=True, text=True, check=True).stdout
    assert all(f" -c {f} " in plan for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp")))
