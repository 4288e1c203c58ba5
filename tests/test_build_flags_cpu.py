"""No GPU code of the repository has packed fp32 arithmetic (v_pk_add / mul / fma_f32): it is not written by hand, and every line that
compiles HIP sources switches it off."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def sources():
    for top in ("tools", os.path.join("scenario-wise-rec_amd", "csrc"), "include"):
        for folder, _, names in os.walk(os.path.join(ROOT, top)):
            for n in names:
                if n.endswith((".hip", ".h", ".sh")):
                    path = os.path.join(folder, n)
                    yield os.path.relpath(path, ROOT), open(path).read()


def test_no_packed_fp32_by_hand():
    bad = [p for p, text in sources() if re.search(r'asm[^;]*"[^"]*v_pk_(add|mul|fma)_f32', text)]
    assert not bad, bad


def test_every_compile_line_switches_it_off():
    import importlib.util
    spec = importlib.util.spec_from_file_location("swr_build_native_flags", os.path.join(ROOT, "scenario-wise-rec_amd", "build_native.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    assert FLAG in " ".join(build.FLAGS)
    bad = [(p, line) for p, text in sources() for line in text.replace("\\\n", " ").split("\n")
           if re.search(r"hipcc\s+--offload-arch", line) and "-shared" not in line and FLAG not in line]
    assert not bad, bad
