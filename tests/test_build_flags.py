"""Every tool that compiles a kernel takes the product library's flags and sources from its Makefile."""
import glob
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))


def test_flags_and_sources_come_from_the_makefile():
    import build_flags
    flags = " ".join(build_flags.cxxflags())
    assert "--offload-arch=gfx950" in flags and "-Xclang -target-feature -Xclang -packed-fp32-ops" in flags
    assert sorted(build_flags.names()) == sorted(os.path.basename(f)[:-4] for f in glob.glob(os.path.join(ROOT, "med-ts-llm_amd", "csrc", "mtl_*.hip")))
    assert len(build_flags.objects("mtl_gemm")) == len(build_flags.names()) - 1


def test_no_tool_has_flags_of_its_own():
    tools = [f for d in ("tools", "tools/diag") for e in ("py", "sh") for f in glob.glob(os.path.join(ROOT, d, "*." + e))]
    compiling = [f for f in tools if re.search(r"hipcc\b.*-c\b|hipcc\b.*\"-[cS]\"|hipcc\b.*-S\b", open(f).read())]
    assert len(compiling) >= 5
    for f in compiling:
        text = open(f).read()
        assert "build_flags" in text and "-O3" not in text, f
