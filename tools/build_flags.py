#!/usr/bin/env python3
"""The product library's compiler flags, sources and objects, as its Makefile has them: what every tool that compiles a kernel takes, so that it looks at the code that is shipped.
usage: tools/build_flags.py flags | names"""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "med-ts-llm_amd", "csrc")


def _ask(target):
    return subprocess.run(["make", "-s", "--no-print-directory", "-C", CSRC, target], capture_output=True, text=True, check=True).stdout.split()


def cxxflags():
    return _ask("flags")


def names():
    """mtl_gemm, mtl_attention, ..."""
    return [s[:-len(".hip")] for s in _ask("sources")]


def objects(*without):
    """the built objects of all sources but the given ones (mtl_gemm, ...)"""
    return [os.path.join(ROOT, "build", "obj", n + ".o") for n in names() if n not in without]


if __name__ == "__main__":
    print(" ".join({"flags": cxxflags, "names": names}[sys.argv[1]]()))
