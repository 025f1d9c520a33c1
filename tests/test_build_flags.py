"""The two builds of the kernels, csrc/build.py and CMakeLists.txt, give every source the same arithmetic."""
import importlib.util
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_accurate_sources_are_the_same_in_both_builds():
    spec = importlib.util.spec_from_file_location("xft_build", os.path.join(ROOT, "csrc", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    text = open(os.path.join(ROOT, "CMakeLists.txt")).read()
    assert not re.search(r"target_compile_options\([^)]*--use_fast_math", text)
    names = re.search(r'list\(FILTER XFT_FAST_SRCS EXCLUDE REGEX "/\((.*)\)\\\\\.cu\$"\)', text).group(1).split("|")
    assert {n + ".cu" for n in names} == build.ACCURATE
    assert all(os.path.exists(os.path.join(ROOT, "csrc", "kernels", n)) for n in build.ACCURATE)
