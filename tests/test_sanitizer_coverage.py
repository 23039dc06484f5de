"""The host sanitizer pass (tests/sanitize) compiles every source of the library and calls every function of its header."""
import os
import re

from q8_kernels_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def read(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


def test_every_source_is_compiled():
    listed = re.search(r"^for f in (.*); do$", read("tests", "sanitize", "run.sh"), re.M).group(1).split()
    assert sorted(listed) == sorted(os.path.splitext(s)[0] for s in build.SOURCES)


def test_every_function_is_called():
    header = re.sub(r"/\*.*?\*/", "", read("include", "q8_hip.h"), flags=re.S)
    functions = set(re.findall(r"\b(q8_\w+)\s*\(", header))
    driver = re.sub(r"//.*", "", read("tests", "sanitize", "abi_driver.cpp"))
    assert len(functions) > 30 and functions <= set(re.findall(r"\b(q8_\w+)\s*\(", driver))
