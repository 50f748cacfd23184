"""Importing the package does not load the library: a process that imports it
and then rebuilds the library runs the new one, and only that."""

import subprocess
import sys

CODE = """
import cube_awq_b200, cube_awq_b200.build
from cube_awq_b200 import _lib
maps = lambda: "libcube_awq.so" in open("/proc/self/maps").read()
assert not maps()
cube_awq_b200.version()
assert maps()
"""


def test_the_library_is_loaded_by_the_first_call_not_by_the_import():
    r = subprocess.run([sys.executable, "-c", CODE], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
