"""CPU: the kernel sources are what the build reads, and profiles are tied to the sources that they were measured on."""
import os

from ai2bmd_amd import build


def test_every_kernel_source_is_built():
    listed = {f for f in build.SOURCES + build.HEADERS if os.sep not in f}
    assert set(os.listdir(build.CSRC)) == listed
