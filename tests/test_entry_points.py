"""The argument kinds that the wrappers give ctypes agree with the library's sources."""
import glob
import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "ferrum_b200", "csrc", "kernels")


def declared(name):
    for f in glob.glob(os.path.join(KERNELS, "*.cu")):
        m = re.search(r"FERRUM_API int " + name + r"\((.*?)\) \{", open(f).read(), re.S)
        if m:
            return "".join("p" if "*" in a or "cudaStream_t" in a else "l" if "long long" in a else "f" if "float" in a else "i" for a in m.group(1).split(","))


@pytest.mark.parametrize("name", ["ferrum_rope_cache_write_packed", "ferrum_unpack_cache", "ferrum_attention_packed", "ferrum_sample_filtered"])
def test_argument_kinds(name):
    from ferrum_b200.ops import lib as ops
    assert ops._ARGUMENTS[name] == declared(name)


def test_every_typed_entry_point_is_looked_at():
    from ferrum_b200.ops import lib as ops
    assert all(declared(name) for name in ops._ARGUMENTS)
