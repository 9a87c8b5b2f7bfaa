"""The key-value cache's bookkeeping under AddressSanitizer and UndefinedBehaviorSanitizer: tests/test_kv_pool.py's pool tests
against the library whose host code clang instrumented, as tests/test_sanitizers.py does for the rest of the host side."""
import glob
import os

import pytest

from test_sanitizers import LIB_SAN, ROOT, _build, _child


def test_pool_bookkeeping_under_asan_ubsan():
    _build(os.path.join(ROOT, "stream-_amd"))
    rts = sorted(glob.glob("/opt/rocm/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not rts:
        pytest.skip("clang's ASan runtime is not installed")
    out = _child(rts[-1], {"ES_HIP_LIB": LIB_SAN}, ["tests/test_kv_pool.py", "-k", "not child and not refusals and not room and not grid"])
    assert "passed" in out
