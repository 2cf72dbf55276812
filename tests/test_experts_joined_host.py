"""mm_expert_joined refuses components that it has no tiles for before it looks for a tile of them (no GPU needed)."""
import os

import pytest
from test_experts_null_host import JOINED

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mace-million_amd", "lib", "libmace_million_amd.so")
pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built (python mace-million_amd/build.py)")


@pytest.mark.timeout(20)
@pytest.mark.parametrize("M", [65, 1000003, 100000007, 2 ** 31 - 1])
@pytest.mark.parametrize("k", [1, 2])
def test_many_components(M, k):
    from mace_onegpu import _lib
    assert _lib.lib().mm_expert_joined(*dict(JOINED, k=k, T=1, M=M).values()) == -3
    assert "64 components" in _lib.last_error()
