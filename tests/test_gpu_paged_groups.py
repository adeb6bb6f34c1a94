"""Groups of query heads of the paged attention that need the most shared memory."""
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu
FIFTEEN = """
import sys
sys.path[:0] = [%r, %r]
from test_gpu_paged import Pool, _check_attention
for act, cache in (("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "f32")):
    for dim, hk in ((64, 1), (40, 2)):
        _check_attention(Pool([63, 64, 65, 0, 200], 32, hk, dim, cache, seed=15), act, 15 * hk, dim ** -0.5)
"""


def test_attention_of_fifteen_heads_per_kv_head_in_a_fresh_process(cuda_ok):
    """No other group of heads has run before: what a kernel needs, its own first call asks for."""
    r = subprocess.run([sys.executable, "-c", FIFTEEN % (ROOT, ROOT + "/tests")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
