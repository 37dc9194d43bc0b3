"""A kernel whose LDS limit cannot be raised at first: the call fails with its error, leaves none behind in the runtime, and the next one tries
again (no GPU needed: the runtime's calls are stood in for, and nothing is launched)."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RUNTIME = """
static int refusals = 1, last, launches, raised;
int hipFuncSetAttribute(const void* f, int attribute, int value) { return refusals-- > 0 ? last = 1 : (++raised, 0); }
int hipGetLastError(void) { int e = last; last = 0; return e; }
int hipPeekAtLastError(void) { return last; }
int hipLaunchKernel(const void* f, ...) { ++launches; return 0; }
int __hipPushCallConfiguration(long a, ...) { return 0; }
int __hipPopCallConfiguration(void* a, void* b, void* c, void* d) { return 0; }
int launched(void) { return launches; }
int limits_raised(void) { return raised; }
"""

CHILD = """
import ctypes as C, sys
sys.path.insert(0, {root!r})
runtime = C.CDLL({stub!r}, mode=C.RTLD_GLOBAL)  # before the library, whose calls it takes
from tensorrt_amd import capi
api, A = capi.api(), 0x10000
if {which!r} == "window":
    p = capi.WindowAttentionParams(q=A, k=A, v=A, out=A, cu_seqlens=A, B=2, T=9, max_tokens=5, q_heads=4, kv_heads=2, d=64, scale=0.125, left=3, right=3)
    call = lambda: api.window_attention(None, C.byref(p))
else:
    c = capi.KvCache(k=A, v=A, k_scale=A, v_scale=A, page_table=A, lengths=A, cu_seqlens=A, data_type=2, pages=9, page_tokens=16, kv_heads=2, d=128,
                     B=1, max_pages=4, max_tokens=40, T=40)
    p = capi.KvCacheAttentionParams(cache=c, q=A, out=A, q_heads=4, scale=0.125)
    call = lambda: api.kv_cache_attention(None, C.byref(p))
assert call() != 0 and "LDS" in api.last_error_str(), api.last_error_str()
assert runtime.hipPeekAtLastError() == 0 and runtime.launched() == 0
for n in (1, 2, 3):
    assert call() == 0, api.last_error_str()
    assert runtime.launched() == n and runtime.limits_raised() == 1
print("sound")
"""


@pytest.mark.parametrize("which", ["window", "cached"])
def test_a_limit_that_is_refused_once(tmp_path, which):
    source, stub = tmp_path / "runtime.c", str(tmp_path / "runtime.so")
    source.write_text(RUNTIME)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-w", "-o", stub, str(source)])
    r = subprocess.run([sys.executable, "-c", CHILD.format(root=ROOT, stub=stub, which=which)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "sound" in r.stdout, r.stdout + r.stderr
