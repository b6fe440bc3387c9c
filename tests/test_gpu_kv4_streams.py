"""The calls around the 4-bit K/V cache on the library's stream (NULL) before its first call and after it was shut down, each in a process of its own."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

COMMON = """
import ctypes as C, sys
sys.path.insert(0, %r)
import l3m_amd as A
import torch
lib = A.lib()
nq, nkv, hd, cap = 4, 2, 64, 40
c = A.KV4()
mem = torch.zeros(lib.l3m_kv4_bytes(A.DTYPES["q4_0"], nkv, hd, cap), dtype=torch.uint8, device="cuda")
assert lib.l3m_kv4_init(C.byref(c), A.DTYPES["q4_0"], nkv, hd, cap, mem.data_ptr()) == 0
g = torch.Generator(device="cuda")
g.manual_seed(1)
rows = torch.randn(cap, (nq + 2 * nkv) * hd, generator=g, device="cuda")
q, k, v, out = (torch.zeros(cap, h, hd, device="cuda") for h in (nq, nkv, nkv, nq))
size = lib.l3m_kv4_work_bytes(C.byref(c), cap, nq)
work = torch.empty(size, dtype=torch.uint8, device="cuda")
torch.cuda.synchronize()
def calls():
    yield lib.l3m_k_qk_norm_rope(q.data_ptr(), k.data_ptr(), rows.data_ptr(), rows.shape[1], cap, nq, nkv, hd, None, None, 0.0, 0, 0, None, None)
    yield lib.l3m_k_kv4_append(C.byref(c), q.data_ptr(), rows.data_ptr(), rows.shape[1], cap, nq, None, None, 0.0, 0, 0, None, None)
    yield lib.l3m_k_kv4_attend(out.data_ptr(), q.data_ptr(), C.byref(c), cap, nq, 0, work.data_ptr(), size, None)
    yield lib.l3m_k_kv4_rows(C.byref(c), k.data_ptr(), v.data_ptr(), 0, cap, None)
""" % str(ROOT)


def run(code):
    done = subprocess.run([sys.executable, "-u", "-c", COMMON + code], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.strip().endswith("well"), done.stdout + done.stderr


def test_first_call():
    """The first call makes the library's stream: synchronizing it waits for the calls."""
    run("""
assert not lib.l3m_dev_stream()
assert list(calls()) == [0] * 4 and lib.l3m_dev_stream()
assert lib.l3m_dev_sync() == 0
assert torch.equal(q.reshape(cap, -1), rows[:, :nq * hd]) and (v.reshape(cap, -1) - rows[:, (nq + nkv) * hd:]).abs().max() < 0.6 and v.any()
assert torch.isfinite(out).all() and (out[0] - v[0].repeat_interleave(nq // nkv, 0)).abs().max() < 1e-5
print("well")
""")


def test_after_shutdown():
    """After the shutdown the calls fail and change nothing."""
    run("""
assert lib.l3m_dev_init() == 0
lib.l3m_dev_shutdown()
for rc in calls():
    assert rc == -1 and b"shut down" in lib.l3m_dev_error(), rc
torch.cuda.synchronize()
assert not q.any() and not k.any() and not v.any() and not out.any() and not mem.any()
print("well")
""")
