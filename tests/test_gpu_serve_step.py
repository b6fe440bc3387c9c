"""Many sequences served: prompts and steps through tables, rotary positions, writer and attention together, forked, cut and compacted on the way; the same
recorded into a graph and replayed, and on several streams at once."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import l3m_amd as A
from serve import PAGE, Blocks, Lists, attended, bf16, from_bf16

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


class Server:
    """What a program keeps: a cache of two layers, tables, buffers for a step's fused bf16 rows [q | k | v], a workspace; and the formulas' side of it."""

    def __init__(self, dev, seqs, nq=6, nkv=2, hd=64, pages=30, width=8, most=600, layers=2):
        self.dev, self.lib = dev, dev.lib
        self.nq, self.nkv, self.hd, self.seqs, self.most, self.layers = nq, nkv, hd, seqs, most, layers
        self.c, self.p = dev.kv8(pages, layers, nkv, hd), dev.pages(pages, seqs, width)
        self.plan = dev.rotary_plan(hd, hd // 2, True, 10000.0, "turns", 4.0, trained=512)
        self.w = (nq + 2 * nkv) * hd
        self.rows, self.out, self.prompt = (dev.alloc(2 * most * n) for n in (layers * self.w, layers * nq * hd, nq * hd))
        self.pos, self.ids, self.starts = dev.alloc(4 * most), dev.alloc(4 * seqs), dev.alloc(4 * (seqs + 1))
        self.size = self.lib.l3m_kv8_work_bytes(C.byref(self.c), most, nq)
        self.work = dev.alloc(self.size)
        self.lists, self.held = Lists(pages, seqs, width), [[[[Blocks(hd) for _ in range(nkv)] for _ in range(2)] for _ in range(layers)] for _ in range(seqs)]
        self.rng = np.random.default_rng(seqs)

    def put(self, at, x):
        assert self.lib.l3m_dev_upload(at, C.c_void_p(x.ctypes.data), x.nbytes) == 0

    def bring(self, ids, counts):
        """The batch and its rows into the program's buffers."""
        n = sum(counts)
        self.put(self.ids, np.int32(ids))
        self.put(self.starts, np.int32(np.cumsum([0] + list(counts))))
        x = bf16(self.rng.standard_normal((self.layers, n, self.w)) * 1.5)
        for layer in range(self.layers):
            self.put(self.rows + 2 * layer * self.most * self.w, x[layer])
        return A.Batch(self.ids, self.starts, len(ids), n), x

    def enqueue(self, b, stream, packed=False):
        """One step's calls."""
        lib, nq, nkv, hd, w, calls = self.lib, self.nq, self.nkv, self.hd, self.w, []
        c, p, bb = C.byref(self.c), C.byref(self.p), C.byref(b)
        calls.append(lib.l3m_k_pages_grow(p, c, bb, self.pos, stream))
        for layer in range(self.layers):
            q = self.rows + 2 * layer * self.most * w
            k, v, out = q + 2 * nq * hd, q + 2 * (nq + nkv) * hd, self.out + 2 * layer * self.most * nq * hd
            calls.append(lib.l3m_k_rotary(C.byref(self.plan), q, w, k, w, A.BF16, q, w, A.BF16, b.n, nq, nkv, self.pos, 0, stream))
            if packed and layer == 0:
                calls.append(lib.l3m_k_attend_packed(self.prompt, nq * hd, q, w, k, v, w, bb, nq, nkv, hd, stream))
            calls.append(lib.l3m_k_kv8_append(c, p, layer, k, v, w, A.BF16, bb, stream))
            calls.append(lib.l3m_k_kv8_attend(out, nq * hd, q, w, A.BF16, c, p, layer, bb, nq, 0, self.work, self.size, stream))
        assert calls == [0] * len(calls)

    def outputs(self, n):
        return np.stack([self.dev.get(self.out + 2 * layer * self.most * self.nq * self.hd, (n, self.nq, self.hd), np.uint16) for layer in range(self.layers)])

    def step(self, ids, counts, packed=False):
        b, x = self.bring(ids, counts)
        self.enqueue(b, None, packed)
        n, nq, nkv, hd = b.n, self.nq, self.nkv, self.hd
        pos, _ = self.lists.grow(ids, counts)
        self.lists.check(self.dev.pages_state(self.p))
        assert list(self.dev.get(self.pos, n, np.int32)) == pos
        got, starts = self.outputs(n), np.cumsum([0] + list(counts))
        for layer in range(self.layers):
            q, k = self.dev.rotary(self.plan, x[layer], nq, nkv, np.int32(pos), out=A.BF16)
            turned = self.dev.get(self.rows + 2 * layer * self.most * self.w, (n, self.w), np.uint16)
            assert np.array_equal(turned[:, :(nq + nkv) * hd].reshape(n, nq + nkv, hd), np.concatenate([q, k], 1))
            assert np.array_equal(turned[:, (nq + nkv) * hd:], x[layer][:, (nq + nkv) * hd:])
            q, k, v = (from_bf16(y) for y in (q, k, turned[:, (nq + nkv) * hd:].reshape(n, nkv, hd)))
            for i, s in enumerate(ids):
                part = slice(starts[i], starts[i + 1])
                for kv, y in ((0, k), (1, v)):
                    for h in range(nkv):
                        self.held[s][layer][kv][h].add(y[part, h])
                kx, vx = (np.stack([self.held[s][layer][kv][h].x for h in range(nkv)], 1) for kv in (0, 1))
                seen = [len(kx) - counts[i] + t + 1 for t in range(counts[i])]
                self.near(got[layer][part], q[part], kx, vx, seen, 2.0 ** -16)
                if packed and layer == 0:
                    self.near(self.dev.get(self.prompt, (n, nq, hd), np.uint16)[part], q[part], k[part], v[part], range(1, counts[i] + 1), 2.0 ** -8)

    @staticmethod
    def near(got, q, k, v, seen, rel):
        want, tol = attended(q, k, v, seen, rel, 2.0 ** -126)
        assert np.all(np.abs(from_bf16(got) - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol))

    def fork(self, sources, to):
        self.dev.pages_fork(self.p, sources, to)
        self.lists.fork(sources, to)
        for a, b in zip(sources, to):
            for layer in range(self.layers):
                for kv in (0, 1):
                    for h in range(self.nkv):
                        x = self.held[b][layer][kv][h]
                        x.x, x.u = self.held[a][layer][kv][h].x.copy(), list(self.held[a][layer][kv][h].u)

    def cut(self, ids, keep):
        self.dev.pages_cut(self.p, ids, keep)
        self.lists.cut(ids, keep)
        for s, n in zip(ids, keep):
            for layer in range(self.layers):
                for kv in (0, 1):
                    for h in range(self.nkv):
                        self.held[s][layer][kv][h].cut(n)

    def compact(self):
        self.dev.pages_compact(self.p, self.c)
        assert self.lists.compact()


def test_serving(dev):
    """Prompts packed, steps, continuations that share a prompt, tokens taken back, sequences that end, the pool compacted, and steps behind it."""
    s = Server(dev, 6)
    s.step([0, 1, 3], [130, 37, 250], packed=True)
    s.step([3, 0, 1], [1, 1, 1])
    s.fork([3, 3], [2, 5])
    s.step([5, 3, 0, 2], [1, 4, 1, 1])
    s.step([2, 5, 1], [2, 130, 1])
    s.cut([5, 3], [300, 249])                         # inside a block that stays
    s.step([4, 5, 3], [128, 1, 3])
    s.cut([2, 0], [0, 0])
    s.compact()
    s.lists.check(dev.pages_state(s.p))
    s.step([3, 1, 5, 0, 4], [1, 1, 1, 90, 1])
    s.step([3, 1, 5, 0, 4], [1, 1, 1, 1, 1])


def hip():
    return C.CDLL("libamdhip64.so")


def streams(n):
    out = []
    for _ in range(n):
        st = C.c_void_p()
        assert hip().hipStreamCreateWithFlags(C.byref(st), 1) == 0
        out.append(st)
    return out


def test_captured_steps(dev):
    """A step recorded once and replayed: each replay takes the lengths, pages and rows that it finds, over ends of blocks and pages, between eager calls on
    the same buffers. Beside a second program that makes the same steps by calls: the same bits."""
    counts, ids = [1, 1, 2, 1], [2, 0, 3, 1]
    one, two = Server(dev, 4, layers=1), Server(dev, 4, layers=1)
    for s in (one, two):
        b, _ = s.bring([0, 1, 2, 3], [127, 31, 254, 1])
        s.enqueue(b, None)
    st, = streams(1)
    b = A.Batch(one.ids, one.starts, len(ids), sum(counts))
    graph, ex = C.c_void_p(), C.c_void_p()
    assert hip().hipStreamBeginCapture(st, 1) == 0
    one.enqueue(b, st)
    assert hip().hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hip().hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    for i in range(6):
        one.bring(ids, counts)
        assert dev.lib.l3m_dev_sync() == 0
        if i == 3:                                    # what a replay finds changes: a sequence cut, another forked
            for s in (one, two):
                dev.pages_cut(s.p, [3, 1], [0, 20])
                dev.pages_fork(s.p, [0], [3])
        assert hip().hipGraphLaunch(ex, st) == 0 and hip().hipStreamSynchronize(st) == 0
        got = one.outputs(b.n)
        b2, _ = two.bring(ids, counts)
        two.enqueue(b2, None)
        assert np.array_equal(got, two.outputs(b2.n)) and got.any()
        for x, y in zip(*(dev.pages_state(s.p).values() for s in (one, two))):
            assert np.array_equal(x, y)
    assert hip().hipGraphExecDestroy(ex) == 0 and hip().hipGraphDestroy(graph) == 0 and hip().hipStreamDestroy(st) == 0


def test_two_streams(dev):
    """Two programs on streams of their own, at once, each with its workspace: what each gives alone."""
    servers = [Server(dev, 4, layers=1), Server(dev, 4, nq=8, nkv=1, hd=128, layers=1)]
    want = []
    for s in servers:
        b, _ = s.bring([0, 1, 2, 3], [500, 30, 60, 10])
        s.enqueue(b, None)
        assert dev.lib.l3m_dev_sync() == 0
        s.put(s.starts, np.int32([0, 1, 2, 3, 4]))
        s.batch = A.Batch(s.ids, s.starts, 4, 4)
        width = s.nq * s.hd

        def attend(stream, s=s, width=width):
            q = s.rows
            assert dev.lib.l3m_k_kv8_attend(s.out, width, q, s.w, A.BF16, C.byref(s.c), C.byref(s.p), 0, C.byref(s.batch), s.nq, 0, s.work, s.size, stream) == 0
            assert dev.lib.l3m_k_attend_packed(s.prompt, width, q, s.w, q + 2 * width, q + 2 * (width + s.nkv * s.hd), s.w, C.byref(A.Batch(None, s.starts, 4, 4)), s.nq, s.nkv, s.hd,
                                               stream) == 0
        s.attend = attend
        attend(None)
        want.append((s.outputs(4), dev.get(s.prompt, (4, width), np.uint16)))
    st = streams(2)
    for _ in range(20):
        for s, x in zip(servers, st):
            s.attend(x)
    assert hip().hipDeviceSynchronize() == 0
    for s, (o, p) in zip(servers, want):
        assert np.array_equal(s.outputs(4), o) and np.array_equal(dev.get(s.prompt, p.shape, np.uint16), p)
    for x in st:
        assert hip().hipStreamDestroy(x) == 0


CODE = """
import ctypes as C, sys
sys.path[:0] = [%r, %r]
import numpy as np
import l3m_amd as A
import torch
lib = A.lib()
first = sys.argv[1] == "first"
if not first:
    assert lib.l3m_dev_init() == 0
    lib.l3m_dev_shutdown()
x = torch.ones(4, 6 * 64, dtype=torch.bfloat16, device="cuda")
o = torch.zeros(4, 4 * 64, dtype=torch.bfloat16, device="cuda")
starts = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
mem = torch.zeros(lib.l3m_kv8_bytes(2, 1, 1, 64), dtype=torch.uint8, device="cuda")
tab = torch.zeros(lib.l3m_pages_bytes(2, 1, 2), dtype=torch.uint8, device="cuda")
work = torch.zeros(lib.l3m_kv8_work_bytes(C.byref(A.KV8(1 << 20, 2, 1, 1, 64)), 4, 4), dtype=torch.uint8, device="cuda")
f = torch.zeros(4, 64, device="cuda")
torch.cuda.synchronize()
r, c, p, b = A.Rotary(), A.KV8(), A.Pages(), A.Batch(None, starts.data_ptr(), 1, 4)
assert lib.l3m_rotary_init(C.byref(r), 64, 64, 0, 1e4, 0, 1.0, 1.0, 4.0, 1) == 0
assert lib.l3m_kv8_init(C.byref(c), 2, 1, 1, 64, mem.data_ptr()) == 0 and lib.l3m_pages_init(C.byref(p), 2, 1, 2, tab.data_ptr()) == 0
X, O, F = x.data_ptr(), o.data_ptr(), f.data_ptr()
calls = [lambda: lib.l3m_k_pages_reset(C.byref(p), None), lambda: lib.l3m_k_pages_clear(C.byref(p), None), lambda: lib.l3m_k_pages_grow(C.byref(p), C.byref(c), C.byref(b), None, None),
         lambda: lib.l3m_k_kv8_append(C.byref(c), C.byref(p), 0, X, X, 384, A.BF16, C.byref(b), None), lambda: lib.l3m_k_kv8_rows(C.byref(c), C.byref(p), 0, F, None, C.byref(b), None),
         lambda: lib.l3m_k_kv8_attend(O, 256, X, 384, A.BF16, C.byref(c), C.byref(p), 0, C.byref(b), 4, 0, work.data_ptr(), work.numel(), None),
         lambda: lib.l3m_k_attend_packed(O, 256, X, 384, X + 512, X + 640, 384, C.byref(b), 4, 1, 64, None), lambda: lib.l3m_k_pages_compact(C.byref(p), C.byref(c), None),
         lambda: lib.l3m_k_pages_fork(C.byref(p), None, None, 0, None), lambda: lib.l3m_k_pages_cut(C.byref(p), starts.data_ptr(), None, 1, None),
         lambda: lib.l3m_k_rotary(C.byref(r), O, 256, None, 0, A.BF16, X, 384, A.BF16, 4, 4, 0, None, 0, None)]
for i, call in enumerate(calls):
    rc = call()
    if first:
        assert rc == 0, (i, lib.l3m_dev_error())
    elif i != 8:
        assert rc == -1 and b"shut down" in lib.l3m_dev_error(), i
        lib.l3m_dev_clear_error()
if first:
    assert lib.l3m_dev_sync() == 0 and (f == 1).all() and o.any()
else:
    torch.cuda.synchronize()
    assert not o.any() and not f.any() and not mem.any() and not tab.any()
print("well")
""" % (str(ROOT), str(ROOT / "tests"))


@pytest.mark.parametrize("when", ["first", "after"])
def test_library_stream(when):
    """Calls without a stream make the library's if they are its first, and after its shutdown fail and change nothing; each in a process of its own."""
    done = subprocess.run([sys.executable, "-u", "-c", CODE, when], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.strip().endswith("well"), done.stdout + done.stderr
