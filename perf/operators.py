"""The operators around a 4-bit K/V cache, as cases that can be timed and compared.

Kinds of case:
  rope    the norm of every query and key head and the position rotation, in one pass (l3m_k_qk_norm_rope).
  append  the same on a step's fused [q | k | v] rows, K and V then stored in a 4-bit cache (l3m_k_kv4_append); the queries
          and the stored rows as the values they stand for (l3m_k_kv4_rows).
  attend  the attention of n tokens at positions pos .. pos + n - 1 over a 4-bit cache (l3m_k_kv4_attend).

The cache's formats per 32 values of a head's row (a last block may hold fewer):
  q4_0   d = (the value of largest magnitude, the first of equal ones) / -8, stored as f16; code = floor(x / d + 8.5) within
         0..15, in float32 with the reciprocal of d; value (code - 8) d.
  mxfp4  2^e with e = floor(log2 of the largest magnitude) - 2 (-126 at least); the nearest e2m1 code, the smaller on ties.
"""
import ctypes
import math

import torch

own = False

# ------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # the start of a reply of the 110M benchmark model (12 heads of 64): launches and latency
        {"name": "attend 1 of 40 q4_0", "kind": "attend", "dtype": "q4_0", "n": 1, "pos": 39, "nq": 12, "nkv": 12, "hd": 64},
        # the end of the 135M benchmark model's context (9 heads over 3)
        {"name": "attend 1 of 256 mxfp4", "kind": "attend", "dtype": "mxfp4", "n": 1, "pos": 255, "nq": 9, "nkv": 3, "hd": 64},
        # an ordinary conversation with grouped heads of 128
        {"name": "attend 1 of 4001 q4_0", "kind": "attend", "dtype": "q4_0", "n": 1, "pos": 4000, "nq": 32, "nkv": 8, "hd": 128},
        # a long document in the cache, and the longest, at an odd length
        {"name": "attend 1 of 32768 mxfp4", "kind": "attend", "dtype": "mxfp4", "n": 1, "pos": 32767, "nq": 32, "nkv": 8, "hd": 128},
        {"name": "attend 1 of 131071 q4_0", "kind": "attend", "dtype": "q4_0", "n": 1, "pos": 131070, "nq": 32, "nkv": 8, "hd": 128},
        # a few guessed tokens checked at once, a head that is no multiple of 32
        {"name": "attend 5 of 1003 hd 80", "kind": "attend", "dtype": "mxfp4", "n": 5, "pos": 998, "nq": 10, "nkv": 2, "hd": 80},
        # a prompt from the start: 480 tokens of the 135M model
        {"name": "attend prompt 480 q4_0", "kind": "attend", "dtype": "q4_0", "n": 480, "pos": 0, "nq": 9, "nkv": 3, "hd": 64},
        # a chunk of a long prompt, with what came before it in the cache
        {"name": "attend 1024 at 2999 mxfp4", "kind": "attend", "dtype": "mxfp4", "n": 1024, "pos": 2999, "nq": 32, "nkv": 8, "hd": 128},
        # one decode step's rows into the cache: the launch and its latency
        {"name": "append 1 q4_0", "kind": "append", "dtype": "q4_0", "n": 1, "pos": 255, "nq": 9, "nkv": 3, "hd": 64, "halves": False},
        # a long prompt's rows, from inside a tile of the cache on
        {"name": "append 1000 mxfp4", "kind": "append", "dtype": "mxfp4", "n": 1000, "pos": 2045, "nq": 32, "nkv": 8, "hd": 128, "halves": True},
        # norm and rotation alone (a program with a cache of its own): one token, and a prompt
        {"name": "rope 1", "kind": "rope", "n": 1, "pos": 100, "nq": 12, "nkv": 12, "hd": 64, "halves": False},
        {"name": "rope 2048", "kind": "rope", "n": 2048, "pos": 0, "nq": 32, "nkv": 8, "hd": 128, "halves": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "rope"])
    hd = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 128, 256])
    nkv = rng.choice([1, 2, 3, 4, 8, 8])
    case = {"kind": kind, "dtype": rng.choice(["q4_0", "mxfp4"]), "nq": nkv * rng.choice([1, 2, 3, 4, 4, 8]), "nkv": nkv, "hd": hd}
    width = case["nq"] * hd
    if kind == "attend":
        one = rng.random() < 0.6
        if one:
            return {**case, "n": 1, "pos": _log(rng, 1, min(131071, 131071 * 1024 // (nkv * hd))) - 1}
        # at most the work of 1024 tokens over 4023 positions of 32 heads of 128
        n = _log(rng, 2, 1024)
        most = 4096 * 3500 * 1024 // (n * width)
        return {**case, "n": n, "pos": max(0, min(_log(rng, 1, 8000) - 1, most - n))} if most > n else {**case, "n": n // 2 + 1, "pos": 0}
    if kind == "rope":
        case.pop("dtype")
    n = 1 if rng.random() < 0.3 else _log(rng, 2, min(2048, 1000 * 6144 // (width + 2 * nkv * hd)))
    return {**case, "n": n, "pos": _log(rng, 1, 4000) - 1, "halves": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------ inputs

EPS = 1e-6
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _randn(shape, seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return torch.randn(shape, generator=g, device="cuda")


def _table(case):
    """[pos + n][hd / 2][2]: cosine and sine of every position's angles, base 10000."""
    i = torch.arange(case["hd"] // 2, device="cuda", dtype=torch.float64)
    a = torch.arange(case["pos"] + case["n"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / case["hd"])
    return torch.stack([a.cos(), a.sin()], -1).float()


def _cached(case, seed):
    """K and V rows [pos + n][nkv][hd] as they enter the cache: keys of unit variance with a few wide channels."""
    shape = (case["pos"] + case["n"], case["nkv"], case["hd"])
    return _randn(shape, seed, 2) * (1 + 2 * (_randn(shape[1:], seed, 4) > 1.5)), _randn(shape, seed, 3) * 0.5


def _q(case, seed):
    return _randn((case["n"], case["nq"], case["hd"]), seed, 1)


def _rows(case, seed):
    """The fused [q | k | v] rows of a step and the norms' weights."""
    width = (case["nq"] + 2 * case["nkv"]) * case["hd"]
    return _randn((case["n"], width), seed, 1) * 1.5, 1 + 0.1 * _randn(case["hd"], seed, 2), 1 + 0.1 * _randn(case["hd"], seed, 3)


def _codes(dtype, x):
    """float32 x [..., hd] as packed codes [..., hd / 2] (value 2j low) and a scale per 32 values."""
    hd = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -hd % 32)).unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    if dtype == "q4_0":
        d = b.gather(-1, (b.abs() == amax).to(torch.uint8).argmax(-1, keepdim=True)) / -8
        r = torch.where(d != 0, 1 / d, torch.zeros_like(d))
        c = torch.floor(b * r + 8.5).clamp(0, 15).to(torch.uint8)
        s = d.to(torch.float16)
    else:
        e = (torch.frexp(amax)[1] - 3).clamp(min=-126)               # frexp: amax = m 2^e, m in [1/2, 1)
        y = torch.ldexp(b, -e)
        c = torch.zeros_like(b, dtype=torch.uint8)
        for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
            c += y.abs() > t
        c += ((y < 0) & (c > 0)).to(torch.uint8) * 8
        s = (e + 127).to(torch.uint8)
    c = c.flatten(-2)[..., :hd].unflatten(-1, (-1, 2))
    return c[..., 0] | c[..., 1] << 4, s.squeeze(-1)


def prepare(case, seed):
    s = {"case": case, "kind": case["kind"]}
    n, nq, nkv, hd, pos = (case[k] for k in ("n", "nq", "nkv", "hd", "pos"))
    if case["kind"] == "attend":
        k, v = _cached(case, seed)
        s["q"] = _q(case, seed)
        if own:
            s.update(_own_cache(case, pos + n))
            _fill(s, k, v)
            s["out"] = torch.empty_like(s["q"])
            size = s["lib"].l3m_kv4_work_bytes(ctypes.byref(s["cache"]), n, nq)
            s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
            s["size"] = size
        else:
            s["k"], s["v"] = (_codes(case["dtype"], t.transpose(0, 1)) for t in (k, v))
    else:
        s["rows"], s["wq"], s["wk"] = _rows(case, seed)
        s["table"] = _table(case)
        if own and case["kind"] == "append":
            s.update(_own_cache(case, pos + n))
            s.update(oq=torch.empty(n, nq, hd, device="cuda"), ok=torch.empty(n, nkv, hd, device="cuda"), ov=torch.empty(n, nkv, hd, device="cuda"))
        elif own:
            import l3m_amd as A
            s.update(lib=A.lib(), oq=torch.empty(n, nq, hd, device="cuda"), ok=torch.empty(n, nkv, hd, device="cuda"))
            if s["lib"].l3m_dev_init():
                raise RuntimeError("no usable device")
    if own:
        s["p"] = {name: t.data_ptr() for name, t in s.items() if isinstance(t, torch.Tensor)}
        torch.cuda.synchronize()
    return s


def _own_cache(case, cap):
    import l3m_amd as A
    lib, c = A.lib(), A.KV4()
    if lib.l3m_dev_init():
        raise RuntimeError("no usable device")
    dt = A.DTYPES[case["dtype"]]
    mem = torch.zeros(lib.l3m_kv4_bytes(dt, case["nkv"], case["hd"], cap), dtype=torch.uint8, device="cuda")
    _ok(lib, lib.l3m_kv4_init(ctypes.byref(c), dt, case["nkv"], case["hd"], cap, mem.data_ptr()))
    return {"lib": lib, "cache": c, "mem": mem}


def _fill(s, k, v):
    """A cache's earlier rows, as its writer stores them."""
    rows = torch.cat([k, v], 1).contiguous()
    torch.cuda.synchronize()
    _ok(s["lib"], s["lib"].l3m_k_kv4_append(ctypes.byref(s["cache"]), None, rows.data_ptr(), rows[0].numel(), len(rows), 0, None, None, 0.0, 0, 0, None, None))
    torch.cuda.synchronize()


# --------------------------------------------------------------------------------------------- run

def _ok(lib, rc):
    if rc:
        raise RuntimeError((lib.l3m_dev_error() or b"?").decode())


def _values(dtype, packed, scale, hd):
    """The values of packed codes [..., hd / 2] in float32."""
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    if dtype == "q4_0":
        v, s = c.float() - 8, scale.float()
    else:
        v = torch.tensor(E2M1 + [-x for x in E2M1], device=c.device)[c.long()]
        s = torch.exp2(scale.float() - 127)
    return v * s.repeat_interleave(32, -1)[..., :hd]


def _norm_rope(x, w, table, halves):
    """Head rows x [n][heads][hd] normalized and rotated, in x's type."""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    a, b = y.chunk(2, -1) if halves else (y[..., 0::2], y[..., 1::2])
    a, b = a * c - b * s, a * s + b * c
    return torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)


def run(s):
    case = s["case"]
    n, nq, nkv, hd, pos = case["n"], case["nq"], case["nkv"], case["hd"], case["pos"]
    if own:
        lib, p = s["lib"], s["p"]
        if s["kind"] == "attend":
            _ok(lib, lib.l3m_k_kv4_attend(p["out"], p["q"], ctypes.byref(s["cache"]), n, nq, pos, p["work"], s["size"], None))
            return s["out"]
        width = (nq + 2 * nkv) * hd
        if s["kind"] == "append":
            c = ctypes.byref(s["cache"])
            _ok(lib, lib.l3m_k_kv4_append(c, p["oq"], p["rows"], width, n, nq, p["wq"], p["wk"], EPS, case["halves"], pos, p["table"], None))
            _ok(lib, lib.l3m_k_kv4_rows(c, p["ok"], p["ov"], pos, n, None))
            return {"q": s["oq"], "k": s["ok"], "v": s["ov"]}
        _ok(lib, lib.l3m_k_qk_norm_rope(p["oq"], p["ok"], p["rows"], width, n, nq, nkv, hd, p["wq"], p["wk"], EPS, case["halves"], pos, p["table"], None))
        return {"q": s["oq"], "k": s["ok"]}
    if s["kind"] == "attend":
        k, v = _values(case["dtype"], *s["k"], hd), _values(case["dtype"], *s["v"], hd)              # [nkv][positions][hd]
        g, seen = nq // nkv, pos + n
        q = s["q"].view(n, nkv, g, hd).permute(1, 2, 0, 3).reshape(nkv, g * n, hd)
        sc = (q @ k.transpose(1, 2) / math.sqrt(hd)).view(nkv, g, n, seen)
        if n > 1:
            at = torch.arange(seen, device="cuda")
            sc = sc.masked_fill(at > at[pos:, None], -math.inf)
        e = torch.exp(sc - sc.amax(-1, keepdim=True))
        e = (e / e.sum(-1, keepdim=True)).view(nkv, g * n, seen)
        return (e @ v).view(nkv, g, n, hd).permute(2, 0, 1, 3).reshape(n, nq, hd)
    x = s["rows"].view(n, nq + 2 * nkv, hd)
    table = s["table"][pos:]
    q = _norm_rope(x[:, :nq], s["wq"], table, case["halves"])
    if s["kind"] == "rope":
        return {"q": q, "k": _norm_rope(x[:, nq:nq + nkv], s["wk"], table, case["halves"])}
    # the stored codes hang on which side of a border a key lies: 64 bits up to the one rounding of the row
    k = _norm_rope(x[:, nq:nq + nkv].double(), s["wk"].double(), table.double(), case["halves"]).float()
    kv = [_values(case["dtype"], *_codes(case["dtype"], t), hd) for t in (k, x[:, nq + nkv:])]
    return {"q": q, "k": kv[0], "v": kv[1]}


# -------------------------------------------------------------------------------------------- work

def work(case):
    n, nq, nkv, hd, pos = case["n"], case["nq"], case["nkv"], case["hd"], case["pos"]
    if case["kind"] == "rope":
        vals = float(n * (nq + nkv) * hd)
        return {"bytes": 8 * vals + 4 * n * hd + 8 * hd, "flops": 9 * vals}
    row = 2.0 * nkv * (hd / 2 + -(-hd // 32) * (2 if case["dtype"] == "q4_0" else 1))    # a position's K and V
    if case["kind"] == "attend":
        return {"bytes": (pos + n) * row + 8.0 * n * nq * hd, "flops": 4.0 * nq * hd * n * (pos + (n + 1) / 2)}
    # the rows in, the queries out, the cache's rows written; and read back as float32 values
    return {"bytes": 4.0 * n * (2 * nq + 2 * nkv) * hd + n * row + n * row + 8.0 * n * nkv * hd + 4.0 * n * hd + 8 * hd,
            "flops": 9.0 * n * (nq + nkv) * hd + 8.0 * n * nkv * hd}


# ------------------------------------------------------------------------------------------- exact

def _stored(dtype, x):
    """What the cache holds for float32 rows x [..., hd], in 64 bits, from the formats' definition, block by block."""
    hd, parts = x.shape[-1], []
    for b in range(0, hd, 32):
        v = x[..., b:b + 32]
        mag, first = v.abs().max(-1).values[..., None], None
        if dtype == "q4_0":
            n = v.shape[-1]
            at = torch.where(v.abs() == mag, torch.arange(n, device=v.device), torch.tensor(n, device=v.device)).min(-1).values
            first = torch.take_along_dim(v, at[..., None], -1)
            d = first / -8.0                                     # a power of two: exact
            r = (1.0 / d.double()).float()                       # one rounding, as the format defines it
            prod = (v.double() * r.double()).float()
            c = torch.floor((prod.double() + 8.5).float()).double()
            c = torch.where(first == 0, torch.full_like(c, 8.0), torch.minimum(torch.maximum(c, torch.zeros_like(c)), torch.full_like(c, 15.0)))
            parts.append((c - 8.0) * d.half().double())
        else:
            e = torch.floor(torch.log2(mag.double().clamp(min=2.0 ** -149))) - 2
            unit = torch.exp2(e.clamp(min=-126))
            grid = torch.tensor(E2M1, device=v.device, dtype=torch.float64)
            near = (v.double().abs()[..., None] - grid * unit[..., None]).abs()
            pick = near.argmin(-1)                               # the first of equals: the smaller
            parts.append(torch.sign(v.double()) * grid[pick] * unit)
    return torch.cat(parts, -1)


def _turned(x, w, case):
    """Norm and rotation of head rows x [n][heads][hd] by complex numbers, in 64 bits."""
    x, hd, n, pos = x.double(), case["hd"], case["n"], case["pos"]
    y = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
    z = torch.view_as_complex((torch.stack([y[..., :hd // 2], y[..., hd // 2:]], -1) if case["halves"] else y.reshape(n, -1, hd // 2, 2)).contiguous())
    t = torch.view_as_complex(_table(case)[pos:].double().contiguous())
    z = torch.view_as_real(z * t[:, None])
    return torch.cat([z[..., 0], z[..., 1]], -1) if case["halves"] else z.reshape(n, -1, hd)


def exact(case, seed):
    n, nq, nkv, hd, pos = case["n"], case["nq"], case["nkv"], case["hd"], case["pos"]
    if case["kind"] == "attend":
        (k, v), q = (_cached(case, seed)), _q(case, seed).double()
        out = torch.empty(n, nq, hd, device="cuda", dtype=torch.float64)
        for h in range(nkv):
            kh, vh = _stored(case["dtype"], k[:, h]), _stored(case["dtype"], v[:, h])
            for j in range(h * nq // nkv, (h + 1) * nq // nkv):
                sc = kh @ q[:, j].T / math.sqrt(hd)                   # [positions][tokens]
                if n > 1:
                    late = torch.arange(pos + n, device="cuda")[:, None] > pos + torch.arange(n, device="cuda")
                    sc[late] = -math.inf
                out[:, j] = torch.softmax(sc, 0).T @ vh
        return out
    rows, wq, wk = _rows(case, seed)
    x = rows.view(n, nq + 2 * nkv, hd)
    q, k = _turned(x[:, :nq], wq, case), _turned(x[:, nq:nq + nkv], wk, case)
    if case["kind"] == "rope":
        return {"q": q, "k": k}
    return {"q": q, "k": _stored(case["dtype"], k.float()), "v": _stored(case["dtype"], x[:, nq + nkv:])}
