"""The operators that serve many sequences from one paged 8-bit K/V cache, as cases that can be timed and compared.

Kinds of case:
  rotary   rotary positions of the query and key heads of fused rows (l3m_k_rotary): pairs (2i, 2i + 1) or halves, the whole head or its first part,
           frequencies scaled for long contexts, a position for each token.
  prompt   causal attention over whole prompts packed one behind the other (l3m_k_attend_packed).
  append   the K and V rows of a batch's new tokens into the cache (l3m_k_kv8_append), and the blocks that they touch read back as values (l3m_k_kv8_rows).
  attend   the attention of a batch's last tokens over the cache (l3m_k_kv8_attend).
  grow     sequences forked (l3m_k_pages_fork) and then all given room for their next tokens, shared pages copied (l3m_k_pages_grow).
  compact  the pages in use moved to the front of the pool (l3m_k_pages_compact).

The cache: pages of 128 positions. A page holds for each layer, one behind the other, nkv units [K codes 128 x HP][V codes HP x 128] (HP: hd rounded up
to 32, the rest zeros), then 8 bytes a head: K's and V's scales of the four blocks of 32 positions; a layer's part is rounded up to 256 bytes. Codes are
OCP e4m3, scales 2^(byte - 127). A block's scale is the smallest power of two, 2^-126 at least, by which its largest finite value is no more than 448; when
rows are added to a block that holds earlier ones it is the larger of the old one and theirs, and the old codes are rounded again. A value that is
not finite is NaN (code 127). The new tokens of a sequence are its last ones: its length counts them already.
"""
import ctypes
import math
import random

import torch

own = False
PAGE, BLOCK = 128, 32
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16}
SCALINGS = ["plain", "linear", "base", "index", "turns"]

# ------------------------------------------------------------------------------------------- cases


def listed():
    heads = {"nq": 32, "nkv": 8, "hd": 128}
    return [
        # one decode step of the 135M benchmark model (9 heads over 3): a launch and its latency
        {"name": "rotary 1 f32", "kind": "rotary", "from": "f32", "to": "f32", "n": 1, "first": 200, "nq": 9, "nkv": 3, "hd": 64, "rd": 64, "halves": False,
         "scaling": "plain", "base": 10000.0, "factor": 1.0, "trained": 2048},
        # packed prompts of a long-context model that turns half of each head
        {"name": "rotary 8192 bf16", "kind": "rotary", "from": "bf16", "to": "bf16", "n": 8192, "first": 100000, **heads, "rd": 64, "halves": True,
         "scaling": "index", "base": 500000.0, "factor": 16.0, "trained": 8192},
        # a few short questions for the 135M benchmark model, at odd lengths
        {"name": "prompt 5 short", "kind": "prompt", "runs": 5, "least": 1, "most": 64, "pick": 5, "nq": 9, "nkv": 3, "hd": 64},
        # prompts of many lengths in one batch
        {"name": "prompt 24 packed", "kind": "prompt", "runs": 24, "least": 16, "most": 2048, "pick": 6, **heads},
        # one long document
        {"name": "prompt 8191", "kind": "prompt", "runs": 1, "least": 8191, "most": 8191, "pick": 0, **heads},
        # a decode step of 48 conversations: one row each
        {"name": "append 48 x 1 bf16", "kind": "append", "dtype": "bf16", "runs": 48, "least": 1, "most": 3000, "count": 1, "pick": 1, **heads},
        # the prompts of six of them at once, from inside a block on, heads that are no multiple of 32
        {"name": "append 6 prompts f32", "kind": "append", "dtype": "f32", "runs": 6, "least": 700, "most": 1200, "count": 600, "pick": 2, "nq": 10, "nkv": 5, "hd": 80},
        # three guessed tokens of one conversation of the 110M benchmark model (12 heads of 64), in float32
        {"name": "attend 3 of 300 f32", "kind": "attend", "dtype": "f32", "runs": 1, "least": 300, "most": 300, "count": 3, "pick": 0, "nq": 12, "nkv": 12, "hd": 64},
        # a decode step of 64 conversations of many lengths
        {"name": "attend 64 x 1 bf16", "kind": "attend", "dtype": "bf16", "runs": 64, "least": 100, "most": 8000, "count": 1, "pick": 3, **heads},
        # a decode step at the end of a very long context
        {"name": "attend 1 of 131071 bf16", "kind": "attend", "dtype": "bf16", "runs": 1, "least": 131071, "most": 131071, "count": 1, "pick": 0, **heads},
        # four continuations of each of eight sequences tried at once, and a step of all of them
        {"name": "grow 8 forked by 4", "kind": "grow", "runs": 8, "children": 4, "least": 100, "most": 4000, "add": 1, "spare": 60, "pick": 4, "layers": 4, "nkv": 8, "hd": 64},
        # a pool that half emptied, before its tail is given back
        {"name": "compact 700 pages", "kind": "compact", "runs": 60, "least": 100, "most": 3000, "pages": 700, "pick": 5, "layers": 2, "nkv": 8, "hd": 128},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["rotary", "prompt", "prompt", "append", "attend", "attend", "attend", "grow", "compact"])
    hd = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 128, 256])
    nkv = rng.choice([1, 2, 3, 4, 8, 8])
    nq = nkv * rng.choice([g for g in (1, 2, 3, 4, 4, 5, 8) if nkv * g * hd <= 4096] or [1])
    heads, dtype, pick = {"nq": nq, "nkv": nkv, "hd": hd}, rng.choice(["f32", "bf16", "bf16"]), rng.randrange(1 << 30)
    if kind == "rotary":
        n = 1 if rng.random() < 0.2 else _log(rng, 2, min(8192, 8192 * 4096 // (nq * hd)))
        to = rng.choice(["f32", "bf16"])
        return {"kind": kind, "from": dtype, "to": to, "n": n, "first": _log(rng, 1, 131072) - 1, **heads, "rd": rng.choice([hd, hd, hd // 2, hd // 4]),
                "halves": rng.random() < 0.5, "scaling": rng.choice(SCALINGS), "base": rng.choice([10000.0, 500000.0]), "factor": rng.choice([2.0, 4.0, 8.0, 16.0]),
                "trained": rng.choice([2048, 4096, 8192])}
    if kind == "prompt":
        runs = 1 if rng.random() < 0.3 else _log(rng, 2, 32)
        most = _log(rng, 16, 8191 if runs == 1 else 2048 if runs <= 16 else 1500)
        return {"kind": kind, "runs": runs, "least": most if runs == 1 else rng.choice([0, 1, 16]), "most": most, "pick": pick, **heads}
    if kind == "append":
        runs = _log(rng, 1, 64)
        count = 1 if rng.random() < 0.4 else _log(rng, 1, min(2048, 8192 // runs))
        return {"kind": kind, "dtype": dtype, "runs": runs, "least": count, "most": count + _log(rng, 1, 2000), "count": count, "pick": pick, **heads}
    if kind == "attend":
        runs = 1 if rng.random() < 0.3 else _log(rng, 2, 64)
        most = _log(rng, 8, min(131071, 131071 * 1024 // (nkv * hd), 500000 // runs))
        count = 1 if rng.random() < 0.6 else rng.randint(1, 8)
        return {"kind": kind, "dtype": dtype, "runs": runs, "least": min(count, most) if runs > 1 else most, "most": most, "count": min(count, most), "pick": pick, **heads}
    layers = rng.choice([1, 2, 4])
    if kind == "grow":
        runs, children = _log(rng, 1, 16), rng.randint(1, 4)
        most = _log(rng, 2, 4000)
        return {"kind": kind, "runs": runs, "children": children, "least": rng.choice([1, most]), "most": most, "add": _log(rng, 1, 300),
                "spare": runs * (children + 1) * 4 + 8, "pick": pick, "layers": layers, "nkv": nkv, "hd": min(hd, 128)}
    runs = _log(rng, 2, 60)
    return {"kind": kind, "runs": runs, "least": 1, "most": _log(rng, 2, 1400), "pages": 700, "pick": pick, "layers": min(layers, 2), "nkv": nkv, "hd": min(hd, 128)}


# ------------------------------------------------------------------------------------------ inputs

def _randn(shape, seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return torch.randn(shape, generator=g, device="cuda")


def _perm(n, seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return torch.randperm(n, generator=g, device="cuda").int()


def _lengths(case):
    """A length for each run, spread over the logarithm between the case's ends."""
    r = random.Random(case["pick"])
    lens = [min(case["most"], max(case["least"], int(math.exp(r.uniform(math.log(max(case["least"], 0.5)), math.log(case["most"] + 1)))))) for _ in range(case["runs"])]
    return [max(lens[0], 1)] + lens[1:]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(counts):
    return _ints([sum(counts[:i]) for i in range(len(counts) + 1)])


def _padded(hd):
    return -(-hd // 32) * 32


def _layer_bytes(nkv, hd):
    return -(-(nkv * (256 * _padded(hd) + 8)) // 256) * 256


def _planes(mem, nkv, hd):
    """Views of units [..., layer bytes]: K codes [..., nkv, 128, HP], V codes [..., nkv, HP, 128], scales [..., nkv, 8]."""
    hp = _padded(hd)
    u = mem[..., :nkv * 256 * hp].unflatten(-1, (nkv, 2, 128 * hp))
    return u[..., 0, :].unflatten(-1, (128, hp)), u[..., 1, :].unflatten(-1, (hp, 128)), mem[..., nkv * 256 * hp:nkv * (256 * hp + 8)].unflatten(-1, (nkv, 8))


def _rows_kv(case, positions, seed):
    """K and V rows [positions][nkv][hd]: keys of unit variance with a few wide channels, values of less."""
    shape = (positions, case["nkv"], case["hd"])
    return _randn(shape, seed, 2) * (1 + 2 * (_randn(shape[1:], seed, 4) > 1.5)), _randn(shape, seed, 3) * 0.5


def _cache(s, case, seed, lens, layer):
    """A pool with the sequences' pages in no order, their positions stored in `layer`; what lies behind a length is what a page held before."""
    nkv, hd = case["nkv"], case["hd"]
    need = [-(-n // PAGE) for n in lens]
    width, used = max(need + [1]), sum(need)
    pages = used + 3
    place = _perm(pages, seed, 9)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    for i, n in enumerate(need):
        table[i, :n] = place[sum(need[:i]):sum(need[:i + 1])]
    mem = torch.zeros(pages, layer + 1, _layer_bytes(nkv, hd), dtype=torch.uint8, device="cuda")
    k, v = (x.unflatten(0, (used, PAGE)).permute(0, 2, 1, 3) for x in _rows_kv(case, used * PAGE, seed))                  # [page][nkv][128][hd]
    (kc, ks), (vc, vs) = (_stored(x.unflatten(2, (4, BLOCK))) for x in (k, v))
    to_k, to_v, to_s = _planes(mem[:, layer], nkv, hd)
    at = place[:used].long()
    to_k[at, :, :, :hd] = kc.flatten(2, 3)
    to_v[at, :, :hd] = vc.flatten(2, 3).transpose(2, 3)
    to_s[at] = torch.cat([ks, vs], -1)
    s.update(mem=mem, table=table, lens=_ints(lens), ids=_ints(list(range(len(lens)))), pages=pages, width=width, layer=layer)


def _counts(case, lens):
    return [min(case["count"], n) for n in lens]


def _batch_rows(case, lens, seed):
    """What a step brings: rows of query heads, key rows, value rows."""
    n, kind = sum(_counts(case, lens)), KINDS[case["dtype"]]
    q = _randn((n, case["nq"], case["hd"]), seed, 21)
    k, v = _randn((n, case["nkv"], case["hd"]), seed, 22) * 1.5, _randn((n, case["nkv"], case["hd"]), seed, 23) * 0.7
    return q.to(kind), k.to(kind), v.to(kind)


def _tables(s, case, lens, seqs, pages, seed):
    """Sequences' pages scattered over a pool, who holds them, and the pool."""
    need = [-(-n // PAGE) for n in lens]
    width = max(-(-(n + case.get("add", 0)) // PAGE) for n in lens) + 1
    place = _perm(pages, seed, 9)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    for i, n in enumerate(need):
        table[i, :n] = place[sum(need[:i]):sum(need[:i + 1])]
    refs[place[:sum(need)].long()] = 1
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7 + 1)
    pool = torch.randint(0, 256, (pages, case["layers"] * _layer_bytes(case["nkv"], case["hd"])), dtype=torch.uint8, device="cuda", generator=g)
    s.update(pool=pool, refs=refs, table=table, lens=_ints(lens + [0] * (seqs - len(lens))), seqs=seqs, pages=pages, width=width)


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case, "kind": kind}
    if kind == "rotary":
        s["rows"], s["pos"] = _rotary_rows(case, seed)
        s["freq"], s["mag"] = _frequencies(case)
    elif kind == "prompt":
        lens = _lengths(case)
        s["starts"], n = _starts(lens), sum(lens)
        s["q"], s["k"], s["v"] = _prompt_rows(case, n, seed)
        s["longest"], s["runs"] = max(lens), len(lens)
    elif kind in ("append", "attend"):
        lens = _lengths(case)
        counts = _counts(case, lens)
        _cache(s, case, seed, lens, layer=1)
        s["q"], s["k"], s["v"] = _batch_rows(case, lens, seed)
        s["starts"], s["most"], s["longest"], s["runs"], s["n"] = _starts(counts), max(counts), max(lens), len(lens), sum(counts)
        back = [min(n, c + BLOCK - 1) for n, c in zip(lens, counts)]          # from the first touched block's start, at the most
        s["back"], s["most_back"], s["n_back"] = _starts(back), max(back), sum(back)
    elif kind == "grow":
        lens, c = _lengths(case), case["children"]
        runs = len(lens)
        _tables(s, case, lens, runs * (c + 1), sum(-(-n // PAGE) for n in lens) + case["spare"], seed)
        s["from"], s["to"] = _ints([i for i in range(runs) for _ in range(c)]), _ints(list(range(runs, runs * (c + 1))))
        ids = list(range(runs, runs * (c + 1))) + list(range(runs))
        s["ids"], s["starts"] = _ints(ids), _starts([case["add"]] * len(ids))
        s["n"] = case["add"] * len(ids)
    else:
        lens = _lengths(case)
        while sum(-(-n // PAGE) for n in lens) > case["pages"] * 3 // 4:
            lens.pop()
        _tables(s, case, lens, len(lens), case["pages"], seed)
    if own:
        _own_state(s)
    torch.cuda.synchronize()
    return s


def _rotary_rows(case, seed):
    """Fused rows and their positions: packed sequences, so positions that start again."""
    rows = _randn((case["n"], (case["nq"] + 2 * case["nkv"]) * case["hd"]), seed, 1).to(KINDS[case["from"]])
    return rows, (torch.arange(case["n"], device="cuda") % (seed % 97 + 1001) + case["first"]).int()


def _prompt_rows(case, n, seed):
    """Fused rows' three parts, as the projection leaves them: views of one tensor."""
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    x = _randn((n, nq + 2 * nkv, hd), seed, 1).bfloat16()
    return x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]


def _own_state(s):
    """The handles that a program keeps beside its data: structs over its device memory, outputs and a workspace."""
    import l3m_amd as A
    case, lib = s["case"], A.lib()
    s["A"], s["lib"] = A, lib
    if lib.l3m_dev_init():
        raise RuntimeError("no usable device")
    nkv, hd = case["nkv"], case["hd"]
    if s["kind"] == "rotary":
        s["plan"] = A.Rotary()
        _ok(lib, lib.l3m_rotary_init(ctypes.byref(s["plan"]), hd, case["rd"], case["halves"], case["base"], SCALINGS.index(case["scaling"]), case["factor"], LOW,
                                     HIGH[case["scaling"]], case["trained"]))
        s["oq"], s["ok"] = (torch.empty(case["n"], h, hd, dtype=KINDS[case["to"]], device="cuda") for h in (case["nq"], nkv))
        return
    if s["kind"] == "prompt":
        s["batch"] = A.Batch(None, s["starts"].data_ptr(), s["runs"], len(s["q"]))
        s["out"] = torch.empty(s["q"].shape, dtype=torch.bfloat16, device="cuda")
        return
    s["cache"], s["tables"] = A.KV8(), A.Pages()
    mem, layers = (s["mem"], s["layer"] + 1) if "mem" in s else (s["pool"], case["layers"])
    _ok(lib, lib.l3m_kv8_init(ctypes.byref(s["cache"]), s["pages"], layers, nkv, hd, mem.data_ptr()))
    seqs = len(s["lens"])
    held = torch.zeros(lib.l3m_pages_bytes(s["pages"], seqs, s["width"]), dtype=torch.uint8, device="cuda")
    _ok(lib, lib.l3m_pages_init(ctypes.byref(s["tables"]), s["pages"], seqs, s["width"], held.data_ptr()))
    _ok(lib, lib.l3m_k_pages_reset(ctypes.byref(s["tables"]), None))
    _ok(lib, lib.l3m_dev_sync())
    s["held"] = held
    for name, field in (("table", "table"), ("refs", "refs"), ("lens", "len")):
        if name in s:
            _ints_at(s, field, s[name].numel()).copy_(s[name].flatten())
    if s["kind"] in ("append", "attend"):
        s["batch"] = A.Batch(s["ids"].data_ptr(), s["starts"].data_ptr(), s["runs"], s["n"])
        if s["kind"] == "append":
            s["batch_back"] = A.Batch(s["ids"].data_ptr(), s["back"].data_ptr(), s["runs"], s["n_back"])
            s["out_k"], s["out_v"] = (torch.empty(s["n_back"], nkv, hd, device="cuda") for _ in range(2))
        else:
            s["size"] = lib.l3m_kv8_work_bytes(ctypes.byref(s["cache"]), s["n"], case["nq"])
            s["work"] = torch.empty(s["size"], dtype=torch.uint8, device="cuda")
            s["out"] = torch.empty_like(s["q"])
        return
    s["saved"] = held.clone()
    if s["kind"] == "grow":
        s["batch"] = A.Batch(s["ids"].data_ptr(), s["starts"].data_ptr(), len(s["ids"]), s["n"])
        s["out_pos"] = torch.empty(s["n"], dtype=torch.int32, device="cuda")


def _ints_at(s, field, n):
    """A plane of the tables as a tensor."""
    at = (getattr(s["tables"], field) - s["held"].data_ptr())
    return s["held"][at:at + 4 * n].view(torch.int32)


# --------------------------------------------------------------------------------------------- run

LOW, HIGH = 1.0, {"plain": 4.0, "linear": 4.0, "base": 4.0, "index": 32.0, "turns": 4.0}


def _ok(lib, rc):
    if rc:
        raise RuntimeError((lib.l3m_dev_error() or b"?").decode())


def _frequencies(case):
    """Radians per position of each pair, and what the turned values are multiplied by: a model's plan, made once."""
    rd, base, factor, trained = case["rd"], case["base"], case["factor"], case["trained"]
    if case["scaling"] == "base":
        base = base * factor ** (rd / (rd - 2))
    i = torch.arange(rd // 2, device="cuda", dtype=torch.float64)
    f = base ** (-2 * i / rd)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "index":
        at = [rd * math.log(trained / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (HIGH["index"], LOW)]
        a, b = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rd - 1)
        slow = ((i - a) / max(b - a, 0.001)).clamp(0, 1)
        f = f * (1 - slow) + f / factor * slow
    if case["scaling"] == "turns":
        keep = ((trained * f / (2 * math.pi) - LOW) / (HIGH["turns"] - LOW)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f, 0.1 * math.log(factor) + 1 if case["scaling"] == "index" else 1.0


def _e4m3(x):
    """The nearest e4m3 value's code for float32 x of at most 448 in size, ties to even; what is not finite is NaN."""
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    e = torch.frexp(a.clamp(min=2.0 ** -6))[1] - 4                 # a value's last place is 2^e
    m = torch.round(a * _pow2(-e)).int()                           # 0 .. 16; 16 of one exponent is 8 of the next
    code = (e + 9) * 8 + m + 128 * ((x < 0) & (m > 0)).int()
    return torch.where(torch.isfinite(x), code, torch.full_like(code, 127)).to(torch.uint8)


def _pow2(e):
    """2^e of whole e, -126 .. 127, as float32."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _scale(x, dims):
    """The exponent byte of float32 x's largest finite magnitude over `dims`."""
    m = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)
    f, e = torch.frexp(m)                                          # m = f 2^e, f in [1/2, 1)
    e = torch.where(m > 0, e - 9 + (f > 0.875).int(), torch.full_like(e, -126)).clamp(min=-126)
    return e + 127


def _value(code):
    """e4m3 codes as float32."""
    c = code.int()
    e, m = c >> 3 & 15, c & 7
    v = torch.where(e > 0, (m + 8).float() * _pow2(e - 10), m.float() / 512)
    v = torch.where((c & 127) == 127, torch.full_like(v, math.nan), v)
    return torch.where(c >= 128, -v, v)


def _stored(x):
    """Blocks of rows x [..., 32, hd] as codes and a scale byte each."""
    b = _scale(x, (-1, -2))
    return _e4m3(x * _pow2(127 - b)[..., None, None]), b.to(torch.uint8)


def _sequences(s):
    """The batch's sequences as values k, v [runs][nkv][positions][hd], positions a whole number of pages."""
    case, hd = s["case"], s["case"]["hd"]
    kc, vc, sc = _planes(s["mem"][s["table"][s["ids"].long()].long().clamp(min=0), s["layer"]], case["nkv"], hd)      # [runs][width][nkv]..
    sc = _pow2(sc.int() - 127).repeat_interleave(BLOCK, -1)                                                                     # [runs][width][nkv][256]
    k = _value(kc[..., :hd]) * sc[..., :128, None]
    v = _value(vc[..., :hd, :]).transpose(-1, -2) * sc[..., 128:, None]
    return [x.transpose(1, 2).flatten(2, 3) for x in (k, v)]


def _spread(x, starts, most):
    """Packed rows as [runs][most]..., and which of them there are."""
    at = starts[:-1, None].long() + torch.arange(most, device="cuda")
    there = at < starts[1:, None]
    return x[at.clamp(max=len(x) - 1)], there


def _softmax_values(sc, hidden, v):
    sc = sc.masked_fill(hidden, -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    return (e @ v) / e.sum(-1, keepdim=True)


def run(s):
    case, kind = s["case"], s["kind"]
    nkv, hd = case["nkv"], case["hd"]
    if own:
        return _own_run(s)
    if kind == "rotary":
        n, nq, rd = case["n"], case["nq"], case["rd"]
        x = s["rows"].view(n, nq + 2 * nkv, hd)[:, :nq + nkv].float()
        a = s["pos"][:, None].double() * s["freq"]
        c, t = (f(a).float()[:, None] * s["mag"] for f in (torch.cos, torch.sin))
        u, w = (x[..., :rd // 2], x[..., rd // 2:rd]) if case["halves"] else (x[..., 0:rd:2], x[..., 1:rd:2])
        u, w = u * c - w * t, u * t + w * c
        y = torch.cat([torch.cat([u, w], -1) if case["halves"] else torch.stack([u, w], -1).flatten(-2), x[..., rd:]], -1).to(KINDS[case["to"]])
        return {"q": y[:, :nq], "k": y[:, nq:]}
    if kind == "prompt":
        nq, most = case["nq"], s["longest"]
        (q, there), (k, _), (v, _) = (_spread(x, s["starts"], most) for x in (s["q"], s["k"], s["v"]))                  # [runs][most][heads][hd]
        g = nq // nkv
        q, k, v = (x.float().transpose(1, 2) for x in (q, k, v))
        q = q.unflatten(1, (nkv, g))
        at = torch.arange(most, device="cuda")
        o = _softmax_values(q @ k[:, :, None].transpose(-1, -2) / math.sqrt(hd), at > at[:, None], v[:, :, None])       # [runs][nkv][g][most][hd]
        return o.flatten(1, 2).transpose(1, 2)[there].bfloat16()
    if kind == "append":
        most, starts = s["most"], s["starts"]
        lens, counts = s["lens"][s["ids"].long()], starts[1:] - starts[:-1]
        first = lens - counts                                                                                           # the first new position
        block0 = first // BLOCK
        blocks = (most + 2 * BLOCK - 2) // BLOCK
        pos = block0[:, None] * BLOCK + torch.arange(blocks * BLOCK, device="cuda")                                     # the touched blocks' positions
        new = (pos >= first[:, None]) & (pos < lens[:, None])
        page = s["table"][s["ids"].long()].gather(1, (pos // PAGE).clamp(max=s["width"] - 1).long()).long().clamp(min=0)
        kc, vc, sc = _planes(s["mem"][:, s["layer"]], nkv, hd)
        rows = (starts[:-1, None] + pos - first[:, None]).clamp(0, s["n"] - 1).long()
        fresh_block = ~((pos < first[:, None]).unflatten(1, (blocks, BLOCK)).any(-1))                                   # [runs][blocks]
        back, back_there = s["back"], s["back"][:-1, None].long() + torch.arange(s["most_back"], device="cuda") < s["back"][1:, None]
        at_back = (lens - (back[1:] - back[:-1]))[:, None] + torch.arange(s["most_back"], device="cuda")
        out = {}
        for name, x, codes, part in (("k", s["k"], kc, 0), ("v", s["v"], vc.transpose(-1, -2), 4)):
            old = codes[page, :, (pos % PAGE).long()][..., :hd]                                                         # [runs][positions][nkv][hd]
            byte = sc[page, :, (part + pos % PAGE // BLOCK).long()].int()[:, ::BLOCK]                                   # [runs][blocks][nkv]
            vals = torch.where(new[..., None, None], x[rows].float(), torch.zeros((), device="cuda")).unflatten(1, (blocks, BLOCK))
            need = _scale(vals, (2, 4))
            held = torch.where(fresh_block[..., None], need, torch.maximum(need, byte))
            up = _pow2(127 - held)[:, :, None, :, None]
            moved = _value(old) * _pow2((byte - held).clamp(-126, 127)).repeat_interleave(BLOCK, 1)[..., None]             # the old codes' values in the new scale
            code = torch.where(new[..., None, None], _e4m3(vals * up).flatten(1, 2), _e4m3(moved))
            y = _value(code) * _pow2(held - 127).repeat_interleave(BLOCK, 1)[..., None]                                      # [runs][positions][nkv][hd]
            # read back: the touched blocks' as they are now, positions before them as they were
            within = at_back - (block0 * BLOCK)[:, None]
            now = y.gather(1, within.clamp(0, blocks * BLOCK - 1).long()[..., None, None].expand(-1, -1, nkv, hd))
            page_b = s["table"][s["ids"].long()].gather(1, (at_back // PAGE).clamp(0, s["width"] - 1).long()).long().clamp(min=0)
            was = _value(codes[page_b, :, (at_back % PAGE).long()][..., :hd]) * _pow2(sc[page_b, :, (part + at_back % PAGE // BLOCK).long()].int() - 127)[..., None]
            out[name] = torch.where((within >= 0)[..., None, None], now, was)[back_there]
        return out
    if kind == "attend":
        nq, most = case["nq"], s["most"]
        g = nq // nkv
        k, v = _sequences(s)
        q, there = _spread(s["q"], s["starts"], most)
        q = q.float().transpose(1, 2).unflatten(1, (nkv, g)).flatten(2, 3)                                              # [runs][nkv][g most][hd]
        lens, counts = s["lens"][s["ids"].long()], s["starts"][1:] - s["starts"][:-1]
        seen = (lens - counts)[:, None] + torch.arange(most, device="cuda") + 1                                         # [runs][most]
        hidden = torch.arange(k.shape[2], device="cuda") >= seen[..., None]
        v = v.masked_fill((torch.arange(k.shape[2], device="cuda") >= lens[:, None])[:, None, :, None], 0)
        o = _softmax_values(q @ k.transpose(-1, -2) / math.sqrt(hd), hidden[:, None].repeat(1, 1, g, 1), v)
        return o.unflatten(2, (g, most)).flatten(1, 2).transpose(1, 2)[there].to(KINDS[case["dtype"]])
    if kind == "grow":
        refs, table, lens = s["refs"].clone(), s["table"].clone(), s["lens"].clone()
        src, dst = s["from"].long(), s["to"].long()
        table[dst], lens[dst] = table[src], lens[src]
        _hold(refs, table[dst], 1)
        ids, add = s["ids"].long(), s["starts"][1:] - s["starts"][:-1]
        was = lens[ids]
        pos = was.repeat_interleave(add) + torch.arange(s["n"], device="cuda", dtype=torch.int32) - s["starts"][:-1].repeat_interleave(add)
        last = table[ids].gather(1, (was // PAGE).long()[:, None])[:, 0]
        split = (was % PAGE > 0) & (add > 0)                                                        # rows that go into a page that has some
        page = torch.where(split, last, torch.zeros_like(last)).long()
        sharers = torch.zeros_like(refs).index_add_(0, page, split.int())
        i = torch.arange(len(ids), device="cuda")
        keeper = torch.full((len(refs),), len(ids), device="cuda").scatter_reduce_(0, page, torch.where(split, i, len(ids)), "amin")
        keeps = (refs[page] == 1) | ((sharers[page] == refs[page]) & (keeper[page] == i))           # where all holders grow, the first in the list keeps it
        copy = split & ~keeps
        more = -(-(was + add) // PAGE) - -(-was // PAGE) + copy.int()
        begin = more.cumsum(0) - more
        free = (refs == 0).nonzero()[:, 0].int()
        slot = torch.arange(table.shape[1], device="cuda")
        from_ = torch.where(copy, was // PAGE, -(-was // PAGE))[:, None]
        taken = (slot >= from_) & (slot < from_ + more[:, None])
        fresh = free[(begin[:, None] + slot - from_).clamp(0, len(free) - 1).long()]
        refs.index_add_(0, page, -copy.int())
        refs.index_add_(0, fresh.flatten().long(), taken.flatten().int())
        table[ids] = torch.where(taken, fresh, table[ids])
        lens[ids] = was + add
        to = fresh.gather(1, (was // PAGE).long()[:, None])[:, 0]
        s["pool"][to[copy].long()] = s["pool"][page[copy]]
        return {"refs": refs, "table": table, "lens": lens, "pos": pos, "pool": s["pool"]}
    refs, table = s["refs"], s["table"]
    live = (refs > 0).sum()
    i = torch.arange(len(refs), device="cuda")
    mover, hole = ((refs > 0) & (i >= live)).nonzero()[:, 0], ((refs == 0) & (i < live)).nonzero()[:, 0]
    s["pool"][hole] = s["pool"][mover]
    to = i.int()
    to[mover] = hole.int()
    table = torch.where(table >= 0, to[table.clamp(min=0).long()], table)
    return {"refs": torch.where(i < live, refs[torch.where(i < live, i, 0)], 0).index_copy(0, hole, refs[mover]), "table": table, "pool": s["pool"]}


def _hold(refs, table, by):
    """`by` more holders of the pages of some rows of the table."""
    refs.index_add_(0, table.flatten().clamp(min=0).long(), by * (table >= 0).flatten().int())


def _own_run(s):
    case, kind, lib = s["case"], s["kind"], s["lib"]
    nkv, hd, byref = case["nkv"], case["hd"], ctypes.byref
    if kind == "rotary":
        f, t = s["A"].DTYPES[case["from"]], s["A"].DTYPES[case["to"]]
        _ok(lib, lib.l3m_k_rotary(byref(s["plan"]), s["oq"].data_ptr(), case["nq"] * hd, s["ok"].data_ptr(), nkv * hd, t, s["rows"].data_ptr(), s["rows"].stride(0), f,
                                  case["n"], case["nq"], nkv, s["pos"].data_ptr(), 0, None))
        return {"q": s["oq"], "k": s["ok"]}
    if kind == "prompt":
        q = s["q"]
        _ok(lib, lib.l3m_k_attend_packed(s["out"].data_ptr(), case["nq"] * hd, q.data_ptr(), q.stride(0), s["k"].data_ptr(), s["v"].data_ptr(), s["k"].stride(0),
                                         byref(s["batch"]), case["nq"], nkv, hd, None))
        return s["out"]
    c, p = byref(s["cache"]), byref(s["tables"])
    if kind == "append":
        dt = s["A"].DTYPES[case["dtype"]]
        _ok(lib, lib.l3m_k_kv8_append(c, p, s["layer"], s["k"].data_ptr(), s["v"].data_ptr(), nkv * hd, dt, byref(s["batch"]), None))
        _ok(lib, lib.l3m_k_kv8_rows(c, p, s["layer"], s["out_k"].data_ptr(), s["out_v"].data_ptr(), byref(s["batch_back"]), None))
        return {"k": s["out_k"], "v": s["out_v"]}
    if kind == "attend":
        dt, width = s["A"].DTYPES[case["dtype"]], case["nq"] * hd
        _ok(lib, lib.l3m_k_kv8_attend(s["out"].data_ptr(), width, s["q"].data_ptr(), width, dt, c, p, s["layer"], byref(s["batch"]), case["nq"], s["longest"],
                                      s["work"].data_ptr(), s["size"], None))
        return s["out"]
    # the tables as a program's snapshot has them, so that each pass does the same
    _ok(lib, lib.l3m_dev_copy(s["held"].data_ptr(), s["saved"].data_ptr(), s["held"].numel(), None))
    if kind == "grow":
        _ok(lib, lib.l3m_k_pages_fork(p, s["from"].data_ptr(), s["to"].data_ptr(), len(s["to"]), None))
        _ok(lib, lib.l3m_k_pages_grow(p, c, byref(s["batch"]), s["out_pos"].data_ptr(), None))
    else:
        _ok(lib, lib.l3m_k_pages_compact(p, c, None))
    got = {"refs": _ints_at(s, "refs", s["pages"]), "table": _ints_at(s, "table", s["seqs"] * s["width"]).view(s["seqs"], s["width"]), "pool": s["pool"]}
    return {**got, "lens": _ints_at(s, "len", s["seqs"]), "pos": s["out_pos"]} if kind == "grow" else got


# -------------------------------------------------------------------------------------------- work

def work(case):
    kind, nkv, hd = case["kind"], case["nkv"], case["hd"]
    size = {"f32": 4.0, "bf16": 2.0}
    if kind == "rotary":
        vals = float(case["n"] * (case["nq"] + nkv) * hd)
        return {"bytes": (size[case["from"]] + size[case["to"]]) * vals + 4.0 * case["n"], "flops": 6.0 * vals * case["rd"] / hd}
    if kind in ("grow", "compact"):
        page = float(case["layers"] * _layer_bytes(nkv, hd))
        lens = _lengths(case)
        if kind == "compact":
            while sum(-(-n // PAGE) for n in lens) > case["pages"] * 3 // 4:
                lens.pop()
            live = sum(-(-n // PAGE) for n in lens)
            return {"bytes": 2 * page * live * (1 - live / case["pages"]) + 12.0 * case["pages"], "flops": 0.0}      # the share of them behind the front
        copies = sum(n % PAGE > 0 for n in lens) * case["children"]
        return {"bytes": 2 * page * copies + 8.0 * sum(-(-n // PAGE) for n in lens) * case["children"], "flops": 0.0}
    lens = _lengths(case)
    if kind == "prompt":
        pairs = sum(n * (n + 1) / 2 for n in lens)
        return {"bytes": 4.0 * sum(lens) * hd * (case["nq"] + nkv), "flops": 4.0 * pairs * case["nq"] * hd}
    counts, s = _counts(case, lens), size[case["dtype"]]
    position = 2.0 * nkv * (hd + 1 / BLOCK)                                                                          # bytes of a position's K and V
    if kind == "append":
        back = sum(min(n, c + BLOCK - 1) for n, c in zip(lens, counts))
        vals = 2.0 * nkv * hd
        return {"bytes": sum(counts) * (s * vals + position) + back * (4 * vals + position), "flops": 3.0 * sum(counts) * vals}
    pairs = sum(c * n - c * (c - 1) / 2 for n, c in zip(lens, counts))
    return {"bytes": sum(lens) * position + 2 * s * sum(counts) * case["nq"] * hd, "flops": 4.0 * pairs * case["nq"] * hd}


# ------------------------------------------------------------------------------------------- exact

def _grid():
    """All e4m3 values from the format's definition: sign, four bits of exponent with bias 7, three of fraction; 0x7F is NaN."""
    v = []
    for c in range(128):
        e, m = divmod(c, 8)
        v.append(math.nan if c == 127 else (1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6)
    return torch.tensor(v + [-x for x in v], dtype=torch.float64, device="cuda")


def _nearest(x):
    """The e4m3 value nearest to x in 64 bits, of two the one with an even code, by a search of the format's values."""
    g = _grid()[:127]
    a = x.abs().contiguous()
    hi = torch.searchsorted(g, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - g[lo], g[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.where(x < 0, -g[pick], g[pick])


def _unit(x):
    """2^e of a block by its definition: the smallest power of two from 2^-126 up by which its largest magnitude is at most 448."""
    m = float(x.abs().max()) if x.numel() else 0.0
    e = -126
    if m > 0:
        e = max(-126, math.ceil(math.log2(m / 448)) - 1)
        while m > 448 * 2.0 ** e:
            e += 1
    return 2.0 ** e


def exact(case, seed):
    kind, nkv, hd = case["kind"], case["nkv"], case["hd"]
    if kind == "rotary":
        rd, nq = case["rd"], case["nq"]
        rows, pos = _rotary_rows(case, seed)
        x = rows.double().view(case["n"], -1, hd)[:, :nq + nkv]
        part = x[..., :rd]
        z = torch.view_as_complex((torch.stack([part[..., :rd // 2], part[..., rd // 2:]], -1) if case["halves"] else part.unflatten(-1, (-1, 2))).contiguous())
        f, mag = _frequencies(case)
        a = pos[:, None].double() * f
        z = z * torch.polar(torch.full_like(a, mag), a)[:, None]
        z = torch.view_as_real(z)
        y = torch.cat([torch.cat([z[..., 0], z[..., 1]], -1) if case["halves"] else z.flatten(-2), x[..., rd:]], -1)
        return {"q": y[:, :nq], "k": y[:, nq:]}
    if kind in ("grow", "compact"):
        return None
    lens = _lengths(case)
    if kind == "prompt":
        q, k, v = (x.double() for x in _prompt_rows(case, sum(lens), seed))
        out, g, at = torch.empty(q.shape, dtype=torch.float64, device="cuda"), case["nq"] // nkv, 0
        for n in lens:
            late = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            for h in range(case["nq"]):
                w = q[at:at + n, h] @ k[at:at + n, h // g].T / math.sqrt(hd)
                w[late] = -math.inf
                out[at:at + n, h] = torch.softmax(w, -1) @ v[at:at + n, h // g]
            at += n
        return out
    need = [-(-n // PAGE) for n in lens]
    counts = _counts(case, lens)
    old = _rows_kv(case, sum(need) * PAGE, seed)
    q, k, v = _batch_rows(case, lens, seed)
    if kind == "append":
        if sum(counts) + 64 * len(lens) > 6000:
            return None
        out = {"k": [], "v": []}
        for name, x, was in (("k", k, old[0]), ("v", v, old[1])):
            for i, (n, c) in enumerate(zip(lens, counts)):
                base, row = sum(need[:i]) * PAGE, sum(counts[:i])
                for b in range((n - min(n, c + BLOCK - 1)) // BLOCK * BLOCK, n, BLOCK):
                    got = torch.zeros(BLOCK, nkv, hd, dtype=torch.float64, device="cuda")
                    for h in range(nkv):
                        before, end = max(0, min(BLOCK, n - c - b)), min(BLOCK, n - b)
                        # what the block was stored as, then with the new rows in it
                        whole = was[base + b:base + b + BLOCK, h].double()
                        u = _unit(whole)
                        held = _nearest(whole / u) * u
                        new = x[row + b + before - (n - c):row + b + end - (n - c), h].double() if before < end else held[:0]
                        if len(new):
                            w = max(_unit(new), u) if before else _unit(new)
                            held = torch.cat([_nearest(held[:before] / w) * w, _nearest(new / w) * w])
                        got[:end, h] = held[:end]
                    lo = max(n - min(n, c + BLOCK - 1), b)
                    out[name].append(got[lo - b:min(BLOCK, n - b)])
        return {name: torch.cat(x) for name, x in out.items()}
    out, g, row = torch.empty(q.shape, dtype=torch.float64, device="cuda"), case["nq"] // nkv, 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        base = sum(need[:i]) * PAGE
        blocks = need[i] * 4
        late = torch.arange(n, device="cuda") > (n - c + torch.arange(c, device="cuda"))[:, None]
        for h in range(nkv):
            held = []
            for x in old:
                y = x[base:base + blocks * BLOCK, h].double().view(blocks, -1)
                m = y.abs().amax(-1, keepdim=True)
                e = torch.ceil(torch.log2(m / 448))
                e = e + (m > 448 * torch.exp2(e)).double() - (m <= 448 * torch.exp2(e - 1)).double()                  # log2's own rounding
                u = torch.exp2(e.clamp(min=-126))
                held.append((_nearest(y / u) * u).view(-1, hd)[:n])
            for j in range(h * g, h * g + g):
                w = q[row:row + c, j].double() @ held[0].T / math.sqrt(hd)
                w[late] = -math.inf
                out[row:row + c, j] = torch.softmax(w, -1) @ held[1]
        row += c
    return out
