"""Attention over packed sequences, a key-value cache in pages, and attention of one new token over it; what they are measured on.

Rows of several sequences lie one behind the other; sequence g has the rows [first[g], first[g + 1]). Query heads share key-value
heads in groups, in their order. The cache is cut into pages, each [kv_heads, page_size, 128] for K and for V; a table names the
pages of every sequence. It holds bf16, or codes of 8 bits: sign, four bits of exponent, three of fraction (e4m3, largest 448),
with one scale, a power of two held as its biased exponent in a byte, for each token's row of a head.

    prompt   attention within every sequence, causal or not; the keys may begin in front of the queries
    token    attention of one query row a sequence over what the cache holds of it
    cache    new rows written into their pages, and whole sequences read back
"""
import math
import random

import torch

own = False

HD = 128
SCALE = 1.0 / math.sqrt(HD)

_dev = None


def _lib():
    global _dev
    if _dev is None:
        import iris_c_amd
        _dev = iris_c_amd.IrisDev()
    return _dev.lib


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    r = random.Random(7)
    prompts, chats, many, fill = _lengths(r, 24, 4, 512), _lengths(r, 48, 1, 4096), _lengths(r, 256, 1, 2048), _lengths(r, 16, 20, 512)
    return [
        # one short prompt; a batch of prompts as users type them; long documents with a short question behind them
        dict(name="prompt_31", kind="prompt", rows="31", keys="", behind=0, heads=32, kv=8, causal=True),
        dict(name="prompt_batch", kind="prompt", rows=prompts, keys="", behind=0, heads=32, kv=8, causal=True),
        dict(name="prompt_documents", kind="prompt", rows="12001,4096,700,1", keys="", behind=0, heads=32, kv=8, causal=True),
        # text and image rows of pictures of several sizes, every row against all of its picture
        dict(name="prompt_pictures", kind="prompt", rows="4608,1536,2627,576", keys="", behind=0, heads=24, kv=24, causal=False),
        # prompts that go on from what is cached: a few new rows against all rows so far
        dict(name="prompt_continued", kind="prompt", rows="64,1,200,17", keys="2064,900,4113,1217", behind=3, heads=32, kv=8, causal=True),
        # a token of one short text; of a batch of texts; of a few long ones, and of many, in 8 bits
        dict(name="token_300", kind="token", lengths="300", page=16, heads=32, kv=8, dtype="bf16"),
        dict(name="token_48", kind="token", lengths=chats, page=64, heads=32, kv=8, dtype="bf16"),
        dict(name="token_long_fp8", kind="token", lengths="131072,70001,4097", page=64, heads=32, kv=8, dtype="fp8"),
        dict(name="token_256_fp8", kind="token", lengths=many, page=32, heads=32, kv=8, dtype="fp8"),
        # the rows of a token's step written; prompts written and read back in 8 bits; a long text read back to go on from it
        dict(name="cache_tokens", kind="cache", lengths=_lengths(r, 48, 1, 512), new="1", page=64, kv=8, dtype="bf16", read=False),
        dict(name="cache_prompts_fp8", kind="cache", lengths=fill, new="all", page=16, kv=8, dtype="fp8", read=True),
        dict(name="cache_long_fp8", kind="cache", lengths="65536,30011", new="64", page=64, kv=8, dtype="fp8", read=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lengths(rng, n, lo, hi):
    return ",".join(str(_log(rng, lo, hi)) for _ in range(n))


def _ints(text):
    return [int(v) for v in text.split(",")] if text else []


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "token", "token", "cache"])
    heads, kv = rng.choice([(32, 8), (32, 8), (24, 24), (16, 2), (30, 6), (8, 1)])
    if kind == "prompt":
        n = _log(rng, 1, 40)
        most = max(4, min(9000, 20000 // n))
        rows = [0 if rng.random() < 0.05 else _log(rng, 1, most) for _ in range(n)]
        if not sum(rows):
            rows[0] = 1
        before = [_log(rng, 1, max(2, 20000 // n)) if rng.random() < 0.8 else 0 for _ in rows] if rng.random() < 0.3 else []
        if before:
            rows = [min(v, _log(rng, 1, 512)) for v in rows]
        keys = ",".join(str(a + b) for a, b in zip(rows, before))
        causal = True if before else rng.random() < 0.7
        return dict(kind=kind, rows=",".join(map(str, rows)), keys=keys, behind=rng.choice([0, 0, rng.randrange(1, 64)]), heads=heads,
                    kv=kv, causal=causal)
    n = _log(rng, 1, 256)
    most = max(2, min(131072, 262144 // n))
    lengths = [0 if rng.random() < 0.03 else _log(rng, 1, most) for _ in range(n)]
    if not sum(lengths):
        lengths[0] = most
    s = dict(kind=kind, lengths=",".join(map(str, lengths)), page=rng.choice([16, 16, 32, 64, 64, 128]), kv=kv,
             dtype=rng.choice(["bf16", "fp8"]))
    if kind == "token":
        return dict(s, heads=heads)
    return dict(s, new=rng.choice(["1", "all", str(_log(rng, 2, 300))]), read=s["dtype"] == "fp8" or rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------------------- inputs
class _Make:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.seed = seed
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(self, *shape, s=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(s).to(torch.bfloat16)

    def keys(self, *shape):
        """K after its norm and rotation: some of the 128 places larger in all rows of a head."""
        x = torch.randn(*shape, generator=self.g, device="cuda")
        x *= 1.0 + 3.0 * (torch.rand(shape[-1], generator=self.g, device="cuda") < 1 / 32)
        return x.to(torch.bfloat16)


def _first(sizes):
    first = [0]
    for v in sizes:
        first.append(first[-1] + v)
    return first


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    s, m = dict(case), _Make(seed)
    if s["kind"] == "prompt":
        s["n"], s["m"] = _ints(s["rows"]), _ints(s["keys"]) or _ints(s["rows"])
        first = _first(s["n"])
        s["total"] = first[-1] + s["behind"]
        s["first"] = _int(first)
        heads, kv = s["heads"], s["kv"]
        # the rows of a fused projection: q | k | v
        s["qkv"] = torch.cat([m.rows(s["total"], heads * HD), m.keys(s["total"], kv * HD), m.rows(s["total"], kv * HD)], 1)
        s["q"], s["k"], s["v"] = s["qkv"].split([heads * HD, kv * HD, kv * HD], 1)
        s["first_key"], s["key_rows"], s["ldkv"] = None, s["total"], s["qkv"].shape[1]
        if s["keys"]:
            at = _first(s["m"])
            s["first_key"], s["key_rows"], s["ldkv"] = _int(at), at[-1], kv * HD
            s["k"], s["v"] = m.keys(at[-1], kv * HD), m.rows(at[-1], kv * HD)
        # what rows behind the last sequence hold stays there
        s["out"] = torch.full((s["total"], heads * HD), 0.0625, dtype=torch.bfloat16, device="cuda")
        return s
    lengths, page, kv = _ints(s["lengths"]), s["page"], s["kv"]
    n = len(lengths)
    per = [(v + page - 1) // page for v in lengths]
    s["n"], s["len"], s["pages"], s["ld"] = n, _int(lengths), sum(per) + 3, max(1, max(per))
    order = list(range(s["pages"]))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for v in per:
        table.append(order[at:at + v] + [-1] * (s["ld"] - v))
        at += v
    s["table"] = _int(table)
    shape = (s["pages"], kv, page, HD)
    if s["kind"] == "token":
        s["k"], s["v"] = m.keys(*shape), m.rows(*shape)
        if s["dtype"] == "fp8":
            (s["k"], s["ks"]), (s["v"], s["vs"]) = _encode(s["k"]), _encode(s["v"])
        s["q"] = m.rows(n, s["heads"] * HD, s=1.3)
        s["out"] = torch.zeros(n, s["heads"] * HD, dtype=torch.bfloat16, device="cuda")
        return s
    new = lengths if s["new"] == "all" else [min(v, int(s["new"])) for v in lengths]
    s["first"], s["rows"] = _int(_first(new)), sum(new)
    s["first_all"], s["rows_all"] = _int(_first(lengths)), sum(lengths)
    s["kn"], s["vn"] = m.keys(s["rows"], kv * HD), m.rows(s["rows"], kv * HD)
    s["k"], s["v"] = m.keys(*shape), m.rows(*shape)
    if s["dtype"] == "fp8":
        (s["k"], s["ks"]), (s["v"], s["vs"]) = _encode(s["k"]), _encode(s["v"])
    if s["read"]:
        s["ko"], s["vo"] = (torch.zeros(s["rows_all"], kv * HD, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    return s


# ------------------------------------------------------------------------------------------------------ the plain forms
def _encode(x):
    """(codes, scales) of the rows in the last dimension: the largest of a row in (224, 448] of its scale"""
    x = x.float()
    mantissa, exponent = torch.frexp(x.abs().amax(-1))                    # the largest is mantissa * 2^exponent, mantissa in [0.5, 1)
    exponent = (exponent - 9 + (mantissa > 0.875).int()).clamp(-127, 127)
    exponent = torch.where(mantissa > 0, exponent, torch.full_like(exponent, -127))
    half = exponent.div(2, rounding_mode="floor")
    v = torch.ldexp(torch.ldexp(x, -half[..., None]), (half - exponent)[..., None])
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v).exponent.clamp(min=-5) - 4)      # 8 steps a power of two, 2^-9 below 2^-6
    return (torch.round(v / step) * step).to(torch.float8_e4m3fn).view(torch.uint8), (exponent + 127).to(torch.uint8)


def _decode(codes, scales):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), (scales.int() - 127)[..., None])


def _slots(s, most):
    """page and place in it of the positions 0 .. most - 1 of every sequence, and which of them there are: [n, most] each"""
    at = torch.arange(most, device="cuda")
    there = at[None, :] < s["len"][:, None]
    return torch.where(there, s["table"][:, at // s["page"]].long(), 0), (at % s["page"])[None, :].expand(s["n"], -1), there


def _softmax(scores, valid):
    """over the last dimension; zeros where nothing is valid"""
    scores = torch.where(valid, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _plain_prompt(s):
    out = s["out"].clone()
    heads, kv = s["heads"], s["kv"]
    i = j = 0
    for n, m in zip(s["n"], s["m"]):
        if n and m:
            k = s["k"][j:j + m].float().reshape(m, kv, HD).permute(1, 2, 0).contiguous()          # [kv, HD, m]
            v = s["v"][j:j + m].float().reshape(m, kv, HD).transpose(0, 1).contiguous()
            key = torch.arange(m, device="cuda")
            for a in range(0, n, 2048):
                b = min(n, a + 2048)
                q = s["q"][i + a:i + b].float().reshape(b - a, kv, heads // kv, HD).permute(1, 2, 0, 3)
                scores = torch.matmul(q.reshape(kv, -1, HD), k).mul_(SCALE).reshape(kv, heads // kv, b - a, m)
                row = torch.arange(a, b, device="cuda")[:, None] + (m - n)
                p = _softmax(scores, key <= row if s["causal"] else key[None, :] >= 0)
                o = torch.matmul(p.reshape(kv, -1, m), v).reshape(kv, heads // kv, b - a, HD)
                out[i + a:i + b] = o.permute(2, 0, 1, 3).reshape(b - a, heads * HD).to(out.dtype)
        elif n:
            out[i:i + n] = 0
        i, j = i + n, j + m
    return out


def _plain_token(s):
    n, kv, group = s["n"], s["kv"], s["heads"] // s["kv"]
    page, place, there = _slots(s, max(1, int(max(_ints(s["lengths"])))))

    def take(codes, scales):
        if s["dtype"] == "fp8":
            return _decode(codes[page, :, place], scales[page, :, place])
        return codes[page, :, place].float()                                                     # [n, most, kv, HD]
    q = s["q"].float().reshape(n, kv, group, HD)
    scores = torch.matmul(q, take(s["k"], s.get("ks")).permute(0, 2, 3, 1).contiguous()).mul_(SCALE)
    p = _softmax(scores, there[:, None, None, :])
    v = torch.where(there[:, None, :, None], take(s["v"], s.get("vs")).transpose(1, 2), 0.0)
    return torch.matmul(p, v).reshape(n, -1).to(torch.bfloat16)


def _of_rows(s, first, rows):
    """sequence and position of every one of the rows that first cuts into sequences: the last of each"""
    row = torch.arange(rows, device="cuda")
    g = torch.bucketize(row, first[1:].long(), right=True)
    at = row - first[g + 1] + s["len"][g]
    return s["table"][g, at // s["page"]].long(), at % s["page"]


def _plain_cache(s):
    page, place = _of_rows(s, s["first"], s["rows"])
    for pages, scales, x in (("k", "ks", "kn"), ("v", "vs", "vn")):
        x = s[x].reshape(s["rows"], s["kv"], HD)
        if s["dtype"] == "fp8":
            codes, exponents = _encode(x)
            s[pages][page, :, place], s[scales][page, :, place] = codes, exponents
        else:
            s[pages][page, :, place] = x
    if not s["read"]:
        return s["k"], s["v"]
    page, place = _of_rows(s, s["first_all"], s["rows_all"])
    for pages, scales, out in (("k", "ks", "ko"), ("v", "vs", "vo")):
        x = s[pages][page, :, place]
        s[out].copy_((_decode(x, s[scales][page, :, place]) if s["dtype"] == "fp8" else x).reshape(s["rows_all"], -1))
    return s["ko"], s["vo"]


# ----------------------------------------------------------------------------------------------------------------- runs
def run(s):
    if own:
        return _run_own(_lib(), s)
    return {"prompt": _plain_prompt, "token": _plain_token, "cache": _plain_cache}[s["kind"]](s)


def _run_own(lib, s):
    def p(name):
        return s[name].data_ptr() if s.get(name) is not None else None
    if s["kind"] == "prompt":
        lib.iris_dev_attention_sequences(p("out"), s["out"].shape[1], p("q"), s["qkv"].shape[1], p("k"), p("v"), s["ldkv"], p("first"),
                                         p("first_key"), len(s["n"]), s["total"], s["key_rows"], s["heads"], s["kv"], HD, SCALE,
                                         int(s["causal"]))
        return s["out"]
    paged = (s["pages"], s["page"], p("table"), s["ld"], p("len"))
    if s["kind"] == "token":
        if s["dtype"] == "fp8":
            lib.iris_dev_attention_paged_fp8(p("out"), s["heads"] * HD, p("q"), s["heads"] * HD, p("k"), p("v"), p("ks"), p("vs"),
                                             *paged, s["n"], s["heads"], s["kv"], HD, SCALE, None)
        else:
            lib.iris_dev_attention_paged_bf16(p("out"), s["heads"] * HD, p("q"), s["heads"] * HD, p("k"), p("v"), *paged, s["n"],
                                              s["heads"], s["kv"], HD, SCALE, None)
        return s["out"]
    new = (s["kv"] * HD, p("first"), s["n"], s["rows"], s["kv"], HD)
    everything = (p("first_all"), s["n"], s["rows_all"], s["kv"], HD)
    if s["dtype"] == "fp8":
        lib.iris_dev_cache_write_fp8(p("k"), p("v"), p("ks"), p("vs"), *paged, p("kn"), p("vn"), *new)
        if s["read"]:
            lib.iris_dev_cache_read_fp8(p("ko"), p("vo"), s["kv"] * HD, p("k"), p("v"), p("ks"), p("vs"), *paged, *everything)
    else:
        lib.iris_dev_cache_write_bf16(p("k"), p("v"), *paged, p("kn"), p("vn"), *new)
        if s["read"]:
            lib.iris_dev_cache_read_bf16(p("ko"), p("vo"), s["kv"] * HD, p("k"), p("v"), *paged, *everything)
    return (s["ko"], s["vo"]) if s["read"] else (s["k"], s["v"])


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "prompt":
        n, m = _ints(case["rows"]), _ints(case["keys"]) or _ints(case["rows"])
        # a causal row i of n over m keys sees i + 1 + m - n of them
        pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(n, m))
        return {"bytes": 2 * HD * (2 * sum(n) * case["heads"] + 2 * sum(m) * case["kv"]), "flops": 4 * HD * case["heads"] * pairs}
    lengths = _ints(case["lengths"])
    row = 2 * case["kv"] * (2 * HD if case["dtype"] == "bf16" else HD + 1)              # K and V of a token in the cache
    if case["kind"] == "token":
        return {"bytes": sum(lengths) * row + 4 * HD * case["heads"] * len(lengths), "flops": 4 * HD * case["heads"] * sum(lengths)}
    new = sum(lengths) if case["new"] == "all" else sum(min(v, int(case["new"])) for v in lengths)
    plain = 4 * HD * case["kv"]
    return {"bytes": new * (plain + row) + (sum(lengths) * (row + plain) if case["read"] else 0), "flops": 0}


# ---------------------------------------------------------------------------------------------------------------- exact
def _exact_values(codes, scales):
    """By the bits of a code: s eeee mmm."""
    c = codes.long()
    e, f = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * torch.exp2((e - 7).double()))
    return torch.where(c >> 7 > 0, -v, v) * torch.exp2(scales.double() - 127)[..., None]


def _exact_quantised(x):
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    # the smallest power of two of which the largest is at most 448
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448.0))
    scale = torch.exp2(torch.where(top > 0, e, -127.0).clamp(-127, 127))
    f = torch.arange(8, dtype=torch.float64, device=x.device)
    grid = torch.cat([f / 8 * 2.0 ** -6] + [(1 + f / 8) * 2.0 ** k for k in range(-6, 9)])[:127]
    middle = (grid[1:] + grid[:-1]) / 2
    r = x.abs() / scale
    up, down = torch.bucketize(r, middle, right=True), torch.bucketize(r, middle, right=False)
    return torch.sign(x) * grid[torch.where(up % 2 == 0, up, down)] * scale


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "prompt":
        out, i, j, group = s["out"].double(), 0, 0, s["heads"] // s["kv"]
        for n, m in zip(s["n"], s["m"]):
            for h in range(s["heads"]) if n else ():
                at = slice(h // group * HD, h // group * HD + HD)
                k, v = s["k"][j:j + m, at].double(), s["v"][j:j + m, at].double()
                for a in range(0, n, 4096):
                    b = min(n, a + 4096)
                    x = s["q"][i + a:i + b, h * HD:h * HD + HD].double() @ k.T * SCALE
                    if s["causal"]:
                        x += torch.full_like(x, -math.inf).triu(m - n + a + 1)
                    out[i + a:i + b, h * HD:h * HD + HD] = torch.softmax(x, -1) @ v
            i, j = i + n, j + m
        return out
    fp8, kv, page = s["dtype"] == "fp8", s["kv"], s["page"]

    def held(pages, scales, g, n):
        """what the cache holds of sequence g, [kv, n, HD]"""
        at = s["table"][g, :(n + page - 1) // page].long()
        x = _exact_values(s[pages][at], s[scales][at]) if fp8 else s[pages][at].double()
        return x.transpose(0, 1).reshape(kv, len(at) * page, HD)[:, :n]
    lengths = _ints(s["lengths"])
    if s["kind"] == "token":
        out = torch.zeros(s["n"], s["heads"], HD, dtype=torch.float64, device="cuda")
        for g, n in enumerate(lengths):
            if n:
                x = s["q"][g].double().reshape(kv, -1, HD) @ held("k", "ks", g, n).transpose(1, 2) * SCALE
                out[g] = (torch.softmax(x, -1) @ held("v", "vs", g, n)).reshape(-1, HD)
        return out.reshape(s["n"], -1)
    outs = []
    for pages, scales, new in (("k", "ks", "kn"), ("v", "vs", "vn")):
        rows = s[new].reshape(-1, kv, HD)
        rows = _exact_quantised(rows) if fp8 else rows.double()
        whole, at = [], 0
        pool = None if s["read"] else s[pages].double()
        for g, n in enumerate(lengths):
            add = int(s["first"][g + 1]) - int(s["first"][g])
            if s["read"]:
                x = held(pages, scales, g, n).transpose(0, 1).clone()
                x[n - add:] = rows[at:at + add]
                whole.append(x.reshape(n, kv * HD))
            else:
                for t in range(add):
                    pos = n - add + t
                    pool[int(s["table"][g, pos // page]), :, pos % page] = rows[at + t]
            at += add
        outs.append(torch.cat(whole) if s["read"] else pool)
    return tuple(outs)
