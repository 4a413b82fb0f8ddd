"""Linear layers in microscaled 4-bit floating point and linear layers over groups of rows, and what they are measured on.

MXFP4: a row is cut into blocks of 32 columns; a block has one scale, a power of two held as its biased exponent in a byte
(s stands for 2^(s - 127), 255 for "not a number"), and 32 codes of four bits, sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; the
even column of a pair sits in the low half of its byte. A row of codes is 16 bytes a block, a row of scales one byte a block;
the last block of a row is filled up with zeros.

    convert         values -> codes and scales -> the values that these stand for
    linear          y[rows, out] = x[rows, in] W[out, in]^T, both held in MXFP4
    grouped         rows [first[g], first[g + 1]) of x take W[g]; bf16
    grouped_mxfp4   the same, both held in MXFP4
"""
import math
import random

import torch

own = False

_dev = None


def _lib():
    global _dev
    if _dev is None:
        import iris_c_amd
        _dev = iris_c_amd.IrisDev()
    return _dev.lib


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    r = random.Random(20)
    experts, tokens, tokens4 = _cut(r, 4000, 64), _cut(r, 16, 128), _cut(r, 40, 64)
    return [
        # a row of conditioning; rows of an odd width out of a wider buffer; the widest rows of a single-stream block
        dict(name="convert_row", kind="convert", rows=1, cols=4096, ld=4096, dtype="f32"),
        dict(name="convert_1000x2565", kind="convert", rows=1000, cols=2565, ld=2600, dtype="f32"),
        dict(name="convert_4608x16384", kind="convert", rows=4608, cols=16384, ld=16384, dtype="bf16"),
        # the modulation of a step from one row; gate | up of a text-encoder layer; sizes with nothing round about them; the
        # fused projection of a single-stream block
        dict(name="linear_1", kind="linear", rows=1, k=4096, n=24576, dtype="f32"),
        dict(name="linear_512", kind="linear", rows=512, k=2560, n=19456, dtype="bf16"),
        dict(name="linear_777_odd", kind="linear", rows=777, k=1000, n=1111, dtype="f32"),
        dict(name="linear_4608", kind="linear", rows=4608, k=4096, n=36864, dtype="bf16"),
        # q | k | v of a double-stream block: text rows and image rows, weights of their own; rows sorted by the expert that
        # they go to, many and few
        dict(name="grouped_streams", kind="grouped", sizes="512,4096", behind=0, k=4096, n=12288, dtype="bf16"),
        dict(name="grouped_experts", kind="grouped", sizes=experts, behind=96, k=2560, n=1536, dtype="bf16"),
        dict(name="grouped_tokens", kind="grouped", sizes=tokens, behind=0, k=2560, n=1536, dtype="f32"),
        # the same in four bits: the two streams, and the rows of a few tokens
        dict(name="mxfp4_streams", kind="grouped_mxfp4", sizes="512,4096", behind=0, k=4096, n=12288, dtype="bf16"),
        dict(name="mxfp4_tokens", kind="grouped_mxfp4", sizes=tokens4, behind=8, k=2560, n=1536, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cut(rng, rows, groups):
    """`rows` rows dealt out to `groups` groups, unevenly, a sixth of the groups empty; as a text."""
    share = [0.0 if rng.random() < 1 / 6 else -math.log(1.0 - rng.random()) for _ in range(groups)]
    if not sum(share):
        share[rng.randrange(groups)] = 1.0
    total, at, sizes, done = sum(share), 0.0, [], 0
    for s in share:
        at += s
        upto = round(rows * at / total)
        sizes.append(upto - done)
        done = upto
    return ",".join(map(str, sizes))


def _sizes(case):
    return [int(v) for v in case["sizes"].split(",")]


def draw(rng):
    kind = rng.choice(["convert", "linear", "linear", "grouped", "grouped", "grouped_mxfp4", "grouped_mxfp4"])
    if kind == "convert":
        rows, cols = _log(rng, 1, 4608), _log(rng, 16, 16384)
        return dict(kind=kind, rows=rows, cols=cols, ld=cols + rng.choice([0, 0, 8, 33]), dtype=rng.choice(["f32", "bf16"]))
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "linear":
        # most widths of a model are multiples of 256
        k, n = (v if rng.random() < 0.3 else max(256, v // 256 * 256) for v in (_log(rng, 64, 16384), _log(rng, 64, 24576)))
        return dict(kind=kind, rows=min(_log(rng, 1, 4608), max(1, int(6e11 / k / n))), k=k, n=n, dtype=dtype)
    groups = rng.choice([1, 2, 2, 3, _log(rng, 4, 128), _log(rng, 4, 128)])
    k, n = (v if rng.random() < 0.25 else max(256, v // 256 * 256) for v in (_log(rng, 64, 8192), _log(rng, 64, 8192)))
    n = max(32, min(n, int(2.5e8 / groups / k)))
    rows = min(_log(rng, 1, 4608), max(1, int(1.5e11 / k / n)))
    return dict(kind=kind, sizes=_cut(rng, rows, groups), behind=rng.choice([0, 0, rng.randrange(1, 64)]), k=k, n=n, dtype=dtype)


# --------------------------------------------------------------------------------------------------------------- inputs
class _Make:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(self, rows, cols):
        """Activations: every row with a size of its own, and one column in 64 eight times as large."""
        x = torch.randn(rows, cols, generator=self.g, device="cuda")
        x *= torch.exp2(torch.randn(rows, 1, generator=self.g, device="cuda"))
        return x.mul_(1.0 + 7.0 * (torch.rand(cols, generator=self.g, device="cuda") < 1 / 64))

    def weight(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(1.0 / math.sqrt(shape[-1]))


DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _blocks(cols):
    return (cols + 31) // 32


def _codes_room(rows, cols):
    return (torch.zeros(rows, 16 * _blocks(cols), dtype=torch.uint8, device="cuda"),
            torch.zeros(rows, _blocks(cols), dtype=torch.uint8, device="cuda"))


def prepare(case, seed):
    s, m = dict(case), _Make(seed)
    if s["kind"] == "convert":
        rows, cols, ld = s["rows"], s["cols"], s["ld"]
        s["x"] = m.rows(rows, ld).to(DTYPE[s["dtype"]])[:, :cols]
        s["codes"], s["scales"] = _codes_room(rows, cols)
        s["y"] = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
        return s
    if s["kind"] == "linear":
        rows, w = s["rows"], m.weight(s["n"], s["k"])
    else:
        sizes = _sizes(s)
        first = [0]
        for v in sizes:
            first.append(first[-1] + v)
        rows, w = first[-1] + s["behind"], m.weight(len(sizes), s["n"], s["k"])
        s["groups"], s["used"], s["most"] = len(sizes), first[-1], max(sizes)
        s["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
    s["rows"] = rows
    x = m.rows(rows, s["k"])
    if s["kind"] == "grouped":
        s["x"], s["w"] = x.to(torch.bfloat16), w.to(torch.bfloat16)
    else:
        s["xc"], s["xs"] = _encode(x)
        c, e = _encode(w.reshape(-1, s["k"]))
        s["wc"], s["ws"] = c.reshape(*w.shape[:-1], -1), e.reshape(*w.shape[:-1], -1)
    # what rows behind the last group hold stays there
    s["y"] = torch.full((rows, s["n"]), 7.0, dtype=DTYPE[s["dtype"]], device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------ the plain forms
def _encode(x):
    """(codes, scales) of x [rows, cols]"""
    rows, cols = x.shape
    nb = _blocks(cols)
    b = torch.nn.functional.pad(x.float(), (0, 32 * nb - cols)).reshape(rows, nb, 32)
    top = b.abs().amax(-1)
    exponent = (torch.frexp(top).exponent - 3).clamp(-127, 127)           # floor(log2(top)) - 2: the largest of a block in [4, 8)
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127))
    v = torch.ldexp(torch.ldexp(b.abs(), -exponent.div(2, rounding_mode="floor")[..., None]),
                    (exponent.div(2, rounding_mode="floor") - exponent)[..., None]).clamp(max=6.0)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = torch.round(v / step) * step                                      # ties to the even code
    code = torch.where(v < 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4)).to(torch.uint8) | (torch.signbit(b).to(torch.uint8) << 3)
    code = code.reshape(rows, nb * 16, 2)
    return code[..., 0] | (code[..., 1] << 4), (exponent + 127).to(torch.uint8)


def _decode(codes, scales, cols):
    """The float32 values [..., cols] that codes and scales stand for."""
    value = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    value = torch.cat([value, -value])
    pair = torch.stack([value.repeat(16), value.repeat_interleave(16)], 1)   # by byte
    v = pair[codes.int()].reshape(*codes.shape[:-1], -1, 32)
    scale = torch.exp2(scales.float() - 127.0)
    scale = torch.where(scales == 255, torch.full_like(scale, math.nan), scale)
    return (v * scale[..., None]).reshape(*codes.shape[:-1], -1)[..., :cols]


def _grouped(x, w, s):
    """x [rows, k], w [groups, n, k] in float32: the rows of a group, filled up to the largest one's, times its weights."""
    at = s["first"][:-1, None] + torch.arange(s["most"], device="cuda")[None, :]
    there = at < s["first"][1:, None]
    y = torch.matmul(x[torch.where(there, at, 0)], w.transpose(1, 2))
    out = s["y"].clone()
    out[:s["used"]] = y[there].to(out.dtype)
    return out


# ----------------------------------------------------------------------------------------------------------------- runs
def run(s):
    return _run_own(_lib(), s) if own else _run_plain(s)


def _run_plain(s):
    if s["kind"] == "convert":
        return _decode(*_encode(s["x"]), s["cols"]).to(torch.bfloat16)
    if s["kind"] == "linear":
        return torch.matmul(_decode(s["xc"], s["xs"], s["k"]), _decode(s["wc"], s["ws"], s["k"]).T).to(DTYPE[s["dtype"]])
    if s["kind"] == "grouped":
        return _grouped(s["x"].float(), s["w"].float(), s)
    return _grouped(_decode(s["xc"], s["xs"], s["k"]), _decode(s["wc"], s["ws"], s["k"]), s)


def _run_own(lib, s):
    p = lambda name: s[name].data_ptr()  # noqa: E731
    if s["kind"] == "convert":
        encode = lib.iris_dev_f32_to_mxfp4 if s["dtype"] == "f32" else lib.iris_dev_bf16_to_mxfp4
        encode(p("codes"), p("scales"), p("x"), s["ld"], s["rows"], s["cols"])
        lib.iris_dev_mxfp4_to_bf16(p("y"), s["cols"], p("codes"), p("scales"), s["rows"], s["cols"])
    elif s["kind"] == "linear":
        call = lib.iris_dev_linear_mxfp4_f32 if s["dtype"] == "f32" else lib.iris_dev_linear_mxfp4_bf16
        call(p("y"), p("xc"), p("xs"), p("wc"), p("ws"), s["rows"], s["k"], s["n"])
    elif s["kind"] == "grouped":
        call = lib.iris_dev_linear_f32_grouped if s["dtype"] == "f32" else lib.iris_dev_linear_bf16_grouped
        call(p("y"), p("x"), p("w"), p("first"), s["groups"], s["rows"], s["k"], s["n"])
    else:
        call = lib.iris_dev_linear_mxfp4_f32_grouped if s["dtype"] == "f32" else lib.iris_dev_linear_mxfp4_bf16_grouped
        call(p("y"), p("xc"), p("xs"), p("wc"), p("ws"), p("first"), s["groups"], s["rows"], s["k"], s["n"])
    return s["y"]


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "bf16": 2}[case["dtype"]]
    if case["kind"] == "convert":
        # the values in, the values that they become out
        return {"bytes": case["rows"] * case["cols"] * (size + 2), "flops": 0}
    if case["kind"] == "linear":
        rows, weights = case["rows"], 1
    else:
        rows, weights = sum(_sizes(case)), sum(v > 0 for v in _sizes(case))
    row = 2 * case["k"] if case["kind"] == "grouped" else 17 * _blocks(case["k"])
    return {"bytes": (rows + weights * case["n"]) * row + rows * case["n"] * size, "flops": 2 * rows * case["k"] * case["n"]}


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "convert":
        x = s["x"].double()
        cols = x.shape[1]
        x = torch.nn.functional.pad(x, (0, -cols % 32)).unflatten(1, (-1, 32))
        top = x.abs().amax(-1, keepdim=True)
        # in 64 bits the logarithm of a power of two is a whole number, and that of the float below it is not
        scale = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2, -127, 127))
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
        middle = (grid[1:] + grid[:-1]) / 2
        r = x.abs() / scale
        # the grid's value below a middle, the one above it, the even code on it
        up, down = torch.bucketize(r, middle, right=True), torch.bucketize(r, middle, right=False)
        near = torch.where(up % 2 == 0, up, down)
        return (torch.sign(x) * grid[near] * scale).flatten(1)[:, :cols]
    if s["kind"] == "grouped":
        x, w = s["x"].double(), s["w"].double()
    else:
        x, w = _exact_values(s["xc"], s["xs"], s["k"]), _exact_values(s["wc"], s["ws"], s["k"])
    if s["kind"] == "linear":
        return x @ w.T
    y, at = s["y"].double(), 0
    for g, n in enumerate(_sizes(s)):
        y[at:at + n] = x[at:at + n] @ w[g].T
        at += n
    return y


def _exact_values(codes, scales, k):
    """By the bits of a code: s e e m."""
    halves = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign = 1 - 2 * torch.floor(halves / 8)
    rest = halves % 8
    e, mant = torch.floor(rest / 2), rest % 2
    v = sign * torch.where(e == 0, mant / 2, (1 + mant / 2) * torch.exp2(e - 1))
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)[..., :k]
