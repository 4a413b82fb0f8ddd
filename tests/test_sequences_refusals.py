"""What the entries for packed sequences and the paged cache refuse, with a message and nothing launched; their numbers on the CPU. No GPU."""
import numpy as np
import pytest

import iris_c_amd
import sequences_reference as sr


@pytest.fixture(scope="module")
def lib():
    return iris_c_amd.load()


A = 4096                                    # an address that nothing is read from: every call here ends before a launch
SEQ = dict(out=A, ldo=1024, q=A, ldq=1024, k=A, v=A, ldkv=256, first_row=A, first_key=None, sequences=2, rows=8, keys=8, heads=8, kv=2, hd=128, scale=0.1, causal=1)
PAGED = dict(out=A, ldo=1024, q=A, ldq=1024, k=A, v=A, pages=4, page=16, table=A, ld=2, lengths=A, sequences=2, heads=8, kv=2, hd=128, scale=0.1, ws=None)
WRITE = dict(k=A, v=A, pages=4, page=16, table=A, ld=2, lengths=A, kn=A, vn=A, ldn=256, first=A, sequences=2, rows=8, kv=2, hd=128)
READ = dict(kn=A, vn=A, ldn=256, k=A, v=A, pages=4, page=16, table=A, ld=2, lengths=A, first=A, sequences=2, rows=8, kv=2, hd=128)


def with_scales(args):
    out = {}
    for name, value in args.items():
        out[name] = value
        if name == "v":
            out["ks"], out["vs"] = A, A
    return out


ENTRIES = {
    "attention_sequences": SEQ, "attention_paged_bf16": PAGED, "attention_paged_fp8": with_scales(PAGED), "cache_write_bf16": WRITE,
    "cache_write_fp8": with_scales(WRITE), "cache_read_bf16": READ, "cache_read_fp8": with_scales(READ),
}
SEQ_BAD = [dict(out=None), dict(q=None), dict(k=None), dict(v=None), dict(first_row=None), dict(keys=9), dict(keys=-1), dict(kv=3), dict(kv=0), dict(kv=-2), dict(hd=0),
           dict(sequences=-1), dict(ldo=1023), dict(ldq=1000), dict(ldkv=255), dict(rows=2 ** 28, keys=2 ** 28), dict(heads=2 ** 24, kv=2 ** 24), dict(first_key=A, keys=2 ** 31 - 63)]
CACHE_BAD = [dict(k=None), dict(v=None), dict(table=None), dict(lengths=None), dict(page=0), dict(page=24), dict(page=-16), dict(pages=-1), dict(ld=-1), dict(sequences=-1),
             dict(kv=0), dict(hd=0), dict(hd=-128), dict(ld=2 ** 27), dict(ld=2, page=2 ** 30)]
ROWS_BAD = [dict(kn=None), dict(vn=None), dict(ldn=255), dict(first=None)]
BAD = [("attention_sequences", b) for b in SEQ_BAD]
BAD += [(e, b) for e in ENTRIES if e != "attention_sequences" for b in CACHE_BAD]
BAD += [(e, b) for e in ENTRIES if e.startswith("cache") for b in ROWS_BAD]
BAD += [(e, b) for e in ENTRIES if "paged" in e for b in (dict(out=None), dict(q=None), dict(ldo=1000), dict(ldq=1), dict(kv=3), dict(ws=A + 8))]
BAD += [(e, b) for e in ENTRIES if e.endswith("fp8") for b in (dict(ks=None), dict(vs=None))]


def call(lib, entry, **changed):
    lib.iris_dev_last_error()
    getattr(lib, "iris_dev_" + entry)(*{**ENTRIES[entry], **changed}.values())
    return lib.iris_dev_last_error()


@pytest.mark.parametrize("entry,bad", BAD, ids=lambda v: str(v))
def test_refused(lib, capfd, entry, bad):
    assert call(lib, entry, **bad) == -1
    line = capfd.readouterr().err
    assert line.startswith("iris_dev: " + entry) and "not initialised" not in line, line


@pytest.mark.parametrize("entry,nothing", [(e, n) for e in ENTRIES for n in ([dict(sequences=0)] + ([dict(rows=0), dict(rows=-3)] if "paged" not in e else []))], ids=str)
def test_nothing_to_do(lib, entry, nothing):
    assert call(lib, entry, **nothing) == 0


@pytest.mark.parametrize("entry", ENTRIES)
def test_no_fallback_without_a_gpu(lib, capfd, entry):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert call(lib, entry) == -1
    assert "not initialised" in capfd.readouterr().err


def test_the_numbers_of_the_tests_against_torch():
    import torch
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(sr.e4m3_value(codes.numpy()), want, equal_nan=True)
    x = np.random.default_rng(0).standard_normal((50, 128)) * np.exp2(np.arange(-25, 25))[:, None]
    x = sr.bf16_value(sr.bf16_round(x.astype(np.float32))).astype(np.float64)
    c, s = sr.quantise(x)
    scale = sr.scale_value(s)[:, None]
    assert (np.abs(x).max(1) <= 448 * scale[:, 0]).all() and (np.abs(x).max(1) > 224 * scale[:, 0]).all()
    assert np.array_equal(c, torch.tensor(x / scale).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    got = sr.e4m3_value(c) * scale
    assert (np.abs(got - x) <= np.maximum(np.abs(x) * 2.0 ** -4, scale * 2.0 ** -10)).all()


PART = 64 << 20                             # the workspace that the parts of a call share with the linear layers


def plan(lib, n, rows, keys, heads, kv, causal, own):
    import ctypes as C
    out = [C.c_int() for _ in range(3)]
    lib.iris_hip_sequences_plan(n, rows, keys, heads, kv, causal, own, *(C.byref(x) for x in out))
    return tuple(x.value for x in out)


def cut(tiles, blocks, heads, most):
    """What the kernel does with the tiles of sequences of so many blocks of keys: blocks of a part, entries of its list"""
    parts = lambda each: sum(t * max(1, -(-b // each)) for t, b in zip(tiles, blocks)) * heads
    work, more = sum(t * b for t, b in zip(tiles, blocks)) * heads, most - sum(tiles) * heads
    few, many, turns = max(4, work // most) - 1, max(4, (work + more - 1) // more), 0
    assert more > 0 and work + more < 2 ** 31
    while many - few > 1 + many // 8:
        each, turns = (few + many) // 2, turns + 1
        assert few < each < many and turns < 32
        if parts(each) <= most:
            many = each
        else:
            few = each
    return many, parts(many)


def test_parts_of_keys_fit_the_workspace(lib):
    """Any sizes: the shape is one that there is a kernel for, and where keys are cut, the list is not longer than the workspace has places for,
    whatever the sequences of those sizes are"""
    rng = np.random.default_rng(0)
    known = 0
    for _ in range(20000):
        kv = int(rng.choice([1, 2, 3, 6, 8, 24, 100]))
        heads = kv * int(rng.choice([1, 2, 4, 5, 8, 16, 60]))
        n, rows = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 18))
        own = bool(rng.integers(2))
        keys = rows if own else int(2 ** rng.uniform(0, 24))
        waves, blocks, parts = plan(lib, n, rows, keys, heads, kv, int(rng.integers(2)), own)
        assert (waves, blocks) in {(2, 1), (4, 1), (8, 1), (4, 2), (8, 2)} and parts in (1, 512)
        if parts == 1:
            continue
        known += 1
        assert n <= 256 and parts * (128 * 130 * 4 + 32) <= PART
        for _ in range(3):
            ends = np.sort(rng.integers(0, rows + 1, n - 1)) if rng.integers(2) else np.minimum(np.arange(1, n), rows)
            tiles = [-(-int(r) * (heads // kv) // 128) for r in np.diff(np.concatenate([[0], ends, [rows]]))]
            k = np.sort(rng.integers(0, keys + 1, n - 1)) if rng.integers(2) else np.full(n - 1, keys * int(rng.integers(2)))
            m = [-(-int(c) // 64) for c in np.diff(np.concatenate([[0], k, [keys]]))]
            each, entries = cut(tiles, m, kv, parts)
            assert each >= 4 and sum(tiles) * kv <= entries <= parts, (n, rows, keys, heads, kv)
    assert known > 1000


def test_shapes_of_known_calls(lib):
    assert plan(lib, 1, 31, 31, 32, 8, 1, 1) == (2, 1, 1)
    assert plan(lib, 1, 512, 512, 32, 8, 1, 1) == (4, 1, 1)
    assert plan(lib, 1, 4608, 4608, 24, 24, 0, 1) == (8, 2, 1)
    assert plan(lib, 4, 16797, 16797, 32, 8, 1, 1) == (4, 2, 1)
    assert plan(lib, 1, 32, 16000, 32, 8, 1, 0)[2] == 512
    assert plan(lib, 1, 64, 200, 32, 8, 1, 0)[2] == 1


def test_sizes_that_the_matrix_core_kernel_has_numbers_for(lib):
    takes = lambda pages, shift, ld, n, heads, kv: lib.iris_hip_paged_hd128_takes(pages, shift, ld, n, heads, kv)
    assert takes(1000, 6, 64, 256, 32, 8) == 1
    assert takes(2 ** 23, 6, 10, 1, 8, 8) == 0                       # 2^32 rows
    assert takes(2 ** 23 - 1, 6, 10, 1, 8, 8) == 1
    assert takes(10, 6, 2 ** 20, 2048, 32, 32) == 0                  # 2^37 tiles, if all were as long as the table
    assert lib.iris_dev_attention_paged_workspace() == 1024 * (2 * (16 * 128 + 32) * 4 + 32)
