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
           dict(sequences=-1), dict(ldo=1023), dict(ldq=1000), dict(ldkv=255), dict(rows=2 ** 28, keys=2 ** 28), dict(heads=2 ** 24, kv=2 ** 24)]
CACHE_BAD = [dict(k=None), dict(v=None), dict(table=None), dict(lengths=None), dict(page=0), dict(page=24), dict(page=-16), dict(pages=-1), dict(ld=-1), dict(sequences=-1),
             dict(kv=0), dict(hd=0), dict(hd=-128)]
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
