"""C ABI of include/mg_attention.h without a GPU: descriptor sizes, refusals
with a status and a message before any device is touched, empty calls."""
import ctypes
import os
import subprocess

import pytest

import macrograd_b200 as mg
from macrograd_b200 import _lib, transformer as T

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = _lib.MG_ERR_INVALID, _lib.MG_ERR_UNSUPPORTED
PTR = ctypes.addressof(ctypes.create_string_buffer(64))


@pytest.fixture(scope="module")
def lib():
    return mg.load(build_if_missing=True)


def test_packed_descriptors_have_the_headers_layout(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mg_attention.h"\nint main(void){printf("%zu %zu %zu %zu %zu %zu\\n",'
                   "sizeof(mg_attention_desc),offsetof(mg_attention_desc,slopes),sizeof(mg_rotary_desc),"
                   "offsetof(mg_rotary_desc,positions),sizeof(mg_paged_desc),offsetof(mg_paged_desc,slopes));return 0;}")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [T._ATTENTION.size, T._ATTENTION.size - 24, T._ROTARY.size, T._ROTARY.size - 16, T._PAGED.size,
            T._PAGED.size - 24]
    assert got == want


def attention(**kw):
    d = dict(dtype=0, B=1, H=2, Hkv=1, Lq=4, Lk=4, D=64, causal=1, scale=0.125, cap=0.0, slopes=0, documents=0, prefix=0)
    d.update(kw)
    lead = [d[n] for n in ("dtype", "B", "H", "Hkv", "Lq", "Lk", "D", "causal", "scale", "cap")]
    return T._ATTENTION.pack(*lead, *([64] * 24), d["slopes"], d["documents"], d["prefix"])


@pytest.mark.parametrize("kw,status,fragment", [
    (dict(dtype=2), INVALID, "dtype"),
    (dict(B=-1), INVALID, "out of range"),
    (dict(H=0), INVALID, "out of range"),
    (dict(H=3, Hkv=2), INVALID, "multiple"),
    (dict(D=0), UNSUPPORTED, "head_dim"),
    (dict(D=129), UNSUPPORTED, "head_dim"),
    (dict(scale=float("nan")), INVALID, "scale"),
    (dict(cap=-1.0), INVALID, "cap"),
    (dict(cap=float("inf")), INVALID, "cap"),
    (dict(cap=1e-31), INVALID, "cap"),
    (dict(scale=2e30), INVALID, "scale"),
    (dict(causal=0, prefix=PTR), INVALID, "prefix"),
    (dict(Lq=1 << 29, Lk=1 << 29), UNSUPPORTED, "too long"),
    (dict(B=1 << 20, H=1 << 10, Lq=256), UNSUPPORTED, "too large"),
    (dict(), INVALID, "NULL"),
])
def test_attention_refusals(lib, kw, status, fragment):
    d = attention(**kw)
    assert lib.mg_attention(d, None, None, None, None, None, None) == status
    assert fragment in lib.mg_last_error().decode()
    assert lib.mg_attention_backward(d, *([None] * 10)) == status
    assert fragment in lib.mg_last_error().decode()


def test_empty_calls_need_no_device(lib):
    for kw in (dict(B=0), dict(Lq=0, Lk=0)):
        assert lib.mg_attention(attention(**kw), None, None, None, None, None, None) == _lib.MG_OK
        assert lib.mg_attention_backward(attention(**kw), *([None] * 10)) == _lib.MG_OK
    assert lib.mg_rotary(rotary(len=0), None, None, None, None, None) == _lib.MG_OK
    assert lib.mg_paged_attention(paged(batch=0), *([None] * 8)) == _lib.MG_OK


def test_null_descriptors(lib):
    assert lib.mg_attention(None, *([None] * 6)) == INVALID
    assert lib.mg_attention_backward(None, *([None] * 10)) == INVALID
    assert lib.mg_rotary(None, *([None] * 5)) == INVALID
    assert lib.mg_paged_attention(None, *([None] * 8)) == INVALID


def rotary(**kw):
    d = dict(dtype=0, batch=1, heads=2, kv_heads=1, len=3, head_dim=64, pairs=32, interleaved=0, inverse=0,
             magnitude=1.0, positions=PTR, frequencies=PTR)
    d.update(kw)
    lead = [d[n] for n in ("dtype", "batch", "heads", "kv_heads", "len", "head_dim", "pairs", "interleaved",
                           "inverse", "magnitude")]
    return T._ROTARY.pack(*lead, *([64] * 12), 0, d["positions"], d["frequencies"])


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=5), "dtype"), (dict(batch=-1), "out of range"), (dict(pairs=33), "do not fit"),
    (dict(pairs=-1), "do not fit"), (dict(magnitude=float("inf")), "magnitude"), (dict(), "NULL")])
def test_rotary_refusals(lib, kw, fragment):
    assert lib.mg_rotary(rotary(**kw), None, None, None, None, None) == INVALID
    assert fragment in lib.mg_last_error().decode()
    assert lib.mg_rotary(rotary(positions=0), PTR, None, PTR, None, None) == INVALID
    assert "positions" in lib.mg_last_error().decode()


def paged(**kw):
    d = dict(dtype=0, batch=1, heads=2, kv_heads=1, head_dim=64, page_size=16, pages=4, table_width=2, scale=0.125,
             cap=0.0, slopes=0, block_table=PTR, lengths=PTR)
    d.update(kw)
    lead = [d[n] for n in ("dtype", "batch", "heads", "kv_heads", "head_dim", "page_size", "pages", "table_width",
                           "scale", "cap")]
    return T._PAGED.pack(*lead, *([64] * 15), d["slopes"], d["block_table"], d["lengths"])


@pytest.mark.parametrize("kw,status,fragment", [
    (dict(dtype=-1), INVALID, "dtype"), (dict(page_size=0), INVALID, "out of range"),
    (dict(heads=3, kv_heads=2), INVALID, "multiple"), (dict(head_dim=200), UNSUPPORTED, "head_dim"),
    (dict(scale=float("inf")), INVALID, "scale"), (dict(cap=-3.0), INVALID, "cap"),
    (dict(table_width=1 << 28), UNSUPPORTED, "too wide"), (dict(), INVALID, "NULL")])
def test_paged_refusals(lib, kw, status, fragment):
    assert lib.mg_paged_attention(paged(**kw), *([None] * 8)) == status
    assert fragment in lib.mg_last_error().decode()
    assert lib.mg_paged_attention(paged(), PTR, PTR, PTR, PTR, PTR, PTR, None, None) == INVALID
    assert "come together" in lib.mg_last_error().decode()


def test_python_refuses_cpu_tensors():
    import torch

    x = torch.zeros((1, 1, 4, 8))
    with pytest.raises(mg.MacrogradError, match="CUDA tensor"):
        mg.attention(x, x, x)
    with pytest.raises(mg.MacrogradError, match="CUDA tensor"):
        mg.rotary(x, None, torch.zeros(4, dtype=torch.int32), mg.rotary_frequencies(8, device="cpu"))
    with pytest.raises(mg.MacrogradError, match="CUDA tensor"):
        mg.paged_attention(x[0], x, x, x, x)


def test_backward_refuses_more_rows_than_its_statistics_number(lib):
    d = attention(B=1 << 26, H=2, Lq=2, Lk=2)
    assert lib.mg_attention_backward(d, *([None] * 10)) == UNSUPPORTED
    assert "too large" in lib.mg_last_error().decode()
    assert lib.mg_attention(d, None, None, None, None, None, None) == INVALID     # the forward pass has none


@pytest.mark.parametrize("x", [1e39, -1e39, float("inf"), float("nan")])
def test_numbers_beyond_fp32_are_refused_as_arguments(x):
    with pytest.raises(mg.MacrogradError, match="scale must be finite"):
        T._number(x, "scale")
    largest = (2 - 2.0 ** -23) * 2.0 ** 127
    assert T._number(largest, "scale") == largest
    assert len(T._ATTENTION.pack(0, 1, 1, 1, 1, 1, 8, 1, largest, 0.0, *([0] * 27))) == T._ATTENTION.size


@pytest.mark.parametrize("kw", [dict(theta=0.0), dict(theta=float("inf")), dict(factor=-1.0), dict(factor=float("nan"))])
def test_rotary_frequencies_refuse_what_is_not_positive_and_finite(kw):
    with pytest.raises(mg.MacrogradError, match="positive"):
        mg.rotary_frequencies(8, device="cpu", **kw)
