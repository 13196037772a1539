"""Overlaps of strided views (macrograd_b200/csrc/mg_overlap.h) on the CPU: the
header that the entry points compile, built into tests/overlap_check.cpp with
g++ and compared with all pairs of elements of small random views; and the
refusals of the C ABI that rest on it, before any device is touched."""
import os
import shutil
import subprocess

import pytest

import macrograd_b200 as mg
from macrograd_b200 import _lib, transformer as T

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "macrograd_b200", "csrc")


def test_views_meet_where_they_share_a_byte(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "overlap_check")
    subprocess.run([cxx, "-std=gnu++17", "-O2", "-Wall", "-Werror", "-I", CSRC, os.path.join(HERE, "overlap_check.cpp"),
                    "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


def has_device():
    import torch

    return torch.cuda.is_available()


@pytest.fixture(scope="module")
def lib():
    if has_device():
        pytest.skip("addresses that are no memory: only where nothing can be launched")
    return mg.load(build_if_missing=True)


B, H, L, D = 2, 4, 8, 64
ROW, SIZE = 3 * H * D, 4 * B * L * 3 * H * D      # a packed projection [B, L, 3, H, D] in fp32: a row's elements, all bytes
STRIDES = [L * ROW, D, ROW]
BASE = 1 << 32


def slot(i, buffer=0, shift=0):
    """Address of the queries, keys or values of packed buffer `buffer`, `shift` elements on."""
    return BASE + buffer * SIZE + 4 * (i * H * D + shift)


def refused(status, lib, fragment):
    assert status == _lib.MG_ERR_INVALID, lib.mg_last_error().decode()
    assert fragment in lib.mg_last_error().decode()


def attention_desc(out=STRIDES):
    return T._ATTENTION.pack(0, B, H, H, L, L, D, 1, 0.125, 0.0, *STRIDES * 3, *out, *STRIDES * 4, 0, 0, 0)


LSE = BASE + 20 * SIZE


@pytest.mark.parametrize("at,fragment", [
    (slot(1), "out overlaps k"), (slot(2), "out overlaps v"), (slot(1, shift=5), "out overlaps k"),
    (slot(2, shift=-1), "out overlaps"), (slot(0, shift=4), "out overlaps q"), (slot(0) + ROW * 4, "out overlaps q")])
def test_attention_refuses_outputs_over_inputs(lib, at, fragment):
    refused(lib.mg_attention(attention_desc(), at, LSE, slot(0), slot(1), slot(2), None), lib, fragment)


def test_attention_refuses_out_over_q_with_other_strides_and_lse_over_anything(lib):
    dense = [H * L * D, L * D, D]
    refused(lib.mg_attention(attention_desc(dense), slot(0), LSE, slot(0), slot(1), slot(2), None), lib, "out overlaps q")
    for at, name in ((slot(0), "q"), (slot(1) + 4 * ROW, "k"), (slot(2), "v"), (slot(0, 5), "out")):
        refused(lib.mg_attention(attention_desc(), slot(0, 5), at, slot(0), slot(1), slot(2), None), lib, f"lse overlaps {name}")


GRADIENTS = ["dq", "dk", "dv"]
INPUTS = ["q", "k", "v", "dout", "out"]


@pytest.mark.parametrize("gradient", GRADIENTS)
@pytest.mark.parametrize("other", INPUTS + ["lse"] + GRADIENTS)
def test_gradients_over_inputs_and_each_other_are_refused(lib, gradient, other):
    if gradient == other:
        return
    at = {n: slot(0, i) for i, n in enumerate(GRADIENTS + INPUTS)}
    at["lse"] = LSE
    at[gradient] = at[other] + (0 if other == "lse" else 4 * D)       # a head on
    status = lib.mg_attention_backward(attention_desc(), *(at[n] for n in GRADIENTS), at["dout"], at["q"], at["k"],
                                       at["v"], at["out"], at["lse"], None)
    refused(status, lib, "overlaps")
    message = lib.mg_last_error().decode()
    assert gradient in message and other in message


def rotary_desc(out=STRIDES):
    return T._ROTARY.pack(0, B, H, H, L, D, D // 2, 0, 0, 1.0, *STRIDES * 2, *out, *STRIDES, 0, BASE, BASE)


def test_rotary_refuses_overlaps_that_are_not_the_input_itself(lib):
    dense = [H * L * D, L * D, D]
    for desc, out_q, out_k, fragment in [
            (rotary_desc(dense), slot(0), slot(1, 3), "out_q overlaps q"),
            (rotary_desc(), slot(0, shift=2), slot(1, 3), "out_q overlaps q"),
            (rotary_desc(), slot(1), slot(1, 3), "out_q overlaps k"),
            (rotary_desc(), slot(0, 3), slot(0), "out_k overlaps q"),
            (rotary_desc(), slot(0, 3), slot(1) + 4 * ROW, "out_k overlaps k"),
            (rotary_desc(), slot(0, 3), slot(0, 3, 8), "out_q overlaps out_k")]:
        refused(lib.mg_rotary(desc, out_q, out_k, slot(0), slot(1), None), lib, fragment)


def test_paged_attention_refuses_outputs_over_inputs(lib):
    pages, page, heads = 6, 16, H
    pool = [page * heads * 2 * D, heads * 2 * D, 2 * D]           # keys and values side by side
    desc = T._PAGED.pack(0, B, H, heads, D, page, pages, 2, 0.125, 0.0, H * D, D, H * D, D, *pool, *pool, H * D, D, H * D,
                         D, 2, 0, BASE, BASE)
    k, v, q, kn, vn, out = BASE, BASE + 4 * D, BASE + SIZE * 8, BASE + SIZE * 9, BASE + SIZE * 10, BASE + SIZE * 11
    call = lambda out=out, lse=LSE, k=k, v=v, kn=kn, vn=vn: lib.mg_paged_attention(desc, out, lse, q, k, v, kn, vn, None)  # noqa: E731
    for kw, fragment in [
            (dict(out=q + 4), "out overlaps q"), (dict(out=k + 4 * D * 8), "out overlaps k_pages"),
            (dict(out=v + 8 * D * 4), "out overlaps"), (dict(out=kn), "out overlaps k_new"),
            (dict(out=vn + 64), "out overlaps v_new"), (dict(lse=q), "lse overlaps q"), (dict(lse=out), "lse overlaps out"),
            (dict(lse=v), "lse overlaps v_pages"), (dict(v=k + 4 * (D - 1)), "k_pages overlaps v_pages"),
            (dict(v=k), "k_pages overlaps v_pages")]:
        refused(call(**kw), lib, fragment)
