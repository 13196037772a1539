"""rotary and rotary_backward against complex multiplication in 64 bits: types,
both layouts, parts of the head, odd sizes, far positions, views, in place,
captured graphs.

Bounds: an angle is off by 2^-32 turns of its fixed point, 2^-25 turns of its
rounding to fp32 (below a quarter turn: 2^-24 relative) and the two of sincospi
itself: 4 * 2^-24 * 2 pi altogether with room; the products and the sum round
three times in fp32, and the result once to its type."""
import math

import pytest

torch = pytest.importorskip("torch")
import macrograd_b200 as mg  # noqa: E402
from attention_reference import half_step, rotate, within  # noqa: E402

pytestmark = pytest.mark.gpu


def bound(x, want, pairs, interleaved, magnitude=1.0):
    u32 = 2.0 ** -24
    y = x.double().abs().clone()
    a = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    b = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    both = (y[..., a] + y[..., b]) * (8 * math.pi + 4) * u32 * magnitude
    tol = torch.zeros_like(y)
    tol[..., a] = tol[..., b] = both
    u = half_step(x.dtype)
    return tol * (1 + u) + u * want.abs() * (1 if x.dtype != torch.float32 else 2) + 1e-30


def check(x, y, positions, f, **kw):
    want = rotate(x, positions, f, **kw)
    tol = bound(x, want, f.numel(), kw.get("interleaved", False), kw.get("magnitude", 1.0))
    tol[..., 2 * f.numel():] = 1e-38          # the rest is copied
    within(y, want, tol, "rotated")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("B,H,Hkv,L,D,part", [
    (1, 1, 1, 1, 2, 2), (2, 3, 1, 5, 16, 16), (2, 4, 2, 33, 64, 32), (1, 8, 2, 130, 128, 128), (3, 2, 2, 7, 80, 24),
    (1, 2, 1, 9, 33, 14), (1, 32, 8, 300, 128, 64), (2, 5, 5, 64, 96, 0)])
def test_rotary_and_its_gradient(B, H, Hkv, L, D, part, interleaved, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((B, L, H, D), generator=g, device="cuda").to(dtype).transpose(1, 2)
    k = torch.randn((B, Hkv, L, D), generator=g, device="cuda").to(dtype)
    positions = torch.randint(0, 5000, (B, L), generator=g, device="cuda").int()
    f = mg.rotary_frequencies(part)
    rq, rk = mg.rotary(q, k, positions, f, interleaved=interleaved)
    check(q, rq, positions, f, interleaved=interleaved)
    check(k, rk, positions, f, interleaved=interleaved)
    bq, bk = mg.rotary_backward(q, k, positions, f, interleaved=interleaved)
    check(q, bq, positions, f, interleaved=interleaved, inverse=True)
    check(k, bk, positions, f, interleaved=interleaved, inverse=True)
    assert rq.stride() == torch.empty_like(q).stride()


@pytest.mark.parametrize("start", [0, 10 ** 6, 2 ** 31 - 40, -(2 ** 31), -7])
def test_far_positions(start):
    """Whole turns drop out exactly, for any int32 position; the frequencies' own 2^-53 is what is left."""
    x = torch.randn((1, 2, 33, 64), device="cuda")
    positions = (torch.arange(33, device="cuda") + start).int()
    f = mg.rotary_frequencies(64)
    y, none = mg.rotary(x, None, positions, f)
    assert none is None
    want = rotate(x, positions, f)
    # the reference's own angle, a double of up to 2^31 radians, is off by 2^-22 radians
    far = (abs(start) + 64) * 2.0 ** -52
    within(y, want, bound(x, want, 32, False) + far * x.abs().max().double() * 2, "far")


@pytest.mark.parametrize("scaling,kw", [("linear", dict(factor=4.0)), ("ntk", dict(factor=8.0)),
                                        ("parts", dict(factor=8.0, trained=4096))])
def test_scalings(scaling, kw):
    base = mg.rotary_frequencies(64, device="cpu")
    f = mg.rotary_frequencies(64, scaling=scaling, device="cpu", **kw)
    factor = kw["factor"]
    if scaling == "linear":
        assert torch.equal(f, base / factor)
    if scaling == "ntk":
        assert f[0] == base[0] and abs(f[-1] * factor / base[-1] - 1) < 1e-12
    if scaling == "parts":
        turns = 4096 * base / (2 * math.pi)
        assert torch.equal(f[turns > 32], base[turns > 32]) and torch.equal(f[turns < 1], base[turns < 1] / factor)
        assert (f[1:] < f[:-1]).all()
    x = torch.randn((1, 2, 65, 64), device="cuda")
    pos = torch.arange(30000, 30065, device="cuda").int()
    y, _ = mg.rotary(x, None, pos, f.cuda(), magnitude=1.25)
    check(x, y, pos, f.cuda(), magnitude=1.25)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_views_and_in_place(dtype):
    """Slices of a packed buffer, turned where they are; the values between them stay."""
    buf = torch.randn((2, 40, 3, 4, 64), device="cuda").to(dtype)
    old = buf.clone()
    q, k = buf[:, :, 0].transpose(1, 2), buf[:, :, 1].transpose(1, 2)
    pos = torch.arange(40, device="cuda").int()
    f = mg.rotary_frequencies(64)
    want = mg.rotary(old[:, :, 0].transpose(1, 2), old[:, :, 1].transpose(1, 2), pos, f)
    got = mg.rotary(q, k, pos, f, out_q=q, out_k=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(buf[:, :, 2], old[:, :, 2])
    odd = torch.randn((1, 2, 9, 65), device="cuda").to(dtype)[..., 1:]      # rows off 16 bytes
    y, _ = mg.rotary(odd, None, pos[:9], f)
    check(odd, y, pos[:9], f)


def test_captured_and_replayed():
    x = torch.randn((4, 8, 1, 128), device="cuda").bfloat16()
    pos = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    f = mg.rotary_frequencies(128)
    mg.rotary(x, x, pos, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = mg.rotary(x, x, pos, f)
    pos.fill_(12345)
    graph.replay()
    torch.cuda.synchronize()
    check(x, y, pos, f)
    assert torch.equal(y, z)


def test_empty():
    f = mg.rotary_frequencies(8)
    x = torch.empty((0, 2, 3, 8), device="cuda")
    y, _ = mg.rotary(x, None, torch.zeros(3, dtype=torch.int32, device="cuda"), f)
    assert y.shape == x.shape


def test_refusals():
    x = torch.zeros((1, 2, 3, 8), device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    f = mg.rotary_frequencies(8)
    for call, fragment in [
            (lambda: mg.rotary(x, None, pos, mg.rotary_frequencies(10)), "do not fit"),
            (lambda: mg.rotary(x, None, pos.long(), f), "positions"),
            (lambda: mg.rotary(x, None, pos[:2], f), "positions"),
            (lambda: mg.rotary(x, None, pos, f.float()), "frequencies"),
            (lambda: mg.rotary(x, x[:, :, :2], pos, f), "Found shapes"),
            (lambda: mg.rotary(x, x.bfloat16(), pos, f), "as the others"),
            (lambda: mg.rotary(x, None, pos, f, out_k=x), "out_k without k"),
            (lambda: mg.rotary(x, None, pos, f, out_q=x[..., :4]), "out_q"),
            (lambda: mg.rotary(x, x, pos, f, out_q=x, out_k=x), "same memory"),
            (lambda: mg.rotary(x, x.clone(), pos, f, out_k=x), "same memory"),
            (lambda: mg.rotary(x, None, pos, f, magnitude=math.nan), "magnitude"),
            (lambda: mg.rotary_frequencies(7), "even"),
            (lambda: mg.rotary_frequencies(8, scaling="other"), "scaling"),
            (lambda: mg.rotary_frequencies(8, scaling="parts"), "trained"),
            (lambda: mg.rotary_frequencies(8, theta=-1.0), "positive")]:
        with pytest.raises(mg.MacrogradError, match=fragment):
            call()


def test_outputs_that_overlap_the_inputs_otherwise_are_refused():
    buf = torch.randn((2, 40, 3, 4, 64), device="cuda")
    q, k = buf[:, :, 0].transpose(1, 2), buf[:, :, 1].transpose(1, 2)
    pos, f = torch.arange(40, device="cuda").int(), mg.rotary_frequencies(64)
    flat = buf.flatten(2)
    between = flat[:, :, 64:320].unflatten(2, (4, 64)).transpose(1, 2)          # queries 1 to 3 and the first key
    for kw, fragment in [(dict(out_q=between), "out_q overlaps q"), (dict(out_k=between), "out_k overlaps k"),
                         (dict(out_q=flat[:, :, 320:576].unflatten(2, (4, 64)).transpose(1, 2)), "out_q overlaps k")]:
        with pytest.raises(mg.MacrogradError, match=fragment):
            mg.rotary(q, k, pos, f, **kw)


def test_one_token_in_place_through_another_view():
    """The stride of a dim of one element says nothing: a token's heads viewed in two ways are the same elements."""
    x = torch.randn((3, 4, 64), device="cuda")
    a, b = x.view(3, 1, 4, 64).transpose(1, 2), x.view(3, 4, 1, 64)
    assert a.stride() != b.stride()
    pos, f = torch.tensor([[5], [6], [1000]], dtype=torch.int32, device="cuda"), mg.rotary_frequencies(64)
    want, _ = mg.rotary(a, None, pos, f)
    got, _ = mg.rotary(a, None, pos, f, out_q=b)
    assert got is b and torch.equal(x.view(3, 4, 1, 64), want)
    with pytest.raises(mg.MacrogradError, match="out_q overlaps q"):
        mg.rotary(x.view(1, 3, 4, 64), None, pos.new_zeros((4,)), f, out_q=x.view(1, 4, 3, 64).transpose(1, 2))
