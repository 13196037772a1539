"""attention and attention_backward against the definition in 64 bits: types,
shared heads, head sizes, lengths from one token on, strided views, caps, biases,
documents, prefixes, rows that see nothing, padding that holds NaN; determinism,
other streams, captured graphs, offsets beyond 32 bits."""
import ctypes
import math
from concurrent.futures import ThreadPoolExecutor

import pytest

torch = pytest.importorskip("torch")
import macrograd_b200 as mg  # noqa: E402
from macrograd_b200 import _lib, transformer  # noqa: E402
from attention_reference import Reference, half_step, within  # noqa: E402

pytestmark = pytest.mark.gpu

SIZES = [  # B, H, Hkv, Lq, Lk, D
    (1, 1, 1, 1, 1, 8),
    (2, 4, 2, 1, 257, 64),
    (3, 2, 1, 5, 7, 16),
    (1, 2, 1, 17, 17, 40),
    (1, 3, 3, 33, 70, 33),
    (2, 2, 2, 64, 64, 64),
    (2, 3, 3, 128, 128, 64),
    (1, 4, 2, 129, 255, 128),
    (1, 2, 2, 200, 100, 64),
    (1, 6, 2, 257, 513, 96),
    (1, 2, 1, 640, 640, 128),
    (2, 1, 1, 385, 385, 80),
    (1, 5, 1, 128, 384, 128),
]
MASKS = ["full", "causal", "cap", "slopes", "documents", "prefix", "all"]


def make(size, mask, dtype, seed=0, strided=True):
    B, H, Hkv, Lq, Lk, D = size
    g = torch.Generator(device="cuda").manual_seed(seed)
    gain = 3.0 if mask in ("cap", "all") else 1.0

    def heads(n, L, gain=1.0):
        if strided:
            return (torch.randn((B, L, n, D), generator=g, device="cuda") * gain).to(dtype).transpose(1, 2)
        return (torch.randn((B, n, L, D), generator=g, device="cuda") * gain).to(dtype)

    q, k, v, dout = heads(H, Lq, gain), heads(Hkv, Lk), heads(Hkv, Lk), heads(H, Lq)
    kw = dict(causal=mask != "full")
    if mask in ("cap", "all"):
        kw["cap"] = 10.0
    if mask in ("slopes", "all"):
        kw["slopes"] = torch.tensor([2.0 ** (-1 - h) for h in range(H)], device="cuda")
    if mask in ("documents", "all"):
        ids = torch.zeros((B, Lk), dtype=torch.int32)
        for b in range(B):
            cuts = sorted(int(x) for x in torch.randint(0, Lk + 1, (3,), generator=torch.Generator().manual_seed(b)))
            for i, c in enumerate(cuts):
                ids[b, c:] = 5 - i           # ids fall along the row
            ids[b, Lk - Lk // 9:] = -1       # padding at the end
        kw["documents"] = ids.cuda()
    if mask in ("prefix", "all"):
        kw["prefix"] = torch.tensor([Lk * (2 * b + 1) // (3 * B) for b in range(B)], dtype=torch.int32, device="cuda")
    return q, k, v, dout, kw


def compare(q, k, v, dout, kw):
    out, lse = mg.attention(q, k, v, **kw)
    ref = Reference(q, k, v, dout, **kw)
    within(out, ref.out, ref.out_tol, "out")
    within(lse, ref.lse, ref.lse_tol, "lse")
    dq, dk, dv = mg.attention_backward(dout, q, k, v, out, lse, **kw)
    within(dv, ref.dv, ref.dv_tol, "dv")
    within(dq, ref.dq, ref.dq_tol, "dq")
    within(dk, ref.dk, ref.dk_tol, "dk")
    assert out.stride() == torch.empty_like(q).stride()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_attention_and_gradients(size, mask, dtype):
    compare(*make(size, mask, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_long_rows(dtype):
    """Several rows of tiles, an odd length, shared heads, documents shorter and longer than a tile."""
    q, k, v, dout, kw = make((1, 4, 2, 1537, 1537, 128), "causal", dtype, 3)
    ids = torch.repeat_interleave(torch.arange(6), torch.tensor([1, 130, 700, 5, 601, 100])).int()[None].cuda()
    kw["documents"] = ids.contiguous()
    compare(q, k, v, dout, kw)


@pytest.mark.parametrize("layout", ["packed", "unaligned", "wide"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_views(layout, dtype):
    """q, k, v as slices of one buffer; rows that do not start on 16 bytes; rows much wider than a head."""
    B, H, L, D = 2, 3, 150, 64
    g = torch.Generator(device="cuda").manual_seed(7)
    if layout == "packed":
        qkv = torch.randn((B, L, 3, H, D), generator=g, device="cuda").to(dtype)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    else:
        pad = 1 if layout == "unaligned" else 448
        q, k, v = (torch.randn((B, H, L, D + pad), generator=g, device="cuda").to(dtype)[..., pad:] for _ in range(3))
    dout = torch.randn((B, L, H, D), generator=g, device="cuda").to(dtype).transpose(1, 2)
    compare(q, k, v, dout, dict(causal=True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 33])
def test_padding_may_hold_anything(dtype, D):
    """NaN and infinity in the keys, values, queries and upstream gradients of padding reach nothing."""
    L = 300
    q, k, v, dout, _ = make((2, 2, 1, L, L, D), "causal", dtype, 11, strided=False)
    ids = torch.zeros((2, L), dtype=torch.int32, device="cuda")
    ids[0, 200:] = -1
    ids[1, 100:140] = -1     # padding in the middle of a row
    ids[1, 140:] = 4
    for t in (q, k, v, dout):
        pad = (ids < 0)[:, None, :, None].expand_as(t)
        t[pad] = float("nan")
        t[0, :, 250] = float("inf")
    kw = dict(causal=True, documents=ids)
    compare(q, k, v, dout, kw)
    out, lse = mg.attention(q, k, v, **kw)
    assert (out[0, :, 200:] == 0).all() and torch.isneginf(lse[0, :, 200:]).all()
    dq, dk, dv = mg.attention_backward(dout, q, k, v, out, lse, **kw)
    for t in (dq, dk, dv):
        assert (t[0, :, 200:] == 0).all() and (t[1, :, 100:140] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_rows_that_see_nothing(dtype):
    """More queries than keys: the first queries stand before every key."""
    q, k, v, dout, kw = make((1, 2, 1, 150, 20, 64), "causal", dtype, 5)
    out, lse = mg.attention(q, k, v, **kw)
    assert (out[:, :, :130] == 0).all() and torch.isneginf(lse[:, :, :130]).all()
    compare(q, k, v, dout, kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("Lq", [1, 9])
def test_no_keys(dtype, Lq):
    q = torch.randn((2, 2, Lq, 64), device="cuda").to(dtype)
    k = torch.empty((2, 1, 0, 64), device="cuda", dtype=dtype)
    out, lse = mg.attention(q, k, k)
    assert (out == 0).all() and torch.isneginf(lse).all()
    dq, dk, dv = mg.attention_backward(q, q, k, k, out, lse)
    assert (dq == 0).all() and dk.numel() == dv.numel() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_no_queries(dtype):
    q = torch.empty((2, 2, 0, 64), device="cuda", dtype=dtype)
    k = torch.randn((2, 1, 130, 64), device="cuda").to(dtype)
    out, lse = mg.attention(q, k, k)
    dq, dk, dv = mg.attention_backward(q, q, k, k, out, lse)
    assert out.numel() == dq.numel() == 0 and (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_scores_of_several_hundred(dtype, cap):
    """Scores of several hundred: the running maximum moves far, sums stay finite."""
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn((1, 2, 400, 64), generator=g, device="cuda").mul(8).to(dtype) for _ in range(2))
    v, dout = (torch.randn((1, 2, 400, 64), generator=g, device="cuda").to(dtype) for _ in range(2))
    k[:, :, 300:] *= 4       # the maximum comes late
    compare(q, k, v, dout, dict(causal=False, cap=cap))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_same_inputs_same_bits(dtype):
    q, k, v, dout, kw = make((1, 4, 1, 300, 300, 64), "all", dtype, 4)
    first = mg.attention(q, k, v, **kw)
    grads = mg.attention_backward(dout, q, k, v, *first, **kw)
    for _ in range(3):
        again = mg.attention(q, k, v, **kw)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert all(torch.equal(a, b) for a, b in zip(grads, mg.attention_backward(dout, q, k, v, *again, **kw)))


def test_scale_is_the_callers():
    q, k, v, dout, kw = make((1, 2, 2, 100, 100, 64), "causal", torch.float32, 8)
    compare(q, k, v, dout, dict(kw, scale=0.3))
    compare(q, k, v, dout, dict(kw, scale=-0.05))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_negative_scale_with_cap_and_slopes(dtype, D):
    q, k, v, dout, kw = make((1, 2, 1, 150, 150, D), "all", dtype, 12)
    compare(q, k, v, dout, dict(kw, scale=-0.1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_scale_of_zero_and_far_caps(dtype):
    """Every seen key weighs the same; a cap far above the scores changes nothing, one far below makes them all its own."""
    q, k, v, dout, kw = make((1, 2, 1, 150, 150, 64), "causal", dtype, 12)
    compare(q, k, v, dout, dict(kw, scale=0.0))
    compare(q, k, v, dout, dict(kw, cap=1e6))
    ref = Reference(q, k, v, scale=0.0, **kw)
    for more in (dict(cap=1e-20), dict(cap=1e-30, scale=1e30)):
        out, lse = mg.attention(q, k, v, **more, **kw)
        within(out, ref.out, ref.out_tol, "out under a cap of nearly nothing")
        assert torch.isfinite(lse).all()
        one, _ = mg.attention(q[:, :, -1:], k, v, **more, **kw)
        within(one, ref.out[:, :, -1:], ref.out_tol[:, :, -1:], "one query under it")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 33])
def test_broadcast_keys_and_values(dtype, D):
    """k and v expanded over the batch and over heads (stride 0)."""
    g = torch.Generator(device="cuda").manual_seed(14)
    q, dout = (torch.randn((3, 4, 140, D), generator=g, device="cuda").to(dtype) for _ in range(2))
    k = torch.randn((1, 2, 200, D), generator=g, device="cuda").to(dtype).expand(3, 2, 200, D)
    v = torch.randn((3, 1, 200, D), generator=g, device="cuda").to(dtype).expand(3, 2, 200, D)
    compare(q, k, v, dout, dict(causal=True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("ids", ["each its own", "any sign", "one", "none"])
def test_kinds_of_documents(dtype, ids):
    """A document to each position, ids of any 32-bit value, a single document, nothing but padding."""
    L = 270
    q, k, v, dout, _ = make((2, 2, 2, L, L, 64), "causal", dtype, 15)
    docs = {"each its own": torch.arange(L), "any sign": torch.randint(-3, 3, (L,), generator=torch.Generator().manual_seed(1))
            * (2 ** 30) + torch.arange(L) // 90, "one": torch.full((L,), 2 ** 31 - 1), "none": torch.full((L,), -7)}[ids]
    kw = dict(documents=docs.int().cuda().expand(2, L).contiguous())
    compare(q, k, v, dout, dict(kw, causal=True))
    compare(q, k, v, dout, dict(kw, causal=False))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_prefixes_out_of_range(dtype):
    q, k, v, dout, _ = make((3, 2, 2, 130, 200, 64), "causal", dtype, 16)
    compare(q, k, v, dout, dict(prefix=torch.tensor([-5, 0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_few_queries_of_a_long_row(dtype):
    q, k, v, dout, kw = make((1, 2, 1, 3, 5000, 64), "causal", dtype, 17)
    compare(q, k, v, dout, kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("mask", ["full", "all"])
@pytest.mark.parametrize("D", [64, 96])
def test_rows_shared_by_several_blocks(dtype, mask, D):
    """Few heads: each row of keys is read in parts and joined; parts without a key that is seen, and rows without any."""
    compare(*make((1, 2, 1, 700, 3100, D), mask, dtype, 18))


def test_two_graphs_at_once():
    """Two captured graphs, each with scratch of its own, replayed on two streams at the same time."""
    sets = [make((1, 8, 2, 900, 900, 64), "all", torch.bfloat16, 40 + i) for i in range(2)]
    want, graphs, got = [], [], []
    for q, k, v, dout, kw in sets:
        f = mg.attention(q, k, v, **kw)
        want.append(f + mg.attention_backward(dout, q, k, v, *f, **kw))
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            f = mg.attention(q, k, v, **kw)
            got.append(f + mg.attention_backward(dout, q, k, v, *f, **kw))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_out_and_its_neighbours():
    """out given as a view: its rows are written, what lies around them stays."""
    q, k, v, _, kw = make((2, 3, 3, 150, 150, 64), "causal", torch.bfloat16, 9)
    room = torch.full((2, 170, 5, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    out = room[:, 10:160, 1:4].transpose(1, 2)
    got, _ = mg.attention(q, k, v, out=out, **kw)
    assert got is out
    assert torch.equal(out, mg.attention(q, k, v, **kw)[0])
    rest = torch.ones_like(room, dtype=torch.bool)
    rest[:, 10:160, 1:4] = False
    assert (room[rest] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("Lq", [1, 140])
def test_captured_and_replayed_with_other_inputs(dtype, Lq):
    size = (2, 2, 1, Lq, 300, 64)
    q, k, v, dout, kw = make(size, "all", dtype, 20)
    mg.attention_backward(dout, q, k, v, *mg.attention(q, k, v, **kw), **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = mg.attention(q, k, v, **kw)
        grads = mg.attention_backward(dout, q, k, v, out, lse, **kw)
    for seed in (21, 22):
        q2, k2, v2, dout2, _ = make(size, "all", dtype, seed)
        for a, b in ((q, q2), (k, k2), (v, v2), (dout, dout2)):
            a.copy_(b)
        kw["documents"].copy_(kw["documents"].roll(seed - 20, 1))
        kw["prefix"].add_(seed)
        graph.replay()
        torch.cuda.synchronize()
        want = mg.attention(q, k, v, **kw)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        for a, b in zip(grads, mg.attention_backward(dout, q, k, v, *want, **kw)):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls on two streams do not share scratch."""
    sets = [make((1, 8, 2, 700, 700, 64), "all", torch.bfloat16, 30 + i) for i in range(2)]
    want = []
    for q, k, v, dout, kw in sets:
        f = mg.attention(q, k, v, **kw)
        want.append(f + mg.attention_backward(dout, q, k, v, *f, **kw))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, (q, k, v, dout, kw) in enumerate(sets):
            f = mg.attention(q, k, v, stream=streams[i], **kw)
            got[i].append(f + mg.attention_backward(dout, q, k, v, *f, stream=streams[i], **kw))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


@pytest.mark.parametrize("Lq", [1, 130])
def test_offsets_beyond_32_bits(Lq):
    """Batches and heads more than 2^32 bytes and 2^31 elements apart."""
    far = (1 << 31) + 4096
    buf = torch.zeros(far + 300 * 64 * 4, dtype=torch.bfloat16, device="cuda")
    k = torch.as_strided(buf, (2, 2, 200, 64), (far, 200 * 64, 64, 1))
    g = torch.Generator(device="cuda").manual_seed(1)
    k.copy_(torch.randn((2, 2, 200, 64), generator=g, device="cuda"))
    q = torch.randn((2, 2, Lq, 64), generator=g, device="cuda").bfloat16()
    dout = torch.randn((2, 2, Lq, 64), generator=g, device="cuda").bfloat16()
    kw = dict(causal=True)
    out, lse = mg.attention(q, k, k, **kw)
    ref = Reference(q, k, k, dout, **kw)
    within(out, ref.out, ref.out_tol, "out")
    within(lse, ref.lse, ref.lse_tol, "lse")
    dq, dk, dv = mg.attention_backward(dout, q, k, k, out, lse, **kw)
    within(dq, ref.dq, ref.dq_tol, "dq")
    within(dk, ref.dk, ref.dk_tol, "dk")
    within(dv, ref.dv, ref.dv_tol, "dv")


@pytest.mark.parametrize("kw", [dict(causal=True), dict(causal=False, cap=4.0)], ids=["causal", "cap"])
def test_gradients_against_differences(kw):
    """Central differences of the forward call itself, in fp32: step h = 2^-6 leaves h^2 / 6 of the third derivative
    (below 2^-13 for these O(1) functions summed over 60 outputs) and 2^-24 * |loss| / h of rounding."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v, dout = (torch.randn((1, 1, 6, 10), generator=g, device="cuda") for _ in range(4))
    out, lse = mg.attention(q, k, v, **kw)
    grads = mg.attention_backward(dout, q, k, v, out, lse, **kw)
    h = 2.0 ** -6
    loss = lambda: float((mg.attention(q, k, v, **kw)[0].double() * dout.double()).sum())  # noqa: E731
    for t, grad in zip((q, k, v), grads):
        flat = t.view(-1)
        for i in range(0, 60, 7):
            x = float(flat[i])
            flat[i] = x + h
            up = loss()
            flat[i] = x - h
            down = loss()
            flat[i] = x
            assert abs((up - down) / (2 * h) - float(grad.view(-1)[i])) < 2e-3


def test_refusals():
    t = lambda *s, **k: torch.zeros(s, device="cuda", **k)  # noqa: E731
    q, kv = t(1, 4, 8, 64), t(1, 2, 8, 64)
    bad = [
        (lambda: mg.attention(q.cpu(), kv, kv), "CUDA tensor"),
        (lambda: mg.attention(q.half(), kv.half(), kv.half()), "float32 or bfloat16"),
        (lambda: mg.attention(q, kv.bfloat16(), kv.bfloat16()), "as the others"),
        (lambda: mg.attention(q[0], kv, kv), "4 dims"),
        (lambda: mg.attention(q, t(1, 3, 8, 64), t(1, 3, 8, 64)), "multiple"),
        (lambda: mg.attention(q, t(1, 2, 8, 32), t(1, 2, 8, 32)), "Found shapes"),
        (lambda: mg.attention(q, kv, t(1, 2, 9, 64)), "Found shapes"),
        (lambda: mg.attention(q.transpose(2, 3).contiguous().transpose(2, 3), kv, kv), "contiguous in its last dim"),
        (lambda: mg.attention(t(1, 4, 8, 136), t(1, 2, 8, 136), t(1, 2, 8, 136)), "head_dim"),
        (lambda: mg.attention(q, kv, kv, cap=-1.0), "cap"),
        (lambda: mg.attention(q, kv, kv, cap=1e31), "cap"),
        (lambda: mg.attention(q, kv, kv, scale=1e31), "scale"),
        (lambda: mg.attention(q, kv, kv, scale=math.inf), "finite"),
        (lambda: mg.attention(q, kv, kv, slopes=t(2)), "slopes"),
        (lambda: mg.attention(q, kv, kv, documents=t(1, 8)), "documents"),
        (lambda: mg.attention(q, kv, kv, causal=False, prefix=t(1, dtype=torch.int32)), "prefix"),
        (lambda: mg.attention(q, kv, kv, out=t(1, 4, 8, 32)), "out"),
        (lambda: mg.attention(q, kv, kv, out=t(1, 1, 8, 64).expand(1, 4, 8, 64)), "overlap"),
        (lambda: mg.attention_backward(q, q, kv, kv, q, t(1, 4, 9)), "lse"),
        (lambda: mg.attention_backward(t(1, 4, 9, 64), q, kv, kv, q, t(1, 4, 8)), "dout"),
    ]
    for call, fragment in bad:
        with pytest.raises(mg.MacrogradError, match=fragment):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(1, 4, 2, 200, 200, 64), (1, 2, 1, 150, 150, 128), (1, 2, 1, 70, 70, 33),
                                  (1, 2, 2, 3, 3000, 64), (1, 2, 1, 1, 2000, 128), (1, 2, 1, 1, 50, 33)], ids=str)
@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("place", ["q", "k", "v", "dout"])
def test_nan_that_is_seen_stays(place, cap, size, dtype):
    """A NaN that a row sees reaches its results, and with them the gradients that the row has a part in."""
    q, k, v, dout, _ = make(size, "causal", dtype, 3)
    Lq, Lk = size[3], size[4]
    row, key = Lq // 2, Lk // 3
    {"q": q, "dout": dout}.get(place, k if place == "k" else v)[0, 0, row if place in ("q", "dout") else key, 5] = math.nan
    out, lse = mg.attention(q, k, v, cap=cap)
    pos = torch.arange(Lq, device="cuda") + Lk - Lq
    hit = (torch.arange(Lq, device="cuda") == row) if place in ("q", "dout") else pos >= key      # rows it reaches
    if place != "dout":
        assert torch.isnan(out[0, 0, hit]).any(-1).all(), "out"
        assert bool(torch.isnan(lse[0, 0, hit]).all()) == (place != "v"), "lse"
    dq, dk, dv = mg.attention_backward(dout, q, k, v, out, lse, cap=cap)
    assert torch.isnan(dq[0, 0, hit]).any(-1).all(), "dq"
    seen = torch.arange(Lk, device="cuda") <= pos[hit].max()
    assert torch.isnan(dk[0, 0, seen]).any(-1).all(), "dk"
    if place != "v":
        assert torch.isnan(dv[0, 0, seen]).any(-1).all(), "dv"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 33])
@pytest.mark.parametrize("power", [20, 26, 40, 100])
def test_large_scores(power, D, dtype):
    """Scores of 2^power: the largest takes its row; rows of equal scores take the mean. Beyond 2^28 rows may be NaN."""
    L, best = 300, 170
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.zeros((1, 1, L, D), device="cuda", dtype=dtype) for _ in range(2))
    v = torch.randn((1, 1, L, D), generator=g, device="cuda").to(dtype)
    q[..., 0] = 2.0 ** (power // 2)
    k[..., 0] = 2.0 ** (power // 2 - 1)
    k[:, :, best, 0] *= 2
    out, lse = mg.attention(q, k, v, scale=1.0)
    want = v.double().cumsum(2) / torch.arange(1, L + 1, device="cuda")[:, None]
    want[:, :, best:] = v[:, :, best].double()
    # a sum of up to L products whose weights are rounded, then a rounding
    u = torch.finfo(dtype).eps / 2
    tol = (2 * u + 8 * 2.0 ** -24 * L ** 0.5) * v.double().abs().cummax(2).values
    tol[:, :, best:] = tol.max()
    nan = torch.isnan(out)
    assert power > 28 or not nan.any()
    assert ((out.double() - want).abs() <= tol)[~nan].all()
    mg.attention(q, k, v, scale=1.0, slopes=torch.tensor([3.0e12], device="cuda"))     # ends
    mg.attention(q, k, v, scale=1.0, causal=False, slopes=torch.tensor([1.0e30], device="cuda"))
    torch.cuda.synchronize()
    assert mg.load().mg_device_status(None, 0) == 0


def test_out_in_the_place_of_keys_or_values_is_refused():
    q, k, v = (torch.randn((1, 2, 8, 64), device="cuda") for _ in range(3))
    for t in (k, v):
        with pytest.raises(mg.MacrogradError, match="same memory"):
            mg.attention(q, k, v, out=t)


SHARED = [  # B, H, Hkv, Lq, Lk, D: few rows of blocks, so that several share a gradient's sum
    (1, 8, 2, 700, 700, 128),
    (1, 2, 1, 1100, 1300, 64),
    (2, 6, 1, 3, 900, 96),
    (1, 1, 1, 2000, 130, 72),
    (1, 16, 1, 150, 150, 64),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("size", SHARED, ids=str)
def test_gradients_of_shared_sums(size, mask, dtype):
    compare(*make(size, mask, dtype, 21))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_gradients_of_shared_sums_repeat(dtype):
    """The same bits every time, and in two captured graphs replayed on two streams."""
    q, k, v, dout, kw = make((1, 8, 2, 700, 700, 64), "documents", dtype, 22)
    out, lse = mg.attention(q, k, v, **kw)
    first = mg.attention_backward(dout, q, k, v, out, lse, **kw)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = mg.attention_backward(dout, q, k, v, out, lse, **kw)
        graphs.append((g, got, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, got, _ in graphs:
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_host_threads_with_heads_of_other_sizes():
    """Two host threads launch the CUDA-core kernels at once, with heads that take different amounts of shared memory:
    through the C ABI, whose calls follow one another closely enough to meet in the launch."""
    lib = mg.load()
    calls = []
    for D in (33, 127):
        q, k, v, _, _ = make((1, 1, 1, 2, 2, D), "causal", torch.float32, 50, strided=False)
        want = mg.attention(q, k, v)
        out, lse = torch.empty_like(q), torch.empty_like(want[1])
        desc = transformer._ATTENTION.pack(0, 1, 1, 1, 2, 2, D, 1, 1 / math.sqrt(D), 0.0, *([2 * D, 2 * D, D] * 4),
                                           *([0] * 12), 0, 0, 0)
        calls.append((desc, q, k, v, out, lse, want, torch.cuda.Stream().cuda_stream))
    torch.cuda.synchronize()

    def repeat(desc, q, k, v, out, lse, want, stream):
        bad = 0
        for _ in range(20000):
            bad += lib.mg_attention(desc, out.data_ptr(), lse.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                    ctypes.c_void_p(stream)) != _lib.MG_OK
        return bad

    with ThreadPoolExecutor(2) as pool:
        refused = sum(f.result() for f in [pool.submit(repeat, *c) for c in calls])
    torch.cuda.synchronize()
    assert refused == 0, f"{refused} of 40000 launches were refused"
    for _, _, _, _, out, lse, want, _ in calls:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


COMMON = [  # B, H, Hkv, Lq, Lk, D, rows off 16 bytes
    (1, 4, 2, 300, 300, 64, False),
    (1, 8, 2, 700, 700, 128, False),         # several blocks share a sum
    (2, 16, 16, 700, 700, 64, False),        # none does
    (1, 2, 1, 3, 900, 96, False),
    (1, 2, 1, 1, 200, 64, False),
    (1, 2, 1, 150, 150, 33, False),
    (2, 4, 2, 130, 200, 64, True),
]


@pytest.mark.parametrize("size", COMMON, ids=str)
@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("short", [False, True], ids=["one document", "documents of 7"])
def test_16_bit_gradients_of_values_with_much_in_common(short, cap, size):
    """Values that differ in their last bit: dP - delta is as small as the rounding of `out` that delta is computed
    from, so a gradient that does not make up for it is wrong by about its own size (taken twice or with the wrong sign,
    by two or three times that).

    Bound, of the norm: half a step (u) each for dS, for the weights of what is made up for (of the size of the
    gradient itself), for the result, and for everything in fp32 (2^-24 * D * 8 of a sum that 2^-7 of is left: less
    than u / 4)."""
    *size, off = size
    B, H, Hkv, Lq, Lk, D = size
    g = torch.Generator(device="cuda").manual_seed(3)

    def heads(n, L, bits=False):
        x = torch.randn((B, n, L, D + off), generator=g, device="cuda")
        return (1 + 2.0 ** -7 * (x > 0) if bits else x).bfloat16()[..., off:]

    q, k, v, dout = heads(H, Lq), heads(Hkv, Lk), heads(Hkv, Lk, True), heads(H, Lq)
    kw = dict(cap=cap)
    if short:
        kw["documents"] = (torch.arange(Lk, device="cuda") // 7).int().expand(B, Lk).contiguous()
    out, lse = mg.attention(q, k, v, **kw)
    ref = Reference(q, k, v, dout, **kw)
    dq, dk, dv = mg.attention_backward(dout, q, k, v, out, lse, **kw)
    for got, want, what in ((dq, ref.dq, "dq"), (dk, ref.dk, "dk"), (dv, ref.dv, "dv")):
        error = float((got.double() - want).norm() / want.norm())
        assert error <= 4 * half_step(torch.bfloat16), f"{what}: {error:.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("top", [2 ** 16, 2 ** 18 + 3, 2 ** 20 + 3, 2 ** 20 + 11])
def test_parts_of_a_row_with_large_scores(top, dtype):
    """One head whose row is shared by several blocks: one half of the keys scores `top`, the other a quarter less, both
    exactly. The halves' weights go by that quarter, whatever the rounding of sums as large as `top`.

    Bound: worst rounding of a part's sum of 4096 equal weights by 64 and tile (128 additions), once above and once
    below the line, two exponentials of 2 ulp each and the logarithm's base in fp32: 300 * 2^-24; 16-bit weights and
    results half a step each."""
    Lq, Lk, D = 130, 8192, 16
    q, k, v = (torch.zeros((1, 1, L, D), device="cuda", dtype=dtype) for L in (Lq, Lk, Lk))
    hi = float(torch.tensor(float(top)).bfloat16())
    q[..., :3] = 1
    k[..., 0], k[..., 1] = hi, top - hi
    k[:, :, Lk // 2:, 2] = -0.25
    v[:, :, :Lk // 2, 0], v[:, :, Lk // 2:, 1] = 1, 1
    out, lse = mg.attention(q, k, v, scale=1.0, causal=False)
    first = 1 / (1 + math.exp(-0.25))
    tol = 300 * 2.0 ** -24 + (2 * half_step(dtype) if dtype == torch.bfloat16 else 0.0)
    for d, want in ((0, first), (1, 1 - first)):
        assert ((out[..., d].double() - want).abs() <= tol * want).all(), float((out[..., d].double() - want).abs().max() / want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("heads", [160, 1], ids=["one block", "parts"])
@pytest.mark.parametrize("top", [2 ** 16, 2 ** 18 + 3, 2 ** 20 + 3, 2 ** 20 + 11])
def test_a_large_maximum_that_comes_late(top, heads, dtype):
    """All keys but four near the end score `top` - 8, those `top`, both exactly: what was summed before the maximum
    moved, and what comes after it, goes by that 8.

    Bound: worst rounding of sums over 4096 keys, 64 additions in a tile and as many tiles, above and below the line,
    and the exponentials' 2 ulp: 300 * 2^-24; e^-8 itself is taken from 8 log2(e) in fp32, off by 12 * 2^-24 and as much
    for log2(e); 16-bit weights and results half a step each."""
    Lq, Lk, D = 128, 4096, 16
    q = torch.zeros((1, heads, Lq, D), device="cuda", dtype=dtype)
    k, v = (torch.zeros((1, 1, Lk, D), device="cuda", dtype=dtype) for _ in range(2))
    hi = float(torch.tensor(float(top)).bfloat16())
    q[..., :3] = 1
    k[..., 0], k[..., 1] = hi, top - hi
    high = slice(Lk - 300, Lk - 296)
    k[..., 2], v[..., 1] = -8, 1
    k[:, :, high, 2], v[:, :, high, 1], v[:, :, high, 0] = 0, 0, 1
    out, lse = mg.attention(q, k, v, scale=1.0, causal=False)
    late = 4 / (4 + (Lk - 4) * math.exp(-8))
    tol = 324 * 2.0 ** -24 + (2 * half_step(dtype) if dtype == torch.bfloat16 else 0.0)
    for d, want in ((0, late), (1, 1 - late)):
        error = float((out[..., d].double() - want).abs().max() / want)
        assert error <= tol, error


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(1, 3, 3, 150, 150, 64), (1, 2, 2, 140, 1500, 128), (2, 2, 2, 70, 70, 33),
                                  (1, 4, 4, 1, 600, 64)], ids=str)
def test_out_in_the_place_of_q(size, dtype):
    """Inside a packed projection too, whose keys and values lie between its queries."""
    B, H, _, Lq, Lk, D = size
    q, k, v, _, kw = make(size, "causal", dtype, 60)
    want = mg.attention(q, k, v, **kw)
    got = mg.attention(q, k, v, out=q, **kw)
    assert got[0] is q and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if Lq != Lk:
        return
    qkv = torch.randn((B, Lq, 3, H, D), device="cuda").to(dtype)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    kept = qkv.clone()
    want = mg.attention(q, k, v, **kw)
    got = mg.attention(q, k, v, out=q, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(qkv[:, :, 1:], kept[:, :, 1:])


def test_out_that_overlaps_an_input_is_refused():
    """Where the views start elsewhere, or are laid out in another way."""
    qkv = torch.randn((2, 8, 3, 4, 64), device="cuda")
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    flat = qkv.flatten(2)
    for out, name in [(flat[:, :, 320:576].unflatten(2, (4, 64)).transpose(1, 2), "k"),
                      (flat[:, :, 500:756].unflatten(2, (4, 64)).transpose(1, 2), "k"),
                      (flat[:, :, 512 + 64:].unflatten(2, (3, 64)).transpose(1, 2), "v"),
                      (flat[:, :, 64:256].unflatten(2, (3, 64)).transpose(1, 2), "q"),
                      (qkv.flatten()[:2 * 4 * 8 * 64].view(2, 4, 8, 64), "q")]:
        n = out.shape[1]
        with pytest.raises(mg.MacrogradError, match=f"out overlaps {name}"):
            mg.attention(q[:, :n], k[:, :n], v[:, :n], out=out)


@pytest.mark.parametrize("op", ["attention", "attention_backward", "rotary", "rotary_backward", "paged_attention"])
def test_operands_let_go_after_a_call_on_another_stream(op):
    """Their memory is not given away while the other stream may still be reading it."""
    dev, dt = "cuda", torch.bfloat16
    heads = lambda n: torch.randn((1, n, 96, 64), device=dev, dtype=dt)  # noqa: E731
    if op.startswith("attention"):
        used = dict(q=heads(4), k=heads(2), v=heads(2), slopes=torch.rand(4, device=dev),
                    documents=torch.zeros((1, 96), dtype=torch.int32, device=dev))
        if op == "attention_backward":
            out, lse = mg.attention(**used)
            used.update(out=out, lse=lse, dout=heads(4))
            del out, lse
        else:
            used["out"] = heads(4)
    elif op.startswith("rotary"):
        names = ("dq", "dk") if op == "rotary_backward" else ("q", "k")
        used = {names[0]: heads(4), names[1]: heads(2), "positions": torch.arange(96, device=dev).int(),
                "frequencies": mg.rotary_frequencies(64)}
    else:
        used = dict(q=heads(4)[:, :, 0], k_pages=torch.randn((6, 16, 2, 64), device=dev, dtype=dt),
                    v_pages=torch.randn((6, 16, 2, 64), device=dev, dtype=dt),
                    block_table=torch.arange(6, device=dev).int()[None].contiguous(),
                    lengths=torch.tensor([90], device=dev).int(), k_new=heads(2)[:, :, 0], v_new=heads(2)[:, :, 0])
    getattr(mg, op)(**used)                  # loads what the call needs, which may wait for the device
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(400_000_000)       # about a fifth of a second
    results = getattr(mg, op)(stream=stream, **used)
    held = {n: (t.untyped_storage().data_ptr(), t.untyped_storage().nbytes()) for n, t in used.items()}
    used.clear()
    fresh = [torch.empty(size, dtype=torch.uint8, device=dev) for _, size in held.values() for _ in range(3)]
    assert not stream.query(), "the stream was done too early for the test to tell"
    places = {t.untyped_storage().data_ptr() for t in fresh}
    assert not [n for n, (at, _) in held.items() if at in places]
    torch.cuda.synchronize()
    assert all(torch.isfinite(t).all() for t in results)


def test_captured_on_another_stream_than_the_graphs():
    """A call on a stream that is forked from the captured one and joined to it, with operands of the graph's own."""
    q, k, v, dout, kw = make((1, 4, 2, 200, 200, 64), "all", torch.bfloat16, 61)
    want = mg.attention(q, k, v, **kw)
    want = want + mg.attention_backward(dout, q, k, v, *want, **kw)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        own = q.clone()
        side.wait_stream(torch.cuda.current_stream())
        got = mg.attention(own, k, v, stream=side, **kw)
        got = got + mg.attention_backward(dout, own, k, v, *got, stream=side, **kw)
        del own
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("size", [(64, 6, 6, 130, 200, 64), (1, 4, 2, 700, 700, 64), (1, 8, 2, 300, 300, 128),
                                  (40, 8, 8, 130, 130, 96), (2, 4, 2, 150, 150, 33), (1, 4, 1, 1, 500, 64)], ids=str)
@pytest.mark.parametrize("top", [2 ** 12 + 3, 2 ** 14 + 7])
def test_fp32_gradients_of_large_scores(top, size):
    """Scores of `top` less 0 to 3, exactly: the weights go by the small part, whatever the rounding of lse, which is some
    2^-24 * top. Of dq and dk the elements that k and q do not hold `top` or its share in, whose own products cancel.

    Bound, of the norm, in steps of 2^-24: exponents of up to 16 powers of two, rounded once (16), exponentials of 2 ulp
    (4), products of 3 pieces (2) and their sums over up to 128 elements and 64 keys truncated at the worst (128), lse's
    part that is taken off (4): below 2^8."""
    B, H, Hkv, Lq, Lk, D = size
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v, dout = (torch.randn((B, n, L, D), generator=g, device="cuda") for n, L in ((H, Lq), (Hkv, Lk), (Hkv, Lk), (H, Lq)))
    q[..., :3] = 1
    k[..., 0], k[..., 1], k[..., 3:] = 2 ** 12, top - 2 ** 12, 0
    k[..., 2] = -torch.randint(0, 25, (B, Hkv, Lk), generator=g, device="cuda") / 8
    out, lse = mg.attention(q, k, v, scale=1.0)
    ref = Reference(q, k, v, dout, scale=1.0)
    dq, dk, dv = mg.attention_backward(dout, q, k, v, out, lse, scale=1.0)
    for got, want, what in ((dq[..., 2:3], ref.dq[..., 2:3], "dq"), (dk, ref.dk, "dk"), (dv, ref.dv, "dv")):
        error = float((got.double() - want).norm() / want.norm())
        assert error <= 2.0 ** -16, f"{what}: {error:.3g}"
