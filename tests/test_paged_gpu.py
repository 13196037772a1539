"""paged_attention against the definition in 64 bits: types, shared heads, page
sizes, ragged lengths with 0 and 1, appended tokens, both pool layouts, bad
pages and lengths; and the chain rotary -> paged cache -> attention as a decoder
uses it, token by token, against one attention over the whole row."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")
import macrograd_b200 as mg  # noqa: E402
from macrograd_b200 import _lib  # noqa: E402
from attention_reference import Reference, half_step, within  # noqa: E402

pytestmark = pytest.mark.gpu


def make(B, H, Hkv, D, page, lengths, dtype, seed=0, append=True, gain=1.0, head_major=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(1, -(-max(lengths) // page)) + 1
    pages = B * width + 2
    shape = (pages, Hkv, page, D) if head_major else (pages, page, Hkv, D)
    kp, vp = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    if head_major:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    table = torch.randperm(pages, generator=g, device="cuda")[:B * width].int().view(B, width)
    q = (torch.randn((B, H, D), generator=g, device="cuda") * gain).to(dtype)
    kn, vn = (torch.randn((B, Hkv, D), generator=g, device="cuda").to(dtype) if append else None for _ in range(2))
    return q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), kn, vn


def compare(args, cap=0.0, slopes=None):
    q, kp, vp, table, lengths, kn, vn = args
    page = kp.shape[1]
    wk, wv = kp.clone(), vp.clone()
    out, lse = mg.paged_attention(q, kp, vp, table, lengths, cap=cap, slopes=slopes, k_new=kn, v_new=vn)
    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            assert (out[b] == 0).all() and torch.isneginf(lse[b]).all()
            continue
        if kn is not None:
            at = int(table[b, (n - 1) // page]), (n - 1) % page
            wk[at], wv[at] = kn[b], vn[b]
        rows = table[b, :-(-n // page)].long()
        k, v = (x[rows].flatten(0, 1)[:n].transpose(0, 1)[None] for x in (wk, wv))
        ref = Reference(q[b][None, :, None], k, v, cap=cap, slopes=slopes)
        within(out[b], ref.out[0, :, 0], ref.out_tol[0, :, 0], f"out[{b}]")
        within(lse[b], ref.lse[0, :, 0], ref.lse_tol[0, :, 0], f"lse[{b}]")
    assert torch.equal(kp, wk) and torch.equal(vp, wv), "the cache beside the new tokens changed"
    return out, lse


def status(reset=True):
    detail = ctypes.c_int32(0)
    return mg.load().mg_device_status(ctypes.byref(detail), int(reset)), detail.value


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,D,page,lengths", [
    (1, 1, 1, 8, 1, [1]),
    (3, 4, 2, 64, 16, [0, 1, 17]),
    (2, 8, 1, 128, 16, [130, 1000]),
    (4, 6, 6, 64, 24, [5, 333, 24, 25]),
    (2, 32, 8, 128, 64, [2049, 64]),
    (1, 12, 4, 96, 7, [777]),
    (2, 20, 1, 80, 256, [300, 3000]),
    (1, 3, 1, 33, 16, [100]),
    (1, 2, 2, 128, 16, [20011])])
@pytest.mark.parametrize("append", [True, False], ids=["append", "read"])
def test_paged(B, H, Hkv, D, page, lengths, append, dtype):
    compare(make(B, H, Hkv, D, page, lengths, dtype, append=append))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_cap_and_slopes(dtype):
    slopes = torch.tensor([2.0 ** (-1 - h) for h in range(8)], device="cuda")
    compare(make(3, 8, 2, 128, 16, [40, 500, 1234], dtype, gain=4.0), cap=5.0)
    compare(make(3, 8, 2, 64, 16, [40, 500, 1234], dtype), slopes=slopes)
    compare(make(3, 8, 4, 128, 16, [40, 500, 1234], dtype, gain=4.0), cap=20.0, slopes=slopes)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_pool_by_heads_and_views(dtype):
    compare(make(2, 4, 2, 64, 16, [100, 33], dtype, head_major=True))
    q, kp, vp, table, lengths, kn, vn = make(2, 4, 2, 64, 16, [100, 33], dtype)
    room = torch.randn((*kp.shape[:3], 2, 64), device="cuda").to(dtype)    # k and v side by side
    room[..., 0, :], room[..., 1, :] = kp, vp
    compare((q, room[..., 0, :], room[..., 1, :], table, lengths, kn, vn))
    wide = torch.randn((*kp.shape[:3], 65), device="cuda").to(dtype)       # rows off 16 bytes
    compare((q, wide[..., 1:], vp, table, lengths, kn, vn))


def test_tokens_beyond_the_length_are_not_read():
    """NaN behind each request's last key, in its last page and in pages of the table beyond it."""
    for dtype in (torch.float32, torch.bfloat16):
        q, kp, vp, table, lengths, kn, vn = make(2, 4, 2, 64, 16, [100, 33], dtype, append=False)
        for b, n in enumerate(lengths.tolist()):
            for j in range(n, table.shape[1] * 16):
                at = int(table[b, j // 16]), j % 16
                kp[at] = vp[at] = float("nan")
        out, lse = mg.paged_attention(q, kp, vp, table, lengths)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        kp[torch.isnan(kp)], vp[torch.isnan(vp)] = 0, 0
        compare((q, kp, vp, table, lengths, None, None))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_bad_pages_and_lengths_are_reported_not_read(dtype):
    q, kp, vp, table, lengths, kn, vn = make(2, 4, 2, 64, 16, [100, 33], dtype)
    assert status()[0] == _lib.MG_OK
    bad = table.clone()
    bad[0, 1], bad[1, 2] = kp.shape[0], -1       # the second is where request 1 appends
    kept = kp.clone(), vp.clone()
    out, lse = mg.paged_attention(q, kp, vp, bad, lengths, k_new=kn, v_new=vn)
    assert status()[0] == _lib.MG_ERR_INVALID
    assert torch.isfinite(out).all()
    rows = table[0, :7].long()
    seen = torch.ones(112, dtype=torch.bool, device="cuda")
    seen[16:32] = seen[100:] = False
    k, v = (x[rows].flatten(0, 1)[seen].transpose(0, 1)[None] for x in (kp, vp))
    ref = Reference(q[0][None, :, None], k, v)
    within(out[0], ref.out[0, :, 0], ref.out_tol[0, :, 0], "out without the bad page")
    changed = (kp != kept[0]).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(table[0, 6])]
    long = lengths.clone()
    long[1] = 10 ** 6
    cut = torch.tensor([100, table.shape[1] * 16], dtype=torch.int32, device="cuda")
    a = mg.paged_attention(q, kp, vp, table, long)
    assert status()[0] == _lib.MG_ERR_INVALID
    b = mg.paged_attention(q, kp, vp, table, cut)
    assert status()[0] == _lib.MG_OK
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    long[1] = -5
    assert (mg.paged_attention(q, kp, vp, table, long)[0][1] == 0).all()
    assert status()[0] == _lib.MG_ERR_INVALID


def test_same_page_twice_and_shared_pages():
    """Requests that share the pages of a common beginning, and a table that names a page twice."""
    q, kp, vp, table, lengths, kn, vn = make(3, 4, 2, 64, 16, [90, 70, 60], torch.bfloat16)
    table[1, :3] = table[0, :3]
    table[2, 1] = table[2, 0]
    compare((q, kp, vp, table, lengths, kn, vn))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_captured_and_replayed_while_requests_grow(dtype):
    args = make(3, 8, 2, 64, 16, [700, 1, 30], dtype)
    q, kp, vp, table, lengths, kn, vn = args
    mg.paged_attention(q, kp, vp, table, lengths, k_new=kn, v_new=vn)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = mg.paged_attention(q, kp, vp, table, lengths, k_new=kn, v_new=vn)
    for step in range(3):
        lengths.add_(1)
        kn.normal_()
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = compare(args)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_same_inputs_same_bits():
    args = make(4, 8, 2, 128, 16, [3000, 7, 129, 4097], torch.bfloat16)
    q, kp, vp, table, lengths, kn, vn = args
    first = mg.paged_attention(q, kp, vp, table, lengths, k_new=kn, v_new=vn)
    for _ in range(3):
        again = mg.paged_attention(q, kp, vp, table, lengths, k_new=kn, v_new=vn)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("lengths", [[900], [1, 128, 129, 1000], [2000] * 40])
def test_chunks_joined_in_a_cluster_and_by_a_kernel(lengths):
    """Few short requests join their chunks in one cluster, many or long ones in a second launch, with a table much wider
    than the requests too."""
    for Hkv in (1, 8):
        args = make(len(lengths), 8, Hkv, 64, 16, lengths, torch.bfloat16, seed=3)
        compare(args)
        wide = torch.cat([args[3], torch.zeros((len(lengths), 500), dtype=torch.int32, device="cuda")], 1)
        compare((*args[:3], wide, *args[4:]))


def test_offsets_beyond_32_bits():
    """Pages more than 2^31 elements into the pool."""
    page, Hkv, D = 256, 1, 128
    pages = (1 << 31) // (page * D) + 8
    kp = torch.empty((pages, page, Hkv, D), dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in table[0].tolist():
        kp[t] = torch.randn((page, Hkv, D), generator=g, device="cuda")
        vp[t] = torch.randn((page, Hkv, D), generator=g, device="cuda")
    q = torch.randn((1, 2, D), generator=g, device="cuda").bfloat16()
    n = 700
    out, lse = mg.paged_attention(q, kp, vp, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    k, v = (x[table[0].long()].flatten(0, 1)[:n].transpose(0, 1)[None] for x in (kp, vp))
    ref = Reference(q[:, :, None], k, v)
    within(out, ref.out[:, :, 0], ref.out_tol[:, :, 0], "out")
    within(lse, ref.lse[:, :, 0], ref.lse_tol[:, :, 0], "lse")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_decoding_token_by_token_is_attention_over_the_row(dtype):
    """A prompt through rotary and attention, its keys put into pages, then tokens one by one through rotary and
    paged_attention: each gives the row that attention over the whole text gives."""
    B, H, Hkv, D, page, prompt, total = 2, 4, 2, 64, 8, 37, 45
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = (torch.randn((B, total, n, D), generator=g, device="cuda").to(dtype).transpose(1, 2)
               for n in (H, Hkv, Hkv))
    f = mg.rotary_frequencies(D // 2, scaling="linear", factor=2.0)
    pos = torch.arange(total, device="cuda").int()
    rq, rk = mg.rotary(q, k, pos, f)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    whole, whole_lse = mg.attention(rq, rk, v, cap=30.0, slopes=slopes)
    ref = Reference(rq, rk, v, cap=30.0, slopes=slopes)
    within(whole, ref.out, ref.out_tol, "whole row")

    width = -(-total // page)
    kp, vp = (torch.zeros((B * width, page, Hkv, D), device="cuda", dtype=dtype) for _ in range(2))
    table = torch.randperm(B * width, generator=g, device="cuda").int().view(B, width)
    for b in range(B):
        for j in range(prompt):
            at = int(table[b, j // page]), j % page
            kp[at], vp[at] = rk[b, :, j], v[b, :, j]
    lengths = torch.full((B,), prompt, dtype=torch.int32, device="cuda")
    for t in range(prompt, total):
        lengths += 1
        tq, tk = mg.rotary(q[:, :, t:t + 1], k[:, :, t:t + 1], (lengths - 1).view(B, 1), f)
        assert torch.equal(tk, rk[:, :, t:t + 1])
        out, lse = mg.paged_attention(tq[:, :, 0], kp, vp, table, lengths, cap=30.0, slopes=slopes,
                                      k_new=tk[:, :, 0], v_new=v[:, :, t])
        within(out, ref.out[:, :, t], ref.out_tol[:, :, t], f"token {t}")
        within(lse, ref.lse[:, :, t], ref.lse_tol[:, :, t], f"lse of token {t}")


def test_refusals():
    q, kp, vp, table, lengths, kn, vn = make(2, 4, 2, 64, 16, [10, 20], torch.float32)
    for call, fragment in [
            (lambda: mg.paged_attention(q[:, :3], kp, vp, table, lengths), "multiple"),
            (lambda: mg.paged_attention(q, kp, vp[:, :8], table, lengths), "Found shapes"),
            (lambda: mg.paged_attention(q, kp.bfloat16(), vp, table, lengths), "as the others"),
            (lambda: mg.paged_attention(q, kp, vp, table.long(), lengths), "block_table"),
            (lambda: mg.paged_attention(q, kp, vp, table[:1], lengths), "block_table"),
            (lambda: mg.paged_attention(q, kp, vp, table, lengths[:1]), "lengths"),
            (lambda: mg.paged_attention(q, kp, vp, table, lengths, k_new=kn), "come together"),
            (lambda: mg.paged_attention(q, kp, vp, table, lengths, k_new=kn[:1], v_new=vn), "k_new"),
            (lambda: mg.paged_attention(q, kp, vp, table, lengths, cap=-2.0), "cap"),
            (lambda: mg.paged_attention(q, kp[:1].expand_as(kp), vp, table, lengths, k_new=kn, v_new=vn), "overlap"),
            (lambda: mg.paged_attention(q, kp, vp, table, lengths, slopes=torch.zeros(3, device="cuda")), "slopes")]:
        with pytest.raises(mg.MacrogradError, match=fragment):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 33])
@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("place", ["q", "k", "v", "new"])
def test_nan_that_is_seen_stays(place, cap, D, dtype):
    q, kp, vp, table, lengths, kn, vn = make(3, 4, 2, D, 16, [1, 40, 2500], dtype)
    for b, n in enumerate(lengths.tolist()):
        if place == "q":
            q[b, 0, 5] = float("nan")
        elif place == "new":
            kn[b, 0, 5] = float("nan")
        elif n > 1:
            (kp if place == "k" else vp)[int(table[b, n // 3 // 16]), n // 3 % 16, 0, 5] = float("nan")
    out, lse = mg.paged_attention(q, kp, vp, table, lengths, k_new=kn, v_new=vn, cap=cap)
    hit = lengths > (1 if place in ("k", "v") else 0)
    assert torch.isnan(out[hit, 0]).any(-1).all()
    assert bool(torch.isnan(lse[hit, 0]).all()) == (place != "v")
    assert torch.isfinite(out[:, 2:]).all()          # heads of the other key-value head


def test_appending_to_one_pool_of_keys_and_values_is_refused():
    q, kp, vp, table, lengths, kn, vn = make(2, 4, 2, 64, 16, [100, 33], torch.bfloat16)
    with pytest.raises(mg.MacrogradError, match="same memory"):
        mg.paged_attention(q, kp, kp, table, lengths, k_new=kn, v_new=vn)
    compare((q, kp, kp, table, lengths, None, None))      # read alone


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 33])
@pytest.mark.parametrize("rows", [16, 176, 6400], ids=["one block", "a cluster", "two launches"])
def test_a_token_beyond_the_table_is_not_appended(rows, D, dtype):
    """A request that has outgrown its table by one token: nothing of the cache changes, and the call attends to what the
    table holds; the requests beside it go on."""
    q, kp, vp, table, lengths, kn, vn = make(2, 4, 2, D, 16, [rows - 15, rows - 20 if rows > 20 else 3], dtype)
    table = table[:, :rows // 16].contiguous()
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    for past in (rows + 1, rows + 17, 2 ** 31 - 1):
        grown = lengths.clone()
        grown[0] = past
        kept = kp.clone(), vp.clone()
        out, lse = mg.paged_attention(q, kp, vp, table, grown, slopes=slopes, k_new=kn, v_new=vn)
        assert status()[0] == _lib.MG_ERR_INVALID
        at = int(table[1, (int(lengths[1]) - 1) // 16]), (int(lengths[1]) - 1) % 16
        kept[0][at], kept[1][at] = kn[1], vn[1]
        assert torch.equal(kp, kept[0]) and torch.equal(vp, kept[1])
        grown[0] = rows
        want = mg.paged_attention(q, kp, vp, table, grown, slopes=slopes)
        assert status()[0] == _lib.MG_OK
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("top", [2 ** 16, 2 ** 18 + 3, 2 ** 20 + 3, 2 ** 20 + 11])
@pytest.mark.parametrize("keys", [512, 16384], ids=["a cluster", "two launches"])
def test_chunks_with_large_scores(keys, top, dtype):
    """One half of the keys scores `top` powers of two, the other a quarter less, both exactly (the scale is ln 2, whose
    product with log2(e) is 1 in fp32): the halves' weights go by that quarter, whatever the rounding of numbers as
    large as `top`.

    Bound: the worst rounding of a chunk's sum of up to 256 equal weights (256 additions), once above and once below the
    line, and of the join (128), exponentials of 2 ulp: 700 * 2^-24; 16-bit weights and results half a step each."""
    D = 64
    scale = float(torch.tensor(math.log(2), dtype=torch.float32))
    q = torch.zeros((1, 2, D), device="cuda", dtype=dtype)
    kp, vp = (torch.zeros((keys // 16, 16, 1, D), device="cuda", dtype=dtype) for _ in range(2))
    hi = float(torch.tensor(float(top)).bfloat16())
    q[..., :3] = 1
    kp[..., 0], kp[..., 1] = hi, top - hi
    kp[keys // 32:, ..., 2] = -0.25
    vp[:keys // 32, ..., 0], vp[keys // 32:, ..., 1] = 1, 1
    table = torch.arange(keys // 16, device="cuda").int()[None].contiguous()
    out, lse = mg.paged_attention(q, kp, vp, table, torch.tensor([keys], dtype=torch.int32, device="cuda"), scale=scale)
    first = 1 / (1 + math.exp(-0.25 * scale))
    tol = 700 * 2.0 ** -24 + (2 * half_step(dtype) if dtype == torch.bfloat16 else 0.0)
    for d, want in ((0, first), (1, 1 - first)):
        error = float((out[..., d].double() - want).abs().max() / want)
        assert error <= tol, error
    assert abs(float(lse[0, 0]) - (top * scale + math.log(keys / 2 / first))) <= 2 * 2.0 ** -24 * top


def test_pools_and_outputs_that_overlap_are_refused():
    q, kp, vp, table, lengths, kn, vn = make(2, 4, 2, 64, 16, [100, 33], torch.bfloat16)
    room = torch.zeros((*kp.shape[:3], 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(mg.MacrogradError, match="k_pages overlaps v_pages"):
        mg.paged_attention(q, room[..., :64], room[..., 32:96], table, lengths, k_new=kn, v_new=vn)
    compare((q, room[..., :64], room[..., 32:96], table, lengths, None, None))          # read alone
    compare((q, room[..., :64], room[..., 64:], table, lengths, kn, vn))
    with pytest.raises(mg.MacrogradError, match="out overlaps v_pages"):
        mg.paged_attention(q, kp, vp, table, lengths, out=vp[3, 4:8, :, :].flatten()[:512].view(2, 4, 64))
    want = mg.paged_attention(q, kp, vp, table, lengths)
    got = mg.paged_attention(q, kp, vp, table, lengths, out=q)
    assert got[0] is q and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("top", [2 ** 16, 2 ** 18 + 3, 2 ** 20 + 3, 2 ** 20 + 11])
@pytest.mark.parametrize("keys", [64, 512, 16384], ids=["one block", "a cluster", "two launches"])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.75])
def test_scores_are_not_rounded_before_the_maximum_is_off_them(scale, keys, top, dtype):
    """As above with scales that leave no score a whole number of powers of two; the two kinds of keys alternate, and a
    single query over a contiguous row is the same call. Bound as above."""
    D = 64
    q = torch.zeros((1, 2, D), device="cuda", dtype=dtype)
    kp, vp = (torch.zeros((keys // 16, 16, 1, D), device="cuda", dtype=dtype) for _ in range(2))
    hi = float(torch.tensor(float(top)).bfloat16())
    q[..., :3] = 1 if scale > 0 else -1
    kp[..., 0], kp[..., 1] = hi, top - hi
    kp[:, 1::2, :, 2] = -0.25
    vp[:, 0::2, :, 0], vp[:, 1::2, :, 1] = 1, 1
    table = torch.arange(keys // 16, device="cuda").int()[None].contiguous()
    out, _ = mg.paged_attention(q, kp, vp, table, torch.tensor([keys], dtype=torch.int32, device="cuda"), scale=scale)
    first = 1 / (1 + math.exp(-0.25 * abs(scale)))
    tol = 700 * 2.0 ** -24 + (2 * half_step(dtype) if dtype == torch.bfloat16 else 0.0)
    k, v = (x.view(1, keys, 1, D).transpose(1, 2) for x in (kp, vp))
    row, _ = mg.attention(q[:, :, None], k, v, scale=scale)
    for got in (out, row[:, :, 0]):
        for d, want in ((0, first), (1, 1 - first)):
            error = float((got[..., d].double() - want).abs().max() / want)
            assert error <= tol, error
