"""Attention over whole rows, rotary positions and paged attention on torch CUDA
tensors, over the C ABI of include/mg_attention.h.

They take the place of the chain that a transformer's attention is made of --
Functional::matmul(Q / sqrt(d), K, mask, false, true), softmax(-1) and
Functional::matmul(P, V) (mini_shakespeare/include/transformer.h:226-244) --
where functional.attention_scores ends: rows of more than 256 keys, scores that
never reach memory, shared key-value heads, 16-bit types, caps, biases by
distance, documents and prefixes.

  attention(q, k, v, ...)                  out and the rows' log-sums
  attention_backward(dout, q, k, v, ...)   dq, dk, dv
  rotary(q, k, positions, frequencies)     positions by turning pairs
  rotary_backward(dq, dk, ...)             its gradient: the opposite turn
  rotary_frequencies(...)                  the pairs' frequencies, also for long contexts
  paged_attention(q, k_pages, ...)         one new token per request over a paged cache

Heads are views [batch, heads, length, head_dim] with a contiguous last dim and
any other strides, float32 or bfloat16, head_dim up to 128; outputs are laid out
as the tensor they belong to (heads split from [batch, length, heads * head_dim]
come back ready to be merged). Sums, softmax statistics and angles are kept in
32 bits or more whatever the type; with bfloat16 tensors the weights P and, in the
gradients, dS are rounded to 16 bits for their products, as the tensors are. Calls run on `stream` (default: the current
one) and can be captured into graphs (but for the library's first call on a
device); nothing is kept from one call for the next. A `stream` that is given has
to be ordered behind whatever writes the operands, as by stream.wait_stream(), and
what comes back belongs to it; the operands may be let go right after the call.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import MacrogradError, check

MG_F32 = 0
MG_BF16 = 1
MAX_HEAD_DIM = 128

_DTYPES = {torch.float32: MG_F32, torch.bfloat16: MG_BF16}
# The descriptors of include/mg_attention.h (native alignment).
_ATTENTION = struct.Struct("@8i2f24q3P")
_ROTARY = struct.Struct("@9if13q2P")
_PAGED = struct.Struct("@8i2f15q3P")
_ZERO3 = (0, 0, 0)
_LARGEST = (2 - 2.0 ** -23) * 2.0 ** 127      # of fp32


# ------------------------------------------------------------------ checks
def _bad(message: str):
    raise MacrogradError(_lib.MG_ERR_INVALID, message)


def _heads(t: torch.Tensor, name: str, dims: int, dtype: Optional[torch.dtype], device) -> None:
    """A float32 or bfloat16 CUDA tensor of `dims` dims with a contiguous last one."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _bad(f"{name} must be a CUDA tensor")
    if t.dim() != dims:
        _bad(f"{name} must have {dims} dims, found shape {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        _bad(f"{name} must be float32 or bfloat16, found {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        _bad(f"{name} must be {dtype} as the others, found {t.dtype}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        _bad(f"{name} must be contiguous in its last dim (strides {t.stride()})")
    if device is not None and t.device != device:
        _bad(f"operands are on different devices: {device}, {t.device}")


def _plain(t: torch.Tensor, name: str, shape, dtype: torch.dtype, device) -> None:
    """A contiguous CUDA tensor of exactly this shape and type."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        _bad(f"{name} must be a tensor on {device}")
    if t.dtype != dtype or t.shape != shape:
        _bad(f"{name} must be {dtype} of shape {tuple(shape)}, found {t.dtype} of shape {tuple(t.shape)}")
    if not t.is_contiguous():
        _bad(f"{name} must be contiguous")


def _written(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    """An output the caller gives: shape and type of `like`, no two elements in one place."""
    _heads(t, name, like.dim(), like.dtype, like.device)
    if t.shape != like.shape:
        _bad(f"{name} must have shape {tuple(like.shape)}, found {tuple(t.shape)}")
    if t.is_contiguous():
        return
    spans = sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1)
    end = 1
    for st, n in spans:
        if st < end:
            _bad(f"{name}'s elements overlap (shape {tuple(t.shape)}, strides {t.stride()})")
        end = st * (n - 1) + end


def _number(x: float, name: str) -> float:
    """A finite number that stays one in the descriptors' fp32."""
    x = float(x)
    if not abs(x) <= _LARGEST:
        _bad(f"{name} must be finite in fp32, found {x}")
    return x


# The raw handle of the current stream, and the current device, without the
# objects around them: a call's host time counts where one token is decoded.
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_device = torch.cuda.current_device


def _on(device: torch.device, stream: Optional[torch.cuda.Stream], call, *used: Optional[torch.Tensor]):
    """call(stream handle) on `stream` (its device current, its allocations the stream's own), by default on the
    current stream of the operands' device. The memory of the tensors `used` is not given to others before a `stream`
    that is given is done with them."""
    if stream is None:
        if _device() == device.index:
            return call(_raw_stream(device.index))
        with torch.cuda.device(device):
            return call(_raw_stream(device.index))
    if torch.device(stream.device) != device:
        _bad(f"operands (and stream) are on different devices: {device}, {stream.device}")
    with torch.cuda.stream(stream):
        results = call(stream.cuda_stream)
    for t in used:
        if t is not None:
            t.record_stream(stream)
    return results


def _cap(cap: float) -> float:
    cap = _number(cap, "cap")
    if cap != 0 and not 1e-30 <= cap <= 1e30:
        _bad("cap must be 0 (none) or within 1e-30..1e30")
    return cap


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# ------------------------------------------------------------------ attention
def _attention_args(q, k, v, scale, causal, cap, slopes, documents, prefix):
    """Checks what both directions share; (dtype, the descriptor's leading values, its pointers)."""
    _heads(q, "q", 4, None, None)
    dt, dev = q.dtype, q.device
    _heads(k, "k", 4, dt, dev)
    _heads(v, "v", 4, dt, dev)
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D or v.shape != k.shape:
        _bad("q, k and v must be [batch, heads, q_len, head_dim] and twice [batch, kv_heads, k_len, head_dim]\n"
             f"Found shapes | q: {tuple(q.shape)} | k: {tuple(k.shape)} | v: {tuple(v.shape)}")
    if Hkv == 0 or H % Hkv:
        _bad(f"the {H} query heads must be a multiple of the {Hkv} key-value heads")
    if not 1 <= D <= MAX_HEAD_DIM:
        raise MacrogradError(_lib.MG_ERR_UNSUPPORTED, f"head_dim {D} is outside 1..{MAX_HEAD_DIM}")
    scale = 1.0 / math.sqrt(D) if scale is None else _number(scale, "scale")
    cap = _cap(cap)
    if slopes is not None:
        _plain(slopes, "slopes", (H,), torch.float32, dev)
    if documents is not None:
        _plain(documents, "documents", (B, Lk), torch.int32, dev)
    if prefix is not None:
        if not causal:
            _bad("a prefix needs causal=True: without it every key is seen already")
        _plain(prefix, "prefix", (B,), torch.int32, dev)
    lead = (_DTYPES[dt], B, H, Hkv, Lq, Lk, D, 1 if causal else 0, scale, cap)
    return dev, lead, (_at(slopes), _at(documents), _at(prefix))


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
              cap: float = 0.0, slopes: Optional[torch.Tensor] = None, documents: Optional[torch.Tensor] = None,
              prefix: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
              stream: Optional[torch.cuda.Stream] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """out = softmax(s) v and lse = log sum exp(s) of each row, without writing s.

    q [B, H, Lq, D], k and v [B, Hkv, Lk, D]; H a multiple of Hkv (query head h reads key-value head h // (H // Hkv)).
    Query i stands at position i + Lk - Lq, key j at position j.
      s = scale * q k^T                      scale: 1 / sqrt(D) by default
      cap > 0:     s = cap * tanh(s / cap)
      slopes [H]:  s -= slopes[h] * |position of the query - position of the key|
    A query sees the keys up to its own position (causal) and, besides, the first prefix[b] keys of its row (int32
    [B]); with documents (int32 [B, Lk], the id of each position) only keys of its own document. Ids below 0 mark
    padding: such keys and queries are left out whatever they hold. A query that sees no key gives out = 0,
    lse = -inf. Everywhere else k, v must be finite also where a mask hides them from some queries. Scores and
    biases are resolved up to 2^28 in size; a row with larger ones may come out as NaN. `out` may be q itself, but must not
    share memory with q in another way, nor with k or v.

    Returns (out, laid out as q, lse [B, H, Lq] in float32)."""
    lib = _lib.load()
    dev, lead, ptrs = _attention_args(q, k, v, scale, causal, cap, slopes, documents, prefix)
    if out is not None:
        _written(out, "out", q)
        for t, name in ((k, "k"), (v, "v")):           # other overlaps are the library's to refuse
            if out.numel() and t.numel() and out.data_ptr() == t.data_ptr():
                _bad(f"out and {name} are the same memory")

    def call(st):
        o = torch.empty_like(q) if out is None else out
        H, Lq = lead[2], lead[4]
        lse = torch.empty_strided(q.shape[:3], (H * Lq, Lq, 1), dtype=torch.float32, device=dev)
        desc = _ATTENTION.pack(*lead, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *o.stride()[:3], *_ZERO3,
                               *_ZERO3, *_ZERO3, *_ZERO3, *ptrs)
        check(lib.mg_attention(desc, o.data_ptr(), lse.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), st))
        return o, lse

    return _on(dev, stream, call, q, k, v, slopes, documents, prefix, out)


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, scale: Optional[float] = None, causal: bool = True, cap: float = 0.0,
                       slopes: Optional[torch.Tensor] = None, documents: Optional[torch.Tensor] = None,
                       prefix: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of sum(dout * out) for attention() called with the same arguments; `out` and `lse`
    are what it returned. Gradients of shared key-value heads are summed over their query heads, in a fixed order:
    the same inputs give the same bits. The slopes are constants (no gradient). Besides k and v, q and dout must be
    finite everywhere but at padding. The weights are exp(s - lse), made to sum to one in each row (but for bfloat16 on
    the tensor cores, where lse's rounding, 2^-24 of its size, is below that of the weights)."""
    lib = _lib.load()
    dev, lead, ptrs = _attention_args(q, k, v, scale, causal, cap, slopes, documents, prefix)
    for t, name in ((dout, "dout"), (out, "out")):
        _heads(t, name, 4, q.dtype, dev)
        if t.shape != q.shape:
            _bad(f"{name} must have q's shape {tuple(q.shape)}, found {tuple(t.shape)}")
    _plain(lse, "lse", q.shape[:3], torch.float32, dev)

    def call(st):
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        desc = _ATTENTION.pack(*lead, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3],
                               *dout.stride()[:3], *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3], *ptrs)
        check(lib.mg_attention_backward(desc, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dout.data_ptr(),
                                        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), st))
        return dq, dk, dv

    return _on(dev, stream, call, dout, q, k, v, out, lse, slopes, documents, prefix)


# ------------------------------------------------------------------ rotary positions
def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       trained: int = 0, low: float = 1.0, high: float = 32.0, device="cuda") -> torch.Tensor:
    """Radians a position of each of the rotary_dim / 2 pairs, float64: theta^(-2p / rotary_dim), scaled for contexts
    `factor` times the trained length:
      "linear"  every frequency divided by factor
      "ntk"     theta raised so that the slowest pair alone is divided by factor
      "parts"   pairs that make fewer than `low` turns over the `trained` positions are divided by factor, those that
                make more than `high` are kept, with a linear ramp in between"""
    if rotary_dim < 0 or rotary_dim % 2:
        _bad(f"rotary_dim must be even, found {rotary_dim}")
    if scaling not in ("none", "linear", "ntk", "parts"):
        _bad(f"scaling must be 'none', 'linear', 'ntk' or 'parts', found {scaling!r}")
    theta, factor = float(theta), float(factor)
    if not (0 < theta < math.inf and 0 < factor < math.inf):
        _bad("theta and factor must be positive and finite")
    if scaling == "parts" and (trained < 1 or not low < high):
        _bad("scaling 'parts' needs trained > 0 and low < high")
    if scaling == "ntk" and rotary_dim > 2:
        theta *= factor ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (-torch.arange(rotary_dim // 2, dtype=torch.float64) * 2 / max(1, rotary_dim))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        keep = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f.to(device)


def _rotary(q, k, positions, frequencies, interleaved, inverse, magnitude, out_q, out_k, stream):
    lib = _lib.load()
    _heads(q, "q", 4, None, None)
    dt, dev = q.dtype, q.device
    B, H, L, D = q.shape
    Hkv = 0
    if k is not None:
        _heads(k, "k", 4, dt, dev)
        Hkv = k.shape[1]
        if k.shape[0] != B or k.shape[2] != L or k.shape[3] != D:
            _bad("k must have q's batch, length and head_dim\n"
                 f"Found shapes | q: {tuple(q.shape)} | k: {tuple(k.shape)}")
    elif out_k is not None:
        _bad("out_k without k")
    if not isinstance(frequencies, torch.Tensor) or frequencies.dim() != 1:
        _bad("frequencies must be a one-dimensional tensor (rotary_frequencies)")
    pairs = frequencies.shape[0]
    _plain(frequencies, "frequencies", (pairs,), torch.float64, dev)
    if 2 * pairs > D:
        _bad(f"{pairs} pairs do not fit a head of {D}")
    if not isinstance(positions, torch.Tensor) or positions.dim() not in (1, 2):
        _bad("positions must be an int32 tensor of shape [length] or [batch, length]")
    shared = positions.dim() == 1
    _plain(positions, "positions", (L,) if shared else (B, L), torch.int32, dev)
    magnitude = _number(magnitude, "magnitude")
    if out_q is not None:
        _written(out_q, "out_q", q)
    if out_k is not None:
        _written(out_k, "out_k", k)
    # other overlaps are the library's to refuse
    for y, other, names in ((out_q, k, "out_q and k"), (out_k, q, "out_k and q"), (out_k, out_q, "out_k and out_q")):
        if y is not None and other is not None and y.numel() and y.data_ptr() == other.data_ptr():
            _bad(f"{names} are the same memory")

    def call(st):
        oq = torch.empty_like(q) if out_q is None else out_q
        ok = torch.empty_like(k) if k is not None and out_k is None else out_k
        desc = _ROTARY.pack(_DTYPES[dt], B, H, Hkv, L, D, pairs, 1 if interleaved else 0, 1 if inverse else 0,
                            magnitude, *q.stride()[:3], *(k.stride()[:3] if Hkv else _ZERO3), *oq.stride()[:3],
                            *(ok.stride()[:3] if Hkv else _ZERO3), 0 if shared else L, positions.data_ptr(),
                            frequencies.data_ptr())
        check(lib.mg_rotary(desc, oq.data_ptr(), _at(ok), q.data_ptr(), _at(k), st))
        return oq, ok

    return _on(dev, stream, call, q, k, positions, frequencies, out_q, out_k)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
           interleaved: bool = False, magnitude: float = 1.0, out_q: Optional[torch.Tensor] = None,
           out_k: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None
           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns pair p of every head of q [B, H, L, D] and k [B, Hkv, L, D] (or None) by the angle positions[b, l] *
    frequencies[p]: (a, b) -> magnitude * (a cos - b sin, a sin + b cos). Pair p is (2p, 2p + 1) if interleaved, else
    (p, p + pairs); what lies behind the 2 * pairs first elements is copied. positions: int32 [L] or [B, L];
    frequencies: float64 (rotary_frequencies). One launch; out_q and out_k may be q and k themselves, but must not
    overlap them in another way.

    Returns (turned q, turned k or None)."""
    return _rotary(q, k, positions, frequencies, interleaved, False, magnitude, out_q, out_k, stream)


def rotary_backward(dq: torch.Tensor, dk: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
                    interleaved: bool = False, magnitude: float = 1.0, out_q: Optional[torch.Tensor] = None,
                    out_k: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None
                    ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of rotary()'s inputs from those of its outputs: the opposite turn, with the same magnitude."""
    return _rotary(dq, dk, positions, frequencies, interleaved, True, magnitude, out_q, out_k, stream)


# ------------------------------------------------------------------ paged attention
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, scale: Optional[float] = None, cap: float = 0.0,
                    slopes: Optional[torch.Tensor] = None, k_new: Optional[torch.Tensor] = None,
                    v_new: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                    stream: Optional[torch.cuda.Stream] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of one new token per request over a cache in pages: attention() for Lq = 1.

    q [B, H, D]; k_pages and v_pages [pages, page_size, Hkv, D] (any strides with a contiguous last dim, so a pool kept
    as [pages, Hkv, page_size, D] is passed transposed); block_table int32 [B, width]: the pages of each request in
    order; lengths int32 [B]: its keys, the new token among them. The query stands at position lengths[b] - 1.
    With k_new and v_new [B, Hkv, D] the token's own key and value come from there, and the call also writes them to
    the cache at that position; requests must not share the page they append to, nor keys and values theirs, and k_new
    and v_new must not lie there. `out` may be q itself, but shares memory with no input otherwise. A length
    of 0 gives out = 0, lse = -inf and writes nothing. A length beyond the table is cut off there (the call attends to
    the keys that the table holds, from the last one's position, and the request appends nothing), a page outside the
    pool is skipped, and mg_device_status() then reports MG_ERR_INVALID.

    Returns (out [B, H, D], lse [B, H] in float32)."""
    lib = _lib.load()
    _heads(q, "q", 3, None, None)
    dt, dev = q.dtype, q.device
    _heads(k_pages, "k_pages", 4, dt, dev)
    _heads(v_pages, "v_pages", 4, dt, dev)
    B, H, D = q.shape
    pages, page, Hkv = k_pages.shape[:3]
    if k_pages.shape != v_pages.shape or k_pages.shape[3] != D or page < 1:
        _bad("k_pages and v_pages must be [pages, page_size, kv_heads, head_dim]\n"
             f"Found shapes | q: {tuple(q.shape)} | k_pages: {tuple(k_pages.shape)} | v_pages: {tuple(v_pages.shape)}")
    if Hkv == 0 or H % Hkv:
        _bad(f"the {H} query heads must be a multiple of the {Hkv} key-value heads")
    if not 1 <= D <= MAX_HEAD_DIM:
        raise MacrogradError(_lib.MG_ERR_UNSUPPORTED, f"head_dim {D} is outside 1..{MAX_HEAD_DIM}")
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        _bad("block_table must be an int32 tensor of shape [batch, width]")
    width = block_table.shape[1]
    _plain(block_table, "block_table", (B, width), torch.int32, dev)
    _plain(lengths, "lengths", (B,), torch.int32, dev)
    scale = 1.0 / math.sqrt(D) if scale is None else _number(scale, "scale")
    cap = _cap(cap)
    if slopes is not None:
        _plain(slopes, "slopes", (H,), torch.float32, dev)
    if (k_new is None) != (v_new is None):
        _bad("k_new and v_new come together")
    for t, name in ((k_new, "k_new"), (v_new, "v_new")):
        if t is not None:
            _heads(t, name, 3, dt, dev)
            if t.shape != (B, Hkv, D):
                _bad(f"{name} must have shape {(B, Hkv, D)}, found {tuple(t.shape)}")
    if k_new is not None:
        _written(k_pages, "k_pages", k_pages)
        _written(v_pages, "v_pages", v_pages)
        if k_pages.numel() and k_pages.data_ptr() == v_pages.data_ptr():
            _bad("k_pages and v_pages are the same memory: nothing can be appended to them")
    if out is not None:
        _written(out, "out", q)

    def call(st):
        o = torch.empty_like(q) if out is None else out
        lse = torch.empty_strided((B, H), (H, 1), dtype=torch.float32, device=dev)
        new = (*k_new.stride()[:2], *v_new.stride()[:2]) if k_new is not None else (0, 0, 0, 0)
        desc = _PAGED.pack(_DTYPES[dt], B, H, Hkv, D, page, pages, width, scale, cap, *q.stride()[:2], *o.stride()[:2],
                           *k_pages.stride()[:3], *v_pages.stride()[:3], *new, width, _at(slopes),
                           block_table.data_ptr(), lengths.data_ptr())
        check(lib.mg_paged_attention(desc, o.data_ptr(), lse.data_ptr(), q.data_ptr(), k_pages.data_ptr(),
                                     v_pages.data_ptr(), _at(k_new), _at(v_new), st))
        return o, lse

    return _on(dev, stream, call, q, k_pages, v_pages, block_table, lengths, slopes, k_new, v_new, out)
