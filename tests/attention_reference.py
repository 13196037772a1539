"""Attention, its gradients and rotary positions in 64 bits, straight from their
definitions (include/mg_attention.h), with element-wise bounds on what a kernel
that rounds as documented may be off by.

Bounds. Let u be half a step of the type, eps / 2 (fp32 2^-24, bf16 2^-8).
* A product of D terms accumulated in fp32 is off by about sqrt(D) * 2^-24 times
  the sum of its terms' magnitudes, and a sum over n keys by sqrt(n) * 2^-24
  (rounding errors of either sign); FACTOR = 8 covers their spread. So a score is
  off by ds = 8 * 2^-24 * (sqrt(D) * top + 4 * |bias|max + 8 * cap), top being the largest
  |q||k| scale, and P relatively by 2 ds + 8 * 2^-24 * sqrt(n).
* With 16-bit tensors P and dS are rounded to 16 bits before their products: each
  term is off by u of itself. delta comes from the rounded out: off by
  u * sum |dout||out|.
* Results are rounded once more: u of themselves.
"""
import math

import torch

FACTOR = 8.0
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def seen_mask(B, Lq, Lk, causal, documents, prefix, device):
    pos = torch.arange(Lq, device=device) + (Lk - Lq)
    j = torch.arange(Lk, device=device)
    seen = torch.ones((B, Lq, Lk), dtype=torch.bool, device=device)
    if causal:
        seen &= (j[None, None] <= pos[None, :, None]) | (
            j[None, None] < (prefix if prefix is not None else torch.zeros(B, device=device))[:, None, None])
    if documents is not None:
        mine = torch.full((B, Lq), -1, dtype=torch.int64, device=device)
        inside = pos >= 0
        mine[:, inside] = documents.long()[:, pos[inside]]
        seen &= (mine[:, :, None] == documents.long()[:, None, :]) & (mine >= 0)[:, :, None]
    return seen


class Reference:
    """Everything about one call, in float64. Padding (documents < 0) is taken as zeros, whatever it holds."""

    def __init__(self, q, k, v, dout=None, scale=None, causal=True, cap=0.0, slopes=None, documents=None, prefix=None):
        dtype = q.dtype
        B, H, Lq, D = q.shape
        Hkv, Lk = k.shape[1], k.shape[2]
        scale = 1 / math.sqrt(D) if scale is None else scale
        dev = q.device
        if documents is not None:
            hide = (documents < 0)[:, None, :, None]
            k, v = k.masked_fill(hide, 0), v.masked_fill(hide, 0)
            pos = torch.arange(Lq, device=dev) + (Lk - Lq)
            pad = torch.ones((B, Lq), dtype=torch.bool, device=dev)
            pad[:, pos >= 0] = (documents < 0)[:, pos[pos >= 0]]
            q = q.masked_fill(pad[:, None, :, None], 0)
            dout = dout.masked_fill(pad[:, None, :, None], 0) if dout is not None else None
        Q, K, V = q.double(), k.double(), v.double()
        G = H // Hkv
        K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
        t = scale * Q @ K.transpose(-1, -2)
        bend = torch.zeros_like(t)
        if cap > 0:
            bend = torch.tanh(t / cap)
            t = cap * bend
        far = ((torch.arange(Lq, device=dev) + (Lk - Lq))[:, None] - torch.arange(Lk, device=dev)[None]).abs().double()
        bias = 0.0
        if slopes is not None:
            t = t - slopes.double()[None, :, None, None] * far
            bias = float(slopes.abs().max() * far.max()) if far.numel() else 0.0
        seen = seen_mask(B, Lq, Lk, causal, documents, prefix, dev)[:, None]
        t = t.masked_fill(~seen, -math.inf)
        if Lk:
            self.lse = torch.logsumexp(t, -1)
            P = torch.where(seen, torch.exp(t - self.lse[..., None]), torch.zeros_like(t))
        else:
            self.lse = torch.full((B, H, Lq), -math.inf, dtype=torch.float64, device=dev)
            P = t
        self.out = P @ V
        u = half_step(dtype)
        u16 = 0.0 if dtype == torch.float32 else u
        top = abs(scale) * float(Q.norm(dim=-1).max() * K.norm(dim=-1).max()) if Q.numel() and K.numel() else 0.0
        # a bias is rounded with the score: a few roundings of its size
        ds = FACTOR * U32 * (math.sqrt(D) * top + 4 * bias + 8 * cap)
        rel = 2 * ds + FACTOR * U32 * math.sqrt(max(1, Lk))
        self.lse_tol = ds + FACTOR * U32 * (math.sqrt(max(1, Lk)) + self.lse.abs().nan_to_num(0, 0, 0))
        self.out_tol = (rel + u16) * (P @ V.abs()) + u * self.out.abs() + 1e-30
        if dout is None:
            return
        dO = dout.double()
        dP = dO @ V.transpose(-1, -2)
        delta = (P * dP).sum(-1, keepdim=True)
        curve = 1 - bend ** 2
        dS = P * (dP - delta) * scale * curve
        self.P, self.dS = P, dS
        shared = lambda x: x.view(B, Hkv, G, Lk, D).sum(2)  # noqa: E731
        self.dq = dS @ K
        self.dk = shared(dS.transpose(-1, -2) @ Q)
        self.dv = shared(P.transpose(-1, -2) @ dO)
        # |error of dS|: of P, of dP (a product of D terms), of delta, of the bend, and the rounding to 16 bits
        mag = dO.abs() @ V.abs().transpose(-1, -2)
        # delta comes from the rounded out, itself within out_tol
        derr = ((dO.abs() * (self.out_tol + u * self.out.abs())).sum(-1, keepdim=True)
                + FACTOR * U32 * math.sqrt(D) * (dO.abs() * self.out.abs()).sum(-1, keepdim=True))
        edS = P * abs(scale) * curve * (rel * (dP - delta).abs() + FACTOR * U32 * math.sqrt(D) * mag + derr) \
            + P * abs(scale) * (dP - delta).abs() * FACTOR * U32 * 4 * (1 if cap else 0) \
            + P * abs(scale) * (dP - delta).abs() * (2 * ds / cap if cap else 0) + u16 * dS.abs()
        long = FACTOR * U32 * math.sqrt(max(Lk, Lq * G, 1))
        self.dq_tol = edS @ K.abs() + long * (dS.abs() @ K.abs()) + u * self.dq.abs() + 1e-30
        self.dk_tol = shared((edS + long * dS.abs()).transpose(-1, -2) @ Q.abs()) + u * self.dk.abs() + 1e-30
        self.dv_tol = shared((P * (rel + u16 + long)).transpose(-1, -2) @ dO.abs()) + u * self.dv.abs() + 1e-30


def within(got, want, tol, what):
    """Every element of `got` within `tol` of `want`; infinities and zeros of empty rows exactly."""
    got = got.double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}"
    if not want.numel():
        return
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got) & (got == want), inf), f"{what}: infinities differ"
    err = torch.where(inf, torch.zeros_like(want), (got - want).abs())
    assert not torch.isnan(err).any(), f"{what}: NaN"
    worst = (err / tol.clamp_min(1e-38)).masked_fill(inf, 0).max()
    assert worst <= 1, f"{what}: error {float(worst):.3g} times its bound"


def rotate(x, positions, frequencies, interleaved=False, inverse=False, magnitude=1.0):
    """x [B, H, L, D] in float64, pairs as complex numbers."""
    pairs = frequencies.numel()
    pos = positions if positions.dim() == 2 else positions[None].expand(x.shape[0], -1)
    angle = pos.double()[:, None, :, None] * frequencies
    turn = torch.polar(torch.full_like(angle, magnitude), -angle if inverse else angle)
    y = x.double().clone()
    a = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    b = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    z = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * turn
    y[..., a], y[..., b] = z.real, z.imag
    return y
