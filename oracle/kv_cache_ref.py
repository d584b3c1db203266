"""Oracle of the paged e4m3 key/value cache and the attention over it, in 64 bits.

Plain torch on whatever device the inputs are on; written from the definitions,
without the package: e4m3 values are decoded and rounded arithmetically.
"""
from __future__ import annotations

import math

import torch

MIN_EXP = -63
NAN_BYTE = 255


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value (ties to the even one) of float64 x with |x| <= 448."""
    power = torch.frexp(x)[1].double() - 1
    step = torch.exp2(power.clamp(min=-6) - 3)
    return torch.round(x / step) * step


def decode_e4m3(codes: torch.Tensor) -> torch.Tensor:
    """float64 values of uint8 codes (0x7f / 0xff are NaN)."""
    c = codes.to(torch.int64)
    e, m = (c >> 3) & 15, (c & 7).double()
    x = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e.double() - 7))
    x = torch.where((c & 0x7f) == 0x7f, torch.full_like(x, math.nan), x)
    return torch.where(c >= 128, -x, x)


def quantise(x: torch.Tensor):
    """(values of the codes, exponent bytes) of rows x (..., D)."""
    x = x.double()
    amax = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    part, power = torch.frexp(torch.where(fine, amax, torch.zeros_like(amax)))
    # amax = part * 2^power <= 448 * 2^e = 0.875 * 2^(e + 9)
    e = power - 9 + (part > 0.875).to(power.dtype)
    e = torch.where(amax == 0, torch.zeros_like(e), e.clamp(min=MIN_EXP))
    x = torch.where(fine.unsqueeze(-1), x, torch.zeros_like(x))
    codes = round_e4m3(x * torch.exp2(-e.double()).unsqueeze(-1))
    byte = torch.where(fine, e + 127, torch.full_like(e, NAN_BYTE))
    return codes, byte.to(torch.uint8)


def factor(byte: torch.Tensor) -> torch.Tensor:
    f = torch.exp2(byte.double() - 127)
    return torch.where(byte == NAN_BYTE, torch.full_like(f, math.nan), f)


def tokens(codes_u8, exps, table_row, first, last):
    """float64 values (H_kv, last - first, D) of tokens first..last-1 of one sequence."""
    page_size = codes_u8.shape[2]
    pos = torch.arange(first, last, device=codes_u8.device)
    page, slot = table_row.long()[pos // page_size], pos % page_size
    x = decode_e4m3(codes_u8[page, :, slot]) * factor(exps[page, :, slot]).unsqueeze(-1)
    return x.transpose(0, 1)


def to_16bit(x: torch.Tensor, dtype) -> torch.Tensor:
    """One rounding to fp16 / bf16, saturating; NaN stays."""
    top = torch.finfo(dtype).max
    return x.clamp(-top, top).to(dtype)


def attention(q, k, v, scale):
    """Queries (H, S_q, D) at the end of keys k, v (H_kv, n, D), all float64.

    Returns out, lse and, for error bounds, A = sum p |v| / sum p, n_eff = sum p /
    max p, and B = the largest sum |q k| * scale of a visible key, per query.
    """
    H, S_q, D = q.shape
    Hkv, n, _ = k.shape
    G = H // Hkv
    kk, vv = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    s = torch.matmul(q, kk.transpose(1, 2)) * scale
    mag = torch.matmul(q.abs(), kk.abs().transpose(1, 2)) * scale
    pos = torch.arange(n - S_q, n, device=q.device)
    seen = torch.arange(n, device=q.device)[None, :] <= pos[:, None]
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    mag = torch.where(seen, mag, torch.zeros_like(mag))
    none = ~seen.any(-1)
    m = torch.where(none, torch.zeros((), dtype=s.dtype, device=s.device), s.amax(-1) if n else 0.0)
    p = torch.exp(s - m.unsqueeze(-1))
    p = torch.where(seen, p, torch.zeros_like(p))
    total = p.sum(-1)
    safe = torch.where(none, torch.ones_like(total), total)
    # A key that a query does not see is no part of its sum, whatever it holds.
    out = torch.zeros(H, S_q, D, dtype=torch.float64, device=q.device)
    A = torch.zeros_like(out)
    for i in range(S_q):
        e = int(min(max(n - S_q + i + 1, 0), n))
        out[:, i] = torch.einsum("hn,hnd->hd", p[:, i, :e], vv[:, :e]) / safe[:, i, None]
        A[:, i] = torch.einsum("hn,hnd->hd", p[:, i, :e], vv[:, :e].abs()) / safe[:, i, None]
    lse = torch.where(none, torch.full_like(m, -math.inf), m + torch.log(safe))
    B = mag.amax(-1) if n else torch.zeros(H, S_q, dtype=torch.float64, device=q.device)
    return out, lse, A, total, B
