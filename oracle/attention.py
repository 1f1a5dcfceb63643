"""Plain restatement of the 8-bit key/value cache and of attention over it (test infrastructure only).

Parity unpinned: the reference has no attention and no cache; the definitions are those of include/jq.h.  The order of the
codes is restated place by place, quantisation is in fp32 with numpy (one rounding per operation), attention in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

TOP = {"int8": np.float32(127), "e4m3": np.float32(448)}
LEAST = np.float32(2.0 ** -60)


def key_place(token: int, d: int, D: int) -> int:
    """Byte of a block's keys that holds value d of a token: a place (g, t) holds values 8t.. of token k and of k + 2."""
    group, kk = divmod(token, 16)
    for g in range(8):
        for j in range(2):
            if 4 * (g // 2) + g % 2 + 2 * j == kk:
                return group * 16 * D + d // 32 * 512 + (4 * g + d % 32 // 8) * 16 + 8 * j + d % 8
    raise AssertionError


def value_place(token: int, d: int, D: int) -> int:
    """The same for values: a place (g, t) holds tokens 4t.. of the values g, g + 8, g + 16, g + 24."""
    group, kk = divmod(token, 16)
    return group * 16 * D + d // 32 * 512 + (4 * (d % 8) + kk // 4) * 16 + 4 * (d % 32 // 8) + kk % 4


def places(T: int, D: int, what: str) -> np.ndarray:
    """[T, D] bytes of a block."""
    f = key_place if what == "keys" else value_place
    return np.array([[f(t, d, D) for d in range(D)] for t in range(T)])


def e4m3_values() -> np.ndarray:
    out = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = np.ldexp(m, -9) if e == 0 else np.ldexp(8 + m, e - 10)
        out[c] = -v if c & 128 else v
    out[0x7F] = out[0xFF] = np.nan
    return out


def decode(codes: np.ndarray, fmt: str) -> np.ndarray:
    """fp32 values at scale 1 (exact)."""
    return (e4m3_values()[codes] if fmt == "e4m3" else codes.astype(np.float64) - 128).astype(np.float32)


def encode(q: np.ndarray, fmt: str) -> np.ndarray:
    """Nearest codes of fp32 values at scale 1, ties to the even code; infinities are the largest, NaN is 0."""
    q = np.clip(np.nan_to_num(q, nan=0.0, posinf=np.inf, neginf=-np.inf), -TOP[fmt], TOP[fmt]).astype(np.float64)
    if fmt == "int8":
        return (np.rint(q) + 128).astype(np.uint8)
    grid = e4m3_values()[:127]                                   # 0 .. 448, rising, code = index
    a = np.abs(q)
    hi = np.searchsorted(grid, a).clip(1, 126)
    lo = hi - 1
    up = (a - grid[lo] > grid[hi] - a) | ((a - grid[lo] == grid[hi] - a) & (hi % 2 == 0))
    return (np.where(up, hi, lo) | np.where(np.signbit(q), 128, 0)).astype(np.uint8)


def append_block(codes, scale, held, fresh, fmt):
    """A block's natural-order codes [T, D] and scale after `fresh` fp32 [n, D] came behind its `held` tokens."""
    codes = codes.copy()
    finite = fresh[np.isfinite(fresh)]
    a = max(LEAST, np.abs(finite).max() if finite.size else np.float32(0)).astype(np.float32)
    old = np.float32(scale if held else 0)
    new = max(old, np.float32(a / TOP[fmt]))
    with np.errstate(invalid="ignore", over="ignore"):
        if held and new > old:
            codes[:held] = encode((decode(codes[:held], fmt) * old).astype(np.float32) / new, fmt)
        codes[held:held + len(fresh)] = encode(fresh.astype(np.float32) / new, fmt)
    return codes, new


def attend(q, keys, values, first, scale, window):
    """64-bit attention of one head: q [n, D] at the positions first.., keys and values [len, D].  Returns outputs, lse, and
    what a bound on the error needs: sum p |v| and the largest sum |q k| scale."""
    q, keys, values = q.double(), keys.double(), values.double()
    n, length = q.shape[0], keys.shape[0]
    pos = first + torch.arange(n, device=q.device)[:, None]
    key = torch.arange(length, device=q.device)
    seen = key <= pos
    if window:
        seen &= key > pos - window
    s = (q @ keys.T * scale).masked_fill(~seen, -torch.inf)
    size = (q.abs() @ keys.abs().T * scale).masked_fill(~seen, 0).amax(-1) if length else torch.zeros(n, device=q.device).double()
    lse = torch.logsumexp(s, -1) if length else torch.full((n,), -torch.inf, device=q.device, dtype=torch.float64)
    p = torch.where(seen, (s - torch.where(lse.isfinite(), lse, 0.0)[:, None]).exp(), 0.0)
    return p @ values, lse, p @ values.abs(), size
