"""64-bit restatement of the row operators (dropout, residual + RMS norm, rows in e4m3) for the tests.

TEST INFRASTRUCTURE.  Written from the definitions in ``include/coda_b200.h``; shares no code with the package.
"""

from __future__ import annotations

import numpy as np
import torch

MASK = np.uint64(0xFFFFFFFF)


def philox(counter: list[np.ndarray], key: tuple[int, int]) -> list[np.ndarray]:
    """Philox4x32-10 on uint64 arrays that hold 32-bit words."""
    c0, c1, c2, c3 = (np.asarray(c, dtype=np.uint64) for c in counter)
    k0, k1 = np.uint64(key[0]), np.uint64(key[1])
    shift = np.uint64(32)
    for _ in range(10):
        p0, p1 = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = (p1 >> shift) ^ c1 ^ k0, p1 & MASK, (p0 >> shift) ^ c3 ^ k1, p0 & MASK
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & MASK, (k1 + np.uint64(0xBB67AE85)) & MASK
    return [c0, c1, c2, c3]


def keep_mask(rows: int, cols: int, p: float, seed: int, step: int, stream: int, first_row: int = 0) -> torch.Tensor:
    """Rows ``first_row ..`` of the mask as a bool tensor on the CPU."""
    blocks = -(-cols // 4)
    b = (np.arange(first_row, first_row + rows, dtype=np.uint64)[:, None] * np.uint64(blocks) + np.arange(blocks, dtype=np.uint64)).reshape(-1)
    one = np.ones_like(b)
    words = philox([b & MASK, b >> np.uint64(32), one * np.uint64(step % 2**32), one * np.uint64(stream)],
                   (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    u = np.stack(words, axis=1).reshape(rows, blocks * 4)[:, :cols]
    return torch.from_numpy(u >= np.uint64(min(round(p * 2**32), 2**32 - 1)))


def dropped(x: torch.Tensor, keep: torch.Tensor, p: float) -> torch.Tensor:
    return torch.where(keep, x / (1.0 - p), torch.zeros_like(x))


def norm(h: torch.Tensor, weight: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(out, rstd)`` of rows in float64."""
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * rstd * weight, rstd


def norm_backward(dout, dh, h, rstd, weight):
    """``(dres, dweight)`` in float64; ``dh`` may be ``None``."""
    g, xh = dout * weight, h * rstd
    dres = rstd * (g - xh * (g * xh).mean(-1, keepdim=True))
    return (dres if dh is None else dres + dh), (dout * xh).reshape(-1, h.shape[-1]).sum(0)


def row_scale(out: torch.Tensor) -> torch.Tensor:
    return torch.clamp(out.abs().amax(-1) / 448.0, min=2.0**-126)
