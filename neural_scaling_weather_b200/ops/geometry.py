"""Window/shift geometry shared by the attention operator and its kernels."""

from __future__ import annotations

from dataclasses import dataclass
from typing import Tuple

import torch


@dataclass(frozen=True)
class WindowGeometry:
    """How a (B, T, H, W) token grid is cut into attention windows.

    window:     (wh, ww) window size in tokens.
    shift:      cyclic shift applied by index arithmetic before partitioning: window
                token (r, c) reads grid token ((r + sh) % H, (c + sw) % W), and its
                output is written back to the same grid position.
    mask:       whether the latitude-wrap mask is active (the block is a shifted one).
    mask_shift: the block's latitude shift; rows r_g >= h_global - mask_shift (global,
                rolled coordinates) form the second region.
    row_offset: global row of this rank's first (rolled) row, in tokens.
    h_global:   global number of token rows.
    """

    window: Tuple[int, int]
    shift: Tuple[int, int] = (0, 0)
    mask: bool = False
    mask_shift: int = 0
    row_offset: int = 0
    h_global: int = 0

    def num_buckets(self, steps: int = 1) -> int:
        """Displacements between two tokens of a window of ``steps`` time steps."""
        return (2 * steps - 1) * (2 * self.window[0] - 1) * (2 * self.window[1] - 1)

    def relative_buckets(self, steps: int = 1) -> torch.Tensor:
        """Bucket of query token i and key token j, (L, L): ``((dt + T - 1) (2 wh - 1) + dy + wh - 1) (2 ww - 1) + dx + ww - 1``
        of the query's time step, row and column less the key's (tokens in window order, columns fastest)."""
        wh, ww = self.window
        at = torch.stack(torch.meshgrid(torch.arange(steps), torch.arange(wh), torch.arange(ww), indexing="ij")).flatten(1)
        d = at[:, :, None] - at[:, None, :] + torch.tensor([steps - 1, wh - 1, ww - 1])[:, None, None]
        return (d[0] * (2 * wh - 1) + d[1]) * (2 * ww - 1) + d[2]
