"""Attention over a paged cache in float64, a sequence and head at a time as whole matrices on the tensors' own device: the
oracle for caches that ``_decoder_ref.attend`` would walk row by row for too long.  Its bounds are that oracle's."""
import math

import torch

from tests._decoder_ref import HALF_STEP


def attend(q, k_cache, v_cache, table, lens, new, kernel=None, dilation=1, scale=None):
    """``(out, lse, out_bound(dtype), lse_bound)`` of float64 tensors; ``new`` within ``[0, L]`` and the lengths."""
    B, L, Hq, D = q.shape
    pages, ps, Hkv, _ = k_cache.shape
    group, scale, dev = Hq // Hkv, D ** -0.5 if scale is None else scale, q.device
    out, spread = [torch.zeros(B, L, Hq, D, dtype=torch.float64, device=dev) for _ in range(2)]
    lse = torch.full((B, L, Hq), -math.inf, dtype=torch.float64, device=dev)
    slack, count = torch.zeros_like(lse), torch.ones_like(lse)
    for b in range(B):
        n, m = int(lens[b]), int(new[b])
        j = torch.arange(min(n, table.shape[1] * ps), device=dev)
        page = table[b].long()[j // ps]
        there = (page >= 0) & (page < pages)
        back = torch.arange(n - m, n, device=dev)[:, None] - j
        seen = (back >= 0) & (back % dilation == 0) & there
        if kernel is not None:
            seen &= back < kernel * dilation
        some = seen.any(-1)
        for h in range(Hq):
            keys, values = [torch.where(there[:, None], c[page.clamp(0, pages - 1), j % ps, h // group], 0.0) for c in (k_cache, v_cache)]
            score = (q[b, :m, h] @ keys.T * scale).masked_fill(~seen, -math.inf)
            lse[b, :m, h] = torch.logsumexp(score, -1)
            w = torch.where(some[:, None], torch.softmax(score, -1), 0.0)
            del score
            out[b, :m, h], spread[b, :m, h] = w @ values, w @ values.abs()
            size = (q[b, :m, h].abs() @ keys.abs().T).masked_fill(~seen, 0.0).amax(-1) * abs(scale)
            slack[b, :m, h] = torch.where(some, (D + 4) * 2.0 ** -24 * size + 2.0 ** -22, 0.0)
            count[b, :m, h] = seen.sum(-1).clamp_min(1)

    def bound(dtype):
        weights = HALF_STEP[dtype] + 2 * slack + 2 * count * 2.0 ** -24
        tiny = (count * 2.0 ** -25)[..., None] * float(v_cache.nan_to_num().abs().max()) if dtype == torch.float16 else 0
        return (spread * weights[..., None] + HALF_STEP[dtype] * out.abs() + tiny + 1e-30).cpu()

    shown = torch.where(torch.isfinite(lse), lse.abs(), 0)
    return out.cpu(), lse.cpu(), bound, (slack + count * 2.0 ** -24 + (shown + 8) * 2.0 ** -22).cpu()
