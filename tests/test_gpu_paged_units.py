"""Attention over a paged cache where a CTA has many units: what one unit leaves behind must not reach the next."""
import math

import pytest
import torch

from natten_mps_b200 import _cabi, functional as F
from tests import _decoder_ref as R, _decoder_rows as rows

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _normal(seed, *shape, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _long(lens, L, Hq, Hkv, D, page, dtype=BF16, seed=0):
    B, width = len(lens), -(-max(lens) // page)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(seed)).int().view(B, width).cuda()
    caches = [_normal(seed + i, B * width, page, Hkv, D, dtype=dtype) for i in (1, 2)]
    return _normal(seed + 3, B, L, Hq, D, dtype=dtype), *caches, table, torch.tensor(lens).int().cuda()


def _check(q, k_cache, v_cache, table, lens, kernel=None, dilation=1, path=None):
    out, lse = F.na1d_paged(q, k_cache, v_cache, table, lens, kernel, dilation, return_lse=True)
    assert path is None or _cabi.last_path() == path
    want, want_lse, bound, lse_bound = rows.attend(q.double(), k_cache.double(), v_cache.double(), table, lens,
                                                   [q.shape[1]] * q.shape[0], kernel, dilation)
    R.check("out", out, want, bound(q.dtype))
    R.check("lse", lse, want_lse, lse_bound)
    return out, lse


@pytest.mark.parametrize("D,kernel,page", [(64, None, 16), (128, None, 64), (64, 2100, 64), (128, 2100, 16)], ids=str)
def test_long_units_of_half_the_rows_in_front_of_whole_ones(D, kernel, page):
    """2080 rows of a group of 4: 32 row tiles of 256 rows and one of 128, in which the second half of the softmax takes no
    part, over up to 32 tiles of keys.  The next sequence's first tiles, which it does take part in, have other keys missing."""
    q, k_cache, v_cache, table, lens = _long([4096, 4000, 4090, 4031], 2080, 16, 4, D, page)
    for b in range(4):
        for n in range(b, 2112 // page, 4 + b):          # holes that differ, in all of the first tiles that a row tile can begin with
            k_cache[table[b, n].long()] = math.nan
            v_cache[table[b, n].long()] = math.nan
            table[b, n] = (-1, 10 ** 9)[n % 2]
    first = _check(q, k_cache, v_cache, table, lens, kernel, path="tcgen05")
    for _ in range(4):
        again = F.na1d_paged(q, k_cache, v_cache, table, lens, kernel, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype,B,L,Hq,Hkv,D,page,context,kernel,dilation,path", [
    # whole prompts through a window: seven units of 256 rows for each of 148 CTAs, taken whole
    (BF16, 2, 4096, 32, 8, 64, 64, 4096, 200, 1, "tcgen05"),
    (F16, 2, 4000, 24, 8, 128, 16, 4096, 130, 1, "tcgen05"),
    (BF16, 2, 4001, 16, 8, 64, 24, 4003, 50, 2, "tcgen05"),
    # ... and shared between CTAs: a window longer than a short unit's tiles
    (BF16, 2, 2500, 32, 8, 128, 16, 2600, 1500, 1, "tcgen05"),
    # 40 rows a unit, split by keys: more columns than threads, and several units a CTA
    (BF16, 600, 10, 4, 1, 64, 16, 90, None, 1, "tcgen05"),
    (F16, 160, 10, 32, 8, 128, 16, 700, None, 1, "tcgen05"),
    (BF16, 300, 20, 8, 4, 128, 7, 400, 33, 1, "tcgen05"),
    # few rows, more short units than SMs (four warps, two CTAs an SM), and more columns than threads
    (BF16, 160, 1, 8, 2, 128, 16, 200, 64, 1, "warp"),
    (F16, 160, 1, 8, 2, 64, 16, 300, 100, 2, "warp"),
    (BF16, 90, 5, 8, 2, 32, 7, 150, None, 1, "warp"),
    (F16, 90, 7, 8, 2, 128, 24, 150, 40, 1, "warp"),
    (BF16, 300, 4, 12, 2, 64, 16, 120, None, 1, "warp"),
    (BF16, 200, 2, 4, 2, 256, 16, 100, None, 1, "warp"),
    # ... and shared: eight warps
    (BF16, 300, 1, 4, 1, 128, 16, 3000, None, 1, "warp"),
    # the FMA pipe
    (F32, 600, 3, 4, 2, 32, 16, 100, None, 1, "simt"),
    (F32, 300, 1, 4, 1, 64, 16, 900, None, 1, "simt"),
    (BF16, 200, 4, 4, 2, 20, 16, 100, 30, 1, "simt"),
], ids=str)
def test_many_units(dtype, B, L, Hq, Hkv, D, page, context, kernel, dilation, path):
    lens = [context - (7 * b) % (context - L + 1) for b in range(B)]
    problem = _long(lens, L, Hq, Hkv, D, page, dtype=dtype)
    a = _check(*problem, kernel, dilation, path=path)
    b = F.na1d_paged(*problem, kernel, dilation, return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
