"""Attention over a paged cache with scores of very different size: a row's maximum has to follow them exactly."""
import pytest
import torch

from natten_mps_b200 import functional as F
from tests import _decoder_ref as R, _decoder_rows as rows

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("first", [-2.0 ** 12, -2.0 ** 40, -2.0 ** 90, 2.0 ** 12, 3 * 2.0 ** 24, 3 * 2.0 ** 39, 5 * 2.0 ** 38, 7 * 2.0 ** 90])
@pytest.mark.parametrize("dtype,L,Hq,Hkv,D", [(BF16, 1, 4, 2, 64), (BF16, 40, 2, 1, 64), (BF16, 70, 4, 1, 128), (BF16, 40, 2, 1, 96),
                                              (torch.float32, 3, 2, 1, 32)], ids=str)
def test_scores_far_from_zero(dtype, L, Hq, Hkv, D, first):
    """The first 256 keys score `first`, all of them, the others between 0 and 288: everything is decided among the higher ones.
    One product a score, so that scores are exact in float32 and in float64."""
    page, n = 16, 32
    table = torch.randperm(2 * n, generator=torch.Generator().manual_seed(0)).int().view(2, n).cuda()
    k_cache = torch.zeros(2 * n, page, Hkv, D, device="cuda", dtype=dtype)
    v_cache = torch.randn(2 * n, page, Hkv, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    j = torch.arange(500, device="cuda")
    for b in range(2):
        at = (table[b].long()[j // page], j % page)
        k_cache[*at, :, 0] = torch.where(j < 256, first, 0.0).to(dtype)[:, None]
        k_cache[*at, :, 1] = torch.where(j < 256, 0.0, (j % 37) * 8.0).to(dtype)[:, None]
    q = torch.zeros(2, L, Hq, D, device="cuda", dtype=dtype)
    q[..., :2] = 1.0
    lens = torch.tensor([500, 500]).int().cuda()
    out, lse = F.na1d_paged(q, k_cache, v_cache, table, lens, scale=1.0, return_lse=True)
    exact = lambda v: rows.attend(q.double(), k_cache.double(), v.double(), table, lens, [L, L], scale=1.0)  # noqa: E731
    want, want_lse = exact(v_cache)[:2]
    # Scores that count lie at most 288 apart: their exponents are off by the roundings of log2(e), of the product with it, of the
    # difference and of the exponential (equal scores by the same); the weights by their rounding, sums by their own.
    slack, count = 4 * 288 * 2.0 ** -24 + 2.0 ** -22, 500
    weight = R.HALF_STEP[dtype] + 2 * slack + 2 * count * 2.0 ** -24
    R.check("out", out, want, exact(v_cache.abs())[0] * weight + R.HALF_STEP[dtype] * want.abs())
    R.check("lse", lse, want_lse, slack + count * 2.0 ** -24 + (want_lse.abs() + 8) * 2.0 ** -22)
