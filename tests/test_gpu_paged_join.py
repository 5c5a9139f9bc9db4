"""Attention over a paged cache whose keys several CTAs share: the kernel that joins their partial results."""
import math

import pytest
import torch

from natten_mps_b200 import functional as F
from tests import _decoder_ref as R, _decoder_rows as rows

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
#        type, new tokens, heads, key/value heads, head dim: one row a head, split keys and two row halves on tcgen05, the FMA pipe
FORMS = [(BF16, 1, 4, 1, 64), (BF16, 40, 4, 2, 64), (F16, 70, 8, 2, 128), (F32, 3, 2, 1, 32)]


def _problem(dtype, L, Hq, Hkv, D, lens=(4100, 2777), page=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    B, width = len(lens), -(-max(lens) // page)
    normal = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    table = torch.randperm(B * width, generator=g).int().view(B, width).cuda()
    return normal(B, L, Hq, D), normal(B * width, page, Hkv, D), normal(B * width, page, Hkv, D), table, torch.tensor(lens).int().cuda()


def _check(q, k_cache, v_cache, table, lens, kernel=None):
    out, lse = F.na1d_paged(q, k_cache, v_cache, table, lens, kernel, return_lse=True)
    want, want_lse, bound, lse_bound = rows.attend(q.double(), k_cache.double(), v_cache.double(), table, lens, [q.shape[1]] * q.shape[0],
                                                   kernel)
    R.check("out", out, want, bound(q.dtype))
    R.check("lse", lse, want_lse, lse_bound)
    return out, lse


@pytest.mark.parametrize("form", [
    (F16, 1, 4, 1, 64), (F16, 3, 8, 2, 128), (BF16, 1, 4, 1, 256), (F16, 2, 4, 2, 160), (BF16, 5, 2, 1, 136),      # warps
    (BF16, 40, 2, 1, 128), (F16, 40, 4, 2, 64), (F16, 70, 8, 2, 64), (BF16, 100, 8, 2, 128),                      # tcgen05
    (F32, 2, 2, 1, 200), (F32, 2, 4, 2, 6), (F16, 1, 2, 1, 5), (BF16, 3, 2, 1, 130), (F32, 17, 2, 2, 129)], ids=str)
@pytest.mark.parametrize("kernel", [None, 2049])
def test_types_and_head_dims(form, kernel):
    """Head dims above 128, not a multiple of 4, every type, split keys."""
    problem = _problem(*form)
    a = _check(*problem, kernel)
    b = _check(*problem, kernel)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_query_that_is_not_a_number_shows(form):
    q, *cache = _problem(*form)
    q[0, -1, 1, 5] = math.nan                            # every score of one row
    out, lse = _check(q, *cache)
    assert bool(out[0, -1, 1].isnan().all()) and bool(lse[0, -1, 1].isnan()) and int(lse.isnan().sum()) == 1


@pytest.mark.parametrize("far_below", [False, True])
@pytest.mark.parametrize("form", [(BF16, 1, 4, 1, 64), (BF16, 40, 2, 1, 64), (F16, 70, 4, 1, 128), (F32, 3, 2, 1, 32)], ids=str)
def test_keys_that_are_not_numbers_show(form, far_below):
    """NaN in just the keys that one CTA sees, in one form or another (two tiles of 128 or 256, 16 of 32), so that its part
    of the sum has no finite score; or only one that is so low that the part's weight against the others vanishes."""
    for start, count in ((896, 256), (768, 512), (1504, 512)):
        q, k_cache, v_cache, table, lens = _problem(*form, lens=(4096,))
        q = q.abs() + 0.5
        where = torch.arange(start, start + count, device="cuda")
        k_cache[table[0].long()[where // 16], where % 16] = math.nan
        if far_below:
            k_cache[table[0, start // 16].long(), start % 16] = -60.0
        out, lse = _check(q, k_cache, v_cache, table, lens)
        assert bool(out.isnan().all()) and bool(lse.isnan().all())
