"""The append to a paged cache refuses tensors that share memory it writes to."""
import pytest
import torch

from natten_mps_b200 import _cabi, functional as F

pytestmark = pytest.mark.gpu


def test_overlapping_tensors_are_refused():
    pool = torch.randn(6, 4, 2, 64, device="cuda")
    k = torch.randn(1, 4, 2, 64, device="cuda")
    table, lens = torch.arange(2).int().view(1, 2).cuda(), torch.tensor([4]).int().cuda()
    keys, values, mine = pool[:3], pool[3:], pool[2:3]               # the last: a page of the keys as new tokens
    before = _cabi.launch_count()
    for args, kw in (((k, k, pool, pool), {}), ((k, k, pool[:4], pool[2:]), {}), ((mine, k, keys, values), {}), ((k, mine, keys, values), {}),
                     ((k, k, keys, values), {"query": mine}), ((k, pool[3:4], keys, values), {})):
        with pytest.raises(RuntimeError, match="memory location"):
            F.na1d_append(*args, table, lens, **kw)
    assert _cabi.launch_count() == before
    # what shares a storage but no element is served: halves of a pool, one behind the other or interleaved; key and value the same
    halves = torch.randn(6, 2, 4, 2, 64, device="cuda")
    want_k, want_v = values.clone(), halves[:, 1].clone()
    F.na1d_append(k, k, keys, values, table, lens)
    want_v[0] = want_k[0] = k[0]
    assert torch.equal(values, want_k) and torch.equal(keys[0], k[0])
    F.na1d_append(k, k, halves[:, 0], halves[:, 1], table, lens)
    assert torch.equal(halves[:, 1], want_v)
