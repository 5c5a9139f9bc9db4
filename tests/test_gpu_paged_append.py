"""The append to a paged cache: new tokens land where the page table says, rotated, and nothing else changes."""
import pytest
import torch

from natten_mps_b200 import functional as F, rotary_frequencies
from tests import _decoder_ref as R

pytestmark = pytest.mark.gpu


def _normal(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _expected(k, v, k_cache, v_cache, table, lens, new, pos, freq, interleaved, magnitude, dtype):
    """Caches after the append, and the bound of each element (0: bit for bit)."""
    pages, ps = k_cache.shape[:2]
    kr, size = R.turn(k.double(), pos, freq, interleaved, magnitude) if freq is not None else (k.double(), None)
    bound = R.turn_bound(kr, size, dtype, pos, freq) if freq is not None else torch.zeros_like(kr)
    want_k, want_v, off = k_cache.double().clone(), v_cache.double().clone(), torch.zeros(k_cache.shape, dtype=torch.float64)
    for b in range(k.shape[0]):
        fresh = min(max(int(new[b]), 0), k.shape[1])
        for i in range(fresh):
            p = max(int(lens[b]), 0) - fresh + i if int(lens[b]) >= 0 else -1
            n = p // ps
            if p < 0 or n >= table.shape[1] or not 0 <= int(table[b, n]) < pages:
                continue
            at = (int(table[b, n]), p % ps)
            want_k[at], want_v[at], off[at] = kr[b, i], v.double()[b, i], bound[b, i]
    return want_k, want_v, off


@pytest.mark.parametrize("dtype,B,L,Hq,Hkv,D,rotary,interleaved,page", [
    (torch.bfloat16, 5, 1, 8, 2, 128, 128, False, 16),
    (torch.bfloat16, 3, 50, 4, 4, 64, 32, True, 7),
    (torch.float16, 4, 9, 6, 3, 64, 64, False, 24),
    (torch.float16, 2, 5, 2, 1, 40, 24, False, 4),
    (torch.float32, 3, 17, 6, 3, 40, 20, True, 24),
    (torch.bfloat16, 2, 6, 3, 1, 33, 10, False, 5),
    (torch.float64, 2, 4, 2, 2, 16, 16, False, 3),
    (torch.bfloat16, 3, 20, 4, 2, 64, 0, False, 16),
])
def test_against_float64(dtype, B, L, Hq, Hkv, D, rotary, interleaved, page):
    width = 12
    freq, magnitude = rotary_frequencies(rotary, scaling="linear", factor=3.0) if rotary else (None, 1.0)
    g = torch.Generator().manual_seed(17)
    k, v, q = _normal(1, B, L, Hkv, D, dtype=dtype), _normal(2, B, L, Hkv, D, dtype=dtype), _normal(3, B, L, Hq, D, dtype=dtype)
    k_cache, v_cache = _normal(4, B * width, page, Hkv, D, dtype=dtype), _normal(5, B * width, page, Hkv, D, dtype=dtype)
    table = torch.randperm(B * width, generator=g).int().view(B, width)
    lens = torch.randint(L, max(L + 1, width * page), (B,), generator=g).int()
    new = torch.randint(0, L + 1, (B,), generator=g).int()
    new[0] = L
    kd, vd = k_cache.cuda(), v_cache.cuda()
    turn = {"frequencies": freq.cuda(), "interleaved": interleaved, "magnitude": magnitude} if rotary else {}
    turned = F.na1d_append(k.cuda(), v.cuda(), kd, vd, table.cuda(), lens.cuda(), new.cuda(), query=q.cuda(), **turn)
    pos = R.new_positions(lens, new, L)
    want_k, want_v, off = _expected(k, v, k_cache, v_cache, table, lens, new, pos, freq, interleaved, magnitude, dtype)
    R.check("keys", kd, want_k, off)
    R.check("values", vd, want_v, torch.zeros_like(off))
    want, size = R.turn(q.double(), pos, freq, interleaved, magnitude) if rotary else (q.double(), None)
    bound = R.turn_bound(want, size, dtype, pos, freq) if rotary else torch.zeros_like(want)
    there = (torch.arange(L) < new[:, None])[..., None, None]
    R.check("query", turned, want * there, bound)


def test_lengths_and_pages_out_of_range_are_dropped():
    """Negative and too large table entries, positions past the table, before the sequence and counts past the batch: none of
    it is written anywhere."""
    B, L, Hkv, D, page, width, pages = 6, 8, 2, 64, 4, 3, 40
    k, v = _normal(1, B, L, Hkv, D, dtype=torch.bfloat16), _normal(2, B, L, Hkv, D, dtype=torch.bfloat16)
    k_cache, v_cache = _normal(3, pages, page, Hkv, D, dtype=torch.bfloat16), _normal(4, pages, page, Hkv, D, dtype=torch.bfloat16)
    table = torch.arange(B * width).int().view(B, width)
    table[0, 1], table[1, 1], table[1, 2] = -1, pages, 2 ** 31 - 1
    lens = torch.tensor([12, 12, 15, 5, 2 ** 31 - 1, 9]).int()       # 15, 2^31 - 1: past the table's 12; 5: three before the start
    new = torch.tensor([8, 8, 8, 8, 8, 100]).int()                   # 100: more than the batch holds
    kd, vd = k_cache.cuda(), v_cache.cuda()
    assert F.na1d_append(k.cuda(), v.cuda(), kd, vd, table.cuda(), lens.cuda(), new.cuda()) is None
    want_k, want_v, off = _expected(k, v, k_cache, v_cache, table, lens, new, None, None, False, 1.0, torch.bfloat16)
    R.check("keys", kd, want_k, off)
    R.check("values", vd, want_v, off)
    # the same with 64-bit tables and lengths
    k2, v2 = k_cache.cuda(), v_cache.cuda()
    F.na1d_append(k.cuda(), v.cuda(), k2, v2, table.long().cuda(), lens.long().cuda(), new.long().cuda())
    assert torch.equal(k2, kd) and torch.equal(v2, vd)


def test_strided_pools_and_tokens():
    """Keys and values as halves of one pool, heads first in the pages; tokens as views of a packed projection; a page table
    that is a slice of a wider one."""
    B, L, Hkv, D, page, width = 3, 11, 2, 64, 8, 4
    freq, _ = rotary_frequencies(D)
    packed = _normal(1, B, L, 2, Hkv, D, dtype=torch.bfloat16).cuda()
    pool = _normal(2, B * width, 2, Hkv, page, D, dtype=torch.bfloat16).cuda()
    k_cache, v_cache = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    before_k, before_v = k_cache.cpu(), v_cache.cpu()
    wide = torch.randperm(B * width, generator=torch.Generator().manual_seed(3)).int().view(B, width).repeat(1, 2).cuda()
    lens = torch.tensor([11, 20, 32]).int()
    F.na1d_append(packed[:, :, 0], packed[:, :, 1], k_cache, v_cache, wide[:, :width], lens.cuda(), frequencies=freq.cuda())
    new = torch.full((B,), L)
    pos = R.new_positions(lens, new, L)
    want_k, want_v, off = _expected(packed[:, :, 0].cpu(), packed[:, :, 1].cpu(), before_k, before_v, wide[:, :width].cpu(), lens, new, pos,
                                    freq, False, 1.0, torch.bfloat16)
    R.check("keys", k_cache, want_k, off)
    R.check("values", v_cache, want_v, torch.zeros_like(off))


def test_offsets_past_32_bits():
    """The last pages of a pool of 2^31 + elements."""
    page, Hkv, D = 128, 8, 128
    pages = (2 ** 31) // (page * Hkv * D) + 3
    k_cache = torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device="cuda")
    v_cache = torch.zeros_like(k_cache)
    k, v = [_normal(i, 1, 3, Hkv, D, dtype=torch.bfloat16).cuda() for i in (1, 2)]
    table = torch.tensor([[pages - 1, pages - 2]]).int().cuda()
    F.na1d_append(k, v, k_cache, v_cache, table, torch.tensor([130]).int().cuda())
    assert torch.equal(k_cache[pages - 1, 127], k[0, 0]) and torch.equal(k_cache[pages - 2, :2], k[0, 1:])
    assert torch.equal(v_cache[pages - 1, 127], v[0, 0]) and torch.equal(v_cache[pages - 2, :2], v[0, 1:])
    assert int((k_cache[:pages - 2] != 0).any()) == 0
    q = _normal(3, 1, 3, 8, D, dtype=torch.bfloat16).cuda()
    out = F.na1d_paged(q, k_cache, v_cache, table, torch.tensor([130]).int().cuda(), 2)
    near = slice(126, 130)
    want, _, bound, _ = R.attend(q.cpu().double(), torch.cat([k_cache[pages - 1], k_cache[pages - 2]])[near].cpu().double()[None],
                                 torch.cat([v_cache[pages - 1], v_cache[pages - 2]])[near].cpu().double()[None], torch.zeros(1, 1).int(),
                                 torch.tensor([4]), torch.tensor([3]), 2)
    R.check("attention", out, want, bound(torch.bfloat16))


def test_refuses_gradients_and_writes_in_place():
    k = torch.randn(1, 2, 2, 64, device="cuda", requires_grad=True)
    cache = torch.zeros(4, 4, 2, 64, device="cuda")
    table, lens = torch.arange(4).int().view(1, 4).cuda(), torch.tensor([2]).int().cuda()
    with pytest.raises(RuntimeError, match="no backward pass"):
        F.na1d_append(k, k.detach(), cache, cache.clone(), table, lens)
    version = cache._version
    with torch.no_grad():
        F.na1d_append(k, k, cache, cache.clone(), table, lens)
    assert cache._version > version                       # autograd sees that the cache was written to
    with torch.inference_mode():
        inference = torch.zeros(4, 4, 2, 64, device="cuda")
        F.na1d_append(k, k, inference, inference.clone(), table, lens)
    assert torch.equal(inference[0, :2], k[0])
    with pytest.raises(ValueError, match="adjacent"):
        F.na1d_append(k.detach(), k.detach(), torch.zeros(4, 4, 64, 2, device="cuda").transpose(2, 3), cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        F.na1d_append(k.detach(), k.detach(), cache, cache, table, lens.cpu())
    with pytest.raises(ValueError, match="dtype"):
        F.na1d_append(k.detach(), k.detach(), cache.half(), cache.half(), table, lens)


@pytest.mark.parametrize("pages,width", [(0, 2), (3, 0), (0, 0)])
def test_no_pages(pages, width):
    """Tokens without a page are dropped where no page is there at all; the query is rotated all the same."""
    k, v, q = [_normal(i, 2, 3, 2, 64, dtype=torch.float32).cuda() for i in (1, 2, 3)]
    cache = [torch.full((pages, 4, 2, 64), 7.0, device="cuda") for _ in range(2)]
    table, lens = torch.zeros(2, width, dtype=torch.int32, device="cuda"), torch.tensor([3, 5]).int().cuda()
    freq = rotary_frequencies(64)[0].cuda()
    got = F.na1d_append(k, v, *cache, table, lens, query=q, frequencies=freq)
    positions = torch.tensor([[0, 1, 2], [2, 3, 4]]).cuda()
    assert torch.equal(got, F.na1d_rotary(q, k, freq, positions)[0])
    assert all(bool((c == 7).all()) for c in cache)
    assert not bool((F.na1d_paged(q, *cache, table, lens, 3) != 0).any())
