"""Operators around a decoder's cache, what needs no GPU: refusals, shape functions, frequencies, the cache's bookkeeping."""
import math

import pytest
import torch

import natten_mps_b200 as nb
from natten_mps_b200 import _cabi, functional as F, rotary_frequencies


def test_frequencies():
    f, m = rotary_frequencies(8)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    g, _ = rotary_frequencies(8, scaling="linear", factor=4.0)
    assert torch.allclose(g * 4, f, rtol=1e-15)
    n, _ = rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert n[0] == f[0] and math.isclose(n[-1] * 4, f[-1], rel_tol=1e-12)
    y, m = rotary_frequencies(128, scaling="yarn", factor=16.0, original_length=4096)
    f, _ = rotary_frequencies(128)
    ratio = f / y
    assert m == 0.1 * math.log(16.0) + 1
    turns = 4096 * f / (2 * math.pi)
    assert torch.allclose(ratio[turns > 40], torch.ones(()).double()) and torch.allclose(ratio[turns < 0.8], torch.tensor(16.0).double())
    assert bool((ratio[1:] >= ratio[:-1] - 1e-12).all())
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="cubic"),
                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="yarn"), dict(rotary_dim=2, scaling="ntk"),
                dict(rotary_dim=8, scaling="yarn", original_length=64, fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def _cache(pages=6, page=4, heads=2, dim=8, batch=2, width=3):
    return [torch.zeros(pages, page, heads, dim), torch.zeros(pages, page, heads, dim), torch.zeros(batch, width, dtype=torch.int32),
            torch.zeros(batch, dtype=torch.int32)]


def test_rotary_refusals():
    q, k, f = torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 2, 8), torch.ones(4).double()
    for args, kw in (((q[0], k, f), {}), ((q, k[:, :2], f), {}), ((q, k[..., :4], f), {}), ((q, k, torch.ones(5).double()), {}),
                     ((q, k, f[:0]), {}), ((q, k, f.half()), {}), ((q, k, f[None]), {}), ((q, k, f, torch.zeros(4).long()), {}),
                     ((q, k, f, torch.zeros(1, 3).long()), {}), ((q, k, f, torch.zeros(3)), {})):
        with pytest.raises(ValueError):
            F.na1d_rotary(*args, **kw)
    with pytest.raises(NotImplementedError):       # no kernel for CPU tensors, and no fallback
        F.na1d_rotary(q, k, f)


def test_append_refusals():
    k = torch.zeros(2, 3, 2, 8)
    kc, vc, table, lens = _cache()
    good = [k, k, kc, vc, table, lens]
    for at, bad in ((0, k[0]), (1, k[:, :2]), (2, kc[..., :4]), (3, vc[:5]), (4, table[:1]), (4, table.float()), (4, table[0]),
                    (5, lens[:1]), (5, lens.float()), (5, lens[:, None])):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            F.na1d_append(*args)
    with pytest.raises(ValueError):
        F.na1d_append(torch.zeros(2, 3, 1, 8), torch.zeros(2, 3, 1, 8), kc, vc, table, lens)      # heads
    for kw in (dict(seq_lens=lens[:1]), dict(seq_lens=lens.float()), dict(query=k[:, :1]), dict(query=k[..., :4]),
               dict(frequencies=torch.ones(5).double())):
        with pytest.raises(ValueError):
            F.na1d_append(*good, **kw)
    with pytest.raises(NotImplementedError):
        F.na1d_append(*good)


def test_attention_refusals():
    q = torch.zeros(2, 3, 4, 8)
    kc, vc, table, lens = _cache()
    good = [q, kc, vc, table, lens]
    for at, bad in ((0, q[0]), (0, torch.zeros(2, 3, 3, 8)), (0, q[..., :4]), (1, kc[:5]), (2, vc[0]), (3, table.float()), (4, lens[:1])):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            F.na1d_paged(*args)
    for args in ((0,), (-3,), (5, 0), (None, 2), (True,), ((3, 4),)):
        with pytest.raises(ValueError):
            F.na1d_paged(*good, *args)
    with pytest.raises(ValueError):
        F.na1d_paged(*good, 3, seq_lens=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(NotImplementedError):
        F.na1d_paged(*good, 3)


def test_meta_shapes():
    m = lambda t: t.to("meta")  # noqa: E731
    q, k, f = m(torch.zeros(2, 3, 4, 8)), m(torch.zeros(2, 3, 2, 8)), m(torch.ones(4).double())
    kc, vc, table, lens = [m(t) for t in _cache()]
    a, b = F.na1d_rotary(q, k, f)
    assert a.shape == q.shape and b.shape == k.shape
    assert F.na1d_append(k, k, kc, vc, table, lens, query=q).shape == q.shape
    assert F.na1d_append(k, k, kc, vc, table, lens) is None
    out, lse = F.na1d_paged(q, kc, vc, table, lens, 3, 1, None, True)
    assert out.shape == q.shape and lse.shape == q.shape[:-1] and lse.dtype == torch.float32


def test_c_abi_checks_without_a_gpu():
    L = _cabi.lib()
    r = _cabi.RotaryParams(dtype=2, batch=1, length=2, heads_q=2, heads_kv=1, dim=8, rotary_dim=8, magnitude=1.0)
    assert L.natten_rotary(None, *[None] * 5) == -1
    assert L.natten_rotary(r, *[None] * 5) == -1                  # no tensors
    r.rotary_dim = 7
    assert L.natten_rotary(r, *[None] * 5) == -1
    r.rotary_dim, r.dim = 8, 2048
    assert L.natten_rotary(r, *[None] * 5) == -2
    r.dim, r.batch = 8, 0
    assert L.natten_rotary(r, *[None] * 5) == 0                   # nothing to do
    p = _cabi.PagedParams(dtype=2, batch=1, length=2, heads_q=2, heads_kv=1, dim=8, pages=4, page_size=4, table_width=2, dilation=1, scale=1.0)
    call = lambda: L.natten_paged_fwd(p, *[None] * 6, 0, None)  # noqa: E731
    assert call() == -1
    for field, bad, code in (("page_size", 0, -1), ("heads_q", 3, -1), ("heads_kv", 2, -1), ("kernel", -1, -1), ("dilation", 0, -1),
                             ("dtype", 9, -1), ("dtype", 3, -2), ("dim", 264, -2), ("length", -1, -1)):
        was = getattr(p, field)
        if field == "heads_q":
            p.heads_kv = 2
        if field == "heads_kv":
            p.heads_q = 3
        setattr(p, field, bad)
        assert call() == code, field
        p.heads_q, p.heads_kv = 2, 1
        setattr(p, field, was)
    assert L.natten_paged_append(p, *[None] * 7) == -1
    p.batch = 0
    assert call() == 0 and L.natten_paged_append(p, *[None] * 7) == 0


def test_cache_bookkeeping():
    c = nb.PagedCache(2, 5, 4, 1, 8, 16, layers=2, dtype=torch.float32, device="cpu")
    c.extend([5, 0])
    assert c.lengths == [5, 0] and c.free_pages == 3 and c.cache_lens.tolist() == [5, 0] and c.seq_lens.tolist() == [5, 0]
    assert c.page_table.tolist() == [[0, 1, -1, -1], [-1] * 4]
    c.extend([3, 4])
    assert c.free_pages == 2 and c.page_table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]]
    before = (c.lengths, c.free_pages, c.page_table.tolist())
    with pytest.raises(RuntimeError, match="free pages"):
        c.extend([8, 1])
    with pytest.raises(ValueError, match="max_length"):
        c.extend([9, 0])
    with pytest.raises(ValueError):
        c.extend([1])
    with pytest.raises(ValueError):
        c.extend(-1)
    assert before == (c.lengths, c.free_pages, c.page_table.tolist())
    c.extend(1)
    assert c.lengths == [9, 5] and c.free_pages == 0 and c.seq_lens.tolist() == [1, 1]
    c.trim(3)                                     # of 9 tokens the last 3 start at 6: page 0 goes, page 1 stays
    assert c.page_table.tolist()[0] == [-1, 1, 3, -1] and c.page_table.tolist()[1] == [2, 4, -1, -1] and c.free_pages == 1
    c.trim(3)
    assert c.free_pages == 1
    c.reset(0)
    assert c.lengths == [0, 5] and c.free_pages == 3 and c.page_table.tolist()[0] == [-1] * 4 and c.seq_lens.tolist() == [0, 1]
    c.extend([12, 0])
    assert c.free_pages == 0 and sorted(p for row in c.page_table.tolist() for p in row if p >= 0) == [0, 1, 2, 3, 4]
    layer = c.layer(1)
    assert layer.key_cache.shape == (5, 4, 1, 8) and layer.page_table is c.page_table
    for bad in (dict(batch=0), dict(page_size=0), dict(num_pages=True)):
        with pytest.raises(ValueError):
            nb.PagedCache(**{**dict(batch=1, num_pages=1, page_size=1, num_kv_heads=1, head_dim=8, max_length=1, device="cpu"), **bad})


def test_module_refusals():
    x = torch.zeros(2, 3, 32)
    cache = nb.PagedCache(2, 4, 4, 4, 8, 8, dtype=torch.float32, device="cpu").layer()
    with pytest.raises(ValueError, match="is_causal"):
        nb.NeighborhoodAttention1D(32, 4, 3)(x, cache=cache)
    with pytest.raises(ValueError, match="is_causal"):
        nb.NeighborhoodAttention1D(32, 4, 3, stride=2, is_causal=True)(x, cache=cache)
    m = nb.NeighborhoodAttention1D(32, 4, 3, is_causal=True, rotary_dim=8)
    with pytest.raises(ValueError, match="one of the two"):
        m(x, torch.tensor([3, 3]), cache)
    with pytest.raises(ValueError, match="input shape"):
        m(x[0], cache=cache)
    with pytest.raises(ValueError, match="rotary_dim"):
        nb.NeighborhoodAttention1D(32, 4, 3, rotary_dim=10)
    assert not any("freq" in name for name in m.state_dict())      # interchangeable with modules without positions


def test_frequencies_first_placed_in_inference_mode_serve_training():
    m = nb.NeighborhoodAttention1D(32, 4, 3, is_causal=True, rotary_dim=8)
    with torch.inference_mode():
        m._rotary.on(torch.device("meta"))
    assert not m._rotary.on(torch.device("meta")).is_inference()
