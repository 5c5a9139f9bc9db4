"""Rotary positions, cache and attention together, as a decoder runs them."""
import pytest
import torch

import natten_mps_b200 as nb
from natten_mps_b200 import functional as F

pytestmark = pytest.mark.gpu


def _module(dtype, dim=64, heads=4, kv=2, kernel=21, dilation=1, **kw):
    torch.manual_seed(3)
    m = nb.NeighborhoodAttention1D(dim * heads, heads, kernel, dilation=dilation, is_causal=True, num_kv_heads=kv, **kw)
    return m.to(device="cuda", dtype=dtype)


# Float32: the same products, summed in another order (1e-5 of values of size one).  16 bits: projections, keys and outputs are
# rounded at the same places, the attention's weights and sums elsewhere: a few half steps of values of size one.
TOL = {torch.float32: 2e-5, torch.bfloat16: 2e-2, torch.float16: 3e-3}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [{}, dict(rotary_dim=64), dict(rotary_dim=32, rotary_interleaved=True, dilation=3),
                                dict(rotary_dim=64, rotary_scaling=dict(scaling="yarn", factor=4.0, original_length=32))], ids=str)
def test_prompt_chunks_and_steps_equal_the_whole_sequence(dtype, kw):
    B, L = 2, 150
    m = _module(dtype, **kw)
    x = torch.randn(B, L, m.embed_dim, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    cache = nb.PagedCache(B, 40, 8, m.num_kv_heads, m.head_dim, 160, dtype=dtype)
    with torch.no_grad():
        want = m(x)
        at = 0
        for n in (90, 37, 1, 1, 5, 1, 15):
            cache.extend(n)
            got = m(x[:, at:at + n], cache=cache.layer())
            err = (got - want[:, at:at + n]).abs().max().item()
            assert err <= TOL[dtype] * max(1.0, want.abs().max().item()), (at, n, err)
            at += n
            # pages that every window has passed go back
            cache.trim((m.kernel_size[0] - 1) * m.dilation[0] + 1)
    assert at == L and cache.free_pages > 0


def test_ragged_batch_and_captured_step():
    """Prompts of different lengths in one padded call, then steps replayed from a captured graph."""
    m = _module(torch.bfloat16, rotary_dim=64)
    prompts, steps = [33, 21, 50], 4
    xs = [torch.randn(1, n + steps, m.embed_dim, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i, n in enumerate(prompts)]
    cache = nb.PagedCache(3, 32, 8, m.num_kv_heads, m.head_dim, 64)
    with torch.no_grad():
        want = [m(x) for x in xs]
        padded = torch.zeros(3, max(prompts), m.embed_dim, device="cuda", dtype=torch.bfloat16)
        for b, n in enumerate(prompts):
            padded[b, :n] = xs[b][0, :n]
        cache.extend(prompts)
        got = m(padded, cache=cache.layer())
        for b, n in enumerate(prompts):
            assert (got[b, :n] - want[b][0, :n]).abs().max().item() <= 2e-2
        x = torch.zeros(3, 1, m.embed_dim, device="cuda", dtype=torch.bfloat16)
        graph = None
        for s in range(steps):
            cache.extend(1)
            for b, n in enumerate(prompts):
                x[b, 0] = xs[b][0, n + s]
            if graph is None:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    m(x, cache=cache.layer())          # warm-up; writes the same slots again
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    y = m(x, cache=cache.layer())
            graph.replay()
            for b, n in enumerate(prompts):
                assert (y[b, 0] - want[b][0, n + s]).abs().max().item() <= 2e-2


def test_training_with_positions():
    """Gradients of the module with rotary positions against the composition of its parts in float64 differences."""
    m = _module(torch.float64, dim=8, heads=2, kv=1, kernel=3, rotary_dim=6, rotary_interleaved=True)
    x = torch.randn(1, 7, m.embed_dim, dtype=torch.float64, device="cuda", requires_grad=True)
    assert torch.autograd.gradcheck(m, (x,), atol=1e-6)
    freq, _ = nb.rotary_frequencies(6)
    q, k, v = m._project(x)
    q, k = F.na1d_rotary(q, k, freq.cuda(), interleaved=True)
    out = F.na1d(q, k, v, 3, is_causal=True, scale=m.scale)
    want = m.proj(out.flatten(2))
    assert (m(x) - want).abs().max().item() <= 1e-12
    plain = _module(torch.float64, dim=8, heads=2, kv=1, kernel=3)
    assert (plain(x) - m(x)).abs().max().item() > 1e-3


def test_cache_needs_no_grad():
    m = _module(torch.bfloat16)
    cache = nb.PagedCache(1, 4, 8, m.num_kv_heads, m.head_dim, 16)
    cache.extend(2)
    x = torch.zeros(1, 2, m.embed_dim, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no backward pass"):
        m(x, cache=cache.layer())


def test_lse_merges_with_other_keys():
    """The log-sum-exp is what merge_attentions takes: a window of the cache and the rest of it make the whole."""
    B, L, n, Hq, Hkv, D = 1, 2, 60, 4, 2, 64
    g = torch.Generator().manual_seed(0)
    q, kc, vc = [torch.randn(*s, generator=g).cuda() for s in ((B, L, Hq, D), (8, 8, Hkv, D), (8, 8, Hkv, D))]
    table, lens = torch.arange(8).int().view(1, 8).cuda(), torch.tensor([n]).int().cuda()
    whole = F.na1d_paged(q[:, :1], kc, vc, table, lens - 1, return_lse=False, seq_lens=torch.ones(1, dtype=torch.int32, device="cuda"))
    near = F.na1d_paged(q[:, :1], kc, vc, table, lens - 1, 20, return_lse=True, seq_lens=torch.ones(1, dtype=torch.int32, device="cuda"))
    far = F.na1d_paged(q[:, :1], kc, vc, table, lens - 1 - 20, return_lse=True, seq_lens=torch.ones(1, dtype=torch.int32, device="cuda"))
    merged, _ = nb.merge_attentions([near[0], far[0]], [near[1], far[1]])
    assert (merged - whole).abs().max().item() <= 1e-5
