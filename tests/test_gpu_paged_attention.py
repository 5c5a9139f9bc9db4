"""Attention of new tokens over a paged cache against float64: windows, dilation, grouped heads, odd pages and head dims,
lengths from nothing to several row tiles, masked places that hold NaN."""
import math

import pytest
import torch

from natten_mps_b200 import _cabi, functional as F
from tests import _decoder_ref as R

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _normal(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _problem(dtype, lens, new, L, Hq, Hkv, D, page, seed=0, poison=True):
    """Caches whose slots hold NaN wherever no token is."""
    B = len(lens)
    width = max(1, -(-max(max(lens), 1) // page))
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(seed)).int().view(B, width)
    k_cache, v_cache = [_normal(seed + i, B * width, page, Hkv, D, dtype=dtype) for i in (1, 2)]
    if poison:
        for b, n in enumerate(lens):
            for p in range(max(n, 0), width * page):
                k_cache[table[b, p // page], p % page] = math.nan
                v_cache[table[b, p // page], p % page] = math.nan
    return _normal(seed + 3, B, L, Hq, D, dtype=dtype), k_cache, v_cache, table, torch.tensor(lens).int(), torch.tensor(new).int()


def _check(problem, kernel, dilation, scale=None, dtype=None, place=lambda t: t.cuda()):
    q, k_cache, v_cache, table, lens, new = problem
    out, lse = F.na1d_paged(place(q), place(k_cache), place(v_cache), place(table), place(lens), kernel, dilation, scale, True,
                            seq_lens=place(new))
    # only keys that are seen enter the result: a NaN that is seen has to show, one that is not must not
    want, want_lse, bound, lse_bound = R.attend(q.double(), k_cache.double(), v_cache.double(), table, lens, new, kernel, dilation, scale)
    assert out.dtype == q.dtype and lse.dtype == F32 and out.is_contiguous()
    R.check("out", out, want, bound(q.dtype))
    R.check("lse", lse, want_lse, lse_bound)
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lens,new,L,Hq,Hkv,D,page,kernel,dilation", [
    ([1, 5, 40], [1, 1, 1], 1, 4, 2, 64, 16, None, 1),
    ([300, 17, 129], [1, 1, 1], 1, 16, 4, 128, 16, None, 1),
    ([300, 17, 129], [1, 1, 1], 1, 8, 8, 128, 24, 33, 1),
    ([300, 17, 129], [1, 0, 1], 1, 6, 2, 64, 7, 33, 3),
    ([90, 33, 8], [4, 4, 2], 4, 8, 2, 64, 16, 15, 1),
    ([90, 33, 8], [5, 3, 5], 5, 3, 1, 32, 8, None, 1),
    ([70, 64], [64, 33], 64, 4, 2, 64, 16, 17, 1),
    ([150, 70], [70, 70], 70, 8, 2, 128, 16, None, 1),
    ([150, 70], [70, 11], 70, 3, 3, 128, 10, 40, 2),
    ([200], [137], 137, 2, 1, 64, 64, 9, 4),
    ([37], [9], 9, 2, 2, 64, 5, 3, 30),               # windows shorter than the dilation reaches; classes of no query
], ids=str)
def test_against_float64(dtype, lens, new, L, Hq, Hkv, D, page, kernel, dilation):
    _check(_problem(dtype, lens, new, L, Hq, Hkv, D, page), kernel, dilation)


@pytest.mark.parametrize("dtype,D", [(BF16, 8), (BF16, 40), (F16, 72), (BF16, 80), (F16, 96), (BF16, 112), (BF16, 160), (F16, 256),
                                     (BF16, 20), (F16, 5), (F32, 40), (F32, 6), (F32, 128), (F32, 200), (F32, 256)])
def test_head_dims(dtype, D):
    _check(_problem(dtype, [50, 21], [1, 1], 1, 4, 2, D, 8), None, 1)
    _check(_problem(dtype, [50, 45], [40, 23], 40, 4, 2, D, 8), 19, 1)


@pytest.mark.parametrize("Hq,Hkv,L", [(40, 1, 1), (64, 1, 2), (5, 1, 7), (7, 7, 3), (96, 2, 3), (12, 4, 33)])
def test_groups(Hq, Hkv, L):
    """Groups larger than a row tile, and groups that no tile holds a whole number of."""
    _check(_problem(BF16, [61, 40], [L, max(1, L - 1)], L, Hq, Hkv, 64, 16), None, 1)
    _check(_problem(BF16, [61, 40], [L, L], L, Hq, Hkv, 128, 16), 12, 2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_see_nothing(dtype):
    """Empty sequences, no new tokens, more new tokens than tokens, lengths past the table, pages that are not there."""
    q, k_cache, v_cache, table, lens, new = _problem(dtype, [0, 12, 3, 30, 30, 9], [0, 0, 6, 6, 6, 6], 6, 4, 2, 64, 4)
    table[3, :] = -1                                  # nothing there
    table[4, 3:6] = torch.tensor([10 ** 6, -5, 2 ** 31 - 1])         # holes
    table[5, 2] = -1                                  # the last page, with the newest token on it
    lens[1] = -7
    out, lse = _check((q, k_cache, v_cache, table, lens, new), None, 1)
    assert int(out[0].abs().sum()) == 0 and bool((lse[3] == -math.inf).all())
    lens[3], lens[4] = 2 ** 31 - 1, 41                # the table ends before the sequence does
    _check((q, k_cache, v_cache, table, lens, new), 5, 1)
    _check((q, k_cache, v_cache, table, lens, new), 5, 3)


@pytest.mark.parametrize("L", [1, 40])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_table_no_pages(dtype, L):
    q = torch.randn(2, L, 4, 64, device="cuda").to(dtype)
    lens = torch.full((2,), 100, dtype=torch.int32, device="cuda")
    for pages, width in ((0, 0), (0, 5), (3, 0)):
        cache = torch.zeros(pages, 16, 2, 64, device="cuda", dtype=dtype)
        out, lse = F.na1d_paged(q, cache, cache, torch.zeros(2, width, dtype=torch.int32, device="cuda"), lens, return_lse=True)
        assert int(out.abs().sum()) == 0 and bool((lse == -math.inf).all())
    for shape in ((0, L), (2, 0)):
        e = torch.empty(*shape, 4, 64, device="cuda", dtype=dtype)
        out = F.na1d_paged(e, cache, cache, torch.zeros(shape[0], 1, dtype=torch.int32, device="cuda"), lens[:shape[0]])
        assert out.shape == e.shape


def test_long_caches_are_shared_between_ctas():
    """Few sequences and many keys: parts of a unit are computed apart and joined; the same twice gives the same bits."""
    for L, kernel in ((1, None), (1, 2500), (3, None), (48, None)):
        p = _problem(BF16, [4100, 2777], [L, L], L, 4, 1, 64, 16, poison=False)
        a, la = _check(p, kernel, 1)
        b, lb = _check(p, kernel, 1)
        assert torch.equal(a, b) and torch.equal(la, lb)
    _check(_problem(F32, [1100, 777], [2, 2], 2, 2, 1, 32, 16, poison=False), None, 1)


@pytest.mark.parametrize("dtype,L", [(BF16, 1), (F16, 1), (BF16, 70), (F16, 70), (F32, 9)])
def test_large_scores(dtype, L):
    """Scores of some hundreds that grow and fall along the keys: running maxima have to follow."""
    for sign in (1, -1):
        q, k_cache, v_cache, table, lens, new = _problem(dtype, [700, 350], [L, L], L, 4, 2, 64, 16, poison=False)
        ramp = torch.linspace(0, 6, table.shape[1] * 16) * sign
        for b in range(2):
            for n in range(table.shape[1]):
                k_cache[table[b, n]] = (k_cache[table[b, n]].float() + ramp[16 * n:16 * n + 16, None, None]).to(dtype)
        q = (q.float() + 3).to(dtype)
        _check((q, k_cache, v_cache, table, lens, new), None, 1)


@pytest.mark.parametrize("L", [1, 33])
def test_strided_tensors(L):
    """Queries as a view of a packed projection; caches as halves of one pool with the heads first; a slice of a wider table."""
    q, k_cache, v_cache, table, lens, new = _problem(BF16, [61, 40], [L, L], L, 4, 2, 64, 16, poison=False)
    packed = torch.stack([q, q + 1, q - 1], dim=2).cuda()[:, :, 0]
    pool = torch.stack([k_cache, v_cache], dim=1).transpose(2, 3).contiguous().cuda().transpose(2, 3)
    wide = torch.cat([table, table], dim=1).cuda()[:, :table.shape[1]]
    got = F.na1d_paged(packed, pool[:, 0], pool[:, 1], wide, lens.cuda(), 20)
    assert torch.equal(got, F.na1d_paged(q.cuda(), k_cache.cuda(), v_cache.cuda(), table.cuda(), lens.cuda(), 20))
    want, _, bound, _ = R.attend(q.double(), k_cache.double(), v_cache.double(), table, lens, new, 20)
    R.check("strided", got, want, bound(BF16))
    # rows that do not start on 16-byte boundaries
    odd = torch.empty(2 * L * 4 * 64 + 1, dtype=BF16, device="cuda")[1:].view(2, L, 4, 64).copy_(q)
    R.check("misaligned", F.na1d_paged(odd, k_cache.cuda(), v_cache.cuda(), table.cuda(), lens.cuda(), 20), want, bound(BF16))
    shifted = torch.empty(k_cache.numel() + 1, dtype=BF16, device="cuda")[1:].view(k_cache.shape).copy_(k_cache)
    R.check("misaligned cache", F.na1d_paged(q.cuda(), shifted, v_cache.cuda(), table.cuda(), lens.cuda(), 20), want, bound(BF16))


@pytest.mark.parametrize("L", [1, 70])
def test_streams_and_graphs(L):
    """Another stream than the default one, and two captured graphs replayed at the same time."""
    p = _problem(BF16, [1500, 800], [L, L], L, 4, 1, 64, 16, poison=False)
    q, k_cache, v_cache, table, lens, new = [t.cuda() for t in p]
    want = F.na1d_paged(q, k_cache, v_cache, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.na1d_paged(q, k_cache, v_cache, table, lens)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs, queries = [], [], [q, (q * 2).contiguous()]
    for x in queries:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F.na1d_paged(x, k_cache, v_cache, table, lens))
        graphs.append(g)
    other = torch.cuda.Stream()
    for _ in range(5):
        side.wait_stream(torch.cuda.current_stream())
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], F.na1d_paged(queries[1], k_cache, v_cache, table, lens))
    # lengths are read when the graph runs
    lens.copy_(torch.tensor([L + 3, L]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], F.na1d_paged(q, k_cache, v_cache, table, lens))


def test_refusals():
    q, k_cache, v_cache, table, lens, new = [t.cuda() for t in _problem(BF16, [20], [2], 2, 4, 2, 64, 16)]
    with pytest.raises(RuntimeError, match="no backward pass"):
        F.na1d_paged(q.requires_grad_(True), k_cache, v_cache, table, lens)
    q = q.detach()
    with pytest.raises(ValueError, match="dtype"):
        F.na1d_paged(q.float(), k_cache, v_cache, table, lens)
    with pytest.raises(NotImplementedError):
        F.na1d_paged(q.double(), k_cache.double(), v_cache.double(), table, lens)
    with pytest.raises(NotImplementedError):
        F.na1d_paged(*[torch.zeros(1, 1, 2, 264, device="cuda") for _ in range(3)], table, lens)
    with pytest.raises(ValueError, match="adjacent"):
        F.na1d_paged(q, torch.zeros(2, 16, 64, 2, device="cuda", dtype=BF16).transpose(2, 3), v_cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        F.na1d_paged(q, k_cache, v_cache, table.cpu(), lens)


def test_equals_attention_on_the_whole_sequence():
    """A cache that holds a whole sequence: the same windows as na1d."""
    L, Hq, Hkv, D, page = 157, 4, 2, 64, 16
    q, k, v = [_normal(i, 1, L, h, D, dtype=F32).cuda() for i, h in enumerate((Hq, Hkv, Hkv))]
    pages = -(-L // page)
    caches = [torch.zeros(pages, page, Hkv, D, device="cuda") for _ in range(2)]
    table, lens = torch.arange(pages).flip(0).int().view(1, -1).cuda(), torch.tensor([L]).int().cuda()
    F.na1d_append(k, v, *caches, table, lens)
    for kernel, dilation in ((11, 1), (11, 5), (31, 2), (1, 1)):
        want, want_lse = F.na1d(q, k, v, kernel, dilation=dilation, is_causal=True, return_lse=True)
        for rows in (L, 1, 40):
            got, lse = F.na1d_paged(q[:, L - rows:], *caches, table, lens, kernel, dilation, return_lse=True)
            assert (got - want[:, L - rows:]).abs().max() <= 1e-5 and (lse - want_lse[:, L - rows:]).abs().max() <= 1e-5


@pytest.mark.parametrize("L,group", [(70, 4), (40, 2)], ids=["rows", "split_keys"])
def test_wait_that_runs_out_is_reported_and_recoverable(L, group):
    """The queries' barrier never fills (made on the host): the kernel gives up, says so, and the next call works again."""
    q, k_cache, v_cache, table, lens, new = [t.cuda() for t in _problem(BF16, [300, 200], [L, L], L, 2 * group, 2, 64, 16, poison=False)]
    call = lambda: F.na1d_paged(q, k_cache, v_cache, table, lens)  # noqa: E731
    try:
        want = call()
        assert _cabi.last_path() == "tcgen05"
        _cabi.lib().natten_debug_wait(400_000, 1)
        call()
        torch.cuda.synchronize()
        assert _cabi.device_status() == -4
        _cabi.lib().natten_debug_wait(0, 0)
        with pytest.raises(RuntimeError, match="bounded wait"):
            call()
        _cabi.clear_status()
        got = call()
        torch.cuda.synchronize()
        assert _cabi.device_status() == 0 and torch.equal(got, want)
    finally:
        _cabi.lib().natten_debug_wait(0, 0)
        _cabi.clear_status()


def test_paths():
    """Which kernels serve a call: rows a class, type, alignment, and the testing flags."""
    def path(dtype, L, Hq, Hkv, D, kernel=None, dilation=1):
        q, k_cache, v_cache, table, lens, new = [t.cuda() for t in _problem(dtype, [100], [L], L, Hq, Hkv, D, 16, poison=False)]
        F.na1d_paged(q, k_cache, v_cache, table, lens, kernel, dilation)
        return _cabi.last_path()

    assert path(BF16, 1, 16, 4, 128) == "warp" and path(F16, 100, 8, 2, 128) == "tcgen05" and path(BF16, 50, 4, 2, 64) == "tcgen05"
    assert path(BF16, 50, 4, 2, 96) == "warp" and path(F32, 1, 4, 2, 64) == "simt" and path(BF16, 1, 4, 2, 20) == "simt"
    assert path(BF16, 64, 2, 2, 64, 5, 64) == "warp"                 # a row a class
    try:
        _cabi.set_force("simt")
        assert path(BF16, 100, 8, 2, 128) == "simt"
        _cabi.set_force("tc")
        with pytest.raises(NotImplementedError):
            path(BF16, 1, 16, 4, 128)
    finally:
        _cabi.set_force(None)


@pytest.mark.parametrize("kernel", [None, 150])
@pytest.mark.parametrize("page,D", [(16, 64), (64, 128), (32, 128), (24, 64)])
@pytest.mark.parametrize("L,Hq,Hkv", [(1, 4, 2), (70, 8, 2), (40, 4, 2)], ids=["warp", "rows", "split_keys"])
def test_missing_pages(L, Hq, Hkv, page, D, kernel):
    """Holes in the page table and slots that no token was written to, NaN in all of them, in the middle of tiles."""
    q, k_cache, v_cache, table, lens, new = _problem(BF16, [700, 333], [L, L - L // 3], L, Hq, Hkv, D, page)
    for b, slots in ((0, (0, 3, 5)), (1, (1, table.shape[1] - 1, 333 // page))):
        for n in slots:
            k_cache[table[b, n]] = math.nan
            v_cache[table[b, n]] = math.nan
            table[b, n] = (-1, 10 ** 9)[n % 2]
    out, _ = _check((q, k_cache, v_cache, table, lens, new), kernel, 1)
    assert not bool(out.isnan().any())


@pytest.mark.parametrize("lens,new,L,Hq,Hkv,D,page,kernel,dilation", [
    ([700], [300], 300, 8, 2, 64, 16, 40, 1),          # several row tiles a sequence, windows shorter than a tile of keys
    ([520, 300], [300, 171], 300, 4, 1, 128, 64, None, 1),
    ([90, 333], [70, 70], 70, 12, 4, 64, 16, None, 1),  # a group that no row tile holds a whole number of
    ([333, 90], [70, 61], 70, 6, 2, 128, 24, 100, 1),
    ([400], [200], 200, 4, 2, 64, 32, 300, 2),
], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_several_row_tiles(dtype, lens, new, L, Hq, Hkv, D, page, kernel, dilation):
    _check(_problem(dtype, lens, new, L, Hq, Hkv, D, page), kernel, dilation)
    assert _cabi.last_path() == "tcgen05"


@pytest.mark.parametrize("dtype,L", [(BF16, 1), (BF16, 40), (BF16, 70), (F32, 3)])
def test_what_is_not_finite_shows(dtype, L):
    """A NaN or Inf in a key or value that the newest query sees reaches it; sequences and heads next to it stay as they were."""
    for tensor, value in ((1, math.nan), (2, math.nan), (2, math.inf)):
        p = list(_problem(dtype, [300, 200], [L, L], L, 4, 2, 64, 16, poison=False))
        q, k_cache, v_cache, table, lens, new = p
        clean = F.na1d_paged(*[t.cuda() for t in (q, k_cache, v_cache, table, lens)], return_lse=False)
        p[tensor][table[0, 3], 5, 1] = value             # sequence 0, position 53, head 1
        out = F.na1d_paged(*[t.cuda() for t in (q, p[1], p[2], table, lens)])
        assert not bool(torch.isfinite(out[0, -1, 2:]).any())
        assert torch.equal(out[1], clean[1]) and torch.equal(out[0, :, :2], clean[0, :, :2])
