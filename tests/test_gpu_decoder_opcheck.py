"""``torch.library.opcheck`` and ``torch.compile`` of the operators around a decoder's cache."""
import pytest
import torch

from natten_mps_b200 import functional as F, rotary_frequencies

pytestmark = pytest.mark.gpu


def _cache(dtype=torch.float32):
    return [torch.randn(6, 4, 2, 32, device="cuda", dtype=dtype), torch.randn(6, 4, 2, 32, device="cuda", dtype=dtype),
            torch.tensor([[0, 3, 5], [1, 2, 4]], dtype=torch.int32, device="cuda"), torch.tensor([9, 12], dtype=torch.int32, device="cuda")]


@pytest.mark.parametrize("op", ["rotary", "append", "paged"])
def test_opcheck(op):
    ops = torch.ops.natten_b200
    q, k = torch.randn(2, 3, 4, 32, device="cuda"), torch.randn(2, 3, 2, 32, device="cuda")
    freq = rotary_frequencies(16)[0].cuda()
    utils = ("test_schema", "test_faketensor")
    if op == "rotary":
        q.requires_grad_(True)
        torch.library.opcheck(ops.na1d_rotary.default, (q, k, freq, None, True, 1.0, False), test_utils=utils + ("test_autograd_registration",))
    elif op == "append":
        torch.library.opcheck(ops.na1d_append.default, (k, k.clone(), *_cache(), None, q, freq, False, 1.0), test_utils=utils)
    else:
        torch.library.opcheck(ops.na1d_paged.default, (q, *_cache(), None, 5, 1, 0.25), test_utils=utils)


def test_under_the_compiler():
    """The operators as nodes of a compiled graph give what they give eagerly (the cache written in place)."""
    freq = rotary_frequencies(16)[0].cuda()
    q, k = torch.randn(2, 3, 4, 32, device="cuda"), torch.randn(2, 3, 2, 32, device="cuda")

    def step(q, k, kc, vc, table, lens):
        turned = F.na1d_append(k, k * 2, kc, vc, table, lens, query=q, frequencies=freq)
        return F.na1d_paged(turned, kc, vc, table, lens, 5)

    a, b = _cache(), None
    b = [t.clone() for t in a]
    with torch.no_grad():
        want = step(q, k, *a)
        got = torch.compile(step, backend="aot_eager")(q, k, *b)
    assert torch.equal(got, want) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    turn = torch.compile(lambda x, y: F.na1d_rotary(x, y, freq), backend="aot_eager")
    x, y = [t.clone().requires_grad_(True) for t in (q, k)]
    out = turn(x, y)
    eager = F.na1d_rotary(q, k, freq)
    assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
    got = torch.autograd.grad(out[0].sum() + (out[1] * 3).sum(), [x, y])
    x2, y2 = [t.clone().requires_grad_(True) for t in (q, k)]
    ref = F.na1d_rotary(x2, y2, freq)
    want = torch.autograd.grad(ref[0].sum() + (ref[1] * 3).sum(), [x2, y2])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refuses_sizes_past_31_bits_and_caches_that_overlap_themselves():
    long = torch.zeros(1, 1, 1, 64, device="cuda").expand(1, 2 ** 32 + 5, 1, 64)         # refused before anything is made of it
    cache = torch.zeros(4, 4, 1, 64, device="cuda")
    table, lens, freq = torch.arange(4).int().view(1, 4).cuda(), torch.tensor([2]).int().cuda(), torch.ones(32).double().cuda()
    for call in (lambda: F.na1d_rotary(long, long, freq), lambda: F.na1d_append(long, long, cache, cache.clone(), table, lens),
                 lambda: F.na1d_paged(long, cache, cache, table, lens, 3)):
        with pytest.raises(ValueError, match="not supported"):
            call()
    k = torch.zeros(1, 2, 1, 64, device="cuda")
    with pytest.raises(RuntimeError):
        F.na1d_append(k, k, cache[:1].expand(4, 4, 1, 64), cache, table, lens)
