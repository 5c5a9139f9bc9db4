"""Rotary positions against float64, with their gradients."""
import pytest
import torch

from natten_mps_b200 import functional as F, rotary_frequencies
from tests import _decoder_ref as R

pytestmark = pytest.mark.gpu


def _normal(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,B,L,Hq,Hkv,D,rotary", [
    (torch.bfloat16, 2, 33, 8, 2, 128, 128),
    (torch.bfloat16, 1, 1, 1, 1, 64, 32),
    (torch.float16, 3, 7, 6, 3, 64, 64),
    (torch.float16, 1, 5, 4, 4, 40, 24),          # half of a pair does not fill 16 bytes
    (torch.bfloat16, 2, 3, 2, 1, 33, 10),         # odd head dim: element by element
    (torch.float32, 2, 65, 4, 4, 32, 32),
    (torch.float32, 1, 9, 3, 1, 20, 2),
    (torch.float64, 2, 11, 2, 2, 16, 12),
    (torch.bfloat16, 5, 400, 16, 4, 128, 64),     # more than one token a block
])
def test_forward_and_gradients(dtype, B, L, Hq, Hkv, D, rotary, interleaved):
    freq, magnitude = rotary_frequencies(rotary, scaling="yarn", factor=4.0, original_length=512)
    q, k, dq, dk = [_normal(i, B, L, h, D, dtype=dtype) for i, h in enumerate((Hq, Hkv, Hq, Hkv))]
    pos = torch.randint(0, 100000, (B, L), generator=torch.Generator().manual_seed(9))
    qd, kd = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
    out = F.na1d_rotary(qd, kd, freq.cuda(), pos.cuda(), interleaved=interleaved, magnitude=magnitude)
    grads = torch.autograd.grad(out, [qd, kd], [dq.cuda(), dk.cuda()])
    for name, got, x, inverse in (("q", out[0], q, False), ("k", out[1], k, False), ("dq", grads[0], dq, True), ("dk", grads[1], dk, True)):
        want, size = R.turn(x.double(), pos, freq, interleaved, magnitude, inverse)
        assert got.dtype == dtype and got.is_contiguous()
        R.check(name, got, want, R.turn_bound(want, size, dtype, pos, freq))


@pytest.mark.parametrize("form", ["none", "shared", "int32", "negative", "far"])
def test_positions(form):
    B, L, D = 2, 37, 64
    freq, _ = rotary_frequencies(D)
    q, k = _normal(1, B, L, 3, D, dtype=torch.float32), _normal(2, B, L, 1, D, dtype=torch.float32)
    pos = torch.arange(L).repeat(B, 1)
    given = None
    if form == "shared":
        pos = pos * 3 + 5
        given = pos[0].cuda()
    elif form == "int32":
        given = pos.int().cuda()
    elif form == "negative":
        pos = -pos
        given = pos.cuda()
    elif form == "far":
        pos = pos + 2 ** 33                      # the angle in 64 bits keeps seven digits here
        given = pos.cuda()
    got = F.na1d_rotary(q.cuda(), k.cuda(), freq.cuda(), given)
    for a, x in zip(got, (q, k)):
        want, size = R.turn(x.double(), pos, freq)
        if form == "far":                        # float64's own angle is off by as much as the kernel's
            R.check(form, a, want, R.turn_bound(want, size, torch.float32, pos, freq) * 2)
        else:
            R.check(form, a, want, R.turn_bound(want, size, torch.float32, pos, freq))


def test_strided_inputs_and_other_streams():
    """Views of a packed projection, channels apart, an expanded batch; a stream other than the default one."""
    B, L, H, D = 2, 19, 4, 64
    freq, _ = rotary_frequencies(D)
    packed = _normal(3, B, L, 3, H, D, dtype=torch.bfloat16).cuda()
    apart = _normal(4, B, L, H, D, 2, dtype=torch.bfloat16).cuda()[..., 0]
    one = _normal(5, 1, L, H, D, dtype=torch.bfloat16).cuda().expand(B, -1, -1, -1)
    pos = torch.arange(L).repeat(B, 1)
    side = torch.cuda.Stream()
    f = freq.cuda()
    for q, k in ((packed[:, :, 0], packed[:, :, 1]), (apart, one), (one, apart)):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = F.na1d_rotary(q, k, f)
        side.synchronize()
        for a, x in zip(got, (q, k)):
            want, size = R.turn(x.cpu().double(), pos, freq)
            R.check("strided", a, want, R.turn_bound(want, size, torch.bfloat16, pos, freq))


def test_gradients_against_differences():
    freq, magnitude = rotary_frequencies(6, scaling="yarn", factor=2.0, original_length=64)
    pos = torch.tensor([[3, 1, 400], [0, 9, 77]]).cuda()
    q = torch.randn(2, 3, 2, 8, dtype=torch.float64, device="cuda", requires_grad=True)
    k = torch.randn(2, 3, 1, 8, dtype=torch.float64, device="cuda", requires_grad=True)
    for interleaved in (False, True):
        f = lambda a, b: F.na1d_rotary(a, b, freq.cuda(), pos, interleaved=interleaved, magnitude=magnitude)  # noqa: E731
        assert torch.autograd.gradcheck(f, (q, k))
        assert torch.autograd.gradgradcheck(f, (q, k))
    # an expanded query: its gradient is the sum over the copies
    one = torch.randn(1, 3, 2, 8, dtype=torch.float64, device="cuda", requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: F.na1d_rotary(a.expand(2, -1, -1, -1), k.detach(), freq.cuda(), pos)[0], (one,))


def test_one_output_unused_and_empty_batches():
    freq, _ = rotary_frequencies(64)
    f = freq.cuda()
    q, k = [torch.randn(2, 3, 2, 64, device="cuda", requires_grad=True) for _ in range(2)]
    qr, kr = F.na1d_rotary(q, k, f)
    gq, gk = torch.autograd.grad(qr.sum(), [q, k], allow_unused=True)
    assert gq.abs().sum() > 0 and (gk is None or gk.abs().sum() == 0)
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64)):
        e = torch.empty(shape, device="cuda", requires_grad=True)
        a, b = F.na1d_rotary(e, e, f)
        assert a.shape == e.shape and b.shape == e.shape
        assert torch.autograd.grad(a.sum() + b.sum(), e)[0].shape == e.shape


def test_captured_in_a_graph():
    freq, _ = rotary_frequencies(128)
    q, k, f = torch.randn(1, 64, 8, 128, device="cuda").bfloat16(), torch.randn(1, 64, 2, 128, device="cuda").bfloat16(), freq.cuda()
    pos = torch.zeros(64, dtype=torch.int64, device="cuda")
    F.na1d_rotary(q, k, f, pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = F.na1d_rotary(q, k, f, pos)
    pos.copy_(torch.arange(64) + 11)
    g.replay()
    torch.cuda.synchronize()
    for a, x in zip(out, (q, k)):
        want, size = R.turn(x.cpu().double(), torch.arange(64)[None] + 11, freq)
        R.check("graph", a, want, R.turn_bound(want, size, torch.bfloat16, torch.arange(75), freq))
