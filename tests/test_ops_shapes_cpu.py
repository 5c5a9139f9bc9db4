"""The CUDA kernels of ``torch.ops.natten_b200`` refuse shapes that do not fit each other.  They are called with CPU tensors past
the dispatcher: shapes come first, then the device, so nothing is launched, and a call whose shapes fit gets as far as the device."""
import pytest
import torch

import natten_mps_b200  # noqa: F401  (registers the operators)
from natten_mps_b200 import functional  # noqa: F401

_CUDA = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)
z = torch.zeros
Q, K, V, VD = z(2, 5, 4, 8), z(2, 5, 2, 8), z(2, 5, 2, 8), z(2, 5, 2, 6)
EK, LENS = z(2, 3, 2, 8), torch.tensor([5, 4], dtype=torch.int32)
OUT, LSE, ATTN, RPB = z(2, 5, 4, 8), z(2, 5, 4), z(2, 5, 4, 3), z(4, 5)
GEO = ([3], [1], [1], [False])


def _fused(q=Q, k=K, v=V, ek=None, ev=None, lens=None, geo=GEO):
    return "na_fused", (q, k, v, ek, ev, lens, *geo, 1.0)


def _fused_bwd(q=Q, k=K, v=V, ek=None, ev=None, lens=None, out=OUT, lse=LSE, dout=OUT, dlse=None, geo=GEO):
    return "na_fused_bwd", (q, k, v, ek, ev, lens, out, lse, dout, dlse, *geo, 1.0)


def _qk(q=Q, k=K, ks=(3,), dil=(1,), st=(1,)):
    return "na_qk", (q, k, list(ks), list(dil), list(st), [False], None)


def _qk_bwd(d=ATTN, q=Q, k=K):
    return "na_qk_bwd", (d, q, k, [3], [1], [1], [False], None)


def _rpb(q=Q, k=Q, rpb=RPB):
    return "na_qk_rpb", (q, k, rpb, [3], [1], None)


def _rpb_bwd(d=ATTN, q=Q, k=Q, shape=(4, 5)):
    return "na_qk_rpb_bwd", (d, q, k, list(shape), [3], [1], None)


def _av(attn=ATTN, v=V):
    return "na_av", (attn, v, [3], [1], [1], [False])


def _av_bwd(dout=OUT, attn=ATTN, v=V):
    return "na_av_bwd", (dout, attn, v, [3], [1], [1], [False])


FIT = [_fused(), _fused(v=VD), _fused(ek=EK, ev=EK, lens=LENS), _fused(geo=([3], [2], [1], [True])), _fused_bwd(), _fused_bwd(dlse=LSE),
       _fused_bwd(ek=EK, ev=EK, lens=LENS), _qk(), _qk(st=(2,)), _qk_bwd(), _rpb(), _rpb_bwd(), _av(), _av_bwd()]
MISFIT = [
    _fused(k=K[:1]), _fused(k=K[:, :4]), _fused(k=K[..., :4]), _fused(k=K[0]), _fused(v=V[:, :4]), _fused(v=V[:1]), _fused(v=V[:, :, :1]),
    _fused(ek=EK), _fused(ek=EK, ev=EK[:, :2]), _fused(ek=EK[:1], ev=EK[:1]), _fused(ek=EK[:, :, :1], ev=EK), _fused(ek=EK[..., :4], ev=EK),
    _fused(geo=([3], [0], [1], [False])), _fused(geo=([0], [1], [1], [False])), _fused(geo=([3], [1], [-1], [False])),
    _fused(geo=([3, 3], [1], [1], [False])), _fused(q=Q[0]),
    _fused_bwd(k=K[:, :4]), _fused_bwd(v=V[:1]), _fused_bwd(out=OUT[:, :4]), _fused_bwd(dout=OUT[:, :, :2]), _fused_bwd(lse=LSE[:1]),
    _fused_bwd(dlse=LSE[..., :2]), _fused_bwd(out=OUT[..., :4]), _fused_bwd(geo=([3], [0], [1], [False])), _fused_bwd(ek=EK),
    _qk(k=K[:1]), _qk(k=K[:, :4]), _qk(k=K[..., :4]), _qk(st=(0,)), _qk(ks=(2 ** 32 + 3,)),
    _qk_bwd(d=ATTN[:, :4]), _qk_bwd(d=ATTN[..., :2]), _qk_bwd(k=K[:, :4]),
    _rpb(k=Q[:1]), _rpb(rpb=RPB[:2]), _rpb(rpb=RPB[:, :4]), _rpb(rpb=RPB[0]), _rpb_bwd(shape=(4, 4)), _rpb_bwd(d=ATTN[..., :2]), _rpb_bwd(k=Q[:1]),
    _av(attn=ATTN[:1]), _av(attn=ATTN[:, :4]), _av(attn=ATTN[..., :2]), _av(v=V[:, :4]),
    _av_bwd(dout=OUT[:, :4]), _av_bwd(dout=OUT[..., :4]), _av_bwd(attn=ATTN[..., :2]), _av_bwd(v=V[:1]),
]


def _call(name, args):
    return getattr(torch.ops.natten_b200, name).default.redispatch(_CUDA, *args)


@pytest.mark.parametrize("name,args", MISFIT, ids=[f"{n}-{i}" for i, (n, _) in enumerate(MISFIT)])
def test_what_does_not_fit_is_refused(name, args):
    with pytest.raises(ValueError, match="natten_b200"):
        _call(name, args)


@pytest.mark.parametrize("name,args", FIT, ids=[f"{n}-{i}" for i, (n, _) in enumerate(FIT)])
def test_what_fits_gets_to_the_device(name, args):
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _call(name, args)
