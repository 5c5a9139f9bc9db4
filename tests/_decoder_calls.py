"""Calls of ``torch.ops.natten_b200`` around a decoder's cache whose shapes do not fit each other."""
import torch


def misfits(device):
    """``(name, call)`` of each; small tensors, and none of the calls may launch anything."""
    ops = torch.ops.natten_b200
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    q, k, f = z(2, 6, 4, 8), z(2, 6, 2, 8), z(4, dtype=torch.float64)
    kc, table, lens = z(6, 4, 2, 8), z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32)
    turned = lambda a, b, c=f: lambda: ops.na1d_rotary(a, b, c, None, False, 1.0, False)  # noqa: E731
    appended = lambda key=k, value=k, cache=kc, pages=table, n=lens, query=None, c=None: lambda: ops.na1d_append(  # noqa: E731
        key, value, cache, cache.clone(), pages, n, None, query, c, False, 1.0)
    attended = lambda query=q, cache=kc, pages=table, n=lens, new=None: lambda: ops.na1d_paged(  # noqa: E731
        query, cache, cache, pages, n, new, 3, 1, 1.0)
    return [
        ("rotary: batch of key", turned(q, k[:1])), ("rotary: tokens of key", turned(q, k[:, :2])),
        ("rotary: head dim of key", turned(q, k[..., :4])), ("rotary: rank of key", turned(q, k[0])), ("rotary: rank of query", turned(q[0], k)),
        ("rotary: frequencies", turned(q, k, z(5, dtype=torch.float64))), ("rotary: rank of frequencies", turned(q, k, f[None])),
        ("append: batch of query", appended(query=q[:1])), ("append: tokens of query", appended(query=q[:, :5])),
        ("append: head dim of query", appended(query=q[..., :4])), ("append: rank of query", appended(query=q[0])),
        ("append: frequencies", appended(c=z(5, dtype=torch.float64))), ("append: value", appended(value=k[:, :5])),
        ("append: heads of cache", appended(cache=z(6, 4, 3, 8))), ("append: head dim of cache", appended(cache=z(6, 4, 2, 4))),
        ("append: table", appended(pages=table[:1])), ("append: lengths", appended(n=lens[:1])),
        ("paged: rank of query", attended(query=q[0])), ("paged: head dim", attended(query=q[..., :4])),
        ("paged: table", attended(pages=table[:1])), ("paged: lengths", attended(n=lens[:1])), ("paged: new", attended(new=lens[:1])),
    ]
