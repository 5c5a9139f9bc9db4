"""What the operators around a decoder's cache are measured on: rotary positions, the append to a paged cache and the
attention of new tokens over it.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` builds what a program has
in hand before a call, ``run`` makes one pass, ``work`` counts the bytes and operations a pass cannot do without and
``exact`` gives the results in 64 bits.  With ``own`` set ``run`` calls the package's operators; without it computes
the same in elementary torch operations.

A case is a flat dict:

    op        rotary   positions of queries and keys              append   new tokens into a paged cache
              paged    attention of new tokens over the cache
    train     (rotary) forward and backward, or forward only
    dtype     float32 | float16 | bfloat16
    batch, length (new tokens a sequence, padded), heads, kv_heads, dim
    rotary    channels of a head that are rotated (0: none)       interleaved, scaling ("none" | "linear" | "ntk" | "yarn"), factor
    far       (rotary) first position
    context   tokens in the longest cache, the new ones among them
    fill      shortest sequence and shortest run of new tokens, percent of the longest
    page      tokens a page
    kernel    (paged) window, 0: all of the past                  dilation
"""
import math

import torch

own = False

_DTYPE = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_WIDTH = {"float32": 4, "float16": 2, "bfloat16": 2}
_BASE = 10000.0
_ORIGINAL = 4096        # length that the scaled frequencies were trained at


def _rotary(name, train, dtype, batch, length, heads, kv_heads, dim, rotary, interleaved=False, scaling="none", factor=1.0, far=0):
    return {"name": name, "op": "rotary", "train": train, "dtype": dtype, "batch": batch, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": interleaved, "scaling": scaling,
            "factor": factor, "far": far}


def _append(name, dtype, batch, length, heads, kv_heads, dim, context, page, rotary, interleaved=False, scaling="none", factor=1.0,
            fill=100):
    return {"name": name, "op": "append", "train": False, "dtype": dtype, "batch": batch, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "context": context, "page": page, "rotary": rotary, "interleaved": interleaved,
            "scaling": scaling, "factor": factor, "fill": fill}


def _paged(name, dtype, batch, length, heads, kv_heads, dim, context, page, kernel=0, dilation=1, fill=100):
    return {"name": name, "op": "paged", "train": False, "dtype": dtype, "batch": batch, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "context": context, "page": page, "kernel": kernel, "dilation": dilation, "fill": fill}


def listed():
    return [
        # A toy or test-sized training step in the default data type: all latency.
        _rotary("rotary_f32_tiny_train", True, "float32", 2, 128, 4, 4, 32, 32, interleaved=True),
        # One layer of a decoder's training step, grouped heads, ragged length.
        _rotary("rotary_bf16_train", True, "bfloat16", 2, 8191, 16, 4, 128, 128),
        # Half of the head rotated, positions far behind the trained length, frequencies scaled for it; forward only.
        _rotary("rotary_f16_part_far", False, "float16", 8, 2049, 16, 16, 64, 32, scaling="yarn", factor=16.0, far=60000),
        # One new token for each of 64 sequences: the step of a serving loop, all latency.
        _append("append_bf16_step", "bfloat16", 64, 1, 16, 4, 128, 1024, 16, 128, fill=25),
        # Prompts into an empty cache.
        _append("append_bf16_prefill", "bfloat16", 2, 8191, 16, 4, 128, 8191, 64, 128, scaling="linear", factor=4.0),
        # Short runs of different lengths, padded, an odd page, part of an odd head, the default data type.
        _append("append_f32_ragged", "float32", 5, 77, 6, 3, 40, 333, 24, 20, interleaved=True, fill=30),
        # One new token against a sliding window, few sequences: latency.
        _paged("paged_bf16_step_window", "bfloat16", 8, 1, 16, 4, 128, 8192, 16, kernel=255, fill=25),
        # One new token against all of the past, many sequences of different lengths: memory.
        _paged("paged_bf16_step_full", "bfloat16", 64, 1, 16, 4, 128, 16384, 64, fill=13),
        # A few proposed tokens to verify, every head its own keys, dilated window, odd page.
        _paged("paged_f16_verify_dilated", "float16", 16, 4, 8, 8, 64, 4096, 24, kernel=1023, dilation=2, fill=50),
        # A chunk of two long prompts over what the cache holds already.
        _paged("paged_bf16_chunk_full", "bfloat16", 2, 2048, 16, 4, 128, 16384, 64),
        # Whole prompts through a sliding window.
        _paged("paged_bf16_prefill_window", "bfloat16", 2, 8191, 16, 4, 128, 8191, 16, kernel=255),
        # A test-sized chunk in the default data type.
        _paged("paged_f32_chunk", "float32", 2, 130, 4, 2, 32, 1021, 16, fill=60),
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm; odd and even alike."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """A family of use first, then sizes over its whole range; too costly ones are drawn again."""
    largest = {}
    for c in listed():
        w = work(c)
        kind = (c["op"], c["dtype"] == "float32")
        largest[kind] = [max(a, b) for a, b in zip(largest.get(kind, [0, 0]), (w["bytes"], w["flops"]))]
    limits = {k: (max(b, 2e8 if k[1] else 1e9 if k[0] == "paged" else b), max(f, 2e9 if k[1] else f)) for k, (b, f) in largest.items()}
    while True:
        c = _draw(rng)
        w, (b, f) = work(c), limits[(c["op"], c["dtype"] == "float32")]
        if w["bytes"] <= 0.9 * b and w["flops"] <= 0.9 * f and _scores(c) < 1.2e9 and _cached(c) < 1.5e9:
            c.pop("name")
            return c


def _scores(c):
    return c["batch"] * c["heads"] * c["length"] * c["context"] if c["op"] == "paged" else 0


def _cached(c):
    """Elements of a cache, keys and values together."""
    return 0 if c["op"] == "rotary" else 2 * c["batch"] * (c["context"] + c["page"]) * c["kv_heads"] * c["dim"]


def _draw(rng):
    family = rng.choice(["rotary", "rotary", "append", "step", "step", "verify", "chunk", "chunk", "window", "float32"])
    half = rng.choice(["bfloat16", "bfloat16", "float16"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128, 24, 7])
    scaling = rng.choice(["none", "none", "linear", "ntk", "yarn"])
    factor = 1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 16]))
    inter = rng.random() < 0.4
    if family == "float32":
        op = rng.choice(["rotary", "append", "paged"])
        dim = rng.choice([32, 40, 64])
        length = _log(rng, 1, 257)
        context = max(length, _log(rng, 64, 2048))
        batch = _log(rng, 1, 8)
        if op == "rotary":
            return _rotary("", rng.random() < 0.6, "float32", batch, length, heads, kv, dim, rng.choice([dim, dim // 2]), inter, scaling, factor)
        if op == "append":
            return _append("", "float32", batch, length, heads, kv, dim, context, page, rng.choice([dim, dim // 2, 0]), inter, scaling,
                           factor, fill=rng.randint(25, 100))
        return _paged("", "float32", batch, length, heads, kv, dim, context, page, kernel=rng.choice([0, _log(rng, 3, 511)]),
                      fill=rng.randint(50, 100))
    if family == "rotary":
        return _rotary("", rng.random() < 0.6, half, _log(rng, 1, 16), _log(rng, 1, 16384), heads, kv, dim, rng.choice([dim, dim, dim // 2]),
                       inter, scaling, factor, far=rng.choice([0, 0, _log(rng, 1, 1000000)]))
    if family == "append":
        length = rng.choice([1, 1, _log(rng, 2, 8191)])
        return _append("", half, _log(rng, 1, 128), length, heads, kv, dim, max(length, _log(rng, 64, 8191)), page,
                       rng.choice([dim, dim, dim // 2, 0]), inter, scaling, factor, fill=rng.randint(25, 100))
    if family in ("step", "verify"):
        length = 1 if family == "step" else rng.randint(2, 9)
        context = max(16, _log(rng, 32, 65536))
        kernel = rng.choice([0, 0, _log(rng, 15, 4095)])
        dilation = rng.choice([1, 1, 1, 2, 3]) if kernel else 1
        return _paged("", half, _log(rng, 1, 128), length, heads, kv, dim, context, page, kernel=kernel, dilation=dilation,
                      fill=rng.randint(13, 100))
    length = _log(rng, 16, 4096 if family == "chunk" else 8191)
    if family == "chunk":
        return _paged("", half, _log(rng, 1, 8), length, heads, kv, dim, max(length, _log(rng, 256, 32768)), page,
                      fill=rng.randint(50, 100))
    return _paged("", half, _log(rng, 1, 8), length, heads, kv, dim, max(length, _log(rng, 256, 8191)), page, kernel=_log(rng, 15, 4095),
                  dilation=rng.choice([1, 1, 1, 2]), fill=rng.randint(50, 100))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _spread(longest, fill, batch):
    """Lengths of a batch's sequences: evenly between the shortest and the longest."""
    shortest = max(1, longest * fill // 100)
    return [longest - (longest - shortest) * i // max(1, batch - 1) for i in range(batch)]


def _frequencies(case):
    """Radians a position, channel pair by channel pair, in 64 bits, and what the rotated channels are multiplied by."""
    half, scaling, factor = case["rotary"] // 2, case["scaling"], case["factor"]
    base = _BASE * factor ** (half / (half - 1)) if scaling == "ntk" else _BASE
    freq = [base ** (-i / half) for i in range(half)]
    magnitude = 1.0
    if scaling == "linear":
        freq = [f / factor for f in freq]
    if scaling == "yarn":
        # pairs that turn more than 32 times within the trained length stay, those that turn less than once are divided
        bounds = [half * math.log(_ORIGINAL / (turns * 2 * math.pi)) / math.log(_BASE) for turns in (32.0, 1.0)]
        low, high = max(0, math.floor(bounds[0])), min(2 * half - 1, math.ceil(bounds[1]))
        share = [min(1.0, max(0.0, (i - low) / max(high - low, 1e-3))) for i in range(half)]
        freq = [f * (1 - s) + f / factor * s for f, s in zip(freq, share)]
        magnitude = 0.1 * math.log(factor) + 1.0
    return torch.tensor(freq, dtype=torch.float64, device="cuda"), magnitude


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, B, L = _DTYPE[case["dtype"]], case["batch"], case["length"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g).to(dtype)

    state = {"case": case}
    if case["op"] == "rotary":
        state["q"], state["k"] = normal(B, L, heads, dim).requires_grad_(case["train"]), normal(B, L, kv, dim).requires_grad_(case["train"])
        state["positions"] = torch.arange(L, device="cuda") + case["far"] + 1000 * torch.randint(0, 8, (B, 1), device="cuda", generator=g)
        if case["train"]:
            state["dq"], state["dk"] = normal(B, L, heads, dim), normal(B, L, kv, dim)
    else:
        # a pool with every sequence's pages in it, in no order
        ps = case["page"]
        lens, new = _spread(case["context"], case["fill"], B), _spread(L, case["fill"], B)
        order = torch.randperm(B, device="cuda", generator=g)
        state["cache_lens"] = torch.tensor(lens, device="cuda", dtype=torch.int32)[order].contiguous()
        state["seq_lens"] = torch.minimum(torch.tensor(new, device="cuda", dtype=torch.int32)[order], state["cache_lens"]).contiguous()
        width = -(-case["context"] // ps)
        state["table"] = torch.randperm(B * width, device="cuda", generator=g).to(torch.int32).view(B, width)
        state["k_cache"], state["v_cache"] = normal(B * width, ps, kv, dim), normal(B * width, ps, kv, dim)
        state["q"] = normal(B, L, heads, dim)
        if case["op"] == "append":
            state["k"], state["v"] = normal(B, L, kv, dim), normal(B, L, kv, dim)
            # the tokens that are there, in the padded batch: what a program that packs its rows keeps
            state["rows"] = (torch.arange(L, device="cuda") < state["seq_lens"][:, None]).flatten().nonzero().flatten()
    if case["op"] != "paged" and case["rotary"]:
        state["freq"], state["magnitude"] = _frequencies(case)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _rotated(x, positions, state):
    """``x [B, L, H, D]`` with its first channels turned by the angles of ``positions [B, L]``, in 32 bits."""
    case, y = state["case"], x.float()
    if not case["rotary"]:
        return y
    angle = positions.double()[..., None, None] * state["freq"]
    cos, sin = torch.cos(angle).float() * state["magnitude"], torch.sin(angle).float() * state["magnitude"]
    turned, rest = y[..., :case["rotary"]], y[..., case["rotary"]:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned.chunk(2, dim=-1)
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_rotary(state):
    q, k = state["q"], state["k"]
    return _rotated(q, state["positions"], state).to(q.dtype), _rotated(k, state["positions"], state).to(k.dtype)


def _new_positions(state):
    length = state["case"]["length"]
    return (state["cache_lens"] - state["seq_lens"])[:, None] + torch.arange(length, device="cuda")


def _plain_append(state):
    case, q, k_cache, v_cache = state["case"], state["q"], state["k_cache"], state["v_cache"]
    pos, rows, ps = _new_positions(state), state["rows"], case["page"]
    there = torch.arange(case["length"], device="cuda") < state["seq_lens"][:, None]
    turned = torch.where(there[..., None, None], _rotated(q, pos, state), 0.0).to(q.dtype)
    key = _rotated(state["k"], pos, state).to(k_cache.dtype)
    page = torch.gather(state["table"], 1, (pos // ps).clamp(0, state["table"].shape[1] - 1)).long()
    slot = (page * ps + pos % ps).flatten()[rows]
    k_cache.view(-1, *k_cache.shape[2:])[slot] = key.flatten(0, 1)[rows]
    v_cache.view(-1, *v_cache.shape[2:])[slot] = state["v"].flatten(0, 1)[rows]
    return turned, k_cache, v_cache


def _plain_paged(state):
    case, q = state["case"], state["q"]
    B, L, heads, dim = q.shape
    kv, group = case["kv_heads"], heads // case["kv_heads"]
    table = state["table"].long()
    keys, values = [c[table].flatten(1, 2).float() for c in (state["k_cache"], state["v_cache"])]
    score = torch.einsum("blhgd,bshd->bhgls", q.float().view(B, L, kv, group, dim) * dim ** -0.5, keys)
    pos, j = _new_positions(state)[..., None], torch.arange(keys.shape[1], device="cuda")
    back = pos - j
    seen = (back >= 0) & (back % case["dilation"] == 0) & (torch.arange(L, device="cuda")[:, None] < state["seq_lens"][:, None, None])
    if case["kernel"]:
        seen &= back < case["kernel"] * case["dilation"]
    seen = seen[:, None, None]
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    weight = torch.exp_(score.sub_(top))
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("bhgls,bshd->bhgld", weight, values) / total.clamp_min(1e-30)
    lse = torch.log(total) + top
    lse = torch.where(total > 0, lse, -math.inf)
    return out.permute(0, 3, 1, 2, 4).reshape(B, L, heads, dim).to(q.dtype), lse[..., 0].permute(0, 3, 1, 2).reshape(B, L, heads)


def _own_rotary(state):
    from natten_mps_b200 import functional as F
    return F.na1d_rotary(state["q"], state["k"], state["freq"], state["positions"], interleaved=state["case"]["interleaved"],
                         magnitude=state["magnitude"])


def _own_append(state):
    from natten_mps_b200 import functional as F
    case = state["case"]
    turn = {"frequencies": state["freq"], "interleaved": case["interleaved"], "magnitude": state["magnitude"]} if case["rotary"] else {}
    turned = F.na1d_append(state["k"], state["v"], state["k_cache"], state["v_cache"], state["table"], state["cache_lens"],
                           state["seq_lens"], query=state["q"], **turn)
    return turned, state["k_cache"], state["v_cache"]


def _own_paged(state):
    from natten_mps_b200 import functional as F
    case = state["case"]
    return F.na1d_paged(state["q"], state["k_cache"], state["v_cache"], state["table"], state["cache_lens"], case["kernel"] or None,
                        case["dilation"], return_lse=True, seq_lens=state["seq_lens"])


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        if not case["train"]:
            with torch.no_grad():
                return _own_rotary(state) if own else _plain_rotary(state)
        out = _own_rotary(state) if own else _plain_rotary(state)
        grads = torch.autograd.grad(out, [state["q"], state["k"]], [state["dq"], state["dk"]])
        return [out[0].detach(), out[1].detach(), *grads]
    with torch.no_grad():
        if case["op"] == "append":
            return _own_append(state) if own else _plain_append(state)
        return _own_paged(state) if own else _plain_paged(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    """Every input read once and every output written once.  Attention counts 4 operations per (query head, key in its
    window, channel) and the keys that any window of a sequence holds; padding rows are written and not read."""
    width, B, L = _WIDTH[case["dtype"]], case["batch"], case["length"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        elements = B * L * (heads + kv) * dim
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * elements * width + 8 * B * L), "flops": passes * 3 * B * L * (heads + kv) * case["rotary"]}
    lens = _spread(case["context"], case["fill"], B)
    new = [min(a, b) for a, b in zip(_spread(L, case["fill"], B), lens)]
    pages = sum(-(-n // case["page"]) for n in (new if case["op"] == "append" else lens))
    if case["op"] == "append":
        bytes_ = width * dim * (sum(new) * (heads + 4 * kv) + B * L * heads) + 4 * pages + 8 * B
        return {"bytes": bytes_, "flops": 3 * sum(new) * (heads + kv) * case["rotary"]}
    pairs = keys = 0
    d = case["dilation"]
    for n, m in zip(lens, new):
        reach = case["kernel"] or n
        for r in range(min(d, m)):                       # new tokens of one dilation class, with the past that they see
            first, last = (n - m + r) // d, (n - m + r) // d + (m - 1 - r) // d
            keys += last - max(0, first - reach + 1) + 1
            full = max(first, reach - 1)                 # from here on windows are whole
            short = max(0, min(last + 1, full) - first)
            pairs += short * first + short * (short + 1) // 2 + (last - first + 1 - short) * reach
    return {"bytes": width * dim * (heads * (sum(new) + B * L) + 2 * kv * keys) + 4 * B * L * heads + 4 * pages + 8 * B,
            "flops": 4 * dim * heads * pairs}


def _exact_turn(x, positions, state, back=False):
    """Rotation as a product with complex numbers."""
    case, y = state["case"], x.double()
    n = case["rotary"]
    if not n:
        return y
    angle = positions.double().unsqueeze(-1) * state["freq"]
    unit = torch.polar(torch.full_like(angle, state["magnitude"]), -angle if back else angle).unsqueeze(-2)
    pairs = y[..., :n].unflatten(-1, (n // 2, 2)) if case["interleaved"] else y[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    z = z if case["interleaved"] else z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), y[..., n:]], dim=-1)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rotary":
            pos = state["positions"]
            out = [_exact_turn(state["q"], pos, state), _exact_turn(state["k"], pos, state)]
            if not case["train"]:
                return tuple(out)
            return out + [_exact_turn(state["dq"], pos, state, True), _exact_turn(state["dk"], pos, state, True)]
        lens, new, table = state["cache_lens"].tolist(), state["seq_lens"].tolist(), state["table"].tolist()
        if case["op"] == "append":
            pos = _new_positions(state)
            turned, key, value = _exact_turn(state["q"], pos, state), _exact_turn(state["k"], pos, state), state["v"].double()
            k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
            for b, (n, m) in enumerate(zip(lens, new)):
                turned[b, m:] = 0
                at = torch.tensor([[table[b][p // case["page"]], p % case["page"]] for p in range(n - m, n)], device="cuda")
                k_cache[at[:, 0], at[:, 1]] = key[b, :m]
                v_cache[at[:, 0], at[:, 1]] = value[b, :m]
            return turned, k_cache, v_cache
        q = state["q"]
        if work(case)["flops"] > 3e12:
            return None
        B, L, heads, dim = q.shape
        group, d = heads // case["kv_heads"], case["dilation"]
        out = torch.zeros(B, L, heads, dim, dtype=torch.float64, device="cuda")
        lse = torch.full((B, L, heads), -math.inf, dtype=torch.float64, device="cuda")
        step = 1024
        for b, (n, m) in enumerate(zip(lens, new)):
            pages = state["table"][b, :-(-n // case["page"])].long()
            keys = state["k_cache"][pages].flatten(0, 1)[:n].double()
            values = state["v_cache"][pages].flatten(0, 1)[:n].double()
            for i in range(0, m, step):                  # some queries at a time, with the stretch of keys that they can see
                stop = min(m, i + step)
                p = torch.arange(n - m + i, n - m + stop, device="cuda")
                low = max(0, n - m + i - (case["kernel"] - 1) * d) if case["kernel"] else 0
                j = torch.arange(low, n - m + stop, device="cuda")
                hidden = (j > p[:, None]) | ((p[:, None] - j) % d != 0)
                if case["kernel"]:
                    hidden |= p[:, None] - j > (case["kernel"] - 1) * d
                for h in range(case["kv_heads"]):
                    s = slice(h * group, (h + 1) * group)
                    x = torch.matmul(q[b, i:stop, s].double().transpose(0, 1), keys[low:n - m + stop, h].T) / math.sqrt(dim)
                    x = x.masked_fill_(hidden, -math.inf)
                    lse[b, i:stop, s] = torch.logsumexp(x, dim=-1).T
                    out[b, i:stop, s] = torch.matmul(torch.softmax(x, dim=-1), values[low:n - m + stop, h]).transpose(0, 1)
        return out, lse
