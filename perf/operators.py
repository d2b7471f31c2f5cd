"""Operators of the hybrid model's attention layers around a key-value cache, measured one by one and as a layer calls them.

Kinds of work
  norm    queries and keys of a training step: RMS norm of every head and position rotation in one pass, and its gradients
          (`ops.qk_norm_rotary`; without `grad` the forward pass alone, as scoring and prompts run it)
  append  a piece of a prompt goes into a paged cache and the sequences are read back (`ops.kv_cache_write`, `ops.kv_cache_read`)
  token   one new token of every sequence in an attention layer: norm, rotation, write, attention over the cache
          (`ops.kv_cache_write`, `ops.paged_attention`)
  attend  the attention of one new token alone (`ops.paged_attention`)

Head counts, head width and lengths are those of the hybrid presets (32 query and 8 key heads of 128 channels, up to 8192
tokens), of the decode benchmark (64 sequences of 2048 tokens) and of the tests' small models; caches hold bfloat16, e4m3 or
int8 with one scale per token and head.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
THETA = 10000.0
TYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
BYTES = {"bf16": 2, "e4m3": 1, "int8": 1}


def _norm(name, batch, tokens, heads, kv_heads, dim, rotary, packed=False, wide=False, grad=True):
    return {"name": name, "kind": "norm", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "packed": packed, "wide": wide, "grad": grad}


def _cache(name, kind, type_, batch, new, length, heads, kv_heads, dim, rotary, page, ragged=False, norm=True):
    return {"name": name, "kind": kind, "type": type_, "batch": batch, "new": new, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "page": page, "ragged": ragged, "norm": norm}


def listed():
    return [
        # a small model's training step on packed texts of an odd length, half of the channels rotated, fp32 norm weights
        _norm("norm_1x257_5+1x64", 1, 257, 5, 1, 64, 32, packed=True, wide=True),
        # hybrid 8B at its 4096-token length, micro-batch 2
        _norm("norm_2x4096_32+8x128", 2, 4096, 32, 8, 128, 128),
        # the longest sequences that the presets train on, micro-batch 4
        _norm("norm_4x8192_32+8x128", 4, 8192, 32, 8, 128, 128),
        # a short chat prompt into an empty cache
        _cache("append_bf16_1x128", "append", "bf16", 1, 128, 0, 32, 8, 128, 128, 16),
        # texts of different lengths behind prompts of different lengths, padded on the right
        _cache("append_e4m3_8x1000+1047", "append", "e4m3", 8, 1000, 1047, 32, 8, 128, 64, 64, ragged=True),
        # a batch of the benchmark's prompts
        _cache("append_int8_16x2048", "append", "int8", 16, 2048, 0, 32, 8, 128, 128, 128),
        # one user in a short conversation: a chain of small kernels
        _cache("token_bf16_1x200", "token", "bf16", 1, 1, 200, 32, 8, 128, 128, 16),
        # the decode benchmark's batch with an 8-bit cache
        _cache("token_e4m3_64x2048", "token", "e4m3", 64, 1, 2048, 32, 8, 128, 128, 64),
        # a few sequences of very different lengths, an odd number of query heads per key head
        _cache("token_bf16_7x5001", "token", "bf16", 7, 1, 5001, 9, 3, 64, 64, 32, ragged=True),
        # one very long document, no rotation, as the hybrid presets have it
        _cache("attend_bf16_1x131072", "attend", "bf16", 1, 1, 131072, 32, 8, 128, 0, 128, norm=False),
        # many query heads on one key head, ragged, int8
        _cache("attend_int8_32x8192", "attend", "int8", 32, 1, 8192, 16, 1, 128, 0, 64, ragged=True, norm=False),
        # the decode benchmark's batch at the longest length of the presets
        _cache("attend_bf16_64x8192", "attend", "bf16", 64, 1, 8192, 32, 8, 128, 0, 64, norm=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "append", "token", "attend"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.randint(1, 8)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 12, 16])
    rotary = rng.choice([0, 16, dim // 2, dim])
    if kind == "norm":
        most = min(32768, (32768 * 40 * 128) // ((heads + kv_heads) * dim))
        tokens = _spread(rng, 1, most)
        batch = rng.randint(1, max(1, min(8, most // tokens)))
        case = _norm("", batch, tokens, heads, kv_heads, dim, rotary, packed=rng.random() < 0.3, wide=rng.random() < 0.3,
                     grad=rng.random() < 0.75)
    else:
        type_ = rng.choice(["bf16", "e4m3", "int8"] if kind != "token" else ["bf16", "e4m3"])
        page = rng.choice([16, 32, 64, 128, 256])
        if kind == "append":
            most = 32768 * 56 * 128 // ((heads + 3 * kv_heads) * dim)
            new = _spread(rng, 1, min(4096, most))
            batch = rng.randint(1, max(1, min(16, most // new)))
            length = rng.choice([0, _spread(rng, 1, max(1, min(2048, most // batch)))])
        else:
            most = 64 * 8192 * 8 * 128 // (kv_heads * dim)
            new, length = 1, _spread(rng, 1, min(131072, most))
            batch = _spread(rng, 1, max(1, min(256, most // length)))
        case = _cache("", kind, type_, batch, new, length, heads, kv_heads, dim, rotary, page, ragged=rng.random() < 0.5,
                      norm=rng.random() < 0.7)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _tables(positions, rotary):
    """fp32 cos / sin of every position and pair of channels; the angles are taken in 64 bits."""
    half = rotary // 2
    inverse = THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") * 2 / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inverse
    return angle.cos().float(), angle.sin().float()


def _activations(g, *shape):
    """Projections as a layer produces them: channels of different sizes, some of them large, rounded to bfloat16."""
    size = torch.empty(shape[-2:], device="cuda").log_normal_(0.0, 0.5, generator=g)
    return (torch.randn(shape, device="cuda", generator=g) * size).to(torch.bfloat16)


def _weight(g, dim, wide):
    w = 1.2 + 0.2 * torch.randn(dim, device="cuda", generator=g)
    return w if wide else w.to(torch.bfloat16)


def _prepare_norm(case, g):
    B, L, H, K, D = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
    # one projection's output, of which queries and keys are views
    qkv = _activations(g, B, L, H + 2 * K, D)
    s = {"case": case, "q": qkv[:, :, :H], "k": qkv[:, :, H:H + K], "qw": _weight(g, D, case["wide"]),
         "kw": _weight(g, D, case["wide"]), "cos": None, "sin": None, "positions": None}
    if case["rotary"]:
        s["cos"], s["sin"] = _tables(L, case["rotary"])
        if case["packed"]:
            # texts of an eighth of the row or less, one behind the other: positions begin again at each
            starts = torch.rand(B, L, device="cuda", generator=g) < 8.0 / L
            at = torch.arange(L, device="cuda").expand(B, L)
            s["positions"] = at - torch.where(starts, at, torch.zeros_like(at)).cummax(dim=1).values
    if case["grad"]:
        s["dq"] = (torch.randn(B, L, H, D, device="cuda", generator=g) * 0.02).to(torch.bfloat16)
        s["dk"] = (torch.randn(B, L, K, D, device="cuda", generator=g) * 0.02).to(torch.bfloat16)
        for name in ("q", "k", "qw", "kw"):
            s[name] = s[name].detach().requires_grad_()
    return s


def _quantised(x, type_):
    """(stored values, scales or None) of rows, in 32 bits."""
    if type_ == "bf16":
        return x.to(torch.bfloat16), None
    scale = x.abs().amax(-1) / LARGEST[type_]
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    return (y.round().to(torch.int8) if type_ == "int8" else y.to(torch.float8_e4m3fn)), scale


def _prepare_cache(case, g):
    B, L, H, K, D, page = (case[k] for k in ("batch", "new", "heads", "kv_heads", "dim", "page"))
    s = {"case": case, "counts": None}
    # lengths before the new tokens, then with them; sequences of a ragged batch are anywhere up to the longest
    longest = case["length"]
    before = torch.full((B,), longest, device="cuda")
    if case["ragged"]:
        before = torch.randint(0, longest + 1, (B,), device="cuda", generator=g)
        before[0] = longest
    if case["kind"] == "append":
        counts = torch.full((B,), L, device="cuda")
        if case["ragged"]:
            counts = torch.randint(1, L + 1, (B,), device="cuda", generator=g)
            s["counts"] = counts.to(torch.int32)
        s["lengths"] = (before + counts).to(torch.int32)
    else:
        s["lengths"] = before.clamp(min=1).to(torch.int32)
    most = longest + L if case["kind"] == "append" else max(1, longest)
    s["most"] = most
    width = -(-most // page)
    pages = B * width + 3
    s["table"] = torch.randperm(pages, device="cuda", generator=g)[:B * width].view(B, width).to(torch.int32)
    held = []
    for _ in range(2):
        if case["kind"] == "append" and longest == 0:
            x = torch.zeros(pages, K, page, D, device="cuda", dtype=torch.bfloat16)
        else:
            x = torch.randn(pages, K, page, D, device="cuda", generator=g, dtype=torch.bfloat16)
            x *= torch.empty(K, 1, D, device="cuda").log_normal_(0.0, 0.4, generator=g).to(torch.bfloat16)
        held.append(x if case["type"] == "bf16" else _quantised(x.float(), case["type"]))
        del x
    if case["type"] == "bf16":
        s["pages"] = (held[0], held[1], None, None)
    else:
        s["pages"] = (held[0][0], held[1][0], held[0][1], held[1][1])
    if case["kind"] == "attend":
        s["q"] = _activations(g, B, 1, H, D)
        return s
    qkv = _activations(g, B, L, H + 2 * K, D)
    s["q"], s["k"], s["v"] = qkv[:, :, :H], qkv[:, :, H:H + K], qkv[:, :, H + K:]
    s["qw"], s["kw"] = (_weight(g, D, False), _weight(g, D, False)) if case["norm"] else (None, None)
    s["cos"], s["sin"] = _tables(most, case["rotary"]) if case["rotary"] else (None, None)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_norm(case, g) if case["kind"] == "norm" else _prepare_cache(case, g)


# ---- one pass -------------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin):
    if cos is None:
        return x
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)


def _normed(x, w):
    """(normed rows, reciprocal root of the mean square) in 32 bits"""
    x = x.float()
    if w is None:
        return x, None
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * r * w.float(), r


def _norm_gradients(x, w, r, dy, cos, sin):
    x, g = x.float(), _rotate(dy.float(), cos, None if sin is None else -sin)
    h = g * w.float()
    dx = r * h - x * (r ** 3 * (h * x).mean(-1, keepdim=True))
    return dx.to(torch.bfloat16), (g * x * r).sum((0, 1, 2)).to(w.dtype)


def _norm_plain(s):
    cos, sin = s["cos"], s["sin"]
    if cos is not None:
        at = s["positions"]
        cos, sin = (cos[:, None], sin[:, None]) if at is None else (cos[at][:, :, None], sin[at][:, :, None])
    with torch.no_grad():
        (q, qr), (k, kr) = _normed(s["q"], s["qw"]), _normed(s["k"], s["kw"])
        out = [_rotate(q, cos, sin).to(torch.bfloat16), _rotate(k, cos, sin).to(torch.bfloat16)]
        if s["case"]["grad"]:
            dq, dqw = _norm_gradients(s["q"], s["qw"], qr, s["dq"], cos, sin)
            dk, dkw = _norm_gradients(s["k"], s["kw"], kr, s["dk"], cos, sin)
            out += [dq, dk, dqw, dkw]
    return out


def _norm_own(s):
    from state_space_models_neuron_b200 import ops
    args = (s["q"], s["k"], s["qw"], s["kw"], EPS, s["cos"], s["sin"], s["positions"])
    if not s["case"]["grad"]:
        with torch.no_grad():
            return list(ops.qk_norm_rotary(*args))
    q, k = ops.qk_norm_rotary(*args)
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["dq"], s["dk"]))]


def _write_plain(s):
    """Queries with norm and rotation; keys and values into the pages."""
    B, L = s["k"].shape[:2]
    page = s["case"]["page"]
    counts = L if s["counts"] is None else s["counts"].long()[:, None]
    at = s["lengths"].long()[:, None] - counts + torch.arange(L, device="cuda")
    real = None if s["counts"] is None else torch.arange(L, device="cuda") < counts
    cos = sin = None
    if s["cos"] is not None:
        rows = at if real is None else at.clamp(max=s["cos"].shape[0] - 1)
        cos, sin = s["cos"][rows][:, :, None], s["sin"][rows][:, :, None]
    q = _rotate(_normed(s["q"], s["qw"])[0], cos, sin).to(torch.bfloat16)
    k, v = _rotate(_normed(s["k"], s["kw"])[0], cos, sin), s["v"].float()
    if real is not None:
        q = torch.where(real[:, :, None, None], q, torch.zeros_like(q))
        seq = torch.arange(B, device="cuda")[:, None].expand(B, L)[real]
        at, k, v = at[real], k[real], v[real]
    else:
        seq = torch.arange(B, device="cuda")[:, None]
    where, slot = s["table"].long()[seq, at // page], at % page
    for x, held, scales in ((k, s["pages"][0], s["pages"][2]), (v, s["pages"][1], s["pages"][3])):
        stored, scale = _quantised(x, s["case"]["type"])
        if stored.dtype == torch.float8_e4m3fn:
            held, stored = held.view(torch.uint8), stored.view(torch.uint8)
        held[where, :, slot] = stored
        if scales is not None:
            scales[where, :, slot] = scale
    return q


def _gathered(s):
    """Keys and values of every sequence in 32 bits, [batch, kv_heads, length, dim]; undefined behind the lengths."""
    both = []
    for held, scales in ((s["pages"][0], s["pages"][2]), (s["pages"][1], s["pages"][3])):
        if held.dtype == torch.float8_e4m3fn:
            x = held.view(torch.uint8)[s["table"].long()].view(torch.float8_e4m3fn).float()
        else:
            x = held[s["table"].long()].float()
        if scales is not None:
            x *= scales[s["table"].long()][..., None]
        both.append(x.transpose(1, 2).flatten(2, 3)[:, :, :s["most"]])
    return both


def _read_plain(s):
    real = (torch.arange(s["most"], device="cuda") < s["lengths"][:, None])[:, :, None, None]
    out = []
    for x in _gathered(s):
        x = x.transpose(1, 2)
        out.append(torch.where(real, x, torch.zeros_like(x)).to(torch.bfloat16))
    return out


def _attend_plain(s, q):
    k, v = _gathered(s)
    B, _, H, D = q.shape
    K = k.shape[1]
    q = q.float().view(B, K, H // K, D) / math.sqrt(D)
    scores = torch.matmul(q, k.transpose(2, 3))
    hidden = torch.arange(s["most"], device="cuda") >= s["lengths"][:, None]
    scores = scores.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(B, 1, H, D).to(torch.bfloat16)


def run(s):
    kind = s["case"]["kind"]
    if kind == "norm":
        return _norm_own(s) if own else _norm_plain(s)
    with torch.no_grad():
        if not own:
            q = s["q"] if kind == "attend" else _write_plain(s)
            if kind == "append":
                return [q, *_read_plain(s)]
            out = [_attend_plain(s, q)]
        else:
            from state_space_models_neuron_b200 import ops
            pages = ops.KVPages(*s["pages"])
            q = s["q"]
            if kind != "attend":
                q = ops.kv_cache_write(s["k"], s["v"], pages, s["table"], s["lengths"], counts=s["counts"], q=q,
                                       q_weight=s["qw"], k_weight=s["kw"], eps=EPS, cos=s["cos"], sin=s["sin"])
            if kind == "append":
                return [q, *ops.kv_cache_read(pages, s["table"], s["lengths"], s["most"])]
            out = [ops.paged_attention(q, pages, s["table"], s["lengths"])]
    if kind == "token":
        out += [q] + [t for t in s["pages"] if t is not None]      # the cache has one token more
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "norm":
        values = case["batch"] * case["tokens"] * (H + K) * D
        return {"bytes": values * (10 if case["grad"] else 4), "flops": values * (25 if case["grad"] else 8)}
    each = BYTES[case["type"]]
    row = D * each + (0 if case["type"] == "bf16" else 4)        # a cached head of a token with its scale
    new = case["batch"] * case["new"]
    # a ragged batch holds about half of the longest, and half of its new tokens are padding
    share = 0.5 if case["ragged"] and case["batch"] > 1 else 1.0
    held = case["batch"] * case["length"] * share
    if case["kind"] == "append":
        new *= share
        moved = new * (H * D * 4 + 2 * K * (D * 2 + row)) + held * 2 * K * row + (held + new) * 2 * K * D * 2
        return {"bytes": moved, "flops": new * (H + 2 * K) * D * 8}
    moved = held * 2 * K * row + new * H * D * 4
    if case["kind"] == "token":
        moved += new * (H * D * 2 + 2 * K * (D * 2 + row))
    return {"bytes": moved, "flops": held * H * D * 4}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _exact_rows(x, w, angle_rows, cos, sin, sign=1.0):
    """RMS norm and rotation of x [..., heads, dim] in 64 bits; pairs of channels as complex numbers."""
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * w.double()
    return _exact_turn(y, angle_rows, cos, sin, sign)


def _exact_turn(y, angle_rows, cos, sin, sign):
    if cos is None:
        return y
    half = cos.shape[-1]
    turn = torch.complex(cos.double()[angle_rows], sign * sin.double()[angle_rows]).unsqueeze(-2)
    z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
    return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)


def _exact_norm(case, s):
    at = s["positions"]
    if at is None:
        at = torch.arange(case["tokens"], device="cuda").expand(case["batch"], -1)
    out, grads, weights = [], [], []
    for x, w, dy in ((s["q"], s["qw"], s.get("dq")), (s["k"], s["kw"], s.get("dk"))):
        x, w = x.detach(), w.detach()
        rows = [_exact_rows(x[b], w, at[b], s["cos"], s["sin"]) for b in range(case["batch"])]
        out.append(torch.stack(rows))
        if dy is None:
            continue
        dw, dx = torch.zeros(case["dim"], dtype=torch.float64, device="cuda"), []
        for b in range(case["batch"]):
            g = _exact_turn(dy[b].double(), at[b], s["cos"], s["sin"], -1.0)
            xd = x[b].double()
            root = (xd.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            unit = xd / root
            dw += (g * unit).sum((0, 1))
            gw = g * w.double()
            dx.append((gw - unit * (gw * unit).mean(-1, keepdim=True)) / root)
        grads.append(torch.stack(dx))
        weights.append(dw)
    return out + grads + weights


def _exact_stored(x, type_):
    if type_ == "bf16":
        return x.to(torch.bfloat16).double()
    scale = (x.abs().amax(-1, keepdim=True) / LARGEST[type_])
    y = x / torch.where(scale == 0, 1.0, scale)
    y = y.round() if type_ == "int8" else y.float().to(torch.float8_e4m3fn).double()
    return y * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(case, s)
    B, L, H, K, D, page = (case[k] for k in ("batch", "new", "heads", "kv_heads", "dim", "page"))
    outs, queries, keys, values = [], [], [], []
    lengths = s["lengths"].tolist()
    counts = [L] * B if s["counts"] is None else s["counts"].tolist()
    for b in range(B):
        n = lengths[b]
        ids = s["table"][b, :-(-n // page)].long()
        kv = []
        for held, scales in ((s["pages"][0], s["pages"][2]), (s["pages"][1], s["pages"][3])):
            x = held.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() if case["type"] == "e4m3" else held[ids].double()
            x = x if scales is None else x * scales[ids].double()[..., None]
            kv.append(x.permute(0, 2, 1, 3).reshape(-1, K, D)[:n])
        q = s["q"][b].double()
        if case["kind"] != "attend":
            c = counts[b]
            at = torch.arange(n - c, n, device="cuda")
            q = torch.zeros(L, H, D, dtype=torch.float64, device="cuda")
            q[:c] = _exact_rows(s["q"][b, :c], s["qw"], at, s["cos"], s["sin"])
            kv[0][n - c:] = _exact_stored(_exact_rows(s["k"][b, :c], s["kw"], at, s["cos"], s["sin"]), case["type"])
            kv[1][n - c:] = _exact_stored(s["v"][b, :c].double(), case["type"])
        queries.append(q)
        if case["kind"] == "append":
            for x, into in zip(kv, (keys, values)):
                into.append(torch.cat([x, x.new_zeros(s["most"] - n, K, D)]))
            continue
        p = torch.softmax(torch.einsum("kgd,tkd->kgt", q[0].view(K, H // K, D), kv[0]) / math.sqrt(D), -1)
        outs.append(torch.einsum("kgt,tkd->kgd", p, kv[1]).reshape(1, H, D))
    if case["kind"] == "append":
        return [torch.stack(queries), torch.stack(keys), torch.stack(values)]
    outs = [torch.stack(outs)]
    if case["kind"] == "token":
        outs += [torch.stack(queries)] + [None] * sum(t is not None for t in s["pages"])
    return outs
