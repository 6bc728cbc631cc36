"""The quantised K/V cache: its operators, one pass at a time.

A static K/V cache of the attention layers held in 4 or 8 bits: rows are
quantised as they are written (``store``; the pass reads the written rows back,
as the values that the codes stand for), read back (``load``), attended by one
new token (``decode``) and by the tokens of a prompt or of a later part of it
(``prompt``).

The form: a row of one head (``dim`` values) has ``dim / 64`` groups of 64
values. A group stands for ``low + step * code`` with codes 0 .. 2^bits - 1,
``low`` its least value, ``step`` its range over 2^bits - 1, both bf16, and
``code`` the whole number nearest to ``(x - low) / step`` (ties to even), held
to that range; a group without a range has step 0 and codes 0. Keys: group g
holds dims 64 g .. 64 g + 63. Values: group g holds the dims d with
``(d mod dim/16) div 4 == g``. Codes are packed in order, in 4 bits the even
dim in a byte's low half; ``key_params`` / ``value_params`` are
``[batch, kv_heads, dim / 64, capacity, (step, low)]``.

Head layouts: 8 query and 2 KV heads of 256 is the 2B decoder of this
repository; the others are generic. Contexts go from one token to 131072.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
# (query heads, KV heads, head dim)
LAYOUTS = [(8, 2, 256), (8, 1, 256), (4, 4, 256), (16, 2, 256), (12, 1, 256), (32, 8, 128), (24, 2, 128),
           (20, 5, 128), (14, 2, 64), (9, 9, 64)]


# ------------------------------------------------------------------ cases
def _case(kind, bits, heads, kv_heads, dim, batch, length, new=1, gate=False, token_major=False):
    return {"kind": kind, "bits": bits, "heads": heads, "kv_heads": kv_heads, "dim": dim, "batch": batch,
            "length": length, "new": new, "gate": gate, "token_major": token_major}


def listed():
    def named(name, *args, **kwargs):
        return {"name": name, **_case(*args, **kwargs)}

    return [
        # the token of a decode step enters the cache (the smallest call)
        named("store 1 token 4bit", "store", 4, 8, 2, 256, 1, 1040),
        # the benchmark's prompt length, less a ragged end, as a projection
        # leaves it (token-major)
        named("store 1000 tokens 8bit", "store", 8, 8, 2, 256, 1, 1000, new=1000, token_major=True),
        # a bf16 cache of a long document moves into the small one
        named("store 100003 tokens 4bit", "store", 4, 8, 2, 256, 1, 100003, new=100003),
        # a chat's cache is read back to go on in bf16
        named("load 777 tokens 4bit", "load", 4, 8, 2, 256, 1, 777),
        # a long document's cache is read back
        named("load 131072 tokens 8bit", "load", 8, 8, 2, 256, 1, 131072),
        # a decode step at the benchmark's context, with the output gate
        named("decode ctx 1088 4bit", "decode", 4, 8, 2, 256, 1, 1088, gate=True),
        # a decode step over a document
        named("decode ctx 16001 8bit", "decode", 8, 8, 2, 256, 1, 16001, gate=True),
        # a decode step over the longest context
        named("decode ctx 131071 4bit", "decode", 4, 8, 2, 256, 1, 131071),
        # a served batch of unequal contexts, one slot of it unused
        named("decode 16 x 8000 4bit", "decode", 4, 32, 8, 128, 16, 8000),
        # a few drafted tokens are checked over a document
        named("prompt 5 after 8192 4bit", "prompt", 4, 8, 2, 256, 1, 8197, new=5),
        # a prompt of ordinary length
        named("prompt 1000 4bit", "prompt", 4, 8, 2, 256, 1, 1000, new=1000),
        # the next part of a long document
        named("prompt 4096 after 28000 8bit", "prompt", 8, 8, 2, 256, 1, 32096, new=4096),
    ]


def _cost(case):
    w = work(case)
    return w["bytes"] / 8e12 + w["flops"] / 2.5e15


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["store", "load", "decode", "decode", "prompt", "prompt"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        heads, kv_heads, dim = rng.choice(LAYOUTS)
        batch = rng.choice([1, 1, 2, 5, 16])
        length = log(1, 131072)
        new = 1
        if kind == "store":
            new = length if rng.random() < 0.6 else log(1, length)
        if kind == "prompt":
            length = log(2, 40000)
            new = log(2, min(length, 6000))
        case = _case(kind, rng.choice([4, 4, 8]), heads, kv_heads, dim, batch, length, new=new,
                     gate=kind == "decode" and rng.random() < 0.5,
                     token_major=kind == "store" and rng.random() < 0.5)
        # memory: the plain form's scores and 32-bit rows of a case
        rows = batch * kv_heads * length * dim
        scores = batch * heads * new * length if kind in ("decode", "prompt") else 0
        if _cost(case) <= most and rows <= 6e8 and scores <= 3e9:
            return case


def _capacity(case):
    return max(512, (case["length"] + 1 + 127) // 128 * 128)


def _lengths(case):
    """Valid tokens of every sequence: unequal ones in a batch, and in a
    batch of 16 the last slot is unused."""
    b, n = case["batch"], case["length"]
    lengths = [max(1, n - i * n // (b + 1)) for i in range(b)]
    if case["kind"] == "decode" and b >= 16:
        lengths[-1] = 0
    if case["kind"] == "prompt":  # at least the new tokens
        lengths = [max(case["new"], x) for x in lengths]
    return lengths


def work(case):
    d, groups = case["dim"], case["dim"] // 64
    row = d * case["bits"] // 8 + 4 * groups  # one token of one head, K or V
    lengths = _lengths(case)
    if case["kind"] in ("store", "load"):
        rows = 2 * case["batch"] * case["kv_heads"] * (case["new"] if case["kind"] == "store" else case["length"])
        passes = 2 if case["kind"] == "store" else 1  # written and read back, or read
        return {"bytes": passes * rows * (row + 2 * d), "flops": 0}
    new = case["new"]
    pairs = sum(sum(n - new + 1 + i for i in (0, new - 1)) * new // 2 if n else 0 for n in lengths)
    io = 2 * case["batch"] * case["heads"] * new * d * 2
    gate = case["batch"] * case["heads"] * d * 2 if case["gate"] else 0
    return {"bytes": 2 * case["kv_heads"] * sum(lengths) * row + io + gate,
            "flops": 4 * d * case["heads"] * pairs}


# ------------------------------------------------------------------ inputs
def _normal(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * std


def _rows(g, case, tokens):
    """Keys with channels of unequal offset, as rotated keys have, and values."""
    shape = (case["batch"], case["kv_heads"], tokens, case["dim"])
    offset = _normal(g, 1, case["kv_heads"], 1, case["dim"])
    k = (_normal(g, *shape) + offset).to(BF16)
    v = _normal(g, *shape, std=0.5).to(BF16)
    return k, v


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    capacity, new = _capacity(case), case["new"]
    state = {"case": dict(case), "scale": case["dim"] ** -0.5}
    if case["kind"] == "store":
        k, v = _rows(g, case, new)
        if case["token_major"]:  # [batch, tokens, heads, dim], seen as [batch, heads, tokens, dim]
            k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
        shape = (case["batch"], case["kv_heads"], capacity)
        packed = [torch.zeros(*shape, case["dim"] * case["bits"] // 8, device=DEV, dtype=torch.uint8)
                  for _ in range(2)]
        params = [torch.zeros(*shape[:2], case["dim"] // 64, capacity, 2, device=DEV, dtype=BF16)
                  for _ in range(2)]
        state.update(k=k, v=v, cache=(*packed, *params),
                     start=torch.tensor(case["length"] - new, device=DEV, dtype=torch.int64))
        return state
    # a cache filled to its capacity: what follows the valid tokens is left from before
    k, v = _rows(g, case, capacity)
    (kc, kp), (vc, vp) = _quantise(k, case["bits"], False), _quantise(v, case["bits"], True)
    state["cache"] = (_pack(kc, case["bits"]), _pack(vc, case["bits"]), kp, vp)
    lengths = _lengths(case)
    state["valid"] = torch.tensor(lengths, device=DEV, dtype=torch.int64)
    if case["kind"] in ("decode", "prompt"):
        state["q"] = _normal(g, case["batch"], case["heads"], new, case["dim"]).to(BF16)
    if case["gate"]:
        width = 2 * case["dim"] * (case["heads"] + case["kv_heads"])
        state["gate"] = _normal(g, case["batch"], 1, width).to(BF16)
    return state


# ------------------------------------------------------------------ plain form
def _grouped(x, values):
    """[..., dim] as [..., groups, 64] (keys) or [..., 16, groups, 4] (values),
    and the axes that a group spans."""
    groups = x.shape[-1] // 64
    if values:
        return x.unflatten(-1, (16, groups, 4)), (-3, -1)
    return x.unflatten(-1, (groups, 64)), (-1,)


def _quantise(x, bits, values):
    """Codes [..., tokens, dim] and params [..., groups, tokens, 2] of bf16 rows."""
    top = 2**bits - 1
    y, axes = _grouped(x.float(), values)
    low, high = y.amin(axes, keepdim=True), y.amax(axes, keepdim=True)
    step = ((high - low) / top).to(BF16)
    # in 64 bits: a code next to a border has to fall on its own side of it
    codes = torch.where(step > 0, (y.double() - low.double()) / step.double(), 0.0).round().clamp(0, top)
    params = torch.stack((step, low.to(BF16)), -1)
    params = params.flatten(-len(axes) - 2 if values else -3, -2).unflatten(-2, (-1,))
    return codes.to(torch.uint8).flatten(-3 if values else -2), params.transpose(-2, -3).contiguous()


def _pack(codes, bits):
    if bits == 8:
        return codes
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _values(packed, params, bits, values):
    """The values that codes stand for, fp32 [..., tokens, dim]."""
    if bits == 4:
        packed = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    y, axes = _grouped(packed.float(), values)
    p = params.float().transpose(-2, -3)  # [..., tokens, groups, 2]
    p = p[..., None, :, None, :] if values else p[..., None, :]
    return (p[..., 1] + p[..., 0] * y).flatten(-len(axes) - 1)


def _attend(state):
    case = state["case"]
    new, heads, kv_heads = case["new"], case["heads"], case["kv_heads"]
    kq, vq, kp, vp = state["cache"]
    n = int(case["length"])  # the longest sequence
    k = _values(kq[:, :, :n], kp[:, :, :, :n], case["bits"], False)
    v = _values(vq[:, :, :n], vp[:, :, :, :n], case["bits"], True)
    q = state["q"].float().unflatten(1, (kv_heads, heads // kv_heads)).flatten(2, 3)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * state["scale"]
    # query row i of a sequence of n tokens sees the tokens 0 .. n - new + i
    last = state["valid"][:, None] - new + torch.arange(new, device=DEV)
    seen = torch.arange(n, device=DEV) <= last[..., None]  # [batch, new, n]
    seen = seen[:, None, None].expand(-1, 1, heads // kv_heads, -1, -1).flatten(2, 3)
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    out = out.unflatten(2, (heads // kv_heads, new)).flatten(1, 2).transpose(1, 2).flatten(2)
    if case["gate"]:
        out = out * torch.sigmoid(_gate(state).float())
    return out.to(BF16)


def _gate(state):
    """The gate of every head from the packed row [q | gate] x heads, k, v."""
    d, heads = state["case"]["dim"], state["case"]["heads"]
    return state["gate"][..., : 2 * heads * d].unflatten(-1, (heads, 2, d))[..., 1, :].flatten(-2)


def _plain(state):
    case = state["case"]
    bits = case["bits"]
    if case["kind"] == "store":
        (kc, kp), (vc, vp) = _quantise(state["k"], bits, False), _quantise(state["v"], bits, True)
        kq, vq = _pack(kc, bits), _pack(vc, bits)
        return _values(kq, kp, bits, False).to(BF16), _values(vq, vp, bits, True).to(BF16)
    if case["kind"] == "load":
        kq, vq, kp, vp = state["cache"]
        n = case["length"]
        return (_values(kq[:, :, :n], kp[:, :, :, :n], bits, False).to(BF16),
                _values(vq[:, :, :n], vp[:, :, :, :n], bits, True).to(BF16))
    return _attend(state)


# ------------------------------------------------------------------ a pass
def run(state):
    if not own:
        return _plain(state)
    from ppu_amd import kernels as K

    case = state["case"]
    cache = K.QuantizedKV(*state["cache"])
    if case["kind"] == "store":
        K.kv_cache_quantize(state["k"], state["v"], cache, cache_start=state["start"])
        return K.kv_cache_dequantize(cache, case["new"], start=case["length"] - case["new"])
    if case["kind"] == "load":
        return K.kv_cache_dequantize(cache, case["length"])
    if case["kind"] == "decode":
        return K.gqa_decode_attention_q(state["q"], cache, state["valid"], state["scale"],
                                        packed_gate=state.get("gate"))
    return K.gqa_prefill_attention_q(state["q"], cache, state["scale"], valid_length=state["valid"])


# ------------------------------------------------------------------ 64 bits
def _exact_groups(dim, values):
    """The dims of every group, one row of 64 a group."""
    d = torch.arange(dim, device=DEV)
    group = (d % (dim // 16)) // 4 if values else d // 64
    return torch.stack([d[group == g] for g in range(dim // 64)])


def _exact_values(packed, params, bits, values):
    packed = packed.long()
    dim = packed.shape[-1] * 8 // bits
    out = torch.empty(*packed.shape[:-1], dim, device=DEV, dtype=torch.float64)
    for g, dims in enumerate(_exact_groups(dim, values)):
        code = packed[..., dims * bits // 8]
        if bits == 4:
            code = torch.where(dims % 2 == 1, code // 16, code % 16)
        p = params[:, :, g].double()
        out[..., dims] = p[..., 1:] + p[..., :1] * code.double()
    return out


def _exact_store(x, bits, values):
    x = x.double()
    out = torch.empty(x.shape, device=DEV, dtype=torch.float64)
    for dims in _exact_groups(x.shape[-1], values):
        y = x[..., dims]
        low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        step = ((high - low) / (2**bits - 1)).float().to(BF16).double()
        code = torch.floor((y - low) / step.clamp_min(1e-300))
        half = (y - low) - (code + 0.5) * step  # its sign says on which side of the border y lies
        code = code + ((half > 0) | ((half == 0) & (code % 2 == 1)))
        out[..., dims] = low + step * code.clamp(max=2**bits - 1)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    bits = case["bits"]
    if case["kind"] == "store":
        return _exact_store(state["k"], bits, False), _exact_store(state["v"], bits, True)
    kq, vq, kp, vp = state["cache"]
    if case["kind"] == "load":
        n = case["length"]
        return (_exact_values(kq[:, :, :n], kp[:, :, :, :n], bits, False),
                _exact_values(vq[:, :, :n], vp[:, :, :, :n], bits, True))
    new, heads, kv_heads, d = case["new"], case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(case["batch"], new, heads, d, device=DEV, dtype=torch.float64)
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        for kvh in range(kv_heads):
            at = slice(b, b + 1), slice(kvh, kvh + 1)
            k = _exact_values(kq[at][:, :, :n], kp[at][:, :, :, :n], bits, False)[0, 0]
            v = _exact_values(vq[at][:, :, :n], vp[at][:, :, :, :n], bits, True)[0, 0]
            for h in range(kvh * heads // kv_heads, (kvh + 1) * heads // kv_heads):
                for i in range(0, new, 1024):
                    rows = state["q"][b, h, i : i + 1024].double()
                    s = rows @ k.t() * state["scale"]
                    row = torch.arange(i, i + rows.shape[0], device=DEV)[:, None]
                    s[torch.arange(n, device=DEV) > n - new + row] = -math.inf
                    out[b, i : i + 1024, h] = torch.softmax(s, -1) @ v
    if case["gate"]:
        packed = state["gate"].double()[:, 0]
        for h in range(heads):
            out[:, 0, h] /= 1 + torch.exp(-packed[:, (2 * h + 1) * d : (2 * h + 2) * d])
    return out.flatten(2)
