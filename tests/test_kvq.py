"""The K/V cache in 4 or 8 bits: write, read back, decode and prompt attention
against oracle/kvq.py (64-bit), and the refusals (host side, CPU).

Tolerances. Codes and params are equal; values read back are the bf16 rounding
of the 64-bit value (equal). An attention output o = sum_t p_t v_t, with s =
sum_t p_t v_t^2 (so sum_t p_t |v_t| <= sqrt(s)), is rounded to bf16 (at most
2^-8 |o|) and its weights may be held in bf16 (each off by at most 2^-8 of
itself: at most 2^-8 sqrt(s) together): 2^-8 (|o| + sqrt(s)) for decode. A
prompt's keys and values may be rounded to bf16 too. A rounding error is spread
over its half step, variance at most 2^-16 / 3 of the square; with scores of
scale dim^-1/2, queries of variance 1 and keys of variance 2, a score's is 2^-16
* 2 / 3. Together the variance is at most 2^-16 (o^2 / 3 + s / 3 (weights) + s /
3 (values) + 2 s / 3 (scores)), as sum p^2 v^2 <= s: the root mean square of all
errors stays below 2^-8 sqrt(mean(o^2 / 3 + 4 s / 3)), and each within 6 of its
standard deviations.
"""

from __future__ import annotations

import random

import pytest
import torch

from oracle import kvq as ref
from ppu_amd import _lib
from ppu_amd import kernels as K
from tests.conftest import KERNEL_SEED, gen

BF = torch.bfloat16
gpu_test = pytest.mark.gpu


def rows(g, *shape):
    """Rows with channels of unequal offset, bf16."""
    return (torch.randn(*shape, generator=g) + torch.randn(shape[-1], generator=g)).to(BF)


def cache_of(k, v, bits, capacity, junk=None):
    """The oracle's cache of ``k, v [B, KVH, n, D]`` with ``capacity`` positions;
    ``junk``: the params of the positions after them, their codes all ones."""
    out = []
    for x, values in ((k, False), (v, True)):
        codes, params = ref.quantise(x, bits, values)
        full = torch.full((*x.shape[:2], capacity, x.shape[3]), 2**bits - 1, dtype=torch.uint8)
        full[:, :, : x.shape[2]] = codes
        par = torch.full((*params.shape[:3], capacity, 2), 0.0 if junk is None else junk, dtype=BF)
        par[:, :, :, : x.shape[2]] = params
        out.append((ref.pack(full, bits).contiguous(), par))
    return K.QuantizedKV(out[0][0], out[1][0], out[0][1], out[1][1])


def to(cache, device):
    return K.QuantizedKV(*(t.to(device) for t in cache))


def values_of(cache):
    """The 64-bit keys and values of a cache."""
    bits = cache.bits
    return (ref.dequantise(ref.unpack(cache.keys, bits), cache.key_params, False),
            ref.dequantise(ref.unpack(cache.values, bits), cache.value_params, True))


def check_attention(got, q, cache, starts, scale, prompt=False, gate=None, skip=None):
    """``got [B, L, H*D]`` bf16 against the oracle on the cache's values;
    ``skip``: an index of rows left out."""
    kd, vd = values_of(cache)
    want, square = ref.attend(q, kd, vd, starts, scale), ref.attend(q, kd, vd.square(), starts, scale)
    if gate is not None:
        want, square = want * gate, square * gate.square()
    got = got.double().cpu()
    if skip is not None:
        for t in (got, want, square):
            t[skip] = 0
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    if prompt:
        var = want.square() / 3 + square * (4 / 3)
        assert err.square().mean().sqrt() <= 2**-8 * var.mean().sqrt()
        bound = 6 * 2**-8 * var.sqrt()
    else:
        bound = 2**-8 * (want.abs() + square.sqrt())
    worst = (err / (bound + 1e-30)).max().item()
    assert worst <= 1.0, f"error {worst:.3f} of its bound"


# ------------------------------------------------------------------ the oracle (CPU)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_oracle_codes_are_nearest(bits, dim):
    """No other code of the group is nearer; the group's least value is exact."""
    g = gen(KERNEL_SEED + 900)
    x = rows(g, 1, 1, 5, dim)
    for values in (False, True):
        codes, params = ref.quantise(x, bits, values)
        back = ref.dequantise(codes, params, values)
        for gi, dims in enumerate(ref.groups(dim, values)):
            low, step = params[0, 0, gi, :, 1].double(), params[0, 0, gi, :, 0].double()
            grid = low[:, None] + step[:, None] * torch.arange(2**bits)
            best = (x[0, 0][:, dims].double()[..., None] - grid[:, None]).abs().amin(-1)
            assert torch.equal((x[0, 0][:, dims].double() - back[0, 0][:, dims]).abs(), best)
            assert torch.equal(low, x[0, 0][:, dims].double().amin(-1))


def test_oracle_known_group():
    x = torch.zeros(64, dtype=BF)
    x[:4] = torch.tensor([-1.5, 13.5, 1.0, 2.0])  # step 1: ties of -1.5 + n + 1/2 go to the even code
    codes, params = ref.quantise(x.view(1, 1, 1, 64), 4, False)
    assert params.flatten().tolist() == [1.0, -1.5]
    assert codes.flatten()[:5].tolist() == [0, 15, 2, 4, 2]
    assert ref.unpack(ref.pack(codes, 4), 4).equal(codes)


def test_oracle_group_layout():
    assert ref.groups(256, True)[1][:8].tolist() == [4, 5, 6, 7, 20, 21, 22, 23]
    assert ref.groups(128, True)[1][:8].tolist() == [4, 5, 6, 7, 12, 13, 14, 15]
    assert ref.groups(64, True)[0].tolist() == list(range(64))
    assert ref.groups(256, False)[2].tolist() == list(range(128, 192))


# ------------------------------------------------------------------ refusals (CPU)
def _empty(bits=4, batch=2, heads=2, capacity=64, dim=128):
    return K.quantized_kv_cache(batch, heads, capacity, dim, bits=bits, device="cpu")


def test_cache_form():
    c = K.quantized_kv_cache(2, 3, 33, 256, bits=8, device="cpu")
    assert (c.capacity, c.head_dim, c.bits) == (64, 256, 8)
    assert c.keys.shape == (2, 3, 64, 256) and c.key_params.shape == (2, 3, 4, 64, 2)
    for bad in (dict(bits=2), dict(head_dim=96), dict(capacity=0), dict(batch=0), dict(kv_heads=0)):
        args = {"batch": 1, "kv_heads": 1, "capacity": 32, "head_dim": 64, **bad}
        with pytest.raises(ValueError):
            K.quantized_kv_cache(**args, device="cpu")


def test_refused_caches():
    c = _empty()
    q = torch.zeros(2, 4, 1, 128, dtype=BF)
    n = torch.ones(1, dtype=torch.int64)
    bad = {
        "K as V": c._replace(values=c.values[:, :1]),
        "K as V ": c._replace(key_params=c.key_params[0]),
        "uint8 codes": c._replace(keys=c.keys.to(torch.int8)),
        "bfloat16 params": c._replace(value_params=c.value_params.float(), key_params=c.key_params.float()),
        "4 or 8 bits": c._replace(keys=c.keys[..., :32], values=c.values[..., :32]),
        "do not match": c._replace(key_params=c.key_params[:, :1], value_params=c.value_params[:, :1]),
        "multiple of 32": c._replace(keys=c.keys[:, :, :33], values=c.values[:, :, :33],
                                     key_params=c.key_params[..., :33, :], value_params=c.value_params[..., :33, :]),
        "contiguous": c._replace(keys=c.keys.transpose(0, 1).contiguous().transpose(0, 1)),
    }
    for message, cache in bad.items():
        for call in (lambda: K.gqa_decode_attention_q(q, cache, n, 1.0),
                     lambda: K.gqa_prefill_attention_q(q, cache, 1.0),
                     lambda: K.kv_cache_quantize(q[:, :2], q[:, :2], cache),
                     lambda: K.kv_cache_dequantize(cache, 1)):
            with pytest.raises(ValueError, match=message.strip()):
                call()
    odd = torch.zeros(c.keys.numel() + 1, dtype=torch.uint8)[1:].view(c.keys.shape)
    if odd.data_ptr() % 16:
        with pytest.raises(ValueError, match="aligned"):
            K.kv_cache_dequantize(c._replace(keys=odd), 1)


def test_refused_operands():
    c = _empty()
    x = torch.zeros(2, 2, 3, 128, dtype=BF)
    n2 = torch.ones(2, dtype=torch.int64)
    refused = [
        ("as the cache", lambda: K.kv_cache_quantize(x[:1], x[:1], c)),
        ("as the cache", lambda: K.kv_cache_quantize(x, x[:, :, :2], c)),
        ("as the cache", lambda: K.kv_cache_quantize(x[..., :64], x[..., :64], c)),
        ("bfloat16", lambda: K.kv_cache_quantize(x.half(), x.half(), c)),
        ("exceed", lambda: K.kv_cache_quantize(x, x, c, start=62)),
        ("exceed", lambda: K.kv_cache_quantize(x, x, c, start=-1)),
        ("exclusive", lambda: K.kv_cache_quantize(x, x, c, start=1, cache_start=n2)),
        ("int64", lambda: K.kv_cache_quantize(x, x, c, cache_start=n2.int())),
        ("int64", lambda: K.kv_cache_quantize(x, x, c, cache_start=torch.ones(3, dtype=torch.int64))),
        ("exceed", lambda: K.kv_cache_dequantize(c, 65)),
        ("exceed", lambda: K.kv_cache_dequantize(c, 1, start=64)),
        ("exceed", lambda: K.kv_cache_dequantize(c, -1)),
        ("head layout", lambda: K.gqa_decode_attention_q(torch.zeros(2, 3, 1, 128, dtype=BF), c, n2, 1.0)),
        ("head layout", lambda: K.gqa_decode_attention_q(torch.zeros(1, 4, 1, 128, dtype=BF), c, n2, 1.0)),
        ("head layout", lambda: K.gqa_prefill_attention_q(torch.zeros(2, 4, 1, 64, dtype=BF), c, 1.0)),
        ("expects q", lambda: K.gqa_decode_attention_q(x, c, n2, 1.0)),
        ("bfloat16", lambda: K.gqa_decode_attention_q(x[:, :, :1].float().contiguous(), c, n2, 1.0)),
        ("contiguous", lambda: K.gqa_prefill_attention_q(x.transpose(1, 2).contiguous().transpose(1, 2), c, 1.0)),
        ("int64", lambda: K.gqa_decode_attention_q(x[:, :, :1].contiguous(), c, n2.float(), 1.0)),
        ("gate", lambda: K.gqa_decode_attention_q(x[:, :, :1].contiguous(), c, n2, 1.0,
                                                  packed_gate=torch.zeros(2, 1, 511, dtype=BF))),
        ("range", lambda: K.gqa_prefill_attention_q(x, c, 1.0, kv_start=62)),
        ("range", lambda: K.gqa_prefill_attention_q(torch.zeros(2, 2, 65, 128, dtype=BF), c, 1.0,
                                                    valid_length=n2)),
        ("exclusive", lambda: K.gqa_prefill_attention_q(x, c, 1.0, kv_start=1, valid_length=n2)),
        ("needs valid_length", lambda: K.gqa_prefill_attention_q(x, c, 1.0, length_is_start=True)),
        # sound operands on the CPU: there is no CPU path
        ("GPU", lambda: K.kv_cache_quantize(x, x, c)),
        ("GPU", lambda: K.kv_cache_dequantize(c, 3)),
        ("GPU", lambda: K.gqa_decode_attention_q(x[:, :, :1].contiguous(), c, n2, 1.0)),
        ("GPU", lambda: K.gqa_prefill_attention_q(x, c, 1.0)),
    ]
    for message, call in refused:
        with pytest.raises(ValueError, match=message):
            call()


def test_refused_entries():
    """The C entries refuse sizes, and null or unaligned buffers, before a launch."""
    lib = _lib.load()
    p = [4096] * 4  # never read: every call below is refused
    ok = dict(B=1, KVH=2, L=3, D=128, bits=4, C=64)

    def write(k=4096, k_sl=128, n_start=0, start_dev=None, **kw):
        a = {**ok, **kw}
        return lib.q35_kv_quantize(k, 768, 384, k_sl, 4096, 768, 384, 128, *p, start_dev, n_start, 0, a["B"],
                                   a["KVH"], a["L"], a["D"], a["bits"], a["C"], None)

    def read(k=4096, start=0, **kw):
        a = {**ok, **kw}
        return lib.q35_kv_dequantize(*p, k, 4096, start, a["B"], a["KVH"], a["L"], a["D"], a["bits"], a["C"], None)

    def attend(q=4096, QH=4, n_len=0, length=None, gate=None, ws=None, floats=0, gate_stride=1024, **kw):
        a = {**ok, **kw}
        return lib.q35_gqa_attention_kvq(q, *p, length, n_len, 0, gate, gate_stride, 1.0, 4096, ws, floats, a["B"], QH,
                                         a["KVH"], a["L"], a["D"], a["bits"], a["C"], None)

    for f in (write, read, attend):
        for bad in (dict(D=96), dict(bits=2), dict(C=33), dict(C=0), dict(KVH=0), dict(L=-1), dict(B=-1),
                    dict(D=256, bits=8, C=1 << 24)):
            assert f(**bad) == 1, (f.__name__, bad)
    assert write(k=None) == 1 and write(k=4104) == 1 and write(k_sl=124) == 1
    assert write(start_dev=4096, n_start=2) == 1
    assert write(B=1 << 20, L=1 << 20) == 1
    assert read(k=None) == 1 and read(k=4104) == 1 and read(start=62) == 1 and read(start=-1) == 1
    assert attend(q=None) == 1 and attend(q=4104) == 1 and attend(QH=3) == 1 and attend(QH=0) == 1
    assert attend(length=4096, n_len=2) == 1 and attend(gate=4096) == 1
    assert attend(gate=4096, L=1, gate_stride=1026) == 1 and attend(gate=4096, L=1, gate_stride=-4) == 1
    assert write(B=1 << 16) == 1 and read(B=1 << 16) == 1 and read(KVH=1 << 15) == 1
    assert lib.q35_gqa_attention_kvq_workspace(1, 3, 2, 1, 128, 4, 64) == -1
    assert lib.q35_gqa_attention_kvq_workspace(1, 4, 2, 1, 96, 4, 64) == -1


# ------------------------------------------------------------------ write and read back
FORMS = [(4, 64), (4, 128), (4, 256), (8, 64), (8, 128), (8, 256)]


@gpu_test
@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("batch,heads,length,start", [(1, 1, 1, 0), (2, 3, 37, 5), (1, 2, 64, 32)])
def test_write_and_read_back(gpu, bits, dim, batch, heads, length, start):
    """Codes, params and values are the oracle's; positions around stay."""
    g = gen(KERNEL_SEED + 901)
    k, v = rows(g, batch, heads, length, dim), rows(g, batch, heads, length, dim)
    cache = K.quantized_kv_cache(batch, heads, 96, dim, bits=bits, device=gpu)
    for t in cache:
        t.fill_(7)
    K.kv_cache_quantize(k.to(gpu), v.to(gpu), cache, start=start)
    kb, vb = K.kv_cache_dequantize(cache, length, start=start)
    inside = torch.zeros(96, dtype=torch.bool)
    inside[start : start + length] = True
    for x, got, packed, params, values in ((k, kb, cache.keys, cache.key_params, False),
                                           (v, vb, cache.values, cache.value_params, True)):
        codes, want = ref.quantise(x, bits, values)
        packed, params = packed.cpu(), params.cpu()
        assert torch.equal(packed[:, :, inside], ref.pack(codes, bits))
        assert torch.equal(params[..., inside, :], want)
        assert (packed[:, :, ~inside] == 7).all() and (params[..., ~inside, :] == 7).all()
        assert torch.equal(got.cpu(), ref.dequantise(codes, want, values).to(BF))


@gpu_test
@pytest.mark.parametrize("bits", [4, 8])
def test_write_special_groups(gpu, bits):
    """Constant, tiny, huge and non-finite groups, ties, a least value far
    below the step, signed zeros."""
    g = gen(KERNEL_SEED + 902)
    x = rows(g, 1, 1, 12, 256)
    x[0, 0, 0] = 3.25
    x[0, 0, 1] = 0.0
    x[0, 0, 2] = torch.linspace(-3.3e38, 3.3e38, 256).to(BF)
    x[0, 0, 3] = (torch.arange(256) % 16 * 2.0**-132).to(BF)
    x[0, 0, 4, 70] = float("inf")
    x[0, 0, 5, 9] = float("-inf")
    x[0, 0, 6, 200] = float("nan")
    x[0, 0, 7] = (torch.arange(256) % 31 * 0.5).to(BF)  # step 1 in 4 bits: every other value a tie
    x[0, 0, 8] = (torch.arange(256) % 64 * 0.25).to(BF)
    x[0, 0, 8, ::64] = -(2.0**-30)  # no tie by 2^-30, one in 32 bits
    x[0, 0, 9] = torch.where(torch.arange(256) % 2 == 0, -0.0, 0.0).to(BF)
    x[0, 0, 10] = 2.0**-133
    x[0, 0, 10, ::5] = 0.0
    x[0, 0, 11] = (torch.arange(256) % 8 * 2.0**-120).to(BF)
    cache = K.quantized_kv_cache(1, 1, 32, 256, bits=bits, device=gpu)
    K.kv_cache_quantize(x.to(gpu), x.to(gpu), cache)
    got = K.kv_cache_dequantize(cache, 12)
    for packed, params, back, values in ((cache.keys, cache.key_params, got[0], False),
                                         (cache.values, cache.value_params, got[1], True)):
        codes, want = ref.quantise(x, bits, values)
        torch.testing.assert_close(params[:, :, :, :12].cpu(), want, rtol=0, atol=0, equal_nan=True)
        assert torch.equal(packed[:, :, :12].cpu(), ref.pack(codes, bits))
        torch.testing.assert_close(back.cpu(), ref.dequantise(codes, want, values).to(BF), rtol=0, atol=0,
                                   equal_nan=True)


@gpu_test
@pytest.mark.parametrize("bits", [4, 8])
def test_write_many_values(gpu, bits):
    """Half a million values, among them narrow ones whose quotients crowd the
    borders: every code as decided in 64 bits."""
    g = gen(KERNEL_SEED + 903)
    x = torch.randn(1, 1, 2048, 256, generator=g)
    x[:, :, 1024:] = torch.randint(-40, 41, (1, 1, 1024, 256), generator=g) / 32
    x = x.to(BF)
    cache = K.quantized_kv_cache(1, 1, 2048, 256, bits=bits, device=gpu)
    K.kv_cache_quantize(x.to(gpu), x.to(gpu), cache)
    for packed, params, values in ((cache.keys, cache.key_params, False), (cache.values, cache.value_params, True)):
        codes, want = ref.quantise(x, bits, values)
        assert torch.equal(params.cpu(), want)
        assert torch.equal(packed.cpu(), ref.pack(codes, bits))


@gpu_test
@pytest.mark.parametrize("bits,dim", FORMS)
def test_write_wide_values(gpu, bits, dim):
    """Values of unlike exponents in a group, groups from the smallest steps to
    the largest, few distinct values (many on the border of two codes)."""
    g = gen(KERNEL_SEED + 936)
    n = 96
    x = torch.randn(3, 1, n, dim, generator=g)
    x[0] *= torch.exp2(torch.randint(-30, 1, (1, n, dim), generator=g).float())  # unlike exponents
    x[1] *= torch.exp2(torch.linspace(-125, 124, n))[:, None]  # every magnitude
    x[2] = torch.randint(-40, 41, (1, n, dim), generator=g) * torch.exp2(torch.randint(-6, 7, (1, n, 1), generator=g).float())
    k = x.to(BF)
    v = k.flip(2).contiguous()
    cache = to(K.quantized_kv_cache(3, 1, n, dim, bits=bits, device="cpu"), gpu)
    K.kv_cache_quantize(k.to(gpu), v.to(gpu), cache)
    want = cache_of(k, v, bits, n)
    for got, w in zip(cache, want):
        assert torch.equal(got.cpu(), w)


@gpu_test
@pytest.mark.parametrize("dim", [64, 256])
def test_write_strides_and_starts(gpu, dim):
    """Token-major views, slices of a packed projection, unaligned rows, rows of
    stride 0, a start per sequence, and positions outside the cache."""
    g = gen(KERNEL_SEED + 904)
    batch, heads, length, capacity = 3, 2, 9, 32
    packed = rows(g, batch, length, heads * dim * 2 + 8)
    views = [
        packed[..., : heads * dim].unflatten(-1, (heads, dim)).transpose(1, 2),
        packed[..., 8 : 8 + heads * dim].unflatten(-1, (heads, dim)).transpose(1, 2),
        packed[..., 1 : 1 + heads * dim].unflatten(-1, (heads, dim)).transpose(1, 2),
        packed[..., : 2 * heads * dim : 2].unflatten(-1, (heads, dim)).transpose(1, 2),
        packed[:1, :1, :dim].unsqueeze(1).expand(batch, heads, length, dim),
    ]
    starts = torch.tensor([0, -4, capacity - 3])
    on_gpu = packed.to(gpu)
    for view in views:
        moved = on_gpu.as_strided(view.shape, view.stride(), view.storage_offset())
        cache = K.quantized_kv_cache(batch, heads, capacity, dim, device=gpu)
        K.kv_cache_quantize(moved, moved, cache, cache_start=starts.to(gpu))
        for back, values in zip(K.kv_cache_dequantize(cache, capacity), (False, True)):
            want = torch.zeros(batch, heads, capacity, dim, dtype=BF)
            rows_of = ref.dequantise(*ref.quantise(view, 4, values), values).to(BF)
            for b in range(batch):
                for t in range(length):
                    pos = int(starts[b]) + t
                    if 0 <= pos < capacity:
                        want[b, :, pos] = rows_of[b, :, t]
            assert torch.equal(back.cpu(), want)


@gpu_test
def test_empty_calls(gpu):
    cache = K.quantized_kv_cache(2, 1, 32, 64, device=gpu)
    none = torch.empty(2, 1, 0, 64, device=gpu, dtype=BF)
    K.kv_cache_quantize(none, none, cache)
    k, v = K.kv_cache_dequantize(cache, 0)
    assert k.shape == v.shape == (2, 1, 0, 64)
    assert K.gqa_prefill_attention_q(none, cache, 1.0).shape == (2, 0, 64)


# ------------------------------------------------------------------ attention
# heads: groups of 1, 2, 3, 4, 7, 8, 12, 16 and 20 query heads
HEADS = [(1, 1), (4, 2), (6, 2), (8, 2), (7, 1), (8, 1), (12, 1), (16, 1), (20, 1)]


@gpu_test
@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_decode_head_layouts(gpu, bits, dim, heads, kv_heads):
    g = gen(KERNEL_SEED + 905)
    n, capacity = 203, 224
    k, v = rows(g, 1, kv_heads, n, dim), rows(g, 1, kv_heads, n, dim)
    cache = cache_of(k, v, bits, capacity, junk=float("nan"))
    q = torch.randn(1, heads, 1, dim, generator=g).to(BF)
    got = K.gqa_decode_attention_q(q.to(gpu), to(cache, gpu), torch.tensor([n], device=gpu), dim**-0.5)
    check_attention(got, q, cache, [n - 1], dim**-0.5)


@gpu_test
@pytest.mark.parametrize("bits,dim", [(4, 256), (8, 128), (4, 64)])
@pytest.mark.parametrize("lengths", [[1, 2, 15], [16, 17, 31], [32, 33, 64], [0, 127, 128], [129, 160, 161],
                                     [-3, 1000, 1], [511, 512, 513]])
def test_decode_lengths(gpu, bits, dim, lengths):
    """Unequal lengths in a batch, with ones that are empty, negative or past
    the capacity; what lies behind a sequence's end is NaN."""
    g = gen(KERNEL_SEED + 906)
    capacity = 544
    k, v = rows(g, 3, 2, capacity, dim), rows(g, 3, 2, capacity, dim)
    cache = cache_of(k, v, bits, capacity)
    for b, n in enumerate(lengths):
        cache.key_params[b, :, :, max(n, 0) :] = float("nan")
        cache.value_params[b, :, :, max(n, 0) :] = float("inf")
    q = torch.randn(3, 8, 1, dim, generator=g).to(BF)
    got = K.gqa_decode_attention_q(q.to(gpu), to(cache, gpu), torch.tensor(lengths, device=gpu), dim**-0.5)
    check_attention(got, q, cache, [n - 1 for n in lengths], dim**-0.5)


@gpu_test
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_gate(gpu, bits):
    """The gate of each head's own half of the packed row, a row per sequence."""
    g = gen(KERNEL_SEED + 907)
    batch, heads, kv_heads, dim, n = 2, 8, 2, 256, 77
    cache = cache_of(rows(g, batch, kv_heads, n, dim), rows(g, batch, kv_heads, n, dim), bits, 96)
    q = torch.randn(batch, heads, 1, dim, generator=g).to(BF)
    packed = (2 * torch.randn(batch, 1, 2 * dim * (heads + kv_heads), generator=g)).to(BF)
    args = q.to(gpu), to(cache, gpu), torch.tensor(n, device=gpu), dim**-0.5
    got = K.gqa_decode_attention_q(*args, packed_gate=packed.to(gpu))
    gate = packed.double()[..., : 2 * heads * dim].unflatten(-1, (heads, 2, dim))[..., 1, :].flatten(2)
    check_attention(got, q, cache, [n - 1] * batch, dim**-0.5, gate=torch.sigmoid(gate))


@gpu_test
def test_decode_gate_many_heads(gpu):
    """More than 128 heads on one KV head in a roomy cache, with a gate: one
    token is the decode kernel's at any size."""
    g = gen(KERNEL_SEED + 930)
    heads, dim, n = 144, 64, 100
    cache = cache_of(rows(g, 1, 1, n, dim), rows(g, 1, 1, n, dim), 4, 128, junk=float("nan"))
    q = torch.randn(1, heads, 1, dim, generator=g).to(BF)
    packed = (2 * torch.randn(1, 1, 2 * dim * heads, generator=g)).to(BF)
    roomier = wide(cache, roomy(heads, 1, dim, 1), gpu, float("nan"))
    got = K.gqa_decode_attention_q(q.to(gpu), roomier, torch.tensor(n, device=gpu), dim**-0.5, packed_gate=packed.to(gpu))
    gate = packed.double().unflatten(-1, (heads, 2, dim))[..., 1, :].flatten(2)
    check_attention(got, q, cache, [n - 1], dim**-0.5, gate=torch.sigmoid(gate))


@gpu_test
@pytest.mark.parametrize("bits,dim", [(4, 256), (8, 128), (4, 64)])
@pytest.mark.parametrize("scale_q,scale_k,scale_v",
                         [(1e20, 1e-20, 1e30), (1e-25, 1e25, 1e-12), (2.0**-100, 2.0**100, 1.0)])
def test_decode_magnitudes(gpu, bits, dim, scale_q, scale_k, scale_v):
    """Far from 1 each, the scores as ever: no power of two is lost."""
    g = gen(KERNEL_SEED + 931)
    n = 301
    k = (rows(g, 1, 2, n, dim).float() * scale_k).to(BF)
    v = (rows(g, 1, 2, n, dim).float() * scale_v).to(BF)
    cache = cache_of(k, v, bits, 320, junk=float("nan"))
    q = (torch.randn(1, 8, 1, dim, generator=g) * scale_q).to(BF)
    got = K.gqa_decode_attention_q(q.to(gpu), to(cache, gpu), torch.tensor(n, device=gpu), dim**-0.5)
    check_attention(got, q, cache, [n - 1], dim**-0.5)


@gpu_test
@pytest.mark.parametrize("bits,dim,length", [(4, 256, 1), (8, 256, 1), (4, 128, 2), (8, 64, 1)])
@pytest.mark.parametrize("lengths", [[4000, 3, 0, 33, 129, 5, 1, 64, 2], [1, 2500], [700] * 3 + [0] * 5])
def test_decode_unequal_lengths(gpu, bits, dim, length, lengths):
    """Sequences that share a KV head's workgroups: one long among short and
    empty ones."""
    g = gen(KERNEL_SEED + 932)
    batch, capacity = len(lengths), 4032
    cache = cache_of(rows(g, batch, 2, max(lengths), dim), rows(g, batch, 2, max(lengths), dim), bits, capacity)
    q = torch.randn(batch, 6, length, dim, generator=g).to(BF)
    got = K.gqa_prefill_attention_q(q.to(gpu), to(cache, gpu), dim**-0.5, valid_length=torch.tensor(lengths, device=gpu))
    check_attention(got, q, cache, [n - length for n in lengths], dim**-0.5)


@gpu_test
def test_decode_large_batches(gpu):
    """More sequences than a wave has lanes, lengths from 0 on."""
    g = gen(KERNEL_SEED + 933)
    batch, dim = 70, 64
    lengths = [(7 * i) % 97 for i in range(batch)]
    cache = cache_of(rows(g, batch, 1, 96, dim), rows(g, batch, 1, 96, dim), 4, 96)
    q = torch.randn(batch, 3, 1, dim, generator=g).to(BF)
    got = K.gqa_decode_attention_q(q.to(gpu), to(cache, gpu), torch.tensor(lengths, device=gpu), dim**-0.5)
    check_attention(got, q, cache, [n - 1 for n in lengths], dim**-0.5)


@gpu_test
@pytest.mark.parametrize("bits,dim", [(4, 256), (8, 256), (4, 128), (8, 64)])
def test_decode_long(gpu, bits, dim):
    """A long cache: many splits and several tiles of every wave."""
    g = gen(KERNEL_SEED + 908)
    n, capacity = 40961, 41024
    k, v = rows(g, 1, 1, n, dim), rows(g, 1, 1, n, dim)
    cache = cache_of(k, v, bits, capacity, junk=float("nan"))
    q = torch.randn(1, 4, 1, dim, generator=g).to(BF)
    got = K.gqa_decode_attention_q(q.to(gpu), to(cache, gpu), torch.tensor([n], device=gpu), dim**-0.5)
    check_attention(got, q, cache, [n - 1], dim**-0.5)


@gpu_test
@pytest.mark.parametrize("scale", [4.0, 0.0, -0.5])
def test_decode_scores(gpu, scale):
    """Peaked, flat and reversed scores; keys that grow along the cache move the
    running maximum in every tile."""
    g = gen(KERNEL_SEED + 909)
    n, dim = 700, 128
    k = (rows(g, 1, 1, n, dim).float() * torch.linspace(0.1, 3, n)[:, None]).to(BF)
    v = rows(g, 1, 1, n, dim)
    cache = cache_of(k, v, 4, 704)
    q = torch.randn(1, 3, 1, dim, generator=g).to(BF)
    got = K.gqa_decode_attention_q(q.to(gpu), to(cache, gpu), torch.tensor([n], device=gpu), scale)
    check_attention(got, q, cache, [n - 1], scale)


@gpu_test
@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 1), (20, 1)])
@pytest.mark.parametrize("length,start", [(2, 0), (5, 60), (17, 0), (33, 31), (70, 100)])
def test_prefill_sizes(gpu, bits, dim, heads, kv_heads, length, start):
    g = gen(KERNEL_SEED + 910)
    n, capacity = start + length, 192
    k, v = rows(g, 1, kv_heads, n, dim), rows(g, 1, kv_heads, n, dim)
    cache = cache_of(k, v, bits, capacity, junk=float("nan"))
    q = torch.randn(1, heads, length, dim, generator=g).to(BF)
    got = K.gqa_prefill_attention_q(q.to(gpu), to(cache, gpu), dim**-0.5, kv_start=start)
    check_attention(got, q, cache, [start], dim**-0.5, prompt=True)


def roomy(heads, kv_heads, dim, length, batch=1):
    """A capacity at which more than 96 rows of a KV head go over the unpacked
    cache whatever it is: rows x batch x KV heads x capacity x dim above 2^32
    (heads of 64: 2^31.5)."""
    capacity = int(2 ** (31.5 if dim == 64 else 32)) // (heads // kv_heads * length * batch * kv_heads * dim) + 1
    return (capacity + 31) // 32 * 32


def wide(cache, capacity, device, junk=0.0):
    """``cache`` on the GPU with ``capacity`` positions, the codes of the others
    all ones and their params ``junk``."""
    out = []
    for t in cache:
        dim, fill = (2, 255) if t.ndim == 4 else (3, junk)
        shape = list(t.shape)
        shape[dim] = capacity
        w = torch.full(shape, fill, dtype=t.dtype, device=device)
        w.narrow(dim, 0, t.shape[dim]).copy_(t)
        out.append(w)
    return K.QuantizedKV(*out)


@gpu_test
@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("heads,kv_heads,length,start", [(8, 2, 33, 0), (8, 2, 65, 63), (3, 1, 70, 100), (12, 1, 50, 7),
                                                         (2, 2, 400, 1), (5, 1, 129, 319)])
def test_prefill_many_rows(gpu, bits, dim, heads, kv_heads, length, start):
    """Row tiles that end inside a token, in the middle of a wave, in several
    tiles; key ranges of one and several blocks; the rest of the cache NaN."""
    g = gen(KERNEL_SEED + 916)
    n = start + length
    k, v = rows(g, 1, kv_heads, n, dim), rows(g, 1, kv_heads, n, dim)
    cache = cache_of(k, v, bits, (n + 31) // 32 * 32, junk=float("nan"))
    q = torch.randn(1, heads, length, dim, generator=g).to(BF)
    roomier = wide(cache, roomy(heads, kv_heads, dim, length), gpu, float("nan"))
    got = K.gqa_prefill_attention_q(q.to(gpu), roomier, dim**-0.5, kv_start=start)
    check_attention(got, q, cache, [start], dim**-0.5, prompt=True)
    valid = torch.tensor([start], device=gpu)
    again = K.gqa_prefill_attention_q(q.to(gpu), roomier, dim**-0.5, valid_length=valid, length_is_start=True)
    assert torch.equal(got, again)


@gpu_test
@pytest.mark.parametrize("bits,dim", [(4, 256), (8, 128), (4, 64)])
@pytest.mark.parametrize("scale_k,scale_v", [(1e-20, 1e20), (1e4, 1e-30), (2.0**100, 2.0**120)])
def test_prefill_many_rows_magnitudes(gpu, bits, dim, scale_k, scale_v):
    """Keys and values far from one, with queries that bring the scores back;
    one row of queries is zero and one has a value 2^20 above the others."""
    g = gen(KERNEL_SEED + 917)
    heads, length = 4, 64
    k, v = rows(g, 1, 1, length, dim), rows(g, 1, 1, length, dim)
    cache = cache_of((k.float() * scale_k).to(BF), (v.float() * scale_v).to(BF), bits, length)
    q = (torch.randn(1, heads, length, dim, generator=g) / scale_k).to(BF)
    q[0, 1, 5] = 0
    q[0, 2, 9] *= 2.0**-20
    q[0, 2, 9, 3] = 1 / scale_k
    roomier = wide(cache, roomy(heads, 1, dim, length), gpu)
    got = K.gqa_prefill_attention_q(q.to(gpu), roomier, dim**-0.5).double().cpu() / scale_v
    # the oracle on the same numbers, brought back in 64 bits
    kd, vd = values_of(cache)
    want = ref.attend(q.double() * scale_k, kd / scale_k, vd / scale_v, [0], dim**-0.5)
    square = ref.attend(q.double() * scale_k, kd / scale_k, (vd / scale_v).square(), [0], dim**-0.5)
    var = want.square() / 3 + square * (4 / 3)
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= 6 * 2**-8 * var.sqrt()).all()


@gpu_test
@pytest.mark.parametrize("bits,dim,length,heads,capacity", [
    (4, 256, 100, 4, None), (8, 128, 100, 4, None), (4, 64, 150, 4, None),
    (4, 256, 100, 16, 768), (8, 128, 150, 16, 768), (4, 64, 150, 32, 768), (8, 256, 130, 24, 2048)])
def test_prefill_batch_many_rows(gpu, bits, dim, length, heads, capacity):
    """As test_prefill_batch, over the unpacked cache: in roomy caches, whose
    greatest values are found by a launch of its own, and in short ones."""
    g = gen(KERNEL_SEED + 918)
    capacity = capacity or roomy(heads, 2, dim, length, 4)
    n = 256
    starts = [0, 77, -length // 2, n - length]
    cache = cache_of(rows(g, 4, 2, n, dim), rows(g, 4, 2, n, dim), bits, n)
    for b, s in enumerate(starts):
        cache.key_params[b, :, :, max(s + length, 0) :] = float("nan")
        cache.value_params[b, :, :, max(s + length, 0) :] = float("nan")
    # the keys of the last token NaN in one sequence, a group of its values in another
    cache.key_params[0, :, :, length - 1] = float("nan")
    cache.value_params[1, :, 0, 77 + length - 1] = float("nan")
    q = torch.randn(4, heads, length, dim, generator=g).to(BF)
    valid = torch.tensor([s + length for s in starts], device=gpu)
    roomier = wide(cache, capacity, gpu, float("inf"))
    got = K.gqa_prefill_attention_q(q.to(gpu), roomier, dim**-0.5, valid_length=valid).cpu()
    kd, vd = values_of(cache)
    assert torch.isnan(got[0, -1]).all()
    want = ref.attend(q[1:2], kd[1:2], vd[1:2], [77], dim**-0.5)[0, -1]
    assert torch.equal(torch.isnan(got[1, -1]), torch.isnan(want))
    for b, t in ((0, length - 1), (1, length - 1)):
        got[b, t] = 0
    want, square = ref.attend(q, kd, vd, starts, dim**-0.5), ref.attend(q, kd, vd.square(), starts, dim**-0.5)
    for t in (want, square):
        t[0, -1] = t[1, -1] = 0
    assert torch.isfinite(got).all()
    var = want.square() / 3 + square * (4 / 3)
    err = (got.double() - want).abs()
    assert err.square().mean().sqrt() <= 2**-8 * var.mean().sqrt()
    assert (err <= 6 * 2**-8 * var.sqrt() + 1e-30).all()
    assert (got[2, : length // 2] == 0).all()


@gpu_test
@pytest.mark.parametrize("bits,dim,length", [(4, 256, 6), (8, 128, 40), (4, 64, 90), (4, 256, 100)])
@pytest.mark.parametrize("length_is_start", [False, True])
def test_prefill_batch(gpu, bits, dim, length, length_is_start):
    """Unequal starts in a batch: one left-padded sequence (rows before its
    first token are zero), one past the capacity, and keys that no row of a
    sequence sees, or only its later rows, NaN or huge."""
    g = gen(KERNEL_SEED + 911)
    capacity = 256
    starts = [0, 77, -length // 2, capacity - length + 3]
    cache = cache_of(rows(g, 4, 2, capacity, dim), rows(g, 4, 2, capacity, dim), bits, capacity)
    for b, s in enumerate(starts):
        cache.key_params[b, :, :, max(s + length, 0) :] = float("nan")
        cache.value_params[b, :, :, max(s + length, 0) :] = float("nan")
    # sequence 1: the last key is infinite and only the last row sees it
    cache.value_params[1, :, :, 77 + length - 1] = float("inf")
    q = torch.randn(4, 4, length, dim, generator=g).to(BF)
    valid = torch.tensor([s if length_is_start else s + length for s in starts], device=gpu)
    got = K.gqa_prefill_attention_q(q.to(gpu), to(cache, gpu), dim**-0.5, valid_length=valid,
                                    length_is_start=length_is_start).cpu()
    assert not torch.isfinite(got[1, -1]).any()
    check_attention(got, q, cache, starts, dim**-0.5, prompt=True, skip=(1, -1))
    assert (got[2, : length // 2] == 0).all()


@gpu_test
@pytest.mark.parametrize("bits,dim", [(4, 256), (8, 256), (4, 128), (8, 64)])
def test_prefill_long(gpu, bits, dim):
    """A part of a prompt over a long cache: several key ranges of a row."""
    g = gen(KERNEL_SEED + 912)
    length, start = 67, 5000
    n = start + length
    cache = cache_of(rows(g, 1, 1, n, dim), rows(g, 1, 1, n, dim), bits, 5088, junk=float("nan"))
    q = torch.randn(1, 4, length, dim, generator=g).to(BF)
    roomier = wide(cache, roomy(4, 1, dim, length), gpu, float("nan"))
    got = K.gqa_prefill_attention_q(q.to(gpu), roomier, dim**-0.5, kv_start=start)
    check_attention(got, q, cache, [start], dim**-0.5, prompt=True)


# ------------------------------------------------------------------ together
@gpu_test
@pytest.mark.parametrize("bits,dim,length,many", [(4, 256, 1, False), (8, 128, 6, False), (4, 64, 90, False),
                                                  (4, 256, 100, True), (8, 128, 100, True), (4, 64, 200, True)])
def test_visible_nan(gpu, bits, dim, length, many):
    """A group of values that is NaN makes NaN of its dims, a key that is NaN of
    every dim, for the rows that see it; the others are as without (a step of
    bf16 apart at most: the greatest value of a head sets its power of two)."""
    g = gen(KERNEL_SEED + 937)
    heads, kv_heads, n = 4, 2, 230
    k, v = rows(g, 1, kv_heads, n, dim), rows(g, 1, kv_heads, n, dim)
    plain = wide(cache_of(k, v, bits, 256), roomy(heads, kv_heads, dim, length) if many else 256, gpu)
    q = torch.randn(1, heads, length, dim, generator=g).to(BF).to(gpu)
    want = K.gqa_prefill_attention_q(q, plain, dim**-0.5, kv_start=n - length).cpu().unflatten(-1, (heads, dim))
    sees = torch.arange(length) + n - length
    for at in {3, n - 1, n - length, n - length // 2 - 1}:
        hit = sees >= at  # the rows that see position `at`
        bad = K.QuantizedKV(*(t.clone() for t in plain))
        bad.value_params[0, 1, 0, at] = float("nan")  # the first group of KV head 1
        got = K.gqa_prefill_attention_q(q, bad, dim**-0.5, kv_start=n - length).cpu().unflatten(-1, (heads, dim))
        dims = ref.groups(dim, True)[0]
        nan = torch.zeros_like(want, dtype=torch.bool)
        nan[:, hit, 2:] = torch.isin(torch.arange(dim), torch.as_tensor(dims))
        assert torch.equal(torch.isnan(got), nan), f"values, position {at}"
        torch.testing.assert_close(got[~nan].float(), want[~nan].float(), rtol=2**-7, atol=1e-6)
        bad = K.QuantizedKV(*(t.clone() for t in plain))
        bad.key_params[0, 0, 0, at] = float("nan")
        got = K.gqa_prefill_attention_q(q, bad, dim**-0.5, kv_start=n - length).cpu().unflatten(-1, (heads, dim))
        nan = torch.zeros_like(want, dtype=torch.bool)
        nan[:, hit, :2] = True
        assert torch.equal(torch.isnan(got), nan), f"keys, position {at}"


@gpu_test
def test_far_offsets(gpu):
    """A cache of 9.7 GB: the last of 72 sequences lies beyond 2^32 bytes of codes
    and 2^31 values; all operators on it give what they give on that sequence
    alone (attention: the same sums in another order, then at most one bf16 step
    apart, 2^-7 of the value, or 1e-5, 2^-18 of the values' range)."""
    g = gen(KERNEL_SEED + 938)
    batch, kv_heads, dim, capacity, new = 72, 2, 256, 131072, 80
    cache = K.quantized_kv_cache(batch, kv_heads, capacity, dim, bits=8, device=gpu)
    for t in cache[:2]:
        t[-1].random_(0, 256)
    for t in cache[2:]:
        t[-1, ..., 0], t[-1, ..., 1] = 0.01, -1.0
    last = K.QuantizedKV(*(t[-1:].clone() for t in cache))
    k, v = (rows(g, 1, kv_heads, new, dim).to(gpu) for _ in range(2))
    start = torch.zeros(batch, dtype=torch.int64, device=gpu)
    start[-1] = capacity - new
    start[:-1] = capacity  # the others' rows are outside
    K.kv_cache_quantize(k.expand(batch, -1, -1, -1), v.expand(batch, -1, -1, -1), cache, cache_start=start)
    K.kv_cache_quantize(k, v, last, start=capacity - new)
    for t, u in zip(cache, last):
        assert torch.equal(t[-1:], u) and not t[-2].any()
    for t, u in zip(K.kv_cache_dequantize(cache, new, start=capacity - new), K.kv_cache_dequantize(last, new, start=capacity - new)):
        assert torch.equal(t[-1:], u) and not t[:-1].any()
    length = torch.where(start == capacity, 0, capacity)
    for n in (1, new):
        q = torch.randn(1, 8, n, dim, generator=g).to(BF).to(gpu)
        got = K.gqa_prefill_attention_q(q.expand(batch, -1, -1, -1).contiguous(), cache, dim**-0.5, valid_length=length)
        want = K.gqa_prefill_attention_q(q, last, dim**-0.5, kv_start=capacity - n)
        assert not got[:-1].any()
        torch.testing.assert_close(got[-1:], want, rtol=2**-7, atol=1e-5)


@gpu_test
def test_operators_together(gpu):
    """A prompt in two parts, then decoded tokens, as a model's attention layer
    uses them: each call's output against the oracle on the cache so far."""
    g = gen(KERNEL_SEED + 913)
    heads, kv_heads, dim, capacity = 8, 2, 256, 160
    cache = K.quantized_kv_cache(1, kv_heads, capacity, dim, device=gpu)
    length = torch.zeros(1, device=gpu, dtype=torch.int64)
    k, v = rows(g, 1, kv_heads, capacity, dim), rows(g, 1, kv_heads, capacity, dim)
    oracle = cache_of(k, v, 4, capacity)
    kd, vd = values_of(oracle)
    at = 0
    for new in (50, 70, 1, 1, 1, 4, 1):
        q = torch.randn(1, heads, new, dim, generator=g).to(BF)
        part = slice(at, at + new)
        K.kv_cache_quantize(k[:, :, part].to(gpu), v[:, :, part].to(gpu), cache, cache_start=length)
        if new > 1:
            got = K.gqa_prefill_attention_q(q.to(gpu), cache, dim**-0.5, valid_length=length, length_is_start=True)
        length += new
        if new == 1:
            got = K.gqa_decode_attention_q(q.to(gpu), cache, length, dim**-0.5)
        check_attention(got, q, oracle, [at], dim**-0.5, prompt=True)
        at += new
    kb, vb = K.kv_cache_dequantize(cache, at)
    assert torch.equal(kb.cpu(), kd[:, :, :at].to(BF)) and torch.equal(vb.cpu(), vd[:, :, :at].to(BF))


@gpu_test
def test_decode_step_captured(gpu):
    """Write and decode of one token captured once, replayed along the cache,
    with eager calls and synchronisations between: the same bits as eager."""
    g = gen(KERNEL_SEED + 914)
    heads, kv_heads, dim, capacity, n0 = 8, 2, 256, 1024, 333
    k, v = rows(g, 1, kv_heads, capacity, dim).to(gpu), rows(g, 1, kv_heads, capacity, dim).to(gpu)
    caches = [K.quantized_kv_cache(1, kv_heads, capacity, dim, device=gpu) for _ in range(2)]
    for c in caches:
        K.kv_cache_quantize(k[:, :, :n0], v[:, :, :n0], c)
    qs = torch.randn(6, 1, heads, 1, dim, generator=g).to(BF).to(gpu)
    length = [torch.tensor([n0], device=gpu) for _ in range(2)]
    q, kn, vn = qs[0].clone(), k[:, :, n0 : n0 + 1].clone(), v[:, :, n0 : n0 + 1].clone()

    def step(cache, length, q, kn, vn):
        K.kv_cache_quantize(kn, vn, cache, cache_start=length)
        length.add_(1)
        return K.gqa_decode_attention_q(q, cache, length, dim**-0.5)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(caches[0], length[0].clone(), q, kn, vn)  # position n0, written again below
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], length[0], q, kn, vn)
    for i in range(6):
        at = slice(n0 + i, n0 + i + 1)
        for dst, src in ((q, qs[i]), (kn, k[:, :, at]), (vn, v[:, :, at])):
            dst.copy_(src)
        graph.replay()
        want = step(caches[1], length[1], qs[i], k[:, :, at].contiguous(), v[:, :, at].contiguous())
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {i}"
    assert int(length[0]) == n0 + 6


@gpu_test
@pytest.mark.parametrize("length,many", [(5, False), (70, True)])
def test_prompt_captured(gpu, length, many):
    """Parts of a prompt, written and attended in one graph that is replayed
    along the cache, with eager calls between: the same bits as eager."""
    g = gen(KERNEL_SEED + 934)
    heads, kv_heads, dim, n0, parts = 8, 2, 128, 40, 4
    capacity = roomy(heads, kv_heads, dim, length) if many else 512
    n = n0 + parts * length
    k, v = rows(g, 1, kv_heads, n, dim).to(gpu), rows(g, 1, kv_heads, n, dim).to(gpu)
    qs = torch.randn(parts, 1, heads, length, dim, generator=g).to(BF).to(gpu)
    caches = [K.quantized_kv_cache(1, kv_heads, capacity, dim, bits=8, device=gpu) for _ in range(2)]
    for c in caches:
        K.kv_cache_quantize(k[:, :, :n0], v[:, :, :n0], c)
    at = [torch.tensor([n0], device=gpu) for _ in range(2)]

    def step(cache, at, q, kn, vn):
        K.kv_cache_quantize(kn, vn, cache, cache_start=at)
        out = K.gqa_prefill_attention_q(q, cache, dim**-0.5, valid_length=at, length_is_start=True)
        at.add_(length)
        return out

    q, kn, vn = qs[0].clone(), k[:, :, n0 : n0 + length].clone(), v[:, :, n0 : n0 + length].clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(caches[0], at[0].clone(), q, kn, vn)  # the same rows again below
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], at[0], q, kn, vn)
    for i in range(parts):
        part = slice(n0 + i * length, n0 + (i + 1) * length)
        for dst, src in ((q, qs[i]), (kn, k[:, :, part]), (vn, v[:, :, part])):
            dst.copy_(src)
        graph.replay()
        want = step(caches[1], at[1], qs[i], k[:, :, part], v[:, :, part])
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {i}"


@gpu_test
def test_entry_without_lengths(gpu):
    """The C entry with no lengths takes their count for nothing."""
    g = gen(KERNEL_SEED + 935)
    batch, dim, n = 3, 128, 64
    cache = cache_of(rows(g, batch, 2, n, dim), rows(g, batch, 2, n, dim), 4, n)
    q = torch.randn(batch, 4, 1, dim, generator=g).to(BF)
    c, qd = to(cache, gpu), q.to(gpu)
    out = torch.empty(batch, 1, 4 * dim, device=gpu, dtype=BF)
    floats = _lib.load().q35_gqa_attention_kvq_workspace(batch, 4, 2, 1, dim, 4, n)
    ws = torch.empty(floats, device=gpu)
    _lib.call("q35_gqa_attention_kvq", qd.data_ptr(), c.keys.data_ptr(), c.values.data_ptr(), c.key_params.data_ptr(),
              c.value_params.data_ptr(), 0, batch, 40, 0, 0, dim**-0.5, out.data_ptr(), ws.data_ptr(), floats,
              batch, 4, 2, 1, dim, 4, n, torch.cuda.current_stream().cuda_stream)
    check_attention(out, q, cache, [40] * batch, dim**-0.5)


@gpu_test
def test_two_streams(gpu):
    """Two attentions at once on two streams give what each gives alone."""
    g = gen(KERNEL_SEED + 915)
    jobs = []
    for heads, kv_heads, dim, length in ((8, 2, 256, 1), (4, 1, 128, 65)):
        cache = wide(cache_of(rows(g, 2, kv_heads, 900, dim), rows(g, 2, kv_heads, 900, dim), 4, 928),
                     roomy(heads, kv_heads, dim, length, 2) if length > 1 else 928, gpu)
        q = torch.randn(2, heads, length, dim, generator=g).to(BF).to(gpu)
        valid = torch.tensor([900, 411], device=gpu)
        jobs.append((q, cache, valid, dim**-0.5))

    def run(q, cache, valid, scale):
        return K.gqa_prefill_attention_q(q, cache, scale, valid_length=valid)

    alone = [run(*job) for job in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (job, s) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(s):
                got[i].append(run(*job))
    torch.cuda.synchronize()
    for want, several in zip(alone, got):
        assert all(torch.equal(want, x) for x in several)


@gpu_test
@pytest.mark.parametrize("seed", range(8))
def test_random_forms(gpu, seed):
    """Drawn layouts, lengths and bits."""
    r = random.Random(7000 + seed)
    g = gen(KERNEL_SEED + 920 + seed)
    bits, dim = r.choice(FORMS)
    kv_heads = r.randint(1, 3)
    heads, batch = kv_heads * r.randint(1, 17), r.randint(1, 3)
    capacity = 32 * r.randint(1, 20)
    length = r.choice([1, 1, r.randint(2, min(9, capacity)), r.randint(2, min(130, capacity))])
    starts = [r.randint(0, capacity - length) for _ in range(batch)]
    cache = cache_of(rows(g, batch, kv_heads, capacity, dim), rows(g, batch, kv_heads, capacity, dim), bits, capacity)
    q = torch.randn(batch, heads, length, dim, generator=g).to(BF)
    got = K.gqa_prefill_attention_q(q.to(gpu), to(cache, gpu), dim**-0.5, valid_length=torch.tensor(starts, device=gpu),
                                    length_is_start=True)
    check_attention(got, q, cache, starts, dim**-0.5, prompt=True)
