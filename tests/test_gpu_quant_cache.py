"""The 8-bit cache: codes and scales bit for bit against the documented fp32 formula, values against 64 bits."""
import pytest
import torch

import kernel_collections_b200 as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
LARGEST = {"int8": 127.0, "e4m3": 448.0}


def encode(x, code):
    """The documented formula in fp32 on the CPU, every operation rounded once."""
    x = x.float()
    C, one = torch.tensor(LARGEST[code]), torch.ones(())
    top = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    scale = top * (one / C)
    held = finite & (scale >= 2.0 ** -126)
    per = torch.where(held, C * (one / top), torch.zeros(()))
    y = torch.where(finite[..., None], x, torch.zeros(())) * per[..., None]
    y = (torch.round(y) if code == "int8" else y).clamp(-C, C)
    codes = y.to(torch.int8 if code == "int8" else torch.float8_e4m3fn)
    return codes, torch.where(finite, torch.where(held, scale, torch.zeros(())), torch.full((), float("nan")))


def bits(t):
    return t.cpu().contiguous().view(torch.uint8)


def rows(seed, b, h, n, d, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, h, n, d, generator=g) * torch.exp(2 * torch.randn(b, h, n, 1, generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("b,h,n,d", [(1, 1, 1, 1), (3, 2, 5, 128), (2, 8, 33, 64), (2, 3, 7, 96), (1, 2, 9, 100),
                                     (1, 1, 4, 256), (1, 2, 3, 1024), (2, 1, 300, 17)])
def test_append_and_read(dtype, code, b, h, n, d):
    k, v = rows(n + d, b, h, n, d, dtype), rows(n + d + 1, b, h, n, d, dtype)
    cap = n + 6
    start = torch.randint(0, 7, (b,), generator=torch.Generator().manual_seed(d), dtype=torch.int32)
    cache = K.quantized_cache(b, h, cap, d, code=code)
    assert K.quantized_cache_append(cache, k.to(DEV), v.to(DEV), start.to(DEV)) is cache
    rk, rv = K.quantized_cache_read(cache, start.to(DEV), n, dtype=dtype)
    for x, codes, scales, back in ((k, cache.key_codes, cache.key_scales, rk), (v, cache.value_codes, cache.value_scales, rv)):
        c, s = encode(x, code)
        for i in range(b):
            at = slice(int(start[i]), int(start[i]) + n)
            assert torch.equal(bits(codes[i, :, at]), bits(c[i])) and torch.equal(scales[i, :, at].cpu(), s[i])
            rest = torch.ones(cap, dtype=torch.bool)
            rest[at] = False
            assert (bits(codes[i][:, rest.to(DEV)]) == 0).all() and (scales[i][:, rest.to(DEV)] == 0).all()
        assert torch.equal(back.cpu(), (c.float() * s[..., None]).to(dtype))
        # against 64 bits: half a step of the code, plus 6 roundings of 2^-24 on values up to top, plus the output's own
        y = x.double()
        top = y.abs().amax(-1, keepdim=True)
        half = top / 254 if code == "int8" else torch.maximum(y.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10)
        tol = half + top * 6 * 2.0 ** -24 + (y.abs() + half) * torch.finfo(dtype).eps / 2 + 2.0 ** -25
        assert ((back.cpu().double() - y).abs() <= tol).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_zero_tiny_infinite_and_nan_rows(code):
    x = torch.zeros(1, 1, 7, 64)
    x[0, 0, 1, 3] = 1e-40                     # below the smallest scale: held as zeros
    x[0, 0, 2] = 5e-36
    x[0, 0, 3, 5] = float("inf")
    x[0, 0, 4, 6] = float("nan")
    x[0, 0, 5] = 3e38
    x[0, 0, 6, 0], x[0, 0, 6, 1] = -2.0, 1.0
    cache = K.quantized_cache(1, 1, 7, 64, code=code)
    K.quantized_cache_append(cache, x.to(DEV), x.to(DEV), 0)
    c, s = encode(x, code)
    assert torch.equal(bits(cache.key_codes), bits(c)) and torch.equal(bits(cache.value_codes), bits(c))
    assert torch.equal(cache.key_scales.cpu().nan_to_num(7.0), s.nan_to_num(7.0))
    k, _ = K.quantized_cache_read(cache, 0, 7, dtype=torch.float32)
    assert (k[0, 0, :2] == 0).all() and k[0, 0, 3:5].isnan().all() and torch.isfinite(k[0, 0, 5:]).all()


def test_ties_round_to_even_and_the_ends_are_reached():
    x = torch.tensor([127.0, -127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5]).view(1, 1, 1, 8)
    cache = K.quantized_cache(1, 1, 1, 8)
    K.quantized_cache_append(cache, x.to(DEV), -x.to(DEV), 0)
    assert cache.key_codes.flatten().tolist() == [127, -127, 0, 2, 2, 0, -2, 126]
    assert cache.value_codes.flatten().tolist() == [-127, 127, 0, -2, -2, 0, 2, -126]


def test_rows_outside_the_cache_padded_prompts_and_no_tokens():
    b, h, n, d, cap = 4, 2, 6, 64, 10
    k = rows(3, b, h, n, d, torch.bfloat16).to(DEV)
    cache = K.quantized_cache(b, h, cap, d)
    cache.key_codes.fill_(55)
    cache.key_scales.fill_(2.0)
    start = torch.tensor([-2, 7, 2 ** 31 - 1, 0], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([6, 2, 6, 9], dtype=torch.int32, device=DEV)
    K.quantized_cache_append(cache, k, k, start, lengths=lengths)
    c, s = encode(k.cpu(), "int8")
    want_c, want_s = torch.full((b, h, cap, d), 55, dtype=torch.int8), torch.full((b, h, cap), 2.0)
    want_c[0, :, :4], want_s[0, :, :4] = c[0, :, 2:], s[0, :, 2:]
    want_c[1, :, 7:9], want_s[1, :, 7:9] = c[1, :, :2], s[1, :, :2]
    want_c[3, :, :6], want_s[3, :, :6] = c[3], s[3]
    assert torch.equal(cache.key_codes.cpu(), want_c) and torch.equal(cache.key_scales.cpu(), want_s)
    rk, _ = K.quantized_cache_read(cache, start, n, dtype=torch.float32)
    assert (rk[0, :, :2] == 0).all() and (rk[1, :, 3:] == 0).all() and (rk[2] == 0).all()
    assert torch.equal(rk[0, :, 2:].cpu(), c[0, :, 2:].float() * s[0, :, 2:, None])
    before = cache.key_codes.clone()
    K.quantized_cache_append(cache, k[:, :, :0], k[:, :, :0], 0)
    K.quantized_cache_append(cache, k, k, 3, lengths=torch.zeros(b, dtype=torch.int32, device=DEV))
    assert torch.equal(before, cache.key_codes)
    assert K.quantized_cache_read(cache, 0, 0)[0].shape == (b, h, 0, d)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_strided_caches_and_unaligned_inputs(code):
    b, h, n, d, cap = 2, 3, 5, 64, 9
    x = rows(4, b, h, n, d + 1, torch.float16).to(DEV)
    k, v = x[..., 1:], rows(5, b, n, h, d, torch.float16).to(DEV).transpose(1, 2)
    assert k.stride(-1) == 1 and k.data_ptr() % 4 == 2
    want = K.quantized_cache(b, h, cap, d, code=code)
    K.quantized_cache_append(want, k.contiguous(), v.contiguous(), 2)
    codes = [torch.zeros(b, cap, h, d, dtype=torch.uint8, device=DEV).view(want.key_codes.dtype).transpose(1, 2) for _ in "kv"]
    scales = [torch.zeros(b, h, cap + 3, device=DEV)[..., 1:cap + 1] for _ in "kv"]
    cache = K.QuantizedCache(codes[0], scales[0], codes[1], scales[1])
    K.quantized_cache_append(cache, k, v, 2)
    for a, c in zip((want.key_codes, want.value_codes), codes):
        assert torch.equal(bits(a), bits(c))
    assert torch.equal(scales[0], want.key_scales) and torch.equal(scales[1], want.value_scales)
    for a, c in zip(K.quantized_cache_read(cache, 1, 7), K.quantized_cache_read(want, 1, 7)):
        assert torch.equal(a, c)


def test_offsets_past_32_bits():
    b, h, d, cap = 1, 1, 256, (1 << 31) // 256 + 64          # the last rows lie past 2^31 codes
    codes = torch.empty(b, h, cap, d, dtype=torch.int8, device=DEV)
    scales = torch.empty(b, h, cap, device=DEV)
    cache = K.QuantizedCache(codes, scales, codes, scales)
    k = rows(6, b, h, 3, d, torch.bfloat16).to(DEV)
    K.quantized_cache_append(cache, k, k, cap - 3)
    c, s = encode(k.cpu(), "int8")
    assert torch.equal(codes[0, 0, -3:].cpu(), c[0, 0]) and torch.equal(scales[0, 0, -3:].cpu(), s[0, 0])
    got, _ = K.quantized_cache_read(cache, cap - 3, 3, dtype=torch.float32)
    assert torch.equal(got.cpu(), c.float() * s[..., None])


def test_cache_refusals():
    cache = K.quantized_cache(2, 3, 8, 64)
    k = torch.zeros(2, 3, 4, 64, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    for kw in [dict(key=k[:1]), dict(value=k[:, :2]), dict(key=k.half()), dict(key=k.double(), value=k.double()),
               dict(position=torch.zeros(2, device=DEV)), dict(position=torch.zeros(3, **i32)), dict(position=2 ** 31),
               dict(lengths=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(lengths=torch.zeros(1, **i32)),
               dict(key=k[..., :32], value=k[..., :32])]:
        with pytest.raises(ValueError):
            K.quantized_cache_append(**{**dict(cache=cache, key=k, value=k, position=0), **kw})
    c, s = cache.key_codes, cache.key_scales
    for bad in [K.QuantizedCache(c, s, c.view(torch.float8_e4m3fn), s), K.QuantizedCache(c.view(torch.uint8), s, c, s),
                K.QuantizedCache(c, s[:, :2], c, s), K.QuantizedCache(c, s.half(), c, s),
                K.QuantizedCache(c.transpose(2, 3), s, c.transpose(2, 3), s), K.QuantizedCache(c, s, c[:, :, :4], s)]:
        with pytest.raises(ValueError):
            K.quantized_cache_read(bad, 0, 1)
    with pytest.raises(ValueError):
        K.quantized_cache_read(cache, 0, -1)
    with pytest.raises(ValueError):
        K.quantized_cache_read(cache, 0, 1, dtype=torch.float64)
    with pytest.raises(ValueError):
        K.quantized_cache(1, 1, 1, 1, code="int4")
    wide = K.quantized_cache(1, 1, 2, 1025)
    with pytest.raises(ValueError):
        K.quantized_cache_append(wide, torch.zeros(1, 1, 1, 1025, device=DEV), torch.zeros(1, 1, 1, 1025, device=DEV), 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.quantized_cache_append(cache, k.cpu(), k.cpu(), 0)
