"""rotary_embedding against the rotation in 64 bits.

Tolerance per element.  The kernel's angle in half turns is rounded once to fp32 (2^-24 of at most 1, times pi), its
sine and cosine are within 2 units in the last place (2^-23), the factor, two products and a sum round once each (2^-24): an
error of at most (pi + 2 + 4) 2^-24 < 10 * 2^-24 on |a| + |b|, times the magnitude, and then half a step of the
output type on the value itself (2^-25 where fp16 is subnormal)."""
import math

import pytest
import torch

import kernel_collections_b200 as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x, inv_freq, pos, interleaved, magnitude):
    """x (b, h, n, d), pos (b, n) -> (rotated, |a| + |b| of the pair) in 64 bits."""
    dim = 2 * inv_freq.numel()
    y, room = x.double().clone(), x.double().abs().mul(0.0)
    j = torch.arange(dim // 2)
    one, two = (2 * j, 2 * j + 1) if interleaved else (j, j + dim // 2)
    ang = pos.double()[:, None, :, None] * inv_freq.cpu().double()
    c, s = torch.cos(ang) * magnitude, torch.sin(ang) * magnitude
    a, b = x.double()[..., one], x.double()[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    room[..., one] = room[..., two] = (a.abs() + b.abs()) * magnitude
    return y, room


def close(got, x, inv_freq, pos, interleaved, magnitude):
    want, room = reference(x.cpu(), inv_freq, pos, interleaved, magnitude)
    u = torch.finfo(got.dtype).eps / 2
    tol = want.abs() * u + room * 10 * 2.0 ** -24 + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    over = (got.cpu().double() - want).abs() - tol
    assert (over <= 0).all(), f"{over.max().item():.3e} over the tolerance"


def inputs(seed, b, H, KVH, n, D, dtype, token_major=False):
    g = torch.Generator().manual_seed(seed)
    make = lambda h: (torch.randn(b, n, h, D, generator=g).transpose(1, 2) if token_major  # noqa: E731
                      else torch.randn(b, h, n, D, generator=g)).to(dtype).to(DEV)
    return make(H), make(KVH)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,H,KVH,n,D,rot", [(1, 4, 1, 1, 64, 64), (3, 12, 4, 37, 80, 32), (2, 8, 8, 5, 128, 64),
                                             (2, 3, 1, 9, 96, 10), (1, 5, 5, 300, 256, 256), (1, 2, 1, 2, 7, 2),
                                             (16, 32, 8, 1, 128, 128), (2, 40, 8, 500, 128, 128)])
def test_rotary_matches_the_formula(dtype, interleaved, b, H, KVH, n, D, rot):
    q, k = inputs(b * n + D, b, H, KVH, n, D, dtype, token_major=n % 2 == 1)
    f, mag = K.rotary_frequencies(rot, 500000.0)
    first = torch.randint(0, 200000, (b,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
    qo, ko = K.rotary_embedding(q, k, f, first.to(DEV), interleaved=interleaved, magnitude=mag)
    pos = first[:, None].long() + torch.arange(n)
    close(qo, q, f, pos, interleaved, mag)
    close(ko, k, f, pos, interleaved, mag)
    assert torch.equal(qo[..., rot:], q[..., rot:]) and torch.equal(ko[..., rot:], k[..., rot:])


@pytest.mark.parametrize("scaling,kw", [("linear", {}), ("base", {}), ("wavelength", dict(original_length=4096)),
                                        ("yarn", dict(original_length=4096))])
def test_scaled_frequencies_and_magnitude(scaling, kw):
    q, k = inputs(5, 2, 4, 2, 33, 64, torch.float32)
    f, mag = K.rotary_frequencies(64, 10000.0, scaling=scaling, factor=8.0, **kw)
    qo, ko = K.rotary_embedding(q, k, f, 30000, magnitude=mag)
    pos = (30000 + torch.arange(33)).expand(2, 33)
    close(qo, q, f, pos, False, mag)
    close(ko, k, f, pos, False, mag)


def test_positions_of_every_token_the_largest_position_and_negative_ones():
    q, k = inputs(6, 2, 4, 2, 4, 64, torch.float32)
    f, _ = K.rotary_frequencies(64)
    pos = torch.tensor([[5, 6, 6, 2 ** 31 - 1], [-3, 0, 100, 7]], dtype=torch.int32)
    qo, ko = K.rotary_embedding(q, k, f, pos.to(DEV))
    close(qo, q, f, pos.long(), False, 1.0)
    close(ko, k, f, pos.long(), False, 1.0)
    # an int counts on from the largest 32-bit position without wrapping
    qo, _ = K.rotary_embedding(q, k, f, 2 ** 31 - 1)
    close(qo, q, f, (2 ** 31 - 1 + torch.arange(4)).expand(2, 4), False, 1.0)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [64, 32])
def test_in_place_and_into_given_tensors(interleaved, rot):
    q, k = inputs(7, 2, 4, 2, 19, 64, torch.bfloat16, token_major=True)
    f, _ = K.rotary_frequencies(rot)
    want = K.rotary_embedding(q, k, f, 11, interleaved=interleaved)
    wide = torch.full((2, 19, 6, 72), 3.0, dtype=torch.bfloat16, device=DEV)      # strided outputs with a border
    oq, ok = wide[:, :, :4, :64].transpose(1, 2), wide[:, :, 4:, :64].transpose(1, 2)
    got = K.rotary_embedding(q, k, f, 11, interleaved=interleaved, out=(oq, ok))
    assert got[0] is oq and torch.equal(oq, want[0]) and torch.equal(ok, want[1])
    assert (wide[..., 64:] == 3).all()
    K.rotary_embedding(q, k, f, 11, interleaved=interleaved, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_queries_alone_unaligned_views_and_no_tokens():
    f, _ = K.rotary_frequencies(32)
    base = torch.randn(2, 3, 8, 67, device=DEV).bfloat16()
    for interleaved in (False, True):
        q = base[..., 1:65]                               # rows start at odd addresses
        qo, ko = K.rotary_embedding(q, None, f, 9, interleaved=interleaved)
        assert ko is None
        close(qo, q, f, (9 + torch.arange(8)).expand(2, 8), interleaved, 1.0)
        t = base.transpose(2, 3)[:, :, :64, :].transpose(2, 3)      # last dim is not the fast one
        x = t.transpose(2, 3).contiguous().transpose(2, 3)
        assert x.stride(-1) != 1
        qo, _ = K.rotary_embedding(x, None, f, 9, interleaved=interleaved)
        close(qo, x, f, (9 + torch.arange(8)).expand(2, 8), interleaved, 1.0)
    qo, ko = K.rotary_embedding(base[:, :, :0, :64], base[:, :1, :0, :64], f, 0)
    assert qo.shape == (2, 3, 0, 64) and ko.shape == (2, 1, 0, 64)


def test_many_tokens_cross_the_grid():
    q, k = inputs(8, 1, 2, 1, 20011, 16, torch.float32)
    f, _ = K.rotary_frequencies(16)
    qo, ko = K.rotary_embedding(q, k, f, 1)
    close(qo, q, f, (1 + torch.arange(20011))[None], False, 1.0)
    close(ko, k, f, (1 + torch.arange(20011))[None], False, 1.0)


def test_a_rotation_turned_back_gives_the_input():
    q, k = inputs(9, 1, 2, 1, 50, 64, torch.float32)
    f, _ = K.rotary_frequencies(64)
    there = K.rotary_embedding(q, k, f, 1000)
    back = K.rotary_embedding(*there, -f, 1000)
    # two rotations: twice the bound on |a| + |b| <= sqrt(2) of the pair's norm, which a rotation keeps
    room = 2 * 10 * 2.0 ** -24 * 2 * q.abs().max().item() * math.sqrt(2)
    assert (back[0] - q).abs().max().item() <= room + 2 * 2.0 ** -24 * q.abs().max().item()


def test_rotary_refusals():
    q, k = inputs(10, 2, 4, 2, 3, 64, torch.bfloat16)
    f, _ = K.rotary_frequencies(64)
    bad = [dict(query=q[0]), dict(key=k[:1]), dict(key=k[..., :32]), dict(key=k.float()), dict(inv_freq=f.float()),
           dict(inv_freq=torch.cat([f, f])), dict(inv_freq=f[:0]), dict(position=torch.zeros(2, device=DEV)),
           dict(position=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(position=2 ** 31),
           dict(out=(q, None)), dict(out=(q[:1], k)), dict(query=q.double(), key=k.double())]
    for kw in bad:
        with pytest.raises(ValueError):
            K.rotary_embedding(**{**dict(query=q, key=k, inv_freq=f, position=0), **kw})
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rotary_embedding(q.cpu(), None, f, 0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_keys_alone(interleaved):
    """No query heads: the keys turn all the same, into a new tensor and into a given one."""
    q, k = inputs(11, 2, 0, 3, 5, 64, torch.bfloat16)
    f, _ = K.rotary_frequencies(32)
    want = K.rotary_embedding(k, None, f, 7, interleaved=interleaved)[0]
    qo, ko = K.rotary_embedding(q, k, f, 7, interleaved=interleaved)
    assert qo.shape == q.shape and torch.equal(ko, want)
    out = (torch.empty_like(q), torch.full_like(k, 3.0))
    got = K.rotary_embedding(q, k, f, 7, interleaved=interleaved, out=out)
    assert got[0] is out[0] and got[1] is out[1] and torch.equal(out[1], want)
    assert K.rotary_embedding(k, q, f, 7, interleaved=interleaved)[1].shape == q.shape


def test_outputs_that_cannot_be_filled_are_refused():
    """The inputs' memory in another order, memory that several elements share, and a position without a batch."""
    q, k = inputs(12, 2, 4, 4, 4, 64, torch.bfloat16)
    f, _ = K.rotary_frequencies(64)
    one = torch.empty(2, 4, 1, 64, dtype=q.dtype, device=DEV).expand(-1, -1, 4, -1)
    for kw in [dict(out=(q.transpose(1, 2), torch.empty_like(k))), dict(out=(torch.empty_like(q), k.transpose(1, 2))),
               dict(out=(one, torch.empty_like(k))), dict(position=torch.zeros((), dtype=torch.int32, device=DEV)),
               dict(position=torch.zeros(2, 4, 1, dtype=torch.int32, device=DEV))]:
        before = q.clone(), k.clone()
        with pytest.raises(ValueError):
            K.rotary_embedding(**{**dict(query=q, key=k, inv_freq=f, position=0), **kw})
        assert torch.equal(q, before[0]) and torch.equal(k, before[1])
