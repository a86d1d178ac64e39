"""Host-side checks of rotary positions, the 8-bit cache and tree attention: frequencies against their formulas, status
codes of bad parameter blocks, refusal of CPU tensors.  No GPU is touched."""
import math

import pytest
import torch

import kernel_collections_b200 as K
from kernel_collections_b200 import _C


def test_frequencies():
    d, theta, s, L0 = 64, 10000.0, 8.0, 4096
    plain = [theta ** (-2 * j / d) for j in range(d // 2)]
    get = lambda **kw: K.rotary_frequencies(d, theta, device="cpu", **kw)  # noqa: E731
    f, m = get()
    assert f.dtype == torch.float64 and f.tolist() == plain and m == 1.0
    assert get(scaling="linear", factor=s)[0].tolist() == [x / s for x in plain]
    base = get(scaling="base", factor=s)[0]
    # the fastest pair keeps its speed, the slowest is slowed by the factor (a few roundings of 2^-53)
    assert base[0] == 1.0 and abs(base[-1] * s / plain[-1] - 1) < 1e-13
    w = get(scaling="wavelength", factor=s, original_length=L0)[0]
    for x, y in zip(plain, w.tolist()):
        length = 2 * math.pi / x
        if length < L0 / 4:
            assert y == x
        elif length > L0:
            assert y == x / s
        else:
            assert x / s <= y <= x
    y, m = get(scaling="yarn", factor=s, original_length=L0)
    assert m == 0.1 * math.log(s) + 1
    turns = [L0 * x / (2 * math.pi) for x in plain]
    assert all(b == a for a, b, t in zip(plain, y.tolist(), turns) if t > 32 * theta ** (2 / d))
    assert all(abs(b * s / a - 1) < 1e-13 for a, b, t in zip(plain, y.tolist(), turns) if t < theta ** (-2 / d))
    assert (y[1:] <= y[:-1]).all()
    for kw in [dict(scaling="yarn"), dict(scaling="wavelength"), dict(scaling="other"), dict(factor=0.5),
               dict(scaling="wavelength", original_length=L0, low=4.0, high=4.0)]:
        with pytest.raises(ValueError):
            get(**kw)
    for dim in (0, 7, -2):
        with pytest.raises(ValueError):
            K.rotary_frequencies(dim, device="cpu")
    with pytest.raises(ValueError):
        K.rotary_frequencies(2, scaling="base", factor=2.0, device="cpu")


A = 0x10000          # a non-null address that the host never follows


def rotary(**kw):
    f = dict(dtype=1, batch=2, heads=4, kv_heads=2, tokens=3, head_dim=64, rot=64, inter=0, pos=0, mag=1.0, positions=0, psb=0,
             pst=0, freq=A, q=A, k=A, qo=A, ko=A)
    f.update(kw)
    s = (64, 64, 64)
    return _C.ROTARY_PARAMS.pack(f["dtype"], f["batch"], f["heads"], f["kv_heads"], f["tokens"], f["head_dim"], f["rot"], f["inter"],
                                 f["pos"], f["mag"], f["positions"], f["psb"], f["pst"], f["freq"], f["q"], *s, f["k"], *s,
                                 f["qo"], *s, f["ko"], *s)


def cache(**kw):
    f = dict(dtype=1, code=1, batch=2, kv_heads=2, tokens=3, cap=8, head_dim=64, k=A, v=A, kc=A, vc=A, ks=A, vs=A)
    f.update(kw)
    s = (64, 64, 64)
    return _C.CACHE_PARAMS.pack(f["dtype"], f["code"], f["batch"], f["kv_heads"], f["tokens"], f["cap"], f["head_dim"], 0, 0, 0,
                                f["k"], *s, f["v"], *s, f["kc"], *s, f["vc"], *s, f["ks"], 8, 8, f["vs"], 8, 8)


def tree(**kw):
    f = dict(dtype=1, code=0, flags=0, batch=2, heads=8, kv_heads=2, tokens=3, kv_len=1000, head_dim=128, splits=0, scale=1.0,
             q=A, k=A, v=A, ks=0, vs=0, out=A)
    f.update(kw)
    d = f["head_dim"]
    s = (f["kv_heads"] * f["kv_len"] * d, f["kv_len"] * d, d)
    return _C.TREE_PARAMS.pack(f["dtype"], f["code"], f["flags"], f["batch"], f["heads"], f["kv_heads"], f["tokens"], f["kv_len"],
                               d, f["splits"], f["scale"], 0, 0, 0, 0, f["q"], f["heads"] * f["tokens"] * d, f["tokens"] * d, d,
                               f["k"], *s, f["v"], *s, f["ks"], 0, 0, f["vs"], 0, 0, f["out"], f["heads"] * f["tokens"] * d, d)


def test_bad_parameter_blocks_are_refused_on_the_host():
    lib = _C.load()
    for kw in [dict(dtype=3), dict(batch=0), dict(heads=0), dict(kv_heads=-1), dict(tokens=0), dict(head_dim=0), dict(rot=0),
               dict(rot=63), dict(rot=66), dict(q=0), dict(qo=0), dict(k=0), dict(ko=0), dict(kv_heads=0), dict(freq=0)]:
        assert lib.xkv_rotary(rotary(**kw), None) == -1, kw
    assert lib.xkv_rotary(None, None) == -1
    for fn in (lib.xkv_cache_append, lib.xkv_cache_read):
        for kw in [dict(dtype=-1), dict(code=0), dict(code=3), dict(batch=0), dict(kv_heads=0), dict(tokens=0), dict(cap=0),
                   dict(head_dim=0), dict(k=0), dict(v=0), dict(kc=0), dict(vc=0), dict(ks=0), dict(vs=0)]:
            assert fn(cache(**kw), None) == -1, kw
        assert fn(cache(head_dim=1025), None) == -2 and fn(None, None) == -1
        assert fn(cache(batch=32768), None) == -2 and fn(cache(kv_heads=65536), None) == -2
    for kw in [dict(dtype=3), dict(code=3), dict(batch=0), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(tokens=0),
               dict(kv_len=0), dict(head_dim=0), dict(splits=-1), dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(code=1),
               dict(code=2, ks=A)]:
        assert lib.xkv_tree_decode(tree(**kw), None, 0, None) == -1, kw
        assert lib.xkv_tree_decode_workspace_bytes(tree(**kw)) == 0 and lib.xkv_tree_decode_plan(tree(**kw)) is None
    assert lib.xkv_tree_decode(tree(head_dim=257), None, 0, None) == -2
    assert lib.xkv_tree_decode(tree(batch=1 << 20, tokens=1 << 10), None, 0, None) == -2
    assert lib.xkv_tree_decode(None, None, 0, None) == -1
    ok = tree()
    need = lib.xkv_tree_decode_workspace_bytes(ok)
    assert need > 0
    assert lib.xkv_tree_decode(ok, None, 0, None) == -4 and lib.xkv_tree_decode(ok, A, need - 1, None) == -4


def test_cpu_tensors_are_rejected():
    q, k = torch.zeros(1, 4, 2, 64), torch.zeros(1, 2, 8, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.group_query_attention_tree(q, k, k)
    c = K.quantized_cache(1, 2, 8, 64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        K.group_query_attention_quantized(q, c)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.quantized_cache_append(c, k, k, 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rotary_embedding(q, k[:, :, :2], K.rotary_frequencies(64, device="cpu")[0], 0)


def test_kernel_selection_follows_the_call():
    lib = _C.load()
    plan = lambda **kw: lib.xkv_tree_decode_plan(tree(**kw))  # noqa: E731
    q8 = dict(code=1, ks=A, vs=A)
    assert plan(tokens=1) == b"stream" and plan(tokens=1, **q8) == b"stream"
    assert plan(head_dim=96) == b"portable" and plan(dtype=0) == b"portable" and plan(k=A + 2) == b"portable"
    assert plan(dtype=0, **q8) == b"stream" and plan(dtype=0, tokens=64, kv_len=100000, **q8) == b"stream"
    assert plan(flags=_C.FLAG_FORCE_GENERIC) == b"portable"
    # more than 16 query rows per KV head: tcgen05 once re-reading the cache costs more than its set-up
    assert plan(tokens=8, kv_len=1000) == b"stream" and plan(tokens=8, kv_len=100000) == b"tree_tc"
    assert plan(tokens=8, kv_len=1000, flags=_C.FLAG_TREE_TCGEN05) == b"tree_tc"
    assert plan(tokens=8, kv_len=100000, flags=_C.FLAG_TREE_MMA_SYNC) == b"stream"
    assert plan(tokens=4, kv_len=100000, flags=_C.FLAG_TREE_TCGEN05) == b"stream"       # 16 rows
    assert plan(tokens=257, kv_len=100000) == b"stream"


def test_status_words_alone_need_the_library_s_own_bytes():
    lib = _C.load()
    short = dict(tokens=1, kv_len=100)                 # one unit of work per strip: no partial results
    assert lib.xkv_tree_decode_workspace_bytes(tree(**short)) == _C.STATUS_BYTES
    assert lib.xkv_tree_decode_workspace_bytes(tree(tokens=1, kv_len=100000)) > _C.STATUS_BYTES
    text = open(_C.__file__.replace("kernel_collections_b200/_C.py", "include/xkv.h")).read()
    assert f"#define XKV_STATUS_BYTES {_C.STATUS_BYTES}u" in text
