"""Tree attention over dense and 8-bit caches against the definition in 64 bits, evaluated on what the cache holds.

Tolerance per output element.  With w the softmax weights and A = sum w |v| (64 bits), an output is off by at most
  u_out |o|                the final rounding, u = eps / 2 of the type
  u_P A                    weights rounded for the matrix product: eps / 2 of the dense cache's 16-bit type; over an 8-bit
                           cache fp16, 2^-11, in two terms (2^-21) for fp32 queries; nothing for fp32 dense caches
  2 d A                    weights off by a factor e^d (numerator and sum): d = X ((D + 8) 2^-24 + 2^-21) + 2^-21, X the
                           largest sum |q||k| scale; D + 8 roundings of a score, 2^-21 relative for queries held in
                           halves and for the logits' change of base, 2^-21 for the exponential
  2 (L + 8) 2^-24 A        fp32 sums over L tokens, numerator and denominator
and 2^-25 where fp16 is subnormal."""
import math

import pytest
import torch

import kernel_collections_b200 as K
from kernel_collections_b200 import _C

pytestmark = pytest.mark.gpu
DEV = "cuda"
PIN = None


@pytest.fixture(autouse=True, params=[None, True], ids=["chosen", "tcgen05"])
def pinned(request):
    """Every test on the kernel that the library chooses, and on the tcgen05 kernel where it covers the call (the
    library keeps it for larger caches than most tests have)."""
    global PIN
    PIN = request.param
    yield


def random_tree(g, n):
    see = torch.eye(n, dtype=torch.bool)
    for t in range(1, n):
        p = int(torch.randint(max(-1, t - 4), t, (1,), generator=g))
        if p >= 0:
            see[t] |= see[p]
    return see


def dense_of(codes, scales):
    return codes.cpu().float().double() * scales.cpu().double()[..., None]


def reference(q, k, v, mask, lens, scale):
    """(output, sum w|v|, largest sum|q||k| scale) in 64 bits; q (b, H, T, D), k / v (b, KVH, L, D), lens list."""
    b, H, T, D = q.shape
    KVH = k.shape[1]
    G = H // KVH
    out, room = torch.zeros(b, H, T, D, dtype=torch.float64), torch.zeros(b, H, T, D, dtype=torch.float64)
    X = 0.0
    for i in range(b):
        n = max(0, min(lens[i], k.shape[2]))
        if n == 0:
            continue
        m = torch.ones(T, T).tril().bool() if mask is None else (mask if mask.dim() == 2 else mask[i])
        at = torch.arange(n)
        u = at - (n - T)
        see = (u < 0)[None] | m[:, u.clamp(min=0)]
        kk = k[i, :, :n].repeat_interleave(G, 0)
        vv = v[i, :, :n].repeat_interleave(G, 0)
        kk = torch.where(see.any(0)[None, :, None], kk, torch.zeros((), dtype=torch.float64))
        vv = torch.where(see.any(0)[None, :, None], vv, torch.zeros((), dtype=torch.float64))
        s = torch.einsum("htd,hld->htl", q[i], kk) * scale
        X = max(X, (torch.einsum("htd,hld->htl", q[i].abs(), kk.abs()) * abs(scale)).max().item())
        s = s.masked_fill(~see[None], -float("inf"))
        w = torch.softmax(s, -1).masked_fill(~see.any(1)[None, :, None], 0.0)
        out[i] = torch.einsum("htl,hld->htd", w, vv)
        room[i] = torch.einsum("htl,hld->htd", w, vv.abs())
    return out, room, X


def close(got, q, k, v, mask, lens, scale, quantised):
    """`k`, `v`: float64 values that the cache holds."""
    want, room, X = reference(q.cpu().double(), k, v, mask, lens, scale)
    dt = got.dtype
    u = torch.finfo(dt).eps / 2
    up = (2.0 ** -21 if dt == torch.float32 else 2.0 ** -11) if quantised else (0.0 if dt == torch.float32 else u)
    D, L = q.shape[-1], k.shape[2]
    d = X * ((D + 8) * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -21
    tol = u * want.abs() + (up + 2 * d + 2 * (L + 8) * 2.0 ** -24) * room + (2.0 ** -25 if dt == torch.float16 else 1e-37)
    assert torch.isfinite(got).all()
    over = (got.cpu().double() - want).abs() - tol
    assert (over <= 0).all(), f"{over.max().item():.3e} over a tolerance of {tol.flatten()[over.argmax()].item():.3e}"


def rows(g, shape, dtype):
    size = torch.exp(0.5 * torch.randn(1, shape[1], 1, shape[3], generator=g))
    return (torch.randn(shape, generator=g) * size + 0.3).to(dtype)


def case(seed, b, H, KVH, T, L, D, dtype, code, mask_kind="tree", lens=None):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, H, T, D, generator=g).to(dtype)
    k, v = rows(g, (b, KVH, L, D), dtype), rows(g, (b, KVH, L, D), dtype)
    mask = {"tree": lambda: random_tree(g, T), "trees": lambda: torch.stack([random_tree(g, T) for _ in range(b)]),
            "chain": lambda: None, "empty": lambda: torch.zeros(T, T, dtype=torch.bool),
            "any": lambda: torch.rand(b, T, T, generator=g) < 0.5}[mask_kind]()
    return q, k, v, mask, lens


def run(q, k, v, mask, lens, code, scale=None, **kw):
    """Through the public entry points; returns the output and the float64 key / value rows that the cache holds."""
    kw.setdefault("tcgen05", PIN)
    lt = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    m = None if mask is None else mask.to(DEV)
    if code == "dense":
        out = K.group_query_attention_tree(q.to(DEV), k.to(DEV), v.to(DEV), m, sm_scale=scale, kv_lens=lt, **kw)
        return out, k.double(), v.double()
    b, KVH, L, D = k.shape
    cache = K.quantized_cache(b, KVH, L, D, code=code)
    K.quantized_cache_append(cache, k.to(DEV), v.to(DEV), 0)
    out = K.group_query_attention_quantized(q.to(DEV), cache, m, sm_scale=scale, kv_lens=lt, **kw)
    return out, dense_of(cache.key_codes, cache.key_scales), dense_of(cache.value_codes, cache.value_scales)


def check(seed, b, H, KVH, T, L, D, dtype, code, mask_kind="tree", lens=None, scale=None, **kw):
    q, k, v, mask, lens = case(seed, b, H, KVH, T, L, D, dtype, code, mask_kind, lens)
    out, kd, vd = run(q, k, v, mask, lens, code, scale, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype
    close(out, q, kd, vd, mask, lens or [L] * b, D ** -0.5 if scale is None else scale, code != "dense")


TYPES = [torch.float32, torch.bfloat16, torch.float16]
CODES = ["dense", "int8", "e4m3"]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256, 80, 33])
def test_one_token_and_a_tree_at_every_head_size(dtype, code, D):
    check(D, 2, 8, 2, 1, 300, D, dtype, code)
    check(D + 1, 2, 8, 2, 5, 300, D, dtype, code)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(1, 1), (1, 16), (5, 3), (4, 4), (1, 17), (8, 4), (4, 16), (3, 21), (8, 16), (1, 129),
                                 (5, 26), (8, 64), (1, 300)])
def test_row_counts(dtype, code, G, T):
    """G heads per KV head times T drafted tokens: below, at and above the row blocks of every kernel."""
    check(G * 100 + T, 2, 2 * G, 2, T, 413, 128, dtype, code, "trees")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4099])
def test_lengths(dtype, code, L):
    check(L, 1, 4, 1, 1, L, 128, dtype, code)
    check(L + 1, 2, 8, 2, min(L, 6), L, 64, dtype, code, "tree")
    check(L + 2, 1, 16, 1, min(L, 9), L, 128, dtype, code, "any")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(4, 1), (4, 3), (8, 12), (8, 40)])
def test_ragged_lengths_short_long_and_none(dtype, code, G, T):
    """Lengths of zero, below the number of drafted tokens, at the tile borders, at and past the capacity."""
    lens = [0, 1, 2, T, T + 1, 64, 63 + T, 128, 700, 701, 5000, -4]
    check(T, len(lens), G * 2, 2, T, 701, 128, dtype, code, "tree", lens)
    check(T, len(lens), G * 2, 2, T, 701, 64, dtype, code, "any", lens)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [2, 7, 33])
def test_chain_by_default_and_rows_that_see_nothing(dtype, code, T):
    check(T, 2, 8, 2, T, 200, 128, dtype, code, "chain")
    check(T, 2, 8, 2, T, 200, 128, dtype, code, "empty")
    q, k, v, mask, _ = case(T, 2, 8, 2, T, T, 128, dtype, code, "empty")        # nothing in front of the drafted rows
    out, _, _ = run(q, k, v, mask, None, code)
    assert (out == 0).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(4, 4), (8, 20)])
def test_what_a_token_does_not_see_does_not_reach_it(dtype, code, G, T):
    """Drafted rows hidden from some tokens and rows past the length hold NaN and infinities."""
    b, KVH, L, D = 3, 2, 300, 128
    q, k, v, mask, lens = case(T, b, KVH * G, KVH, T, L, D, dtype, code, "trees", [300, 150, 64 + T])
    mask[:, :, T - 1] = False                                     # token T-1's row: only token T-1 sees it
    mask[:, T - 1, T - 1] = True
    clean, _, _ = run(q, k, v, mask, lens, code)
    for bad in (float("nan"), float("inf"), -float("inf")):
        kb, vb = k.clone(), v.clone()
        for i, n in enumerate(lens):
            for x in (kb, vb):
                x[i, :, n - 1, 5:9] = bad
                x[i, :, n:] = bad
        out, _, _ = run(q, kb, vb, mask, lens, code)
        assert torch.equal(out[:, :, :T - 1], clean[:, :, :T - 1])
        assert out[:, :, T - 1, 5:9].isnan().all() or bad != bad or code == "dense"
        if bad != bad:
            assert out[:, :, T - 1].isnan().all()
    # a NaN in front of the drafted rows is seen by all of that sequence's tokens, and by no other sequence's
    kb = k.clone()
    kb[1, 0, 7, 0] = float("nan")
    out, _, _ = run(q, kb, v, mask, lens, code)
    assert out[1, :G].isnan().all() and torch.equal(out[0], clean[0]) and torch.equal(out[1, G:], clean[1, G:])
    assert torch.equal(out[2], clean[2])


@pytest.mark.parametrize("dtype", TYPES)
def test_an_infinite_value_reaches_only_its_column(dtype):
    """Dense values: a visible drafted row with an infinity in one element gives that element alone."""
    T, G = 4, 4
    q, k, v, mask, _ = case(3, 1, 2 * G, 2, T, 100, 128, dtype, "dense", "tree")
    mask[:, T - 1] = torch.tensor([False] * (T - 1) + [True])
    clean, _, _ = run(q, k, v, mask, None, "dense")
    v[:, :, 99, 17] = float("inf")
    out, _, _ = run(q, k, v, mask, None, "dense")
    assert (out[:, :, T - 1, 17] == float("inf")).all()
    keep = torch.ones(128, dtype=torch.bool)
    keep[17] = False
    assert torch.equal(out[..., keep.to(DEV)], clean[..., keep.to(DEV)]) and torch.equal(out[:, :, :T - 1], clean[:, :, :T - 1])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_growing_logits(dtype, code):
    """Scores that climb along the cache (the running maximum moves at every tile), and a scale that makes one token
    take everything."""
    b, H, KVH, T, L, D = 1, 8, 2, 3, 700, 128
    q, k, v, mask, _ = case(4, b, H, KVH, T, L, D, dtype, code, "tree")
    ramp = torch.linspace(0, 4, L)[None, None, :, None]
    q = q.abs()
    k = (k.abs() * 0.05 + ramp).to(dtype)
    for scale in (0.05, 0.5, -0.05):
        out, kd, vd = run(q, k, v, mask, None, code, scale)
        close(out, q, kd, vd, mask, [L], scale, code != "dense")


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_very_different_scales(dtype, code):
    """Value rows whose scales span eight decades, and growing: the product's common factor moves along the cache.  The
    weights are rounded relative to the largest scale so far, so the room is that of the largest row."""
    b, H, KVH, T, L, D = 1, 8, 2, 2, 500, 128
    q, k, v, mask, _ = case(5, b, H, KVH, T, L, D, torch.float32, code, "tree")
    v = v * torch.logspace(-6, 2, L)[None, None, :, None]
    v = v.clamp(-60000, 60000).to(dtype)
    q, k = q.to(dtype), k.to(dtype)
    for x in (v, v.flip(2)):
        out, kd, vd = run(q, k, x, mask, None, code)
        close(out, q, kd, vd, mask, [L], D ** -0.5, True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
def test_queries_of_any_magnitude(dtype, code):
    q, k, v, mask, _ = case(6, 1, 8, 2, 2, 300, 128, torch.float32, code, "tree")
    for size in (1e-3, 1.0, 3e4 if dtype == torch.float16 else 1e8):
        x = (q.clamp(-2, 2) * size).to(dtype)
        out, kd, vd = run(x, k.to(dtype), v.to(dtype), mask, None, code, 0.05 / size)
        close(out, x, kd, vd, mask, [300], 0.05 / size, True)
    x = q.to(dtype)
    x[0, 3] = 0.0
    x[0, 5, 1, 7] = float("inf")
    out, _, _ = run(x, k.to(dtype), v.to(dtype), mask, None, code)
    clean, _, _ = run(q.to(dtype), k.to(dtype), v.to(dtype), mask, None, code)
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(out[:, keep], clean[:, keep]) and torch.equal(out[0, 5, 0], clean[0, 5, 0]) and out[0, 5, 1].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 6, 30])
def test_strided_and_unaligned_caches_and_queries(dtype, T):
    b, H, KVH, L, D = 2, 16, 2, 333, 128
    q, k, v, mask, _ = case(7, b, H, KVH, T, L, D, dtype, "dense", "trees")
    want, _, _ = run(q, k, v, mask, None, "dense")
    m = mask.to(DEV)
    tok = lambda t: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)  # noqa: E731
    wide = lambda t: torch.cat([t, t], -1).to(DEV)[..., :D]  # noqa: E731
    odd = lambda t: torch.cat([t[..., :1], t], -1).to(DEV)[..., 1:]  # noqa: E731
    flip = lambda t: t.transpose(2, 3).contiguous().to(DEV).transpose(2, 3)  # noqa: E731
    for f in (tok, wide, flip):
        assert torch.equal(K.group_query_attention_tree(f(q), f(k), f(v), m, tcgen05=PIN), want)
    out = K.group_query_attention_tree(odd(q), odd(k), odd(v), m)      # another kernel: compare with 64 bits
    close(out, q, k.double(), v.double(), mask, [L] * b, D ** -0.5, False)
    m2 = torch.zeros(b, T, 2 * T, dtype=torch.bool, device=DEV)
    m2[:, :, ::2] = m
    assert torch.equal(K.group_query_attention_tree(q.to(DEV), k.to(DEV), v.to(DEV), m2[:, :, ::2], tcgen05=PIN), want)
    shared = K.group_query_attention_tree(q.to(DEV), k[:1].to(DEV).expand(b, -1, -1, -1), v[:1].to(DEV).expand(b, -1, -1, -1), m,
                                          tcgen05=PIN)
    assert torch.equal(shared[0], want[0])


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_strided_quantised_cache(code, T):
    b, H, KVH, L, D = 2, 16, 2, 333, 128
    q, k, v, mask, _ = case(8, b, H, KVH, T, L, D, torch.bfloat16, code, "trees")
    c = K.quantized_cache(b, KVH, L, D, code=code)
    K.quantized_cache_append(c, k.to(DEV), v.to(DEV), 0)
    want = K.group_query_attention_quantized(q.to(DEV), c, mask.to(DEV), tcgen05=PIN)
    tok = lambda t: t.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(t.dtype)  # noqa: E731
    pad = lambda t: torch.cat([t, t[..., :5]], -1)[..., :L]  # noqa: E731
    c2 = K.QuantizedCache(tok(c.key_codes), pad(c.key_scales), tok(c.value_codes), pad(c.value_scales))
    assert torch.equal(K.group_query_attention_quantized(q.to(DEV), c2, mask.to(DEV), tcgen05=PIN), want)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T", [1, 5, 40])
def test_split_counts_repeats_and_the_portable_kernel_agree(code, T):
    b, H, KVH, L, D = 1, 8, 2, 2000, 128
    q, k, v, mask, _ = case(9, b, H, KVH, T, L, D, torch.bfloat16, code, "tree")
    first, kd, vd = run(q, k, v, mask, None, code)
    again, _, _ = run(q, k, v, mask, None, code)
    assert torch.equal(first, again)
    for kw in (dict(num_splits=1), dict(num_splits=3), dict(num_splits=64), dict(force_generic=True), dict(tcgen05=False)):
        out, _, _ = run(q, k, v, mask, None, code, **kw)
        close(out, q, kd, vd, mask, [L], D ** -0.5, code != "dense")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("G,T", [(4, 1), (8, 32)])
def test_captured_calls_replay_and_two_graphs_run_side_by_side(code, G, T):
    b, KVH, L, D = 2, 2, 1500, 128
    sets = []
    for seed in (10, 11):
        q, k, v, mask, _ = case(seed, b, KVH * G, KVH, T, L, D, torch.bfloat16, code, "tree")
        want, _, _ = run(q, k, v, mask, None, code)
        qd, kd, vd, md = q.to(DEV), k.to(DEV), v.to(DEV), mask.to(DEV)
        if code == "dense":
            call = lambda qd=qd, kd=kd, vd=vd, md=md: K.group_query_attention_tree(qd, kd, vd, md, tcgen05=PIN)  # noqa: E731
        else:
            c = K.quantized_cache(b, KVH, L, D, code=code)
            K.quantized_cache_append(c, kd, vd, 0)
            call = lambda qd=qd, c=c, md=md: K.group_query_attention_quantized(qd, c, md, tcgen05=PIN)  # noqa: E731
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        sets.append((graph, out, want, torch.cuda.Stream(), call))       # `call` keeps the captured inputs alive
    junk = [torch.full((1 << 22,), float("nan"), device=DEV) for _ in range(4)]       # other allocations in between
    for _ in range(5):
        for graph, out, _, stream, _ in sets:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                out.fill_(float("nan"))
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _, _ in sets:
            assert torch.equal(out, want)
    del junk


def test_another_stream_and_no_sync_between_calls():
    q, k, v, mask, _ = case(12, 2, 8, 2, 9, 900, 128, torch.float16, "dense", "tree")
    want, _, _ = run(q, k, v, mask, None, "dense")
    qd, kd, vd, md = q.to(DEV), k.to(DEV), v.to(DEV), mask.to(DEV)
    torch.cuda.synchronize()
    outs = []
    for _ in range(6):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(4):
                outs.append(K.group_query_attention_tree(qd, kd, vd, md, tcgen05=PIN))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_two_host_threads_at_once():
    """Calls of several shapes from two threads, on one stream and on two: none sees the other's partial results."""
    import threading
    cases = []
    for i, (T, L, code) in enumerate([(1, 5000, "int8"), (9, 700, "dense"), (1, 300, "e4m3"), (30, 2000, "dense")]):
        q, k, v, mask, _ = case(20 + i, 2, 8, 2, T, L, 128, torch.bfloat16, code, "tree")
        want, _, _ = run(q, k, v, mask, None, code)
        qd, kd, vd, md = q.to(DEV), k.to(DEV), v.to(DEV), mask.to(DEV)
        if code == "dense":
            cases.append((lambda qd=qd, kd=kd, vd=vd, md=md: K.group_query_attention_tree(qd, kd, vd, md, tcgen05=PIN), want))
        else:
            c = K.quantized_cache(2, 2, L, 128, code=code)
            K.quantized_cache_append(c, kd, vd, 0)
            cases.append((lambda qd=qd, c=c, md=md: K.group_query_attention_quantized(qd, c, md, tcgen05=PIN), want))
    torch.cuda.synchronize()
    wrong = []

    def work(first, stream):
        try:
            with torch.cuda.stream(stream):
                outs = [(n, cases[n][0]()) for i in range(60) for n in [(first + i) % len(cases)]]
            stream.synchronize()
            wrong.extend(n for n, o in outs if not torch.equal(o, cases[n][1]))
        except Exception as e:      # a thread's exception is not the test's
            wrong.append(repr(e))

    for streams in ((torch.cuda.current_stream(),) * 2, (torch.cuda.Stream(), torch.cuda.Stream())):
        # (first = 1, 3: dense caches, whose tensor maps are the threads' first CUDA calls)
        threads = [threading.Thread(target=work, args=(2 * i + 1, s)) for i, s in enumerate(streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong, wrong


def test_a_long_cache_past_32_bit_offsets():
    """The last rows of the second sequence lie past 2^31 elements."""
    KVH, D, L = 8, 128, 1_050_000
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.zeros(2, KVH, L, D, dtype=torch.float16, device=DEV)
    assert k.numel() > 2 ** 31
    n = 70
    tail = torch.randn(2, KVH, n, D, generator=g, device=DEV).half()
    k[:, :, L - n:] = tail
    q = (torch.randn(2, 16, 2, D, generator=g, device=DEV) * 4).half()
    out = K.group_query_attention_tree(q, k, k, sm_scale=1.0, tcgen05=PIN)
    s = torch.einsum("bhgtd,bhld->bhgtl", q.double().view(2, KVH, 2, 2, D), tail.double())
    s[:, :, :, 0, n - 1] = -float("inf")
    zeros = float(L - n)
    m = s.amax(-1, keepdim=True).clamp(min=0)
    w = torch.exp(s - m)
    total = w.sum(-1, keepdim=True) + zeros * torch.exp(-m)
    want = torch.einsum("bhgtl,bhld->bhgtd", w / total, tail.double()).reshape(2, 16, 2, D)
    room = torch.einsum("bhgtl,bhld->bhgtd", w / total, tail.double().abs()).reshape(2, 16, 2, D)
    X = torch.einsum("bhgtd,bhld->bhgtl", q.double().abs().view(2, KVH, 2, 2, D), tail.double().abs()).max().item()
    # the zero rows' weights are equal: their sum is within the tolerance's terms for 64 splits of 32-bit sums
    d = X * ((D + 8) * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -21
    tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * d + 2 * L * 2.0 ** -24) * room + 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all()


def test_a_verification_step_rotates_writes_and_attends():
    """The operators together, twice in a row: prompts written, then two trees rotated, appended and attended to."""
    b, H, KVH, D, cap, T = 3, 8, 2, 128, 400, 7
    g = torch.Generator().manual_seed(13)
    f, mag = K.rotary_frequencies(64, 500000.0, scaling="yarn", factor=4.0, original_length=128)
    lens = torch.tensor([120, 0, 301], dtype=torch.int32)
    cache = K.quantized_cache(b, KVH, cap, D, code="int8")
    kd, vd = torch.zeros(b, KVH, cap, D, dtype=torch.float64), torch.zeros(b, KVH, cap, D, dtype=torch.float64)

    def rotate64(x, pos):
        y = x.double().clone()
        ang = pos.double()[:, None, :, None] * f.cpu()
        c, s = torch.cos(ang) * mag, torch.sin(ang) * mag
        a, w = x.double()[..., 0:64:2], x.double()[..., 1:64:2]
        y[..., 0:64:2], y[..., 1:64:2] = a * c - w * s, w * c + a * s
        return y

    def step(n, pos, at, lengths):
        q = torch.randn(b, H, n, D, generator=g).bfloat16()
        k, v = (torch.randn(b, KVH, n, D, generator=g).bfloat16() for _ in "kv")
        qr, kr = K.rotary_embedding(q.to(DEV), k.to(DEV), f, pos.to(DEV), interleaved=True, magnitude=mag)
        K.quantized_cache_append(cache, kr, v.to(DEV), at.to(DEV), lengths=lengths)
        for src, x in ((q, qr), (k, kr)):
            want = rotate64(src, pos)
            assert ((x.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 20 * 2.0 ** -24 * mag * 8).all()
        return qr

    n = 310
    pos = torch.arange(n, dtype=torch.int32).expand(b, n)
    step(n, pos, torch.zeros(b, dtype=torch.int32), lens.to(DEV))
    for _ in range(2):
        mask = torch.stack([random_tree(g, T) for _ in range(b)])
        depth = mask.sum(-1).to(torch.int32) - 1
        qr = step(T, lens[:, None] + depth, lens, None)
        lens = lens + T
        out = K.group_query_attention_quantized(qr, cache, mask.to(DEV), kv_lens=lens.to(DEV), tcgen05=PIN)
        kd, vd = dense_of(cache.key_codes, cache.key_scales), dense_of(cache.value_codes, cache.value_scales)
        close(out, qr, kd, vd, mask, lens.tolist(), D ** -0.5, True)
    # what was written reads back as what the attention saw
    rk, rv = K.quantized_cache_read(cache, 0, cap, dtype=torch.float32)
    assert torch.equal(rk.cpu(), kd.float()) and torch.equal(rv.cpu(), vd.float())


def test_tree_refusals():
    b, H, KVH, T, L, D = 2, 8, 2, 3, 20, 64
    q, k, v, mask, _ = (x if x is None else x.to(DEV) for x in case(14, b, H, KVH, T, L, D, torch.bfloat16, "dense", "tree"))
    i32 = dict(dtype=torch.int32, device=DEV)
    for kw in [dict(query=q[0]), dict(query=q[:1]), dict(query=q.float()), dict(query=q[..., :32]), dict(query=q[:, :3]),
               dict(key=k[:, :1]), dict(value=v[:, :, :5]), dict(value=v.float()), dict(tree_mask=mask.float()),
               dict(tree_mask=mask[:2]), dict(tree_mask=mask[None]), dict(kv_lens=torch.zeros(2, device=DEV)),
               dict(kv_lens=torch.zeros(3, **i32)), dict(key=k[:, :, :0], value=v[:, :, :0]), dict(num_splits=-1)]:
        with pytest.raises(ValueError):
            K.group_query_attention_tree(**{**dict(query=q, key=k, value=v, tree_mask=mask), **kw})
    big = torch.zeros(1, 1, 2, 260, device=DEV)
    with pytest.raises(ValueError):
        K.group_query_attention_tree(big, big, big)
    c = K.quantized_cache(b, KVH, L, D)
    for kw in [dict(query=q[:1]), dict(query=q[..., :32]), dict(query=q[:, :3]), dict(query=q.double()), dict(tree_mask=mask.int())]:
        with pytest.raises(ValueError):
            K.group_query_attention_quantized(**{**dict(query=q, cache=c, tree_mask=mask), **kw})


def test_status_check_passes_on_good_calls():
    prev = _C.set_check_status(True)
    try:
        check(15, 2, 8, 2, 20, 300, 128, torch.bfloat16, "dense")
        check(15, 2, 8, 2, 20, 300, 128, torch.bfloat16, "int8")
    finally:
        _C.set_check_status(prev)


def test_calls_that_need_no_scratch_leave_other_memory_alone():
    """A device's first small call comes on a stream whose freed tensor is still being read there; a second small call on
    another stream does not wait for it.  Neither stores anything in the tensor's memory."""
    q, k, v, mask, _ = case(30, 1, 8, 2, 2, 60, 128, torch.bfloat16, "dense", "tree")
    want, _, _ = run(q, k, v, mask, None, "dense", tcgen05=False)
    qd, kd, vd, md = q.to(DEV), k.to(DEV), v.to(DEV), mask.to(DEV)
    call = lambda: K.group_query_attention_tree(qd, kd, vd, md, tcgen05=False, check_status=False)  # noqa: E731
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for nbytes in (256, 512):
        _C._status_scratch.clear()
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            x = torch.full((nbytes,), 7, dtype=torch.uint8, device=DEV)
            torch.cuda._sleep(20_000_000)              # some 10 ms
            y = x.clone()
            del x
            first = call()
        with torch.cuda.stream(two):
            second = call()
        torch.cuda.synchronize()
        assert (y == 7).all() and torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("G,T", [(4, 8), (8, 40)])
def test_runs_of_idle_sequences(code, G, T):
    """Slots of a serving batch that hold nothing, one after the other within a block's share of the work: no tiles, and
    still a row of zeros each; the sequences in between are as they are alone."""
    b, KVH, L, D = 700, 2, 260, 64
    lens = [0] * b
    for i, n in ((0, 260), (5, 130), (6, 41), (350, 129), (699, 260)):
        lens[i] = n
    q, k, v, mask, _ = case(T, b, KVH * G, KVH, T, L, D, torch.bfloat16, code, "tree")
    out, kd, vd = run(q, k, v, mask, lens, code, check_status=True)
    busy = [i for i in range(b) if lens[i]]
    idle = torch.tensor([n == 0 for n in lens], device=DEV)
    assert (out[idle] == 0).all()
    close(out[busy], q[busy], kd[busy], vd[busy], mask, [lens[i] for i in busy], D ** -0.5, code != "dense")


def scattered(v, lens, T, kinds):
    """`v` with one element of every drafted row replaced by one of `kinds` in turn, and the places: (sequence, drafted token,
    column, kind)."""
    v = v.clone()
    places = []
    for i, n in enumerate(lens):
        for u in range(T):
            if n - T + u < 0:
                continue
            col, kind = (7 * u + 31 * (u % 2)) % v.shape[3], kinds[u % len(kinds)]
            v[i, :, n - T + u, col] = kind
            places.append((i, u, col, kind))
    return v, places


def expected_with(clean, places, mask, T):
    """`clean` (the output with zeros in those places) plus what each token sees of them."""
    want = clean.cpu().clone()
    for i, u, col, kind in places:
        sees = (mask if mask.dim() == 2 else mask[i])[:, u]
        want[i, :, sees, col] += torch.tensor(kind, dtype=want.dtype)
    return want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T,D", [(4, 3, 128), (4, 8, 128), (4, 8, 64), (8, 40, 128), (8, 40, 64), (1, 250, 128)])
def test_values_that_are_not_finite_reach_their_column_of_the_rows_that_see_them(dtype, G, T, D):
    """Dense drafted rows, every one with a NaN or an infinity somewhere; the tree hides most from any one token."""
    b, KVH, L = 2, 2, 300
    lens = [300, max(T - 2, 1)]
    q, k, v, mask, _ = case(T + D, b, KVH * G, KVH, T, L, D, dtype, "dense", "trees")
    bad, places = scattered(v, lens, T, [float("inf"), float("nan"), -float("inf"), float("inf")])
    zero, _ = scattered(v, lens, T, [0.0])
    clean, _, _ = run(q, k, zero, mask, lens, "dense")
    out, _, _ = run(q, k, bad, mask, lens, "dense")
    want = expected_with(clean, places, mask, T)
    out = out.cpu()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(5.0, 6.0, 7.0), want.nan_to_num(5.0, 6.0, 7.0))
    assert want.isnan().any() and want.isinf().any() and want.isfinite().any()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(4, 1), (4, 4), (8, 20)])
def test_keys_with_one_large_channel(dtype, code, G, T):
    """One channel sets the scale of every key row and the queries hardly look at it: the codes they do look at are 0 and
    +-1, and the queries share a sign, so that an offset of the codes would add up to much more than the score."""
    L, D = 400, 128
    g = torch.Generator().manual_seed(T)
    q = torch.rand(1, 2 * G, T, D, generator=g) + 0.5
    q[..., 77] = 2.0 ** -10
    k = 8.0 * torch.randint(-1, 2, (1, 2, L, D), generator=g).float()
    k[..., 77] = 8.0 * 127
    v = torch.randn(1, 2, L, D, generator=g)
    q = q.to(dtype)
    mask = random_tree(g, T)
    out, kd, vd = run(q, k, v, mask, None, code)
    close(out, q, kd, vd, mask, [L], D ** -0.5, True)


def weighed(seed, G, T, L, low, dtype):
    """Queries and keys whose scores are ordinary but for the rows `low`, which lie that many bits (log2) below.  The
    offset is a channel of its own: 1 in every query, negative in those keys."""
    D = 128
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(1, 2 * G, T, D, generator=g)
    k = torch.randn(1, 2, L, D, generator=g) * 0.3
    v = torch.randn(1, 2, L, D, generator=g)
    q[..., 0], k[..., 0] = 1.0, 0.0
    for row, bits in low.items():
        k[:, :, row] = 0.0
        k[:, :, row, 0] = -bits * math.log(2.0) * D ** 0.5
    return q.to(dtype), k, v, random_tree(g, T)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(4, 1), (4, 4), (4, 8), (8, 20)])
@pytest.mark.parametrize("L", [60, 700])
@pytest.mark.parametrize("bits,size", [(60, 24), (60, 32), (100, 60)])
def test_large_values_that_carry_no_weight_take_no_bits(dtype, code, G, T, L, bits, size):
    """Rows whose values are 2^size times the others' and whose weights are 2^-bits: all others keep their precision."""
    at = [0, 17, L // 2]
    q, k, v, mask = weighed(bits + T, G, T, L, {i: bits for i in at}, dtype)
    for i in at:
        v[:, :, i] *= 2.0 ** size
    out, kd, vd = run(q, k, v, mask, None, code)
    close(out, q, kd, vd, mask, [L], 128 ** -0.5, True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,T", [(4, 1), (4, 4), (4, 8), (8, 20)])
@pytest.mark.parametrize("size", [-60, -110])
def test_small_values_that_carry_all_the_weight(dtype, code, G, T, size):
    """One row takes all the weight and its values are 2^size of the others', whose weights are near 2^-40: what they add
    is most of the output.  Then the row's values are zeros."""
    L = 300
    q, k, v, mask = weighed(T, G, T, L, {i: 40 for i in range(L) if i != 5}, dtype)
    for factor in (2.0 ** size, 0.0):
        x = v.clone()
        x[:, :, 5] *= factor
        out, kd, vd = run(q, k, x, mask, None, code)
        close(out, q, kd, vd, mask, [L], 128 ** -0.5, True)
        assert (out != 0).any()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(4, 1), (4, 4), (4, 8), (8, 20)])
def test_rows_of_zeros_before_and_between_values(dtype, code, G, T):
    """Value rows of zeros have no scale to be relative to: first all of them, then the first 300, then every second."""
    L = 500
    q, k, v, mask = weighed(T, G, T, L, {}, dtype)
    out, _, _ = run(q, k, v * 0.0, mask, None, code)
    assert (out == 0).all()
    for zeros in (slice(0, 300), slice(0, L, 2)):
        x = v.clone()
        x[:, :, zeros] = 0.0
        out, kd, vd = run(q, k, x, mask, None, code)
        close(out, q, kd, vd, mask, [L], 128 ** -0.5, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T,D", [(4, 3, 128), (4, 8, 128), (4, 8, 64), (8, 40, 128), (8, 40, 64)])
@pytest.mark.parametrize("generic", [False, True])
def test_nan_codes_reach_their_column_of_the_rows_that_see_them(dtype, G, T, D, generic):
    """e4m3 codes 0x7f and 0xff (a cache may come from anywhere) in one element of every drafted value row, and of a row
    in front of them: the same rule in every kernel."""
    b, KVH, L = 2, 2, 300
    lens = [300, max(T - 2, 1)]
    q, k, v, mask, _ = case(T + D, b, KVH * G, KVH, T, L, D, dtype, "e4m3", "trees")
    c = K.quantized_cache(b, KVH, L, D, code="e4m3")
    K.quantized_cache_append(c, k.to(DEV), v.to(DEV), 0)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kw = dict(force_generic=True) if generic else dict(tcgen05=PIN)
    call = lambda: K.group_query_attention_quantized(q.to(DEV), c, mask.to(DEV), kv_lens=lt, **kw).cpu()  # noqa: E731
    held = c.value_codes.view(torch.uint8).cpu()
    zero, places = scattered(held, lens, T, [0x00])
    bad, _ = scattered(held, lens, T, [0x7f, 0xff])
    c.value_codes.view(torch.uint8).copy_(zero)
    clean = call()
    want = expected_with(clean, [(i, u, col, float("nan")) for i, u, col, _ in places], mask, T)
    c.value_codes.view(torch.uint8).copy_(bad)
    out = call()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(5.0), want.nan_to_num(5.0))
    assert want.isnan().any() and want.isfinite().any()
    bad = zero.clone()
    bad[0, 0, 290 - T, 3] = bad[0, 0, 20, 9] = 0x7f                  # in the drafted rows' tile (or the one before), and far in front
    c.value_codes.view(torch.uint8).copy_(bad)
    out = call()
    assert out[0, :G][..., [3, 9]].isnan().all()
    out[0, :G, :, 3], out[0, :G, :, 9] = clean[0, :G, :, 3], clean[0, :G, :, 9]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(4, 4), (8, 20)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_an_infinite_key_that_a_token_sees(dtype, G, T, sign):
    """Dense caches, one infinite key element in a row that only the last token sees: a score of +inf makes its output
    NaN, as inf - inf does in the definition; a score of -inf leaves the row without weight."""
    L = 300
    q, k, v, mask, _ = case(T, 1, 2 * G, 2, T, L, 128, dtype, "dense", "tree")
    q = torch.where(q == 0, torch.ones_like(q), q)
    mask[:, T - 1] = False
    hidden, _, _ = run(q, k, v, mask, None, "dense")
    mask[T - 1, T - 1] = True
    clean, _, _ = run(q, k, v, mask, None, "dense")
    k[:, :, L - 1, 40] = sign * float("inf")
    out, _, _ = run(q, k, v, mask, None, "dense")
    assert torch.equal(out[:, :, :T - 1], clean[:, :, :T - 1])
    up = (q[:, :, T - 1, 40] * sign > 0).to(DEV)
    last = out[:, :, T - 1]
    assert up.any() and (~up).any()
    assert last[up].isnan().all() and torch.equal(last[~up], hidden[:, :, T - 1][~up])


def test_no_key_heads_and_counts_past_32_bits_are_refused():
    q = torch.zeros(2, 8, 3, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(2, 2, 20, 64, dtype=torch.bfloat16, device=DEV)
    c = K.quantized_cache(2, 2, 20, 64)
    for kw in [dict(key=k[:, :0], value=k[:, :0]), dict(num_splits=2 ** 31)]:
        with pytest.raises(ValueError):
            K.group_query_attention_tree(**{**dict(query=q, key=k, value=k), **kw})
    with pytest.raises(ValueError):
        K.group_query_attention_quantized(q, K.quantized_cache(2, 0, 20, 64))
    with pytest.raises(ValueError):
        K.quantized_cache_read(c, 0, 2 ** 31)
