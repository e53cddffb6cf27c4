"""GPU: attention over the paged 4-bit KV cache (acb_attn_kv_q4) against the 64-bit softmax over the values it holds.

Bar, per element, with A = sum_j p_j |v_j| and S = max_j |scale| * sum_d |q_d k_jd|: a score is a sum of D products in f32, so it
is off by at most (D + 4) 2^-24 S (D roundings, the scale, the exponent's argument twice, its power), a weight by e^that, the
output by twice that times A (weight and sum); the sums of P and PV over n keys in f32 add (n + D) 2^-24 A in the worst case,
taken as 2^-15 A (n <= 400 here; longer ones are checked at sqrt(n)). For 16-bit types P may be an f16 number (half a step
2^-11 of each weight: 2^-11 A) and q may be scaled into f16 (2^-11 of an f16 step below the row's largest: 2^-22 S). Then half
a step of the output.
P is held in f16 as 2^6 p / p_ref, p_ref at most the largest weight met: a weight below f16's normal range keeps an absolute
error of half of its smallest number, 2^-25, against a largest weight of 2^6 or more, so of at most 2^-31 of the largest weight
(which is at most the sum): 2^-31 sum_j |v_j| in the output. It shows only where the keys that weigh have a value of zero."""
import numpy as np
import pytest

import acb
import serving_ref as S

pytestmark = pytest.mark.gpu


def _cache(rng, n_seq, max_len, page, Nkv, D, spare=2, big=1.0):
    import torch
    mp = -(-max_len // page)
    n_pages = n_seq * mp + spare
    table = torch.from_numpy(rng.permutation(n_pages)[:n_seq * mp].reshape(n_seq, mp).astype(np.int32)).cuda()
    t = []
    for _ in "kv":
        t.append(torch.from_numpy(rng.integers(0, 256, (n_pages, Nkv, page, D // 2), dtype=np.uint8)).cuda())
        d = S.bf16((big * rng.uniform(0.02, 0.2, (n_pages, Nkv, page, D // 32)) * rng.choice([-1, 1], (n_pages, Nkv, page, D // 32)))
                   .astype(np.float32)).astype(np.float16)
        t.append(torch.from_numpy(d).cuda())
    return acb.KVCacheQ4(*t, table)


def _held(cache, s, n):
    kc, ks, vc, vs, table = (t.cpu().numpy() for t in cache.tensors)
    P = kc.shape[2]
    pg = table[s, np.arange(n) // P]
    at = np.arange(n) % P
    return S.values(kc[pg, :, at], ks[pg, :, at]), S.values(vc[pg, :, at], vs[pg, :, at])


def _check(cache, q, o, q_lens, kv_lens, window, scale, kind, starts=None):
    q, o = q.float().cpu().numpy().astype(np.float64), o.float().cpu().numpy().astype(np.float64)
    T, H, D = q.shape
    G = H // cache.n_kv_heads
    at = 0
    for s, (n, m) in enumerate(zip(q_lens, kv_lens)):
        r0 = starts[s] if starts else at
        at += n
        if n == 0:
            continue
        k, v = _held(cache, s, m)
        for h in range(H):
            ref, A, s1, av = S.attention(q[r0:r0 + n, h], k[:, h // G], v[:, h // G], m - n, window, scale)
            ds = (D + 4) * 2.0 ** -24 * s1 + (2.0 ** -21 * s1 if kind != "f32" else 0)
            tol = A * (2 * ds + 2.0 ** -15 + (2.0 ** -11 if kind != "f32" else 0)) + 2.0 ** -31 * av
            tol = tol + S.HALF_STEP[kind] * (np.abs(ref) + tol) + (2.0 ** -25 if kind == "f16" else 0)
            d = np.abs(o[r0:r0 + n, h] - ref)
            assert (d <= tol).all(), (s, h, float(d.max()), float((d / (tol + 1e-30)).max()))


def _run(rng, q_lens, kv_lens, page, Nkv, G, D, kind, window=0, scale=None, max_len=None, **kw):
    import torch
    n_seq, T, H = len(q_lens), sum(q_lens), Nkv * G
    cache = _cache(rng, n_seq, max_len or max(max(kv_lens), 1), page, Nkv, D)
    q = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    start = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32).cuda()
    ln = torch.tensor(kv_lens, dtype=torch.int32).cuda()
    err = torch.zeros(1, dtype=torch.int32).cuda()
    o = cache.attention(q, ln, start, max(max(q_lens), 1), window=window, scale=scale, err=err, **kw)
    assert int(err) == 0
    _check(cache, q, o, q_lens, kv_lens, window, D ** -0.5 if scale is None else scale, kind)
    return cache, q, ln, start, o


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,Nkv,G,page", [(128, 2, 2, 64), (64, 1, 7, 16), (256, 2, 4, 32), (128, 1, 1, 16), (128, 1, 9, 128),
                                          (64, 3, 16, 16), (256, 1, 17, 16)])
def test_single_tokens(cuda, kind, D, Nkv, G, page):
    """One new token each, lengths around every boundary of a page and a tile, zero and one among them."""
    rng = np.random.default_rng(D + G)
    kv = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 129, 255, 256, 257, 400]
    _run(rng, [1] * len(kv), kv, page, Nkv, G, D, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 5, 16, 100, 10000])
def test_windows(cuda, kind, window):
    rng = np.random.default_rng(window)
    _run(rng, [1, 4, 1, 40, 150], [77, 77, 300, 301, 150], 16, 2, 4, 64, kind, window=window)
    _run(rng, [1, 3, 1, 140], [77, 77, 300, 301], 32, 1, 2, 128, kind, window=window)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,Nkv,G,page", [(128, 2, 2, 64), (64, 2, 7, 16), (256, 1, 3, 32), (128, 1, 8, 16), (128, 1, 5, 256)])
def test_chunks_and_drafts(cuda, kind, D, Nkv, G, page):
    """Rows of many counts over pasts of many lengths, none and whole prompts among them."""
    rng = np.random.default_rng(D * G)
    _run(rng, [3, 1, 0, 17, 64, 130, 8], [3, 1, 50, 170, 65, 130, 333], page, Nkv, G, D, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_that_see_nothing(cuda, kind):
    """No keys, fewer keys than rows: zeros; rows outside every sequence stay as they were."""
    import torch
    rng = np.random.default_rng(2)
    for q_len, big in ((4, 4), (100, 100)):
        cache = _cache(rng, 3, 200, 16, 2, 128)
        T = 3 * q_len + 9
        q = torch.randn(T, 4, 128).to(S.torch_type(kind)).cuda()
        o = torch.full_like(q, 7.0)
        start = torch.tensor([5, 5 + q_len, 5 + 2 * q_len, 5 + 3 * q_len], dtype=torch.int32).cuda()
        kv = [0, 2, q_len + 9]
        err = torch.zeros(1, dtype=torch.int32).cuda()
        cache.attention(q, torch.tensor(kv, dtype=torch.int32).cuda(), start, big, out=o, err=err)
        assert int(err) == 0
        assert bool((o[:5] == 7).all()) and bool((o[5 + 3 * q_len:] == 7).all())
        assert bool((o[5:5 + q_len] == 0).all()) and bool((o[5 + q_len:5 + 2 * q_len - 2] == 0).all())
        _check(cache, q, o, [q_len] * 3, kv, 0, 128 ** -0.5, kind, [5, 5 + q_len, 5 + 2 * q_len])


@pytest.mark.parametrize("kind,D,G", [("f32", 128, 2), ("bf16", 128, 4), ("f16", 64, 7), ("bf16", 256, 2)])
def test_long_sequences_with_and_without_splits(cuda, kind, D, G):
    """The split over the keys gives what the unsplit pass gives; the answer is the same twice."""
    import torch
    rng = np.random.default_rng(11)
    cache, q, ln, start, o = _run(rng, [1, 1, 2], [9000, 37, 5001], 64, 1, G, D, kind)
    again = cache.attention(q, ln, start, 2)
    assert torch.equal(o, again)
    one = torch.empty(1, dtype=torch.uint8).cuda()
    plain = cache.attention(q, ln, start, 2, work=one)
    _check(cache, q, plain, [1, 1, 2], [9000, 37, 5001], 0, D ** -0.5, kind)


def test_workspace_contents_do_not_matter(cuda):
    import torch
    rng = np.random.default_rng(12)
    cache = _cache(rng, 2, 6000, 64, 2, 128)
    q = torch.randn(2, 4, 128).cuda()
    ln = torch.tensor([6000, 100], dtype=torch.int32).cuda()
    w = cache.attn_workspace(2, 4, 1, 6000)
    ref = cache.attention(q, ln)
    for fill in (0, 255):
        if w is not None:
            w.fill_(fill)
        assert torch.equal(cache.attention(q, ln, work=w, max_kv_len=6000), cache.attention(q, ln, max_kv_len=6000))
    _check(cache, q, ref, [1, 1], [6000, 100], 0, 128 ** -0.5, "f32")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 130])
def test_garbage_behind_the_keys(cuda, kind, n):
    """NaN and infinite scales behind the last key, before the window and on other pages do not show."""
    import torch
    rng = np.random.default_rng(13)
    L = 200
    cache = _cache(rng, 1, 256, 32, 1, 128)
    q = torch.randn(n, 2, 128).to(S.torch_type(kind)).cuda()
    start, ln = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([L], dtype=torch.int32).cuda()
    ref = cache.attention(q, ln, start, n, window=40)
    kc, ks, vc, vs, table = cache.tensors
    t = table.cpu().numpy()[0]
    mine = set(t[:-(-L // 32)].tolist())
    for sc in (ks, vs):
        for pg in range(sc.shape[0]):
            if pg not in mine:
                sc[pg] = float("nan")
        sc[t[L // 32], :, L % 32:] = float("inf")
        first = max(0, L - n - 40 + 1)
        for j in range(first):
            sc[t[j // 32], :, j % 32] = float("nan")
    got = cache.attention(q, ln, start, n, window=40)
    assert torch.equal(got, ref) and bool(got.isfinite().all())


@pytest.mark.parametrize("n", [1, 130])
def test_nan_of_a_seen_key_shows(cuda, n):
    import torch
    rng = np.random.default_rng(14)
    cache = _cache(rng, 1, 256, 32, 1, 128)
    cache.tensors[1][int(cache.tensors[4][0, 1]), :, 3, 0] = float("nan")
    q = torch.randn(n, 1, 128).bfloat16().cuda()
    o = cache.attention(q, torch.tensor([200], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), n)
    assert bool(o.isnan().all())


@pytest.mark.parametrize("kind,D", [("f32", 128), ("bf16", 128), ("f16", 64), ("bf16", 256)])
@pytest.mark.parametrize("n", [3, 100])
def test_nan_values_reach_only_the_rows_that_see_them(cuda, kind, D, n):
    """A value scale that is NaN: the block's dimensions of the rows that see its key, and nothing else."""
    import torch
    rng = np.random.default_rng(21)
    cache = _cache(rng, 1, 256, 16, 1, D)
    q = torch.randn(n, 2, D).to(S.torch_type(kind)).cuda()
    start, ln = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([200], dtype=torch.int32).cuda()
    ref = cache.attention(q, ln, start, n)
    j, blk = 198, 1  # the last row but one is the first to see it
    t = cache.tensors[4][0]
    cache.tensors[3][int(t[j // 16]), 0, j % 16, blk] = float("nan")
    o = cache.attention(q, ln, start, n)
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[n - 2:, :, blk * 32:blk * 32 + 32] = True
    assert bool(o[hit].isnan().all())
    assert torch.equal(o[~hit], ref[~hit])
    w = cache.attention(q, ln, start, n, window=1)  # only row n - 2 sees key 198
    hit[n - 1:] = False
    assert bool(w[hit].isnan().all()) and bool(w[~hit].isfinite().all())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 140])
def test_peaked_and_flat_scores(cuda, kind, n):
    """Scores of hundreds (one key holds nearly all), of zero, and increasing or decreasing along the keys."""
    import torch
    rng = np.random.default_rng(15)
    D = 128
    for scale in (0.0, 3.0, -2.0):
        _run(rng, [n], [300], 16, 1, 2, D, kind, scale=scale)
    for step in (1, -1):
        cache = _cache(rng, 1, 512, 16, 1, D)
        kc, ks = cache.tensors[0], cache.tensors[1]
        kc.fill_(0xFF)  # code 15: +7
        j = torch.arange(512).cuda()
        d = ((j if step > 0 else 511 - j).float() / 512).bfloat16().half()
        t = cache.tensors[4].long()[0]
        ks[t[j // 16], 0, j % 16] = d[:, None].expand(512, D // 32).contiguous()
        q = torch.full((n, 1, D), 0.5).to(S.torch_type(kind)).cuda()
        ln = torch.tensor([500], dtype=torch.int32).cuda()
        o = cache.attention(q, ln, torch.tensor([0, n], dtype=torch.int32).cuda(), n, scale=0.3)
        _check(cache, q, o, [n], [500], 0, 0.3, kind)


@pytest.mark.parametrize("kind,size", [("f16", 60000.0), ("f16", 1e-6), ("bf16", 1e30), ("bf16", 1e-30), ("f32", 1e30), ("f32", 1e-30)])
@pytest.mark.parametrize("n", [1, 130])
def test_queries_of_any_size(cuda, kind, size, n):
    """Queries near the ends of their type, the scale taking them back to scores of a few units."""
    import torch
    rng = np.random.default_rng(16)
    cache = _cache(rng, 1, 256, 16, 1, 64)
    q = torch.from_numpy((rng.uniform(-1, 1, (n, 2, 64)) * size).astype(np.float32)).to(S.torch_type(kind)).cuda()
    o = cache.attention(q, torch.tensor([250], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), n,
                        scale=0.125 / size)
    scale = float(np.float32(0.125 / size))
    if (kind, size) == ("f16", 1e-6):  # subnormal queries hold few bits: the reference uses the ones given
        assert bool((q != 0).any())
    _check(cache, q, o, [n], [250], 0, scale, kind)


def test_bounds_errors(cuda):
    import torch
    rng = np.random.default_rng(17)
    for n in (1, 130):
        cache = _cache(rng, 3, 256, 16, 1, 64)
        ref_q = torch.randn(3 * n, 2, 64).bfloat16().cuda()
        start = torch.arange(4, dtype=torch.int32).cuda() * n
        good = cache.attention(ref_q, torch.tensor([200, 201, 202], dtype=torch.int32).cuda(), start, n)
        for bad in (-1, 257, 2 ** 31 - 1):
            err = torch.zeros(1, dtype=torch.int32).cuda()
            o = cache.attention(ref_q, torch.tensor([200, bad, 202], dtype=torch.int32).cuda(), start, n, err=err)
            assert int(err) == 32 and bool((o[n:2 * n] == 0).all())
            assert torch.equal(o[:n], good[:n]) and torch.equal(o[2 * n:], good[2 * n:])
        err = torch.zeros(1, dtype=torch.int32).cuda()
        o = torch.full_like(ref_q, 7.0)
        far = torch.tensor([0, n, 2 * n, 2 * n + 5 * n], dtype=torch.int32).cuda()
        cache.attention(ref_q, torch.tensor([200, 201, 202], dtype=torch.int32).cuda(), far, n, out=o, err=err)
        assert int(err) == 32 and torch.equal(o[:2 * n], good[:2 * n]) and bool((o[2 * n:] == 0).all())
        back = torch.tensor([0, n, n - 1, 2 * n - 1], dtype=torch.int32).cuda()
        o = torch.full_like(ref_q, 7.0)
        err.zero_()
        cache.attention(ref_q, torch.tensor([200, 201, 202], dtype=torch.int32).cuda(), back, n, out=o, err=err)
        assert int(err) == 32 and torch.equal(o[:n - 1], good[:n - 1]) and bool((o[2 * n:] == 7).all())
        # a page outside the pool: its keys take no part
        cache.tensors[4][1, 2] = 10 ** 6
        cache.tensors[4][2, 0] = -1
        err.zero_()
        o = cache.attention(ref_q, torch.tensor([200, 201, 202], dtype=torch.int32).cuda(), start, n, err=err)
        assert int(err) == 16 and torch.equal(o[:n], good[:n]) and bool(o.isfinite().all())
        assert not torch.equal(o[n:2 * n], good[n:2 * n])


def test_strided_rows(cuda):
    import torch
    rng = np.random.default_rng(18)
    for n in (1, 130):
        cache = _cache(rng, 2, 256, 16, 2, 64)
        wide = torch.randn(2 * n, 700).half().cuda()
        out = torch.full((2 * n, 300), 7.0).half().cuda()
        start, ln = torch.arange(3, dtype=torch.int32).cuda() * n, torch.tensor([150, 256], dtype=torch.int32).cuda()
        for off in (0, 1, 4, 9):
            q = wide[:, off:off + 256].unflatten(1, (4, 64))
            ref = cache.attention(q.contiguous(), ln, start, n)
            cache.attention(q, ln, start, n, out=out[:, off:off + 256].unflatten(1, (4, 64)))
            assert torch.equal(out[:, off:off + 256].unflatten(1, (4, 64)), ref)
            assert bool((out[:, :off] == 7).all()) and bool((out[:, off + 256:] == 7).all())
            out.fill_(7.0)


def test_captured_graph_follows_the_lengths(cuda):
    """Two graphs that share a workspace, replayed in turn while lengths and queries change."""
    import torch
    rng = np.random.default_rng(19)
    cache = _cache(rng, 4, 4000, 64, 2, 128)
    ln = torch.tensor([4000, 3, 700, 0], dtype=torch.int32).cuda()
    work = cache.attn_workspace(4, 4, 1, 4000)
    qs = [torch.randn(4, 4, 128).cuda() for _ in range(2)]
    outs, graphs = [torch.zeros_like(qs[0]) for _ in qs], []
    cache.attention(qs[0], ln, max_kv_len=4000, work=work)
    for q, o in zip(qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.attention(q, ln, max_kv_len=4000, out=o, work=work)
        graphs.append(g)
    for lens in ([4000, 3, 700, 0], [1, 2000, 64, 65], [0, 0, 0, 4000]):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        for q in qs:
            q.normal_()
        for g in graphs + graphs[::-1]:
            g.replay()
        for q, o in zip(qs, outs):
            assert torch.equal(o, cache.attention(q, ln, max_kv_len=4000))
            _check(cache, q, o, [1] * 4, lens, 0, 128 ** -0.5, "f32")


def test_two_streams_at_once(cuda):
    import torch
    rng = np.random.default_rng(20)
    cache = _cache(rng, 2, 5000, 64, 2, 128)
    q = [torch.randn(2, 8, 128).bfloat16().cuda() for _ in range(4)]
    ln = torch.tensor([5000, 4999], dtype=torch.int32).cuda()
    ref = [cache.attention(x, ln) for x in q]
    work = [cache.attn_workspace(2, 8, 1, 5120) for _ in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in q], [None] * 4
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = cache.attention(q[i], ln, work=work[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("n", [1, 5, 130])
def test_pages_behind_4_gb(cuda, n):
    """The same keys on the first pages of a pool and on its last, codes past 32-bit offsets: the same output."""
    import torch
    n_pages, page, Nkv, D = 8300, 4096, 2, 128
    table = torch.tensor([[0, 1], [n_pages - 1, n_pages - 2]], dtype=torch.int32).cuda()
    cache = acb.KVCacheQ4.empty(n_pages, page, Nkv, D, table)
    kc, ks, vc, vs, _ = cache.tensors
    for t in (kc, vc):
        t[:2] = torch.randint(0, 256, (2, Nkv, page, D // 2), dtype=torch.uint8).cuda()
        t[[n_pages - 1, n_pages - 2]] = t[:2].clone()
    for t in (ks, vs):
        t[:2] = (0.02 + 0.1 * torch.rand(2, Nkv, page, D // 32)).bfloat16().half().cuda()
        t[[n_pages - 1, n_pages - 2]] = t[:2].clone()
    q = torch.randn(n, 4, D).bfloat16().cuda()
    o = cache.attention(torch.cat([q, q]), torch.tensor([5000, 5000], dtype=torch.int32).cuda(),
                        torch.tensor([0, n, 2 * n], dtype=torch.int32).cuda(), n)
    assert torch.equal(o[:n], o[n:]) and bool((o != 0).any())


def test_wrappers_refuse_what_would_be_misread(cuda):
    import torch
    rng = np.random.default_rng(22)
    cache = _cache(rng, 2, 64, 16, 1, 64)
    q = torch.randn(2, 2, 64).cuda()
    ln = torch.tensor([10, 20], dtype=torch.int32).cuda()
    cache.attention(q, ln)
    for bad in (lambda: cache.attention(q[:1].expand(2, 2, 64), ln), lambda: cache.attention(q, ln.long()),
                lambda: cache.attention(q, ln.cpu()), lambda: cache.attention(q, ln[:1]), lambda: cache.attention(q[..., ::2], ln),
                lambda: cache.attention(q, ln, out=q.half()), lambda: cache.attention(q.cpu(), ln),
                lambda: acb.KVCacheQ4(*cache.tensors[:4], cache.tensors[4][:1].expand(2, 4)),
                lambda: acb.KVCacheQ4(*cache.tensors[:4], cache.tensors[4].long()),
                lambda: acb.KVCacheQ4(cache.tensors[0], cache.tensors[1][:, :, :, :1].contiguous(), *cache.tensors[2:]),
                lambda: cache.append(torch.randn(1, 256).cuda().expand(2, 256), 2, ln, ln),
                lambda: cache.append(torch.randn(2, 255).cuda(), 2, ln, ln),
                lambda: cache.read(ln, ln, k_out=torch.zeros(2, 1, 64).cuda(), v_out=torch.zeros(2, 1, 64).half().cuda())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(acb.AcbError):
        cache.attention(torch.randn(2, 2, 64).cuda(), ln, max_kv_len=65)
    with pytest.raises(acb.AcbError):
        cache.attention(torch.randn(3, 2, 64).cuda(), ln)  # three rows, two sequences and no q_start


@pytest.mark.parametrize("kind,D,G", [("bf16", 128, 1), ("f16", 128, 2), ("bf16", 64, 1), ("f32", 128, 1)])
@pytest.mark.parametrize("n", [70, 300])
def test_references_that_keep_moving(cuda, kind, D, G, n):
    """Scores that rise by 60 along 2400 keys, in steps of one page: the reference moves in nearly every block, while products of
    the blocks before are under way."""
    import torch
    rng = np.random.default_rng(D + n)
    L = 2400
    cache = _cache(rng, 1, L, 16, 1, D)
    kc, ks = cache.tensors[0], cache.tensors[1]
    kc.fill_(0xFF)  # code 15: +7
    j = torch.arange(L).cuda()
    d = ((j // 16 + 1).float() * 16 / L).bfloat16().half()
    t = cache.tensors[4].long()[0]
    ks[t[j // 16], 0, j % 16] = d[:, None].expand(L, D // 32).contiguous()
    q = torch.full((n, G, D), 0.5).to(S.torch_type(kind)).cuda()
    scale = 60 / (3.5 * D)
    for work in (None, torch.empty(1, dtype=torch.uint8).cuda()):  # the keys cut into chunks, and not
        o = cache.attention(q, torch.tensor([L], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), n, scale=scale,
                            work=work)
        _check(cache, q, o, [n], [L], 0, scale, kind)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64), ("f32", 128)])
@pytest.mark.parametrize("window", [0, 900])
def test_holes_and_nan_values_along_many_blocks(cuda, kind, D, window):
    """Pages outside the pool and value scales that are NaN, in blocks far apart and next to each other, for 300 rows of two heads
    over 2400 keys: the holes take no part, a NaN reaches the rows that see its key in its dimensions."""
    import torch
    rng = np.random.default_rng(D + window)
    n, L, P, scale = 300, 2400, 16, 0.1
    cache = _cache(rng, 1, L, P, 1, D)
    k, v = _held(cache, 0, L)
    k, v = k[:, 0], v[:, 0].copy()
    holes = [1, 9, 76, 77, 90, 141, 149]  # pages
    nans = [(1160, 0), (1250, 1), (1300, 0), (2200, 1), (2201, 0), (2350, 1)] if window else [(2150, 0), (2200, 1), (2201, 0), (2350, 1)]
    t = cache.tensors[4][0]
    for j, b in nans:
        cache.tensors[3][int(t[j // P]), 0, j % P, b] = float("nan")
        v[j, 32 * b:32 * b + 32] = 0
    for i, pg in enumerate(holes):
        t[pg] = 10 ** 6 if i % 2 else -1
    q = torch.from_numpy(rng.standard_normal((n, 2, D)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    for work in (None, torch.empty(1, dtype=torch.uint8).cuda()):  # the keys cut into chunks, and not
        err = torch.zeros(1, dtype=torch.int32).cuda()
        o = cache.attention(q, torch.tensor([L], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), n, window=window,
                            scale=scale, err=err, work=work).float().cpu().numpy().astype(np.float64)
        assert int(err) == 16
        key, pos = np.arange(L), L - n + np.arange(n)
        seen = (key[None] <= pos[:, None]) & ~np.isin(key // P, holes)[None]
        if window:
            seen &= key[None] > pos[:, None] - window
        nan = np.zeros((n, D), bool)
        for j, b in nans:
            nan[seen[:, j], 32 * b:32 * b + 32] = True
        for h in range(2):
            x = q[:, h].float().cpu().numpy().astype(np.float64)
            s = np.where(seen, scale * (x @ k.T), -np.inf)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            ref, A = w @ v, w @ np.abs(v)
            s1 = (scale * (np.abs(x) @ np.abs(k).T)).max(1)[:, None]
            ds = (D + 4) * 2.0 ** -24 * s1 + (2.0 ** -21 * s1 if kind != "f32" else 0)
            tol = A * (2 * ds + 2.0 ** -15 + (2.0 ** -11 if kind != "f32" else 0)) + 2.0 ** -31 * np.abs(v).sum(0)
            tol = tol + S.HALF_STEP[kind] * (np.abs(ref) + tol) + (2.0 ** -25 if kind == "f16" else 0)
            assert np.isnan(o[:, h][nan]).all() and (np.abs(o[:, h] - ref) <= tol)[~nan].all()


@pytest.mark.parametrize("n_seq,Nkv,G,n,L", [(24, 8, 4, 4, 700), (24, 8, 4, 8, 700), (24, 8, 4, 12, 700), (2, 2, 2, 64, 900),
                                             (12, 16, 2, 40, 600), (3, 1, 7, 100, 1500)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_sizes_around_the_forms_borders(cuda, kind, n_seq, Nkv, G, n, L):
    """Mean rows and sequences on both sides of where the form for chunks of prompts takes over, lengths and rows ragged."""
    rng = np.random.default_rng(n_seq * n)
    q_lens = [max(0, n - int(x)) for x in rng.integers(0, 3, n_seq)]
    q_lens[0] = n
    _run(rng, q_lens, [L - int(x) for x in rng.integers(0, L // 3, n_seq)], 64, Nkv, G, 64, kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,kv_lens,Nkv,G,D,window", [
    ([1], [300], 1, 7, 128, 0), ([1], [2100], 1, 71, 64, 0), ([1], [1300], 3, 3, 128, 0), ([3, 1, 1], [279, 50, 200], 1, 9, 64, 0),
    ([1, 1, 1], [300, 200, 1], 1, 7, 128, 0), ([1] * 19, [2352] + [100] * 18, 1, 5, 128, 0), ([1] * 3, [700, 699, 3], 1, 5, 256, 200),
    ([1] * 3, [2000, 1999, 3], 1, 11, 64, 200)])
def test_odd_counts_of_parts(cuda, kind, q_lens, kv_lens, Nkv, G, D, window):
    """Tokens, heads and chunks of keys that are all odd: the parts' rows stay on 16 bytes."""
    _run(np.random.default_rng(G * D), q_lens, kv_lens, 16, Nkv, G, D, kind, window=window)


@pytest.mark.parametrize("kind,n_seq,Nkv,G,D,n,L,whole", [("f32", 16, 8, 2, 128, 9, 8192, False), ("f32", 16, 8, 2, 128, 15, 8192, False),
                                                          ("f16", 24, 2, 7, 64, 7, 4000, True), ("bf16", 1, 1, 4, 256, 200, 3000, False),
                                                          ("f32", 24, 2, 7, 64, 7, 4000, False)])
def test_the_workspace_is_enough_to_split(cuda, kind, n_seq, Nkv, G, D, n, L, whole):
    """The workspace of these sizes, one made within and one with room for anything: the same chunks of keys, so the same bits.
    whole: 24 sequences of 2 kv heads and 4 tiles of 16 rows go to the form that does not cut the keys."""
    import torch
    rng = np.random.default_rng(n)
    cache = _cache(rng, n_seq, L, 64, Nkv, D)
    q = torch.from_numpy(rng.standard_normal((n_seq * n, Nkv * G, D)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    start = torch.arange(n_seq + 1, dtype=torch.int32).cuda() * n
    ln = torch.from_numpy(rng.integers(L // 2, L + 1, n_seq).astype(np.int32)).cuda()
    kw = dict(q_start=start, max_q_len=n, max_kv_len=L)
    ample = cache.attention(q, ln, work=torch.empty(1 << 30, dtype=torch.uint8).cuda(), **kw)
    plain = cache.attention(q, ln, work=torch.empty(1, dtype=torch.uint8).cuda(), **kw)
    assert torch.equal(ample, plain) == whole
    assert torch.equal(cache.attention(q, ln, work=cache.attn_workspace(n_seq * n, Nkv * G, n, L), **kw), ample)
    assert torch.equal(cache.attention(q, ln, **kw), ample)


@pytest.mark.parametrize("kind,n_seq,Nkv,G,D,n,pad,window", [
    ("f32", 8, 8, 2, 128, 1, 56, 0), ("bf16", 8, 8, 2, 128, 1, 2040, 0), ("f16", 3, 1, 7, 64, 5, 6, 0), ("f32", 5, 2, 3, 256, 3, 1, 0),
    ("f32", 3, 1, 5, 64, 2, 100, 700), ("bf16", 2, 2, 2, 64, 100, 1848, 0)])
def test_padded_batches_are_as_the_batch_alone(cuda, kind, n_seq, Nkv, G, D, n, pad, window):
    """Rows in front of, and behind, all sequences change neither the chunks nor the bits, and stay as they were."""
    import torch
    rng = np.random.default_rng(pad)
    L, H = 5000, Nkv * G
    cache = _cache(rng, n_seq, L, 64, Nkv, D)
    lens = [n - i % 2 * (n > 1) for i in range(n_seq)]
    lens[0] = n
    T = sum(lens)
    q = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    start = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32).cuda()
    kv = [L - int(x) for x in rng.integers(0, L // 2, n_seq)]
    kw = dict(kv_len=torch.tensor(kv, dtype=torch.int32).cuda(), max_q_len=n, max_kv_len=L, window=window)
    ref = cache.attention(q, q_start=start, **kw)
    ample = cache.attention(q, q_start=start, work=torch.empty(1 << 28, dtype=torch.uint8).cuda(), **kw)
    assert torch.equal(ref, ample)
    front = pad // 3
    wide = torch.full((T + pad, H, D), float("nan"), dtype=q.dtype).cuda()
    wide[front:front + T] = q
    for work in (None, cache.attn_workspace(T + pad, H, n, L)):
        o = torch.full_like(wide, 7.0)
        cache.attention(wide, q_start=start + front, out=o, work=work, **kw)
        assert torch.equal(o[front:front + T], ref)
        assert bool((o[:front] == 7).all()) and bool((o[front + T:] == 7).all())
    _check(cache, q, ref, lens, kv, window, D ** -0.5, kind)


@pytest.mark.parametrize("kind,D", [("f32", 128), ("bf16", 128), ("f16", 64), ("bf16", 256)])
@pytest.mark.parametrize("n,window", [(1, 100), (5, 1), (130, 100), (300, 17), (300, 333), (700, 40)])
def test_pages_behind_the_window_may_be_gone(cuda, kind, D, n, window):
    """A server frees the pages that lie wholly before the first row's window: no error, and the same answer."""
    import torch
    rng = np.random.default_rng(n + window)
    P = 16
    cache = _cache(rng, 2, 1000, P, 1, D)
    q = torch.from_numpy(rng.standard_normal((2 * n, 2, D)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    start, lens = torch.tensor([0, n, 2 * n], dtype=torch.int32).cuda(), [1000, 901]
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    ref = cache.attention(q, ln, start, n, window=window)
    freed = 0
    for s, m in enumerate(lens):
        first = max(0, m - n - window + 1)
        cache.tensors[4][s, :first // P] = torch.tensor([-1, 10 ** 6], dtype=torch.int32).cuda().repeat(100)[:first // P]
        freed += first // P
    assert freed > 0
    err = torch.zeros(1, dtype=torch.int32).cuda()
    o = cache.attention(q, ln, start, n, window=window, err=err)
    assert int(err) == 0 and torch.equal(o, ref)
    cache.tensors[4][0, (1000 - n - window + 1) // P] = -1  # the first page that the first row sees
    cache.attention(q, ln, start, n, window=window, err=err)
    assert int(err) == 16


@pytest.mark.parametrize("kind,n,L", [("f32", 8, 3), ("bf16", 8, 3), ("bf16", 130, 100), ("f16", 300, 290), ("f32", 130, 100)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, 1000])
def test_windows_of_more_than_all_keys(cuda, kind, n, L, window):
    """The largest windows, over fewer keys than rows: the bits of no window."""
    import torch
    rng = np.random.default_rng(n)
    cache = _cache(rng, 2, 400, 16, 1, 128)
    q = torch.from_numpy(rng.standard_normal((2 * n, 2, 128)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    start, ln = torch.tensor([0, n, 2 * n], dtype=torch.int32).cuda(), torch.tensor([L, L // 2], dtype=torch.int32).cuda()
    ref = cache.attention(q, ln, start, n)
    assert torch.equal(cache.attention(q, ln, start, n, window=window), ref)
    _check(cache, q, ref, [n, n], [L, L // 2], 0, 128 ** -0.5, kind)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64), ("f32", 128), ("bf16", 256)])
def test_repeated_calls_give_the_same_bits(cuda, kind, D):
    """Prompts and single tokens, in either form, cut and not."""
    import torch
    rng = np.random.default_rng(D)
    for q_lens, kv_lens in (([300, 200, 259], [2000, 300, 1111]), ([1, 1, 1], [4000, 3, 700])):
        cache, q, ln, start, o = _run(rng, q_lens, kv_lens, 16, 4, 2, D, kind)
        for _ in range(10):
            assert torch.equal(cache.attention(q, ln, start, max(q_lens)), o)
