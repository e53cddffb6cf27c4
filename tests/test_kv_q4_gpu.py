"""GPU: the paged 4-bit KV cache: append (norm, rotation, quantisation, scatter), rows read back.

Bars: the codes and scales are equal, bit for bit, to the definition in single precision applied to the f32 values that
are quantised (for keys these are seen through q_out, whose heads then hold the same numbers); q is within 2^-24 times 8 of the
products' magnitudes of the 64-bit norm and rotation (scale, two products of the norm, two of the rotation, a sum: under 8 half
steps) plus half a step of its type."""
import numpy as np
import pytest

import acb
import serving_ref as S

pytestmark = pytest.mark.gpu


def _table(rng, n_seq, max_pages, n_pages):
    import torch
    return torch.from_numpy(rng.permutation(n_pages)[:n_seq * max_pages].reshape(n_seq, max_pages).astype(np.int32)).cuda()


def _rows(cache, seq, pos):
    kc, ks, vc, vs, table = (t.cpu().numpy() for t in cache.tensors)
    P = kc.shape[2]
    pg = table[seq, pos // P]
    return [a[pg, :, pos % P] for a in (kc, ks, vc, vs)]


@pytest.mark.parametrize("kind,qkind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("D,Nh,Nkv,page,layout,R,norm", [
    (128, 16, 8, 64, "half", 128, True), (64, 3, 1, 16, "interleaved", 32, True), (256, 2, 2, 32, "half", 256, False),
    (128, 8, 8, 16, "half", 50, True), (64, 2, 2, 128, "half", 64, False), (256, 4, 1, 16, "interleaved", 256, True),
    (128, 5, 1, 16, "interleaved", 2, True), (64, 7, 1, 64, "half", 10, True), (128, 2, 1, 32, None, 0, True)])
def test_append_matches_the_definition(cuda, kind, qkind, D, Nh, Nkv, page, layout, R, norm):
    import torch
    rng = np.random.default_rng(D + Nh + R)
    T, n_seq, max_pages = 41, 3, 5
    table = _table(rng, n_seq, max_pages, 17)
    cache = acb.KVCacheQ4.empty(17, page, Nkv, D, table)
    x = torch.from_numpy(rng.standard_normal((T, (Nh + 2 * Nkv) * D)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    at = rng.permutation(n_seq * max_pages * page)[:T]  # distinct places in any order
    seq, pos = at // (max_pages * page), at % (max_pages * page)
    d_seq, d_pos = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (seq, pos))
    rope = acb.rope_table_scaled(max_pages * page, R, 1e4).cuda() if layout else None
    w = [torch.from_numpy((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)).cuda() if norm else None for _ in "qk"]
    kw = dict(layout=layout or "half", eps=1e-5)
    q = cache.append(x, Nh, d_seq, d_pos, rope, q_norm=w[0], k_norm=w[1], q_dtype=S.torch_type(qkind), **kw)
    xs = x.float().cpu().numpy().reshape(T, Nh + 2 * Nkv, D)
    # q
    ref = S.rms(xs[:, :Nh], w[0].cpu().numpy(), 1e-5) if norm else xs[:, :Nh].astype(np.float64)
    mag = np.abs(ref)
    if layout:
        ref, m2 = S.rotate(ref, pos, rope.cpu().numpy(), layout)
        mag = np.maximum(mag, m2)
    tol = 8 * 2.0 ** -24 * mag + S.HALF_STEP[qkind] * (np.abs(ref) + 8 * 2.0 ** -24 * mag) + (2.0 ** -25 if qkind == "f16" else 0)
    assert (np.abs(q.float().cpu().numpy() - ref) <= tol).all()
    # the f32 keys that are quantised, as q heads of a second call without a cache of its own rows
    xk = torch.cat([x[:, Nh * D:(Nh + Nkv) * D], x[:, Nh * D:]], 1).contiguous()
    k32 = cache.append(xk, Nkv, d_seq, d_pos, rope, q_norm=w[1], k_norm=w[1], q_dtype=torch.float32, **kw).cpu().numpy()
    kc, ks, vc, vs = _rows(cache, seq, pos)
    rk, rv = S.quantise(k32), S.quantise(xs[:, Nh + Nkv:])
    for got, want in ((kc, rk[0]), (ks.view(np.uint16), rk[1].view(np.uint16)), (vc, rv[0]), (vs.view(np.uint16), rv[1].view(np.uint16))):
        assert np.array_equal(got, want)
    # nothing else was written
    used = np.zeros((17, page), bool)
    used[table.cpu().numpy()[seq, pos // page], pos % page] = True
    assert not cache.tensors[0].cpu().numpy().transpose(0, 2, 1, 3)[~used].any()
    assert not cache.tensors[3].cpu().numpy().transpose(0, 2, 1, 3)[~used].any()
    # read back: f32 and f16 exact, bf16 rounded once
    val = [S.values(*rk), S.values(*rv)]
    for t in ("f32", "f16", "bf16"):
        got = [o.float().cpu().numpy() for o in cache.read(d_seq, d_pos, dtype=S.torch_type(t))]
        for g, v in zip(got, val):
            assert np.array_equal(g, S.bf16(v.astype(np.float32)) if t == "bf16" else v.astype(np.float32))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_extreme_blocks(cuda, kind):
    """Zeros, one value, values past the scale's range, the smallest numbers, infinities, ties of both signs; NaN."""
    import torch
    rng = np.random.default_rng(1)
    b = np.zeros((12, 64), np.float32)
    b[1, 5] = 3.0
    b[2, :32], b[2, 32:] = -1.0, 60000.0
    b[3] = rng.standard_normal(64) * 1e-7
    b[4] = rng.standard_normal(64) * 1e-4
    b[5, 3], b[5, 9] = 2.5, -2.5
    b[6, 3], b[6, 9] = -2.5, 2.5
    b[7] = rng.standard_normal(64)
    b[7, 11], b[7, 40] = np.inf, -np.inf
    b[8] = np.linspace(-8, 7.75, 64)
    b[9] = rng.standard_normal(64) * 21760
    b[10] = -np.abs(rng.standard_normal(64))
    b[11] = 1e-30
    x = torch.from_numpy(b).to(S.torch_type(kind))
    qkv = torch.cat([x, x], 1).cuda()  # no q, one kv head
    table = torch.zeros((1, 1), dtype=torch.int32).cuda()
    cache = acb.KVCacheQ4.empty(1, 16, 1, 64, table)
    pos = torch.arange(12, dtype=torch.int32).cuda()
    assert cache.append(qkv, 0, torch.zeros_like(pos), pos) is None
    codes, d = S.quantise(x.float().numpy())
    assert np.array_equal(cache.tensors[0].cpu().numpy()[0, 0, :12], codes)
    assert np.array_equal(cache.tensors[2].cpu().numpy()[0, 0, :12], codes)
    assert np.array_equal(cache.tensors[1].cpu().numpy()[0, 0, :12].view(np.uint16), d.view(np.uint16))
    val = S.values(codes, d)
    assert np.abs(val[8] - b[8]).max() <= 0.5 + 2.0 ** -8 * 8
    k, _ = cache.read(torch.zeros_like(pos), pos)
    assert np.array_equal(k.cpu().numpy()[:, 0].astype(np.float64), val) and np.isfinite(val).all()
    bad = torch.ones(1, 128).to(S.torch_type(kind))
    bad[0, 3] = float("nan")
    cache.append(bad.cuda(), 0, torch.zeros(1, dtype=torch.int32).cuda(), torch.full((1,), 15, dtype=torch.int32).cuda())
    k, v = cache.read(torch.zeros(1, dtype=torch.int32).cuda(), torch.full((1,), 15, dtype=torch.int32).cuda())
    assert bool(k[0, 0, :32].isnan().all()) and bool(k[0, 0, 32:].isfinite().all()) and bool(v.isfinite().all())


def test_padding_and_range_errors(cuda):
    import torch
    table = torch.tensor([[0, 1], [2, 99], [-5, 3]], dtype=torch.int32).cuda()
    cases = [((-1, 0), 0, "pad"), ((-7, 10 ** 6), 0, "pad"), ((0, 31), 0, "ok"), ((0, 32), 2, "bad"), ((0, -1), 2, "bad"),
             ((3, 0), 1, "bad"), ((1, 16), 16, "bad"), ((1, 15), 0, "ok"), ((2, 0), 16, "bad"), ((2, 31), 0, "ok"),
             ((2 ** 31 - 1, 2 ** 31 - 1), 3, "bad")]
    rope = acb.rope_table_scaled(64, 64, 1e4).cuda()
    for (s, p), flag, what in cases:
        cache = acb.KVCacheQ4.empty(4, 16, 1, 64, table)
        x = torch.randn(1, 4 * 64).cuda()
        seq, pos = (torch.tensor([v], dtype=torch.int32).cuda() for v in (s, p))
        err = torch.zeros(1, dtype=torch.int32).cuda()
        q = torch.full((1, 2, 64), 5.0).cuda()
        cache.append(x, 2, seq, pos, rope, q_out=q, err=err)
        assert int(err) == flag, (s, p)
        wrote = bool((cache.tensors[0] != 0).any())
        assert wrote == (what == "ok")
        assert bool((q == 5).all()) if what == "pad" else bool((q == 0).all()) == (what == "bad")
        err.zero_()
        k = torch.full((1, 1, 64), 5.0).cuda()
        v = k.clone()
        cache.read(seq, pos, k_out=k, v_out=v, err=err)
        assert int(err) == flag and bool((k == 5).all()) == (what == "pad") and bool((v == 0).all()) == (what == "bad")
    # positions past the rope table
    cache = acb.KVCacheQ4.empty(4, 16, 1, 64, table)
    err = torch.zeros(1, dtype=torch.int32).cuda()
    cache.append(torch.randn(1, 256).cuda(), 2, torch.zeros(1, dtype=torch.int32).cuda(),
                 torch.full((1,), 20, dtype=torch.int32).cuda(), rope[:20].contiguous(), err=err)
    assert int(err) == 2 and not bool((cache.tensors[0] != 0).any())


def test_strided_rows_and_one_output(cuda):
    import torch
    rng = np.random.default_rng(5)
    table = torch.arange(4, dtype=torch.int32).view(2, 2).cuda()
    wide = torch.from_numpy(rng.standard_normal((9, 700)).astype(np.float32)).cuda()
    seq, pos = torch.tensor([0, 1] * 4 + [0], dtype=torch.int32).cuda(), torch.arange(9, dtype=torch.int32).cuda()
    a = acb.KVCacheQ4.empty(4, 16, 2, 64, table)
    b = acb.KVCacheQ4.empty(4, 16, 2, 64, table)
    rope = acb.rope_table_scaled(32, 64, 1e4).cuda()
    for off in (0, 3):
        x = wide[:, off:off + 6 * 64]
        out = torch.full((9, 200), 9.0).cuda()
        qa = a.append(x, 2, seq, pos, rope, q_out=out[:, 1:129].unflatten(1, (2, 64)))
        qb = b.append(x.contiguous(), 2, seq, pos, rope)
        assert torch.equal(qa, qb) and bool((out[:, 0] == 9).all()) and bool((out[:, 129:] == 9).all())
        for s, t in zip(a.tensors, b.tensors):
            assert torch.equal(s, t)
        ko = torch.full((9, 150), 9.0).cuda()
        a.read(seq, pos, k_out=ko[:, 1:129].unflatten(1, (2, 64)))
        k, v = b.read(seq, pos, dtype=torch.float32)
        assert torch.equal(ko[:, 1:129].unflatten(1, (2, 64)), k) and bool((ko[:, 129:] == 9).all())
        vo = torch.empty(9, 2, 64).cuda()
        a.read(seq, pos, v_out=vo)
        assert torch.equal(vo, v)


def test_offsets_past_32_bits(cuda):
    """A pool whose codes are over 4 GB: the first and the last page, written and read."""
    import torch
    n_pages, page, Nkv, D = 8300, 4096, 2, 128
    assert n_pages * page * Nkv * D // 2 > 2 ** 32
    table = torch.tensor([[n_pages - 1, 0]], dtype=torch.int32).cuda()
    cache = acb.KVCacheQ4.empty(n_pages, page, Nkv, D, table)
    x = torch.randn(3, 6 * D, generator=torch.Generator().manual_seed(1))
    pos = torch.tensor([4095, 4096, 17], dtype=torch.int32).cuda()
    cache.append(x.cuda(), 2, torch.zeros_like(pos), pos)
    k, v = cache.read(torch.zeros_like(pos), pos, dtype=torch.float32)
    xs = x.numpy().reshape(3, 6, D)
    assert np.array_equal(k.cpu().numpy(), S.values(*S.quantise(xs[:, 2:4])).astype(np.float32))
    assert np.array_equal(v.cpu().numpy(), S.values(*S.quantise(xs[:, 4:])).astype(np.float32))
    assert bool((cache.tensors[0][n_pages - 1, :, 4095] != 0).any()) and bool((cache.tensors[0][n_pages - 1, :, 17] != 0).any())
    o = cache.attention(x[:1, :2 * D].reshape(1, 2, D).cuda(), torch.tensor([18], dtype=torch.int32).cuda(), window=1)
    assert float((o[0].float() - v[2]).abs().max()) <= 2.0 ** -22 * float(v[2].abs().max())  # one key: its value


@pytest.mark.parametrize("T", [700, 1500, 4000])
@pytest.mark.parametrize("kind,D,layout,R", [("bf16", 128, "half", 128), ("f16", 64, "interleaved", 32), ("f32", 256, "half", 64)])
def test_many_tokens(cuda, kind, D, layout, R, T):
    """More tokens than the GPU holds with all their warps at once, with padding among them, next to the same tokens few at a time."""
    import torch
    rng = np.random.default_rng(T + D)
    Nh, Nkv, page = 3, 2, 64
    n_pages = -(-T // page)
    table = torch.from_numpy(rng.permutation(n_pages).reshape(1, -1).astype(np.int32)).cuda()
    x = torch.from_numpy(rng.standard_normal((T, (Nh + 2 * Nkv) * D)).astype(np.float32)).to(S.torch_type(kind)).cuda()
    pos = torch.from_numpy(rng.permutation(T).astype(np.int32)).cuda()
    seq = torch.from_numpy(np.where(rng.random(T) < 0.05, -1, 0).astype(np.int32)).cuda()
    rope = acb.rope_table_scaled(T, R, 1e4).cuda()
    w = torch.from_numpy((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)).cuda()
    all_at_once, few = (acb.KVCacheQ4.empty(n_pages, page, Nkv, D, table) for _ in range(2))
    q = torch.zeros((T, Nh, D), dtype=x.dtype).cuda()
    q2 = torch.zeros_like(q)
    all_at_once.append(x, Nh, seq, pos, rope, layout, w, w, q_out=q)
    for a in range(0, T, 100):
        b = min(T, a + 100)
        few.append(x[a:b], Nh, seq[a:b], pos[a:b], rope, layout, w, w, q_out=q2[a:b])
    assert torch.equal(q, q2)
    for s, t in zip(all_at_once.tensors[:4], few.tensors[:4]):
        assert torch.equal(s, t)
