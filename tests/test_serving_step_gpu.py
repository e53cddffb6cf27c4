"""GPU: the serving operators together, as a decode loop uses them: prompts of several sequences appended and attended in one
ragged batch, then single tokens, each step's logits through the rules and the greedy sampler, against a 64-bit loop that holds
the same 4-bit values."""
import numpy as np
import pytest

import acb
import serving_ref as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_prompt_then_tokens(cuda, graph):
    import torch
    rng = np.random.default_rng(7)
    Nh, Nkv, D, page, V, n_seq, R = 4, 2, 128, 16, 500, 3, 64
    H = Nh * D
    emb = (rng.standard_normal((V, H)) * 0.5).astype(np.float32)
    wqkv = (rng.standard_normal((H, (Nh + 2 * Nkv) * D)) / np.sqrt(H)).astype(np.float32)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, D))).astype(np.float32)
    prompts = [rng.integers(0, V, n).tolist() for n in (5, 40, 17)]
    n_new, mp = 12, 6
    table = torch.from_numpy(rng.permutation(n_seq * mp + 2)[:n_seq * mp].reshape(n_seq, mp).astype(np.int32)).cuda()
    cache = acb.KVCacheQ4.empty(n_seq * mp + 2, page, Nkv, D, table)
    rope = acb.rope_table_scaled(mp * page, R, 1e4, acb.ROPE_SCALE_YARN, 4.0, orig_max_pos=32).cuda()
    g_emb, g_w, g_qn, g_kn = (torch.from_numpy(a).cuda() for a in (emb, wqkv, qn, kn))
    allowed = rng.random((1, V)) < 0.6
    pad = np.zeros((1, 512), bool)
    pad[:, :V] = allowed
    mask = torch.from_numpy(np.packbits(pad, axis=1, bitorder="little").view(np.int32)).cuda()
    mask_row = torch.zeros(n_seq, dtype=torch.int32).cuda()
    hist = torch.full((n_seq, 64), -1, dtype=torch.int32).cuda()
    for s, p in enumerate(prompts):
        hist[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    plen = torch.tensor([len(p) for p in prompts], dtype=torch.int32).cuda()
    hlen, kv_len = plen.clone(), plen.clone()
    rep, pres = torch.full((n_seq,), 1.2).cuda(), torch.full((n_seq,), 0.3).cuda()

    def layer(ids, seq, pos, start, max_q):
        qkv = g_emb[ids] @ g_w
        q = cache.append(qkv, Nh, seq, pos, rope, q_norm=g_qn, k_norm=g_kn)
        return cache.attention(q, kv_len, start, max_q, max_kv_len=mp * page)

    def pick(o):
        lg = (o.reshape(n_seq, H) @ g_emb.T).contiguous()
        lg = acb.logits_rules(lg, hist, hlen, plen, rep=rep, pres=pres, mask=mask, mask_row=mask_row)
        ids = torch.empty(n_seq, dtype=torch.int32, device="cuda")
        acb.argmax(lg, ids, scratch=scratch)
        return lg, ids

    scratch = torch.zeros(acb.lib().acb_argmax_scratch_bytes(n_seq, V), dtype=torch.uint8, device="cuda")
    start = torch.tensor(np.concatenate([[0], np.cumsum([len(p) for p in prompts])]), dtype=torch.int32).cuda()
    seq = torch.cat([torch.full((len(p),), s) for s, p in enumerate(prompts)]).int().cuda()
    pos = torch.cat([torch.arange(len(p)) for p in prompts]).int().cuda()
    o = layer(torch.tensor(sum(prompts, [])).cuda(), seq, pos, start, 40)
    lg, ids = pick(o[(start[1:] - 1).long()])
    logits, picked = [lg.clone()], [ids.clone()]
    seq1, rows = torch.arange(n_seq, dtype=torch.int32).cuda(), torch.arange(n_seq).cuda()
    cur = ids.long()
    one_out, one_lg, one_ids = None, None, None

    def step():
        hist[rows, hlen.long()] = cur.int()
        hlen.add_(1)
        kv_len.add_(1)
        return pick(layer(cur, seq1, kv_len - 1, None, 1))

    if graph:
        keep = hist.clone(), hlen.clone(), kv_len.clone(), [t.clone() for t in cache.tensors]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()  # the library's matmul set up outside the capture
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            one_lg, one_ids = step()
        hist.copy_(keep[0]), hlen.copy_(keep[1]), kv_len.copy_(keep[2])
        for t, k in zip(cache.tensors, keep[3]):
            t.copy_(k)
    for _ in range(n_new - 1):
        if graph:
            gr.replay()
        else:
            one_lg, one_ids = step()
        logits.append(one_lg.clone())
        picked.append(one_ids.clone())
        cur.copy_(one_ids)
    torch.cuda.synchronize()
    picked = torch.stack(picked).cpu().numpy()
    logits = torch.stack(logits).cpu().numpy().astype(np.float64)
    # the 64-bit loop on the tokens that were picked, over the values that the cache holds
    kc, ks, vc, vs = (t.cpu().numpy() for t in cache.tensors[:4])
    tb, rp = table.cpu().numpy(), rope.cpu().numpy()
    for s, p in enumerate(prompts):
        toks = p + picked[:-1, s].tolist()
        n = len(toks)
        j = np.arange(n)
        pg, at = tb[s, j // page], j % page
        k, v = S.values(kc[pg, :, at], ks[pg, :, at]), S.values(vc[pg, :, at], vs[pg, :, at])
        qkv = (emb[toks].astype(np.float64) @ wqkv.astype(np.float64)).reshape(n, Nh + 2 * Nkv, D)
        q, _ = S.rotate(S.rms(qkv[:, :Nh], qn, 1e-6), j, rp, "half")
        kk, _ = S.rotate(S.rms(qkv[:, Nh:Nh + Nkv], kn, 1e-6), j, rp, "half")
        for val, held in ((kk, k), (qkv[:, Nh + Nkv:], v)):
            top = np.abs(val.reshape(n, Nkv, -1, 32)).max(-1, keepdims=True)
            # a code is at most half a step of top / 8 off, the far end of the range (7 against 8) a whole one, d 2^-9 of 8 steps
            assert (np.abs((val - held).reshape(n, Nkv, -1, 32)) <= top / 8 * (1 + 2.0 ** -8 * 8)).all()
        for step_i in range(n_new):
            i = len(p) + step_i - 1
            o = np.stack([S.attention(q[i:i + 1, h], k[:, h // 2], v[:, h // 2], i, 0, D ** -0.5)[0][0] for h in range(Nh)])
            lg = (o.reshape(-1) @ emb.astype(np.float64).T)
            ref, mag = S.rules(lg, toks[:i + 1], len(p), float(np.float32(1.2)), None, float(np.float32(0.3)), (), allowed[0])
            # 512 products in f32 through attention and head: 2^-13 of the row's size is over sqrt(512) half steps of each
            tol = 2.0 ** -13 * np.abs(o).max() * np.abs(emb).max() * 8
            got = logits[step_i, s]
            assert np.array_equal(np.isneginf(got), np.isneginf(ref))
            fin = np.isfinite(ref)
            assert np.abs(got[fin] - ref[fin]).max() <= tol
            assert picked[step_i, s] == int(np.argmax(got)) and allowed[0, picked[step_i, s]]


def _calls(rng):
    """One call of every operator, to be made on a given stream"""
    import torch
    table = torch.arange(64, dtype=torch.int32).view(1, 64).cuda()
    cache = acb.KVCacheQ4.empty(64, 64, 2, 128, table)
    cache.tensors[0].random_(0, 256), cache.tensors[2].random_(0, 256)
    for t in (cache.tensors[1], cache.tensors[3]):
        t.copy_((0.02 + 0.2 * torch.rand(t.shape)).bfloat16().half())
    x = torch.from_numpy(rng.standard_normal((2, 8, 128)).astype(np.float32)).cuda()
    pos, seq = torch.tensor([4094, 4095], dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda()
    before = pos - 100  # (a caller's tensors live until the stream is done with them)
    ln, start = torch.tensor([4090], dtype=torch.int32).cuda(), torch.tensor([0, 2], dtype=torch.int32).cuda()
    rope = acb.rope_table_scaled(4096, 128, 1e4).cuda()
    lg = torch.from_numpy(rng.standard_normal((2, 5000)).astype(np.float32)).cuda()
    hist = torch.from_numpy(rng.integers(0, 5000, (2, 40)).astype(np.int32)).cuda()
    two = torch.full((2,), 1.5).cuda()
    return [lambda st: acb.rope(x, pos, rope, stream=st),
            lambda st: cache.append(x.reshape(2, -1), 4, seq, pos, rope, stream=st),
            lambda st: cache.read(seq, before, stream=st),
            lambda st: cache.attention(x, ln, start, 2, stream=st),
            lambda st: acb.logits_rules(lg, hist, rep=two, stream=st)]


@pytest.mark.parametrize("as_number", [False, True])
def test_what_a_call_makes_belongs_to_its_stream(cuda, monkeypatch, as_number):
    import torch
    side, made, empty = torch.cuda.Stream(), [], torch.empty

    def noted(*a, **kw):
        made.append(torch.cuda.current_stream().cuda_stream)
        return empty(*a, **kw)
    for call in _calls(np.random.default_rng(1)):
        torch.cuda.synchronize()
        monkeypatch.setattr(torch, "empty", noted)
        made.clear()
        call(side.cuda_stream if as_number else side)
        monkeypatch.undo()
        assert made and set(made) == {side.cuda_stream}
        assert torch.cuda.current_stream().cuda_stream != side.cuda_stream
    torch.cuda.synchronize()


def test_a_late_stream_and_new_memory_on_the_current_one(cuda):
    """The call's stream is busy; what the current stream is given and fills in the meantime is none of the call's memory."""
    import torch
    for call in _calls(np.random.default_rng(2)):
        ref = call(None)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            a = torch.ones(2048, 2048, device="cuda")
            for _ in range(50):
                a = (a @ a).clamp_(-1, 1)
        got = call(side)
        junk = [torch.full((n,), float("nan"), device="cuda") for n in (64, 512, 4096, 1 << 15, 1 << 18, 1 << 20) for _ in range(20)]
        torch.cuda.synchronize()
        # (looked at after the synchronisation only: read gives two tensors)
        got, ref = (v if isinstance(v, tuple) else (v,) for v in (got, ref))
        assert all(torch.equal(g, r) for g, r in zip(got, ref)) and len(junk) == 120


def test_flag_words_that_would_be_misread_are_refused(cuda):
    """A flag on the host, of another type or without an element: refused before anything is launched."""
    import torch
    x, pos = torch.randn(1, 4, 64).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    table, rope = torch.zeros((1, 1), dtype=torch.int32).cuda(), acb.rope_table_scaled(16, 64, 1e4).cuda()
    cache = acb.KVCacheQ4.empty(1, 16, 1, 64, table)
    good = torch.zeros(1, dtype=torch.int32).cuda()
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64).cuda(), torch.zeros(4, dtype=torch.uint8).cuda(),
                torch.zeros(0, dtype=torch.int32).cuda()):
        for call in (lambda e: acb.rope(x, pos, rope, err=e), lambda e: cache.append(x.view(1, 256), 2, pos, pos, rope, err=e),
                     lambda e: cache.read(pos, pos, err=e), lambda e: cache.attention(x, pos + 1, err=e),
                     lambda e: acb.logits_rules(x.view(1, 256), err=e)):
            with pytest.raises(ValueError):
                call(bad)
            call(good), call(good.data_ptr()), call(None)
    assert int(good) == 0


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,D,R,layout", [(1, 128, 128, "half"), (3, 64, 10, "half"), (5, 256, 64, "interleaved"), (400, 128, 128, "half"),
                                          (1500, 64, 64, "interleaved")])
def test_queries_in_place(cuda, kind, n, D, R, layout):
    """q written over the q part of qkv, and the attention's output over q: what separate buffers give."""
    import torch
    import serving_ref as S
    g = torch.Generator().manual_seed(n + D)
    Nh, Nkv, P, past = 10, 2, 16, 777
    pages = -(-(n + past) // P)
    table = torch.arange(pages, dtype=torch.int32).view(1, -1).cuda()
    cache = acb.KVCacheQ4.empty(pages, P, Nkv, D, table)
    rope = acb.rope_table_scaled(pages * P, R, 1e4).cuda()
    w = (1 + 0.1 * torch.randn(D, generator=g)).cuda()
    x = torch.randn(past + n, (Nh + 2 * Nkv) * D, generator=g).to(S.torch_type(kind)).cuda()
    pos, seq = torch.arange(past + n, dtype=torch.int32).cuda(), torch.zeros(past + n, dtype=torch.int32).cuda()
    cache.append(x[:past], Nh, seq[:past], pos[:past], rope, layout, w, w)
    new, ln, start = x[past:], torch.tensor([past + n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    q = cache.append(new, Nh, seq[past:], pos[past:], rope, layout, w, w)
    held = [t.clone() for t in cache.tensors[:4]]
    o = cache.attention(q, ln, start, n)
    buf = new.clone()
    view = buf[:, :Nh * D].unflatten(1, (Nh, D))
    assert cache.append(buf, Nh, seq[past:], pos[past:], rope, layout, w, w, q_out=view) is view
    assert torch.equal(view, q) and torch.equal(buf[:, Nh * D:], new[:, Nh * D:])
    assert all(torch.equal(a, b) for a, b in zip(held, cache.tensors))
    for work in (None, torch.empty(1, dtype=torch.uint8).cuda()):  # the keys cut into chunks, and not
        ref = cache.attention(q, ln, start, n, work=work)
        view.copy_(q)
        cache.attention(view, ln, start, n, out=view, work=work)
        assert torch.equal(view, ref) and torch.equal(buf[:, Nh * D:], new[:, Nh * D:])
    assert bool(o.isfinite().all())
