"""GPU: rules on logits (acb_logits_rules) against 64 bits.

Bar: every step (repetition, frequency's product and difference, presence, bias) is rounded in f32: 5 half steps of the largest
magnitude met, 5 * 2^-24, plus half a step of the output's type. -inf and whole rows of it exactly."""
import numpy as np
import pytest

import acb
import serving_ref as S

pytestmark = pytest.mark.gpu


def _words(bits):
    import torch
    n, V = bits.shape
    pad = np.zeros((n, -(-V // 32) * 32), bool)
    pad[:, :V] = bits
    return torch.from_numpy(np.packbits(pad, axis=1, bitorder="little").view(np.int32)).cuda()


def _check(y, x, R, kind, hist=None, lens=None, prompt=None, rep=None, freq=None, pres=None, bias=None, bits=None, mrow=None):
    for r in range(R):
        h = hist[r, :max(0, min(lens[r], hist.shape[1])) if lens is not None else hist.shape[1]] if hist is not None else None
        b = [(int(t), float(v)) for t, v in zip(bias[0][r if bias[0].ndim == 2 else slice(None)],
                                                bias[1][r if bias[1].ndim == 2 else slice(None)])] if bias else ()
        m = r if mrow is None else mrow[r]
        ref, mag = S.rules(x[r], h, prompt[r] if prompt is not None else 0, None if rep is None else float(rep[r]),
                           None if freq is None else float(freq[r]), None if pres is None else float(pres[r]), b,
                           bits[m] if bits is not None and 0 <= m < len(bits) else None)
        closed = np.isneginf(ref)
        assert np.array_equal(np.isneginf(y[r]), closed)
        tol = 5 * 2.0 ** -24 * mag + S.HALF_STEP[kind] * (np.abs(ref) + 5 * 2.0 ** -24 * mag) + (2.0 ** -25 if kind == "f16" else 0)
        with np.errstate(invalid="ignore"):
            d = np.abs(y[r] - ref)
        assert (d[~closed] <= tol[~closed]).all()


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("R,V,L,B,M", [(1, 1, 1, 1, 1), (3, 33, 5, 2, 2), (2, 4096, 300, 7, 1), (5, 4097, 50, 20, 3),
                                       (1, 50001, 9000, 300, 1), (7, 8191, 64, 0, 0), (4, 12345, 0, 9, 2)])
def test_everything(cuda, kind, out, R, V, L, B, M):
    import torch
    rng = np.random.default_rng(R * V + L)
    x = torch.from_numpy((rng.standard_normal((R, V)) * 4).astype(np.float32)).to(S.torch_type(kind))
    hist = rng.integers(-2, V, (R, L)).astype(np.int32)
    hist[:, ::3] = rng.integers(0, min(V, 7), hist[:, ::3].shape)
    lens, prompt = rng.integers(0, L + 1, R).astype(np.int32), rng.integers(0, L + 1, R).astype(np.int32)
    rep, freq, pres = (rng.uniform(a, b, R).astype(np.float32) for a, b in ((0.7, 1.6), (-0.5, 0.9), (-1, 1)))
    bias = [rng.integers(-1, V, (R, B)).astype(np.int32), rng.standard_normal((R, B)).astype(np.float32)] if B else None
    bits = rng.random((M, V)) < rng.random((M, 1)) if M else None
    mrow = rng.integers(-1, M, R).astype(np.int32) if M else None
    c = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    err = torch.zeros(1, dtype=torch.int32).cuda()
    y = acb.logits_rules(x.cuda(), c(hist), c(lens), c(prompt), c(rep), c(freq), c(pres), c(bias[0]) if B else None,
                         c(bias[1]) if B else None, _words(bits) if M else None, c(mrow), out_dtype=S.torch_type(out), err=err)
    assert int(err) == 0
    if L == 0:
        hist = None
    _check(y.float().cpu().numpy().astype(np.float64), x.float().numpy(), R, out, hist, lens, prompt, rep, freq, pres, bias, bits, mrow)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_each_part_alone(cuda, kind):
    import torch
    rng = np.random.default_rng(3)
    R, V, L = 3, 5000, 40
    x = torch.from_numpy(rng.standard_normal((R, V)).astype(np.float32)).to(S.torch_type(kind))
    xs = x.float().numpy()
    hist = rng.integers(0, V, (R, L)).astype(np.int32)
    d_h, par = torch.from_numpy(hist).cuda(), rng.uniform(0.5, 2, R).astype(np.float32)
    d_p = torch.from_numpy(par).cuda()
    same = acb.logits_rules(x.cuda())
    assert torch.equal(same, x.cuda())
    for name in ("rep", "freq", "pres"):
        y = acb.logits_rules(x.cuda(), d_h, **{name: d_p})
        _check(y.float().cpu().numpy().astype(np.float64), xs, R, kind, hist, **{name: par})
    ids, val = rng.integers(0, V, 9).astype(np.int32), rng.standard_normal(9).astype(np.float32)
    y = acb.logits_rules(x.cuda(), bias_ids=torch.from_numpy(ids).cuda(), bias_val=torch.from_numpy(val).cuda())
    _check(y.float().cpu().numpy().astype(np.float64), xs, R, kind, bias=[ids, val])
    bits = rng.random((R, V)) < 0.3
    y = acb.logits_rules(x.cuda(), mask=_words(bits))
    _check(y.float().cpu().numpy().astype(np.float64), xs, R, kind, bits=bits)


@pytest.mark.parametrize("R,V,L", [(1, 3000, 20000), (300, 9000, 6000), (2, 40, 5000)])
def test_histories_that_name_nearly_every_column(cuda, R, V, L):
    import torch
    rng = np.random.default_rng(V)
    x = torch.from_numpy(rng.standard_normal((R, V)).astype(np.float32))
    hist = rng.integers(0, V, (R, L)).astype(np.int32)
    rep, freq = (rng.uniform(0.1, 1.5, R).astype(np.float32) for _ in "rf")
    prompt = np.full(R, L // 4, np.int32)
    bias = [rng.integers(0, V, (R, 2047)).astype(np.int32), rng.standard_normal((R, 2047)).astype(np.float32)]
    c = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    y = acb.logits_rules(x.cuda(), c(hist), None, c(prompt), c(rep), c(freq), None, c(bias[0]), c(bias[1]))
    rows = [0, R - 1]
    _check(y.cpu().numpy().astype(np.float64)[rows], x.numpy()[rows], len(rows), "f32", hist[rows], None, prompt[rows], rep[rows],
           freq[rows], None, [b[rows] for b in bias])


def test_in_place_strides_and_rows_around(cuda):
    import torch
    rng = np.random.default_rng(4)
    R, V = 4, 999
    for kind in ("f32", "f16"):
        for off in (0, 1, 3, 4):
            buf = torch.from_numpy(rng.standard_normal((R + 2, V + 9)).astype(np.float32)).to(S.torch_type(kind)).cuda()
            keep = buf.clone()
            x = buf[1:R + 1, off:off + V]
            hist = torch.from_numpy(rng.integers(0, V, (R, 30)).astype(np.int32)).cuda()
            rep, bits = torch.full((R,), 1.3).cuda(), rng.random((1, V)) < 0.5
            row = torch.zeros(R, dtype=torch.int32).cuda()
            ref = acb.logits_rules(x.contiguous(), hist, rep=rep, mask=_words(bits), mask_row=row)
            acb.logits_rules(x, hist, rep=rep, mask=_words(bits), mask_row=row, out=x)
            assert torch.equal(x, ref)
            buf[1:R + 1, off:off + V] = keep[1:R + 1, off:off + V]
            assert torch.equal(buf, keep)  # nothing around it


def test_closed_rows_nan_and_infinities(cuda):
    """A mask closes NaN and infinities too and may close a whole row; open ones go through."""
    import torch
    x = torch.zeros(3, 70).cuda()
    x[:, 3], x[:, 4], x[:, 5], x[:, 6] = float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min
    bits = np.zeros((2, 70), bool)
    bits[1, 3:8] = True
    row = torch.tensor([0, 1, -1], dtype=torch.int32).cuda()
    hist = torch.tensor([[3, 4, 5, 6]] * 3, dtype=torch.int32).cuda()
    y = acb.logits_rules(x, hist, rep=torch.full((3,), 2.0).cuda(), mask=_words(bits), mask_row=row).cpu()
    assert bool((y[0] == -float("inf")).all())
    for r in (1, 2):
        assert bool(y[r, 3].isnan()) and y[r, 4] == float("inf") and y[r, 5] == -float("inf") and y[r, 6] == -float("inf")
        assert y[r, 7] == 0
    assert bool((y[1, 8:] == -float("inf")).all()) and bool((y[2, 7:] == 0).all())


def test_range_errors_and_padding(cuda):
    import torch
    V = 100
    x = torch.ones(2, V).cuda()

    def go(**kw):
        err = torch.zeros(1, dtype=torch.int32).cuda()
        return acb.logits_rules(x, err=err, **kw), int(err)
    two, i = torch.full((2,), 2.0).cuda(), lambda *a: torch.tensor(a, dtype=torch.int32).cuda()  # noqa: E731
    y, e = go(hist=i([5, -1, -9], [6, 6, -1]), rep=two)
    assert e == 0 and y[0, 5] == 0.5 and y[1, 6] == 0.5 and int((y != 1).sum()) == 2
    y, e = go(hist=i([V, 2 ** 31 - 1, 5], [6, 6, 6]), rep=two)
    assert e == 1 and y[0, 5] == 0.5 and int((y != 1).sum()) == 2
    y, e = go(hist=i([7, V, 5], [6, 6, 6]), hist_len=i(1, -4), rep=two)  # behind the length nothing is looked at
    assert e == 0 and y[0, 7] == 0.5 and int((y != 1).sum()) == 1
    y, e = go(hist=i([7, 8, 5], [6, 6, 6]), hist_len=i(99, 3), pres=two, prompt_len=i(-3, 99))
    assert e == 0 and y[0, [5, 7, 8]].tolist() == [-1, -1, -1] and int((y != 1).sum()) == 3
    y, e = go(bias_ids=i(V, -1, 3, 3), bias_val=torch.tensor([1.0, 1, 5, 2]).cuda())
    assert e == 1 and bool((y[:, 3] == 3).all()) and int((y != 1).sum()) == 2
    y, e = go(mask=torch.zeros((1, 4), dtype=torch.int32).cuda(), mask_row=i(1, -1))
    assert e == 1 and bool((y == 1).all())


def test_streams_graph_and_repeats(cuda):
    import torch
    rng = np.random.default_rng(6)
    R, V = 8, 30000
    x = torch.randn(R, V).cuda()
    hist = torch.from_numpy(rng.integers(0, 50, (R, 500)).astype(np.int32)).cuda()
    lens, f = torch.full((R,), 300, dtype=torch.int32).cuda(), torch.full((R,), 0.1).cuda()
    out = torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        acb.logits_rules(x, hist, lens, freq=f, out=out)
    for n in (300, 7, 500):
        lens.fill_(n)
        x.normal_()
        g.replay()
        ref = acb.logits_rules(x, hist, lens, freq=f)
        assert torch.equal(out, ref)
        assert all(torch.equal(ref, acb.logits_rules(x, hist, lens, freq=f)) for _ in range(5))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = acb.logits_rules(x, hist, lens, freq=f)
    s.synchronize()
    assert torch.equal(y, ref)


@pytest.mark.parametrize("V,L,B,pad", [(40008, 4000, 2000, 0), (40001, 4100, 7, 0), (40008, 1, 1, 4), (33000, 2500, 0, 8)])
def test_long_slices_of_many_rows(cuda, V, L, B, pad):
    """Enough rows that a block has tens of thousands of columns and few of its warps look at the history; with pad 4 the
    output's rows lie 16 but not 32 bytes apart from a boundary."""
    import torch
    rng = np.random.default_rng(V + L)
    R = 128
    x = torch.from_numpy((rng.standard_normal((R, V)) * 4).astype(np.float32)).to(torch.bfloat16)
    hist = rng.integers(-1, V, (R, L)).astype(np.int32)
    hist[:, ::5] = rng.integers(V // 2, V // 2 + 600, hist[:, ::5].shape)  # often named, next to one another
    lens, prompt = rng.integers(0, L + 1, R).astype(np.int32), rng.integers(0, L + 1, R).astype(np.int32)
    lens[:2] = L
    rep, freq, pres = (rng.uniform(a, b, R).astype(np.float32) for a, b in ((0.7, 1.6), (-0.5, 0.9), (-1, 1)))
    bias = [rng.integers(-1, V, (R, B)).astype(np.int32), rng.standard_normal((R, B)).astype(np.float32)] if B else None
    bits = rng.random((2, V)) < 0.6
    mrow = rng.integers(-1, 2, R).astype(np.int32)
    c = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    out = torch.full((R, V + pad), 7.0).cuda()
    err = torch.zeros(1, dtype=torch.int32).cuda()
    acb.logits_rules(x.cuda(), c(hist), c(lens), c(prompt), c(rep), c(freq), c(pres), c(bias[0]) if B else None,
                     c(bias[1]) if B else None, _words(bits), c(mrow), out=out[:, :V], err=err)
    assert int(err) == 0 and (out[:, V:] == 7).all()
    some = [0, 1, 50, R - 1]
    _check(out[some, :V].cpu().numpy().astype(np.float64), x[some].float().numpy(), len(some), "f32", hist[some], lens[some], prompt[some],
           rep[some], freq[some], pres[some], [b[some] for b in bias] if B else None, bits, mrow[some])


def test_host_threads_of_long_and_short_histories(cuda):
    """Calls from several threads at once, each on a stream of its own and straight into the library, so that they meet
    there: no call's size limits another's launch."""
    import ctypes as C
    import threading
    import torch
    rng = np.random.default_rng(8)
    V, calls, fn = 4096, 5000, acb.lib().acb_logits_rules
    x = torch.randn(2, V).cuda()
    rep = torch.full((2,), 1.5).cuda()
    jobs = []
    for L in (6000, 3, 5000, 40):
        hist = torch.from_numpy(rng.integers(0, V, (2, L)).astype(np.int32)).cuda()
        out = torch.empty_like(x)
        r = acb._LogitRules(hist=hist.data_ptr(), hist_stride=L, rep=rep.data_ptr())
        st = torch.cuda.Stream()
        args = (x.data_ptr(), acb.F32, V, out.data_ptr(), acb.F32, V, 2, V, C.addressof(r), None, st.cuda_stream)
        jobs.append((args, acb.logits_rules(x, hist, rep=rep), out, st, set(), (hist, r)))
    torch.cuda.synchronize()
    go = threading.Barrier(len(jobs))

    def run(args, ref, out, st, seen, keep):
        go.wait()
        for _ in range(calls):
            seen.add(fn(*args))
    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for args, ref, out, st, seen, keep in jobs:
        assert seen == {0} and torch.equal(out, ref)


def test_bias_lists_of_unlike_shapes_are_refused(cuda):
    import torch
    x = torch.zeros(2, 50).cuda()
    i = lambda *s: torch.ones(s, dtype=torch.int32).cuda()  # noqa: E731
    v = lambda *s: torch.ones(s).cuda()  # noqa: E731
    for ids, val in ((i(2, 3), v(3, 2)), (i(2, 3), v(6)), (i(3), v(2, 3)), (i(2, 3), v(1, 3)), (i(3), v(2)), (i(1, 3), v(1, 3))):
        with pytest.raises(ValueError):
            acb.logits_rules(x, bias_ids=ids, bias_val=val)
    for ids, val in ((i(2, 3), v(2, 3)), (i(3), v(3)), (i(3, 3), v(2, 3).repeat(2, 1)), (i(3), v(1, 3)), (i(2, 0), v(2, 0))):
        y = acb.logits_rules(x, bias_ids=ids, bias_val=val)
        assert bool((y[:, 1] == (1 if ids.numel() else 0)).all()) and int((y != 0).sum()) == (2 if ids.numel() else 0)
