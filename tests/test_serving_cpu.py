"""CPU: the serving operators' refusals (every bad argument is a status before a device is touched) and the host table of
angles for long contexts."""
import ctypes as C
import math

import numpy as np
import pytest

import acb

BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 15) // 16 * 16  # a 16-byte aligned address: no call here gets as far as using it


def cache(**kw):
    d = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, page_table=P, table_stride=4, n_pages=8, page_size=16, n_kv_heads=2,
             head_dim=64, n_seq=3, max_pages=4)
    d.update(kw)
    return acb._KvQ4(**d)


BAD_CACHES = [(dict(k_codes=None), 1), (dict(v_scales=None), 1), (dict(page_table=None), 1), (dict(k_codes=P + 8), 1),
              (dict(n_pages=0), 1), (dict(n_seq=0), 1), (dict(n_kv_heads=0), 1), (dict(max_pages=0), 1),
              (dict(table_stride=3), 1), (dict(page_size=0), 1), (dict(page_size=-16), 1), (dict(page_size=8), 2),
              (dict(page_size=48), 2), (dict(page_size=8192), 2), (dict(head_dim=96), 2), (dict(head_dim=512), 2),
              (dict(max_pages=1 << 20, table_stride=1 << 20, page_size=4096), 2)]


def append(kv, qkv=P, type=acb.F32, stride=4 * 64 + 128, n_tok=1, n_heads=2, table=P, max_pos=9, rope_dim=64, layout=0, seq=P,
           pos=P, q_out=P, q_type=acb.F32, q_stride=128):
    return acb.lib().acb_kv_q4_append(C.addressof(kv) if kv is not None else None, qkv, type, stride, n_tok, n_heads, None, None,
                                      1e-6, table, max_pos, rope_dim, layout, seq, pos, q_out, q_type, q_stride, None, None)


def read(kv, seq=P, pos=P, n_tok=1, k=P, v=P, type=acb.F16, stride=128):
    return acb.lib().acb_kv_q4_read(C.addressof(kv) if kv is not None else None, seq, pos, n_tok, k, v, type, stride, None, None)


def attn(kv, q=P, type=acb.F32, q_stride=256, n_tok=3, n_heads=4, q_start=None, kv_len=P, max_q=1, max_kv=64, window=0,
         scale=1.0, o=P, o_stride=256):
    return acb.lib().acb_attn_kv_q4(C.addressof(kv) if kv is not None else None, q, type, q_stride, n_tok, n_heads, q_start,
                                    kv_len, max_q, max_kv, window, scale, o, o_stride, None, 0, None, None)


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_bad_caches_are_refused(kw, status):
    kv = cache(**kw)
    assert append(kv) == status and read(kv) == status and attn(kv) == status
    assert acb.lib().acb_attn_kv_q4_work_bytes(C.addressof(kv), 4, 4, 1, 64) == 0


def test_null_cache_is_refused():
    assert append(None) == 1 and read(None) == 1 and attn(None) == 1


@pytest.mark.parametrize("kw,status", [(dict(qkv=None), 1), (dict(seq=None), 1), (dict(pos=None), 1), (dict(q_out=None), 1),
                                       (dict(n_tok=-1), 1), (dict(n_heads=-1), 1), (dict(stride=383), 1),
                                       (dict(q_stride=127), 1), (dict(max_pos=0), 1), (dict(rope_dim=66), 1),
                                       (dict(rope_dim=3), 1), (dict(rope_dim=0), 1), (dict(layout=2), 1), (dict(layout=4), 1),
                                       (dict(type=acb.Q8_0), 2), (dict(q_type=acb.I32), 2), (dict(n_tok=1 << 40), 2)])
def test_append_refusals(kw, status):
    assert append(cache(), **kw) == status


def test_no_tokens_is_nothing_to_do():
    assert append(cache(), n_tok=0) == 0 and read(cache(), n_tok=0) == 0
    assert attn(cache(), n_tok=0, q_start=P) == 0


@pytest.mark.parametrize("kw,status", [(dict(seq=None), 1), (dict(pos=None), 1), (dict(k=None, v=None), 1), (dict(n_tok=-1), 1),
                                       (dict(stride=127), 1), (dict(type=acb.Q4_K), 2)])
def test_read_refusals(kw, status):
    assert read(cache(), **kw) == status


@pytest.mark.parametrize("kw,status", [(dict(q=None), 1), (dict(o=None), 1), (dict(kv_len=None), 1), (dict(n_tok=-1), 1),
                                       (dict(n_heads=0), 1), (dict(n_heads=3, q_stride=256), 1), (dict(max_q=0), 1),
                                       (dict(max_q=2), 1), (dict(n_tok=4), 1), (dict(max_kv=-1), 1), (dict(window=-1), 1),
                                       (dict(scale=math.nan), 1), (dict(scale=math.inf), 1), (dict(q_stride=255), 1), (dict(o_stride=255), 1),
                                       (dict(max_kv=65), 4), (dict(type=acb.Q8_0), 2)])
def test_attention_refusals(kw, status):
    assert attn(cache(), **kw) == status


def rope(src=P, sts=128, shs=64, dst=P, dts=128, dhs=64, type=acb.F32, n_tok=2, n_heads=2, D=64, R=64, layout=0, pos=P, table=P,
         max_pos=4):
    return acb.lib().acb_rope(src, sts, shs, dst, dts, dhs, type, n_tok, n_heads, D, R, layout, pos, table, max_pos, None, None)


@pytest.mark.parametrize("kw,status", [(dict(src=None), 1), (dict(dst=None), 1), (dict(pos=None), 1), (dict(table=None), 1),
                                       (dict(n_tok=-1), 1), (dict(n_heads=0), 1), (dict(D=63), 1), (dict(R=66), 1),
                                       (dict(R=0), 1), (dict(R=31), 1), (dict(layout=4), 1), (dict(layout=-1), 1),
                                       (dict(max_pos=0), 1), (dict(dts=256), 1), (dict(shs=0, dhs=0), 1),
                                       (dict(sts=64, dts=64), 1), (dict(dst=P + 64, dhs=32), 1),
                                       (dict(type=acb.Q8_0), 2), (dict(D=1026, R=2, sts=4096, dts=4096, shs=2048, dhs=2048), 2),
                                       (dict(n_tok=1 << 40), 2), (dict(n_heads=16385, sts=1 << 21, dts=1 << 21), 2)])
def test_rope_refusals(kw, status):
    assert rope(**kw) == status


def test_rope_of_nothing():
    assert rope(n_tok=0) == 0


def logits(x=P, type=acb.F32, ld=100, y=P, out_type=acb.F32, ldo=100, rows=2, V=100, null_rules=False, **rules):
    r = acb._LogitRules(**rules)
    return acb.lib().acb_logits_rules(x, type, ld, y, out_type, ldo, rows, V, None if null_rules else C.addressof(r), None, None)


@pytest.mark.parametrize("kw,status", [(dict(x=None), 1), (dict(y=None), 1), (dict(null_rules=True), 1), (dict(rows=-1), 1),
                                       (dict(V=0), 1), (dict(ld=99), 1), (dict(ldo=99), 1), (dict(hist=P, hist_stride=-1), 1),
                                       (dict(rep=P), 1), (dict(freq=P), 1), (dict(pres=P), 1), (dict(bias_ids=P), 1),
                                       (dict(bias_val=P), 1), (dict(bias_ids=P, bias_val=P, n_bias=-1), 1),
                                       (dict(bias_ids=P, bias_val=P, n_bias=5, bias_stride=4), 1), (dict(mask=P), 1),
                                       (dict(mask=P, n_masks=2, mask_stride=3), 1), (dict(mask_row=P), 1),
                                       (dict(out_type=acb.F16), 1), (dict(ldo=101), 1), (dict(type=acb.Q8_0, y=P + 16), 2),
                                       (dict(y=P + 16, out_type=acb.I32), 2), (dict(rows=65536), 2)])
def test_logits_refusals(kw, status):
    assert logits(**kw) == status


def test_logits_of_nothing():
    assert logits(rows=0) == 0


# ---- tables -----------------------------------------------------------------------------------------

def _ref(max_pos, R, base, f):
    a = np.arange(max_pos)[:, None] * f(np.arange(R // 2), base ** (-2.0 * np.arange(R // 2) / R))
    return a


# the double angle p f is off by at most 2^-52 p f (f's power, the product), so cos and sin by that, and the float by half a
# step: 2^-24; the values are at most m
@pytest.mark.parametrize("R,base,max_pos", [(128, 1e6, 8192), (64, 1e4, 300), (2, 1e4, 50), (6, 500.0, 20000)])
@pytest.mark.parametrize("kind,factor", [(0, 1.0), (1, 8.0), (2, 4.0), (3, 16.0)])
def test_scaled_tables(R, base, max_pos, kind, factor):
    if kind == acb.ROPE_SCALE_NTK and R < 4:
        with pytest.raises(acb.AcbError):
            acb.rope_table_scaled(max_pos, R, base, kind, factor)
        return
    t = acb.rope_table_scaled(max_pos, R, base, kind, factor, orig_max_pos=4096).numpy()
    i = np.arange(R // 2)
    f, m = float(base) ** (-2.0 * i / R), 1.0
    if kind == 1:
        f = f / factor
    elif kind == 2:
        f = (base * factor ** (R / (R - 2))) ** (-2.0 * i / R)
        assert R == 2 or f[-1] == pytest.approx(base ** (-2.0 * i[-1] / R) / factor, rel=1e-12)
    elif kind == 3:
        m = 0.1 * math.log(factor) + 1
        turns = [R * math.log(4096 / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0)]
        lo, hi = max(0, math.floor(turns[0])), min(R - 1, math.ceil(turns[1]))
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        f = f * (1 - ramp) + f / factor * ramp
    a = np.arange(max_pos)[:, None] * f
    tol = m * (2.0 ** -24 + max_pos * 2.0 ** -50)
    assert np.abs(t[:, 0::2] - m * np.cos(a)).max() <= tol and np.abs(t[:, 1::2] - m * np.sin(a)).max() <= tol


@pytest.mark.parametrize("args", [(0, 64, 1e4, 0, 1.0, 0, 32.0, 1.0), (8, 63, 1e4, 0, 1.0, 0, 32.0, 1.0),
                                  (8, 64, 1.0, 0, 1.0, 0, 32.0, 1.0), (8, 64, math.inf, 0, 1.0, 0, 32.0, 1.0),
                                  (8, 64, 1e4, 4, 1.0, 0, 32.0, 1.0), (8, 64, 1e4, 1, 0.5, 0, 32.0, 1.0),
                                  (8, 64, 1e4, 1, math.nan, 0, 32.0, 1.0), (8, 64, 1e4, 3, 2.0, 0, 32.0, 1.0),
                                  (8, 64, 1e4, 3, 2.0, 100, 1.0, 1.0), (8, 64, 1e4, 3, 2.0, 100, 32.0, 0.0)])
def test_scaled_table_refusals(args):
    assert acb.lib().acb_rope_table_scaled_host(P, *args) == 1
    assert acb.lib().acb_rope_table_scaled_host(None, 8, 64, 1e4, 0, 1.0, 0, 32.0, 1.0) == 1


def test_wrappers_refuse_cpu_tensors():
    import torch
    with pytest.raises(ValueError):
        acb.rope(torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), torch.zeros(4, 64))
    with pytest.raises(ValueError):
        acb.logits_rules(torch.zeros(2, 8), mask=torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError):
        acb.logits_rules(torch.zeros(2, 8), rep=torch.ones(2))


def test_workspaces_cover_every_smaller_call():
    """acb_attn_kv_q4_work_bytes: what it gives for sizes holds for all smaller rows and lengths, and a workspace is only asked
    where there is something to split."""
    f = acb.lib().acb_attn_kv_q4_work_bytes
    for n_seq, heads in ((1, 4), (3, 14), (64, 32)):
        kv = cache(n_seq=n_seq, n_kv_heads=2, head_dim=128, max_pages=1 << 12, table_stride=1 << 12, n_pages=1 << 13)
        ref = C.addressof(kv)
        full = f(ref, n_seq * 40, heads, 40, 60000)
        for q in (1, 2, 3, 7, 39):
            for n in (1, 500, 59999):
                assert f(ref, n_seq * q, heads, q, n) <= full
        assert f(ref, n_seq, heads, 1, 100) == 0
        assert f(ref, 0, heads, 1, 60000) == 0 and f(ref, n_seq, heads, 0, 60000) == 0 and f(ref, n_seq, 3, 1, 60000) == 0


def test_append_refuses_more_tokens_than_a_grid_has_blocks():
    assert append(cache(), n_heads=0, n_tok=2 ** 31) == 2


@pytest.mark.parametrize("n_seq,n_kv,heads,D,first,last,keys", [
    (16, 8, 16, 128, 9, 16, 8192), (24, 2, 14, 64, 5, 6, 4000), (24, 2, 14, 64, 7, 9, 4000), (1, 1, 1, 128, 1009, 1024, 60000),
    (5, 4, 12, 256, 51, 53, 20000)])
def test_workspaces_cover_every_count_of_rows(n_seq, n_kv, heads, D, first, last, keys):
    """Calls of first..last rows a sequence fill the same number of row tiles, so their keys are cut alike and they need the same
    bytes a row; what is enough for the most of them is enough for all in that measure."""
    kv = cache(n_seq=n_seq, n_kv_heads=n_kv, head_dim=D, max_pages=1 << 12, table_stride=1 << 12, n_pages=1 << 13)
    tile = 8 if D == 256 else 16
    assert -(-first * heads // n_kv // tile) == -(-last * heads // n_kv // tile)
    f = lambda q: acb.lib().acb_attn_kv_q4_work_bytes(C.addressof(kv), n_seq * q, heads, q, keys)  # noqa: E731
    assert f(last) > 0
    for q in range(first, last):
        assert f(q) * last >= f(last) * q and f(q) <= f(last)


@pytest.mark.parametrize("kw", [dict(q_stride=256), dict(q_type=acb.F16, q_stride=384)])
def test_append_in_place_wants_one_layout(kw):
    assert append(cache(), q_out=P, qkv=P, n_tok=2, stride=384, **kw) == 1


def test_attention_in_place_wants_one_layout():
    assert attn(cache(), q_stride=256, o_stride=300) == 1


@pytest.mark.parametrize("heads", [(1 << 25) - 4, (1 << 25) - 3, 1 << 30, 2 ** 31 - 1])
def test_append_refuses_rows_of_2_to_the_31_elements(heads):
    assert append(cache(), n_heads=heads, stride=1 << 40, q_stride=1 << 40, q_out=P + 16) == 2
