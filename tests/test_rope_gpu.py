"""GPU: rotary positions in every layout (acb_rope) against the 64-bit rotation.

Bar: the two products and their sum are rounded in f32, so a result is within 3 * 2^-24 of the sum of the products'
magnitudes (two products and a sum, half a step each, the sum at most that large), plus half a step of the output's type."""
import numpy as np
import pytest

import acb
import serving_ref as S

pytestmark = pytest.mark.gpu


def _table(max_pos, R, seed=0):
    return acb.rope_table_scaled(max_pos, R, 1e4, acb.ROPE_SCALE_LINEAR, 4.0)


def _check(y, x, pos, table, layout, inverse, kind):
    ref, mag = S.rotate(x, pos, table.numpy(), layout, inverse)
    R = table.shape[1]
    tol = 3 * 2.0 ** -24 * mag + S.HALF_STEP[kind] * (np.abs(ref) + 3 * 2.0 ** -24 * mag)
    if kind == "f16":
        tol = tol + 2.0 ** -25  # a subnormal's half step
    d = np.abs(y.astype(np.float64) - ref)
    assert (d <= tol).all(), float((d - tol).max())
    assert np.array_equal(y[..., R:], x[..., R:])  # what is not rotated is copied


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 2, 2), (1, 24, 128, 128), (7, 5, 64, 32), (33, 3, 192, 64), (130, 2, 50, 30),
                                     (5, 9, 1024, 1022), (3, 4, 80, 16), (2, 3, 256, 6), (600, 8, 96, 96)])
def test_rope_matches_64_bits(cuda, kind, layout, T, H, D, R):
    import torch
    g = torch.Generator().manual_seed(T * 1000 + D + R)
    x = torch.randn(T, H, D, generator=g).to(S.torch_type(kind))
    pos = torch.randint(0, 900, (T,), generator=g, dtype=torch.int32)
    table = _table(900, R)
    for inverse in (False, True):
        y = acb.rope(x.cuda(), pos.cuda(), table.cuda(), layout, inverse)
        _check(y.float().cpu().numpy(), x.float().numpy(), pos.numpy(), table, layout, inverse, kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,R,off,pad", [(64, 64, 0, 0), (64, 32, 1, 3), (128, 128, 8, 8), (96, 48, 2, 6), (66, 34, 0, 1)])
def test_strides_offsets_and_in_place(cuda, kind, D, R, off, pad):
    """Columns of a wider row at any offset, heads of tokens or tokens of heads, into themselves or into gaps that stay."""
    import torch
    T, H = 11, 3
    g = torch.Generator().manual_seed(D + off)
    wide = torch.randn(T, H * D + off + pad, generator=g).to(S.torch_type(kind)).cuda()
    x = wide[:, off:off + H * D].unflatten(1, (H, D))
    pos = torch.randint(0, 50, (T,), generator=g, dtype=torch.int32)
    table = _table(50, R)
    for layout in ("half", "interleaved"):
        ref = acb.rope(x.contiguous(), pos.cuda(), table.cuda(), layout)
        _check(ref.float().cpu().numpy(), x.float().cpu().numpy(), pos.numpy(), table, layout, False, kind)
        out = torch.full((H, T, D + 5), 7.0, dtype=x.dtype, device=x.device)  # tokens of heads, gaps behind each row
        acb.rope(x, pos.cuda(), table.cuda(), layout, out=out[:, :, :D].transpose(0, 1))
        assert torch.equal(out[:, :, :D].transpose(0, 1), ref) and bool((out[:, :, D:] == 7).all())
        w2 = wide.clone()
        x2 = w2[:, off:off + H * D].unflatten(1, (H, D))
        acb.rope(x2, pos.cuda(), table.cuda(), layout, out=x2)
        assert torch.equal(x2, ref)
        assert torch.equal(w2[:, :off], wide[:, :off]) and torch.equal(w2[:, off + H * D:], wide[:, off + H * D:])


def test_broadcast_source(cuda):
    """One row for every token (stride 0): rotated by each token's position."""
    import torch
    x = torch.randn(1, 2, 64).cuda().expand(40, 2, 64)
    pos, table = torch.arange(40, dtype=torch.int32), _table(40, 64)
    y = acb.rope(x, pos.cuda(), table.cuda())
    _check(y.cpu().numpy(), x.cpu().numpy(), pos.numpy(), table, "half", False, "f32")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_inverse_is_the_gradient(cuda, layout):
    """<g, rope(x + h e) - rope(x - h e)> / 2h against <rope_inverse(g), e>: the map is linear, so the difference quotient is
    its derivative up to f32 rounding: 4 roundings of 2^-24 on each of D terms of magnitude |g||y|/h."""
    import torch
    T, H, D, R, h = 4, 2, 64, 32, 0.5
    gen = torch.Generator().manual_seed(3)
    x, e, g = (torch.randn(T, H, D, generator=gen).cuda() for _ in range(3))
    pos, table = torch.tensor([0, 3, 17, 49], dtype=torch.int32).cuda(), _table(50, R).cuda()
    up, dn = acb.rope(x + h * e, pos, table, layout), acb.rope(x - h * e, pos, table, layout)
    num = ((up - dn).double() * g.double()).sum() / (2 * h)
    ana = (acb.rope(g, pos, table, layout, inverse=True).double() * e.double()).sum()
    bound = 8 * 2.0 ** -24 * float((g.abs().double() * (up.abs() + dn.abs() + x.abs() + e.abs()).double()).sum() / h)
    assert abs(float(num - ana)) <= bound
    back = acb.rope(acb.rope(x, pos, table, layout), pos, table, layout, inverse=True)
    # c^2 + s^2 is 1 within 2^-23 (each a rounded float), and two rotations round six times: 10 * 2^-24 of the pair's size
    assert float((back - x).abs().max()) <= 10 * 2.0 ** -24 * float(x.abs().max()) * 2


def test_far_positions_flag_and_zero(cuda):
    import torch
    x = torch.randn(5, 2, 64).cuda()
    pos = torch.tensor([0, -1, 3, 4, 2 ** 31 - 1], dtype=torch.int32).cuda()
    err = torch.zeros(1, dtype=torch.int32).cuda()
    y = acb.rope(x, pos, _table(4, 64).cuda(), err=err)
    assert int(err) == 2
    assert bool((y[[1, 3, 4]] == 0).all()) and bool((y[[0, 2]] != 0).any(-1).all())
    z = x.clone()
    acb.rope(z, pos, _table(4, 32).cuda(), out=z)  # no flag given
    assert bool((z[[1, 3, 4]] == 0).all())


def test_nan_and_inf_stay_in_their_pair(cuda):
    import torch
    x = torch.ones(1, 1, 64).cuda()
    x[0, 0, 5], x[0, 0, 60] = float("nan"), float("inf")
    y = acb.rope(x, torch.tensor([7], dtype=torch.int32).cuda(), _table(8, 32).cuda(), "half")
    bad = ~torch.isfinite(y[0, 0])
    assert bad.nonzero().flatten().tolist() == [5, 21, 60]


def test_streams_graphs_and_empty(cuda):
    import torch
    x, table = torch.randn(64, 4, 128).cuda(), _table(100, 128).cuda()
    pos = torch.randint(0, 100, (64,), dtype=torch.int32).cuda()
    ref = acb.rope(x, pos, table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = acb.rope(x, pos, table)
    s.synchronize()
    assert torch.equal(y, ref)
    out = torch.zeros_like(x)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        acb.rope(x, pos, table, out=out)
    x.mul_(2)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, acb.rope(x, pos, table))
    assert acb.rope(x[:0], pos[:0], table).shape == (0, 4, 128)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,R", [(3001, 24, 128, 64), (5003, 1, 64, 64), (1100, 9, 192, 16), (2500, 3, 50, 30)])
def test_more_tokens_than_fit_at_once(cuda, kind, layout, T, H, D, R):
    import torch
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, D, generator=g).to(S.torch_type(kind))
    pos = torch.randint(0, 900, (T,), generator=g, dtype=torch.int32)
    table = _table(900, R)
    y = acb.rope(x.cuda(), pos.cuda(), table.cuda(), layout)
    _check(y.float().cpu().numpy(), x.float().numpy(), pos.numpy(), table, layout, False, kind)
    z = x.cuda()
    acb.rope(z, pos.cuda(), table.cuda(), layout, out=z)
    assert torch.equal(z, y)
