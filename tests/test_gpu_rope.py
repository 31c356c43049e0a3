"""Rotary positions on the GPU (sixi_qk_rope) against the definition in 64 bits.

The bound of a rotated element with its pair (x0, x1), r = |x0| + |x1|: cos and sin are f32 values of an angle reduced
in 64 bits (the remainder rounded to f32, 2^-24 of at most half a turn: pi 2^-24 radians; the functions themselves a
few units of 2^-24), times mscale, and the two products' sum: within 16 * 2^-24 of mscale * r.  The norm's factor is an
f32 sum of D squares, a square root and a division: D/8 serial sums in a lane and a tree, within 16 * 2^-24 more.
Plus half a step of the output's type."""
import sys

import numpy as np
import pytest
import torch

import sixi_attn as sa

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _say(msg):
    print(f"[gpu-case] {msg}", file=sys.stderr, flush=True)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _reference(x, freqs, pos, layout, mscale, norm, inverse=False):
    """(values, size): x [S, n, H, D] float64, pos [S, n]; `size` is what the bound is relative to."""
    x = x.copy()
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * norm
    r = 2 * len(freqs)
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == sa.ROPE_HALF else (x[..., 0:r:2], x[..., 1:r:2])
    t = pos[..., None, None].astype(np.float64) * freqs * (-1 if inverse else 1)
    y0, y1 = mscale * (a * np.cos(t) - b * np.sin(t)), mscale * (b * np.cos(t) + a * np.sin(t))
    big = mscale * (np.abs(a) + np.abs(b))
    out, size = x.copy(), np.abs(x)
    if layout == sa.ROPE_HALF:
        out[..., :r // 2], out[..., r // 2:r] = y0, y1
        size[..., :r // 2] = size[..., r // 2:r] = big
    else:
        out[..., 0:r:2], out[..., 1:r:2] = y0, y1
        size[..., 0:r:2] = size[..., 1:r:2] = big
    return out, size


def _check(got, want, size, live, what):
    g = got.cpu().double().numpy()
    half = 2.0 ** -11 if got.dtype == torch.float16 else 2.0 ** -24
    tol = 32 * 2.0 ** -24 * size + half * np.abs(want) * (1 + 1e-3) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    off = (np.abs(g - want) / tol)[live]
    _say(f"  {what}: worst {off.max() if off.size else 0:.3f} of the bound")
    assert (off <= 1).all()
    assert np.isnan(g[~live]).all()


CASES = [
    # streams, rows, H, heads, D, n_rot, kv_len, q_len
    (1, 1, 24, 4, 256, 64, [9000], None),
    (2, 5, 24, 4, 128, 128, [0, 131071], [5, 3]),
    (3, 2, 8, 8, 64, 32, [7, 1, 0], [2, 0, 1]),
    (1, 33, 5, 1, 96, 48, [1 << 20], None),
    (1, 3, 4, 2, 80, 16, [100], None),
    (2, 4, 7, 3, 256, 256, [2000000000, 5], None),
    (1, 2, 3, 1, 16, 16, [3], None),
    (1, 2, 3, 1, 128, 0, [3], None),
]


@pytest.mark.parametrize("s,n,H,heads,d,rot,kv,ql", CASES)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float32, torch.float16), (torch.float16, torch.float16)])
def test_rope(s, n, H, heads, d, rot, kv, ql, layout, norm, types):
    _say(f"rope s={s} n={n} H={H} heads={heads} d={d} rot={rot} kv={kv} ql={ql} layout={layout} norm={norm} types={types}")
    gen = torch.Generator().manual_seed(d + rot + n)
    q, k = (torch.randn((s, n, h, d), generator=gen).to(types[0]) for h in (H, heads))
    wq, wk = (1 + 0.3 * torch.randn(d, generator=gen) for _ in range(2)) if norm else (None, None)
    freqs, m = sa.rope_frequencies(rot, 1e6, sa.ROPE_SCALE_YARN, 4.0, 4096) if rot else (torch.zeros(0, dtype=torch.float64, device="cuda"), 1.0)
    qo, ko = (torch.full(x.shape, float("nan"), dtype=types[1], device="cuda") for x in (q, k))
    sa.qk_rope(q.cuda(), k.cuda(), freqs, qo, ko, kv_len=_i32(kv), q_len=None if ql is None else _i32(ql), layout=layout,
               mscale=m, q_norm=None if wq is None else wq.cuda(), k_norm=None if wk is None else wk.cuda(), eps=EPS)
    pos = np.asarray(kv)[:, None] + np.arange(n)
    live = np.arange(n) < np.asarray([n] * s if ql is None else ql)[:, None]
    for got, x, w, what in ((qo, q, wq, "q"), (ko, k, wk, "k")):
        want, size = _reference(x.double().numpy(), freqs.cpu().numpy(), pos, layout, m, None if w is None else w.double().numpy())
        _check(got, want, size, live, what)


def test_rope_in_place_positions_and_strides():
    """In place on the halves of a wider tensor, positions given (a tree's), no K; then turned back."""
    gen = torch.Generator().manual_seed(1)
    s, n, H, d, rot = 2, 6, 4, 128, 64
    wide = torch.randn((s, n, H, 2 * d), generator=gen).cuda()
    before = wide.clone()
    pos = torch.tensor([[10, 11, 11, 12, 12, 12, 0], [0, 70000, 3, 3, 4, 5, 0]], dtype=torch.int32, device="cuda")[:, :n]
    freqs, m = sa.rope_frequencies(rot, 1e4)
    sa.qk_rope(wide[..., :d], None, freqs, pos=pos)
    want, size = _reference(before[..., :d].double().cpu().numpy(), freqs.cpu().numpy(), pos.cpu().numpy(), 0, 1.0, None)
    _check(wide[..., :d], want, size, np.ones((s, n), bool), "in place")
    assert torch.equal(wide[..., d:], before[..., d:])
    sa.qk_rope(wide[..., :d], None, freqs, pos=pos, inverse=True)
    # two rotations, each within its bound
    assert float((wide - before).abs().max()) <= 4 * 32 * 2.0 ** -24 * 2 * float(before.abs().max())


def test_rope_gradient_is_the_inverse_rotation():
    """The rotation's transpose: <R x, g> = <x, R^-1 g> for mscale 1, and against differences of the formula."""
    gen = torch.Generator().manual_seed(2)
    x, g = (torch.randn((1, 3, 2, 64), generator=gen) for _ in range(2))
    freqs, _ = sa.rope_frequencies(64, 1e4, sa.ROPE_SCALE_LINEAR, 2.0)
    kv = _i32([1000])
    for layout in (0, 1):
        got = torch.empty_like(g, device="cuda")
        sa.qk_rope(g.cuda(), None, freqs, got, kv_len=kv, layout=layout, inverse=True)
        pos, f = 1000 + np.arange(3)[None], freqs.cpu().numpy()
        grad = np.zeros(x.shape)
        for i in range(64):  # the map is linear: differences are exact up to rounding
            e = np.zeros(x.shape)
            e[..., i] = 0.5
            up, _ = _reference(x.double().numpy() + e, f, pos, layout, 1.0, None)
            down, _ = _reference(x.double().numpy() - e, f, pos, layout, 1.0, None)
            grad[..., i] = ((up - down) * g.double().numpy()).sum(-1)
        assert np.abs(got.cpu().double().numpy() - grad).max() <= 32 * 2.0 ** -24 * 2 * float(g.abs().max()) + 1e-9


def test_rope_rows_past_32_bits():
    """Rows three GiB apart, in place."""
    d, step = 64, 3 << 28                                 # in f32 elements
    wide = torch.empty(2 * step + 2 * d, device="cuda")
    q = wide.as_strided((1, 3, 2, d), (wide.numel(), step, d, 1))
    q.copy_(torch.randn((1, 3, 2, d), generator=torch.Generator().manual_seed(5)))
    before = q.clone()
    freqs, _ = sa.rope_frequencies(32, 1e4)
    sa.qk_rope(q, None, freqs, kv_len=_i32([77]))
    want, size = _reference(before.double().cpu().numpy(), freqs.cpu().numpy(), 77 + np.arange(3)[None], 0, 1.0, None)
    _check(q, want, size, np.ones((1, 3), bool), "far rows")


def test_rope_writes_rows_of_their_own_only():
    """Every second row of a buffer: the rows between stay."""
    q = torch.randn((1, 4, 3, 128), device="cuda")
    buf = torch.full((1, 8, 3, 128), 9.0, device="cuda", dtype=torch.float16)
    freqs, _ = sa.rope_frequencies(128, 1e4)
    sa.qk_rope(q, None, freqs, buf[:, ::2], kv_len=_i32([5]))
    assert bool((buf[:, 1::2] == 9).all()) and not bool((buf[:, ::2] == 9).all(-1).any())


def test_rope_many_rows_and_streams():
    gen = torch.Generator().manual_seed(3)
    q, k = torch.randn((5, 700, 6, 128), generator=gen), torch.randn((5, 700, 2, 128), generator=gen)
    freqs, _ = sa.rope_frequencies(128, 1e7)
    qo, ko = torch.empty_like(q, device="cuda"), torch.empty_like(k, device="cuda")
    kv = [0, 5, 1000, 100000, 32768]
    sa.qk_rope(q.cuda(), k.cuda(), freqs, qo, ko, kv_len=_i32(kv))
    pos = np.asarray(kv)[:, None] + np.arange(700)
    for got, x in ((qo, q), (ko, k)):
        want, size = _reference(x.double().numpy(), freqs.cpu().numpy(), pos, 0, 1.0, None)
        _check(got, want, size, np.ones((5, 700), bool), "rows")
