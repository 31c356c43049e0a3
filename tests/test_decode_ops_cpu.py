"""The 8-bit cache, rotary positions and draft verification on any host: what their entry points refuse, with which
status, before they touch a device; the frequency tables; what the Python binding refuses."""
import ctypes
import math
import re

import numpy as np
import pytest
import torch

import sixi_attn as sa
from test_asm_hazards import _asm_of, kernels_with_scratch

FAKE = 0x7F0000000000  # aligned addresses far apart; validation never reads through them


def _at(i):
    return FAKE + (i << 40)


def _lib():
    return sa.load_library()


def _view(i, kind, es, ne):
    """A contiguous view of ne elements (ne[0] fastest)."""
    nb = [es]
    for n in ne[:3]:
        nb.append(nb[-1] * n)
    return sa.make_view(_at(i), kind, ne, nb)


def _cache8(D=128, heads=4, blocks=64, n=2):
    c = sa.SixiKv8Cache()
    c.k, c.v, c.k_exp, c.v_exp = _at(1), _at(2), _at(3), _at(4)
    code, exp = (32 * D, 32 * D * blocks, 32 * D * blocks * heads), (1, blocks, blocks * heads)
    c.k_nb = c.v_nb = (ctypes.c_int64 * 3)(*code)
    c.k_exp_nb = c.v_exp_nb = (ctypes.c_int64 * 3)(*exp)
    c.head_dim, c.n_heads, c.n_blocks, c.n = D, heads, blocks, n
    return c


def _set(p, path, value):
    """p.a.b[i] = value for the path "a.b.i"."""
    *head, last = path.split(".")
    for name in head:
        p = p[int(name)] if name.isdigit() else getattr(p, name)
    if last.isdigit():
        p[int(last)] = value
    else:
        setattr(p, last, value)


# ---- store and read-back ----

def _rows(D=128, heads=4, n_rows=16, S=2, kind=sa.TYPE_F32):
    p = sa.SixiKv8RowsParams()
    es = 4 if kind == sa.TYPE_F32 else 2
    p.k, p.v = (_view(i, kind, es, [D, n_rows, heads, S]) for i in (5, 6))
    p.cache = _cache8(D, heads, n=S)
    p.kv_len, p.q_len = _at(7), _at(8)
    return p


def _rows_rc(p, read):
    return _lib().sixi_kv8_rows_validate(ctypes.byref(p), int(read))


@pytest.mark.parametrize("read", [False, True])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", [sa.TYPE_F32, sa.TYPE_F16])
def test_rows_descriptions_pass(read, D, kind):
    assert _rows_rc(_rows(D=D, kind=kind), read) == sa.OK
    p = _rows(D=D, kind=kind)
    p.kv_len = p.q_len = None
    assert _rows_rc(p, read) == sa.OK
    p.cache.n_blocks, p.cache.n, p.page_table, p.page_table_stride = 8, 100, _at(9), 7
    assert _rows_rc(p, read) == sa.OK


ROWS_REFUSED = [
    ({"flags": 1}, sa.E_INVALID_ARGUMENT),
    ({"cache.head_dim": 64}, sa.E_UNSUPPORTED),
    ({"cache.head_dim": 256}, sa.E_INVALID_ARGUMENT),          # blocks of 128 dims overlap then
    ({"cache.k": None}, sa.E_INVALID_ARGUMENT),
    ({"cache.v_exp": None}, sa.E_INVALID_ARGUMENT),
    ({"cache.k": _at(1) + 8}, sa.E_ALIGNMENT),
    ({"cache.v_nb.0": 32 * 128 + 8}, sa.E_ALIGNMENT),
    ({"cache.k_nb.0": -16}, sa.E_INVALID_ARGUMENT),
    ({"cache.k_nb.0": 1 << 31}, sa.E_UNSUPPORTED),
    ({"cache.n_heads": 0}, sa.E_INVALID_ARGUMENT),
    ({"cache.n_heads": 5000}, sa.E_UNSUPPORTED),
    ({"cache.n_blocks": 0}, sa.E_INVALID_ARGUMENT),
    ({"cache.n": 3}, sa.E_INVALID_ARGUMENT),                    # streams of the cache and of the rows
    ({"cache.k_nb.2": 1 << 62, "cache.n": 4, "k.ne.3": 4, "v.ne.3": 4}, sa.E_INTEGER_OVERFLOW),
    ({"k.ne.0": 64}, sa.E_INVALID_ARGUMENT),
    ({"k.ne.2": 2}, sa.E_INVALID_ARGUMENT),
    ({"v.ne.1": 8}, sa.E_INVALID_ARGUMENT),
    ({"k.type": sa.TYPE_Q8_0}, sa.E_INVALID_ARGUMENT),
    ({"k.type": sa.TYPE_BF16}, sa.E_INVALID_ARGUMENT),
    ({"k.nb.0": 8}, sa.E_INVALID_ARGUMENT),
    ({"k.nb.1": -512}, sa.E_INVALID_ARGUMENT),
    ({"k.nb.1": 520}, sa.E_ALIGNMENT),
    ({"v.data": _at(6) + 4}, sa.E_ALIGNMENT),
    ({"v.data": None}, sa.E_INVALID_ARGUMENT),
    ({"kv_len": _at(7) + 2}, sa.E_ALIGNMENT),
    ({"k.data": _at(1) + 4096}, sa.E_INVALID_ARGUMENT),         # rows inside the cache
    ({"page_table": _at(9), "page_table_stride": 4}, sa.E_INVALID_ARGUMENT),   # blocks of a page: 8
    ({"page_table": _at(9), "page_table_stride": 0, "cache.n_blocks": 8}, sa.E_INVALID_ARGUMENT),
    ({"page_table": _at(9) + 1, "page_table_stride": 4, "cache.n_blocks": 8}, sa.E_ALIGNMENT),
]


@pytest.mark.parametrize("change,want", ROWS_REFUSED, ids=lambda c: ",".join(c) if isinstance(c, dict) else "")
@pytest.mark.parametrize("read", [False, True])
def test_rows_refusals(change, want, read):
    p = _rows()
    for path, value in change.items():
        _set(p, path, value)
    assert _rows_rc(p, read) == want
    assert (_lib().sixi_kv8_read if read else _lib().sixi_kv8_write)(ctypes.byref(p)) == want


def test_rows_of_nothing_and_a_null_description():
    for fn in (_lib().sixi_kv8_write, _lib().sixi_kv8_read):
        assert fn(None) == sa.E_INVALID_ARGUMENT
        p = _rows(n_rows=0)
        p.k.data = p.v.data = None
        assert fn(ctypes.byref(p)) == sa.OK  # nothing to do: nothing is launched
    assert _rows_rc(_rows(S=2), False) == sa.OK


def test_written_ranges_are_apart():
    """What a call writes meets nothing else that it reads or writes: the write's cache, the read's rows."""
    p = _rows()
    p.cache.v = _at(1) + 32 * 128        # K's and V's codes interleaved in one range
    assert _rows_rc(p, False) == sa.E_INVALID_ARGUMENT
    p = _rows()
    p.cache.k_exp = p.cache.v_exp
    assert _rows_rc(p, False) == sa.E_INVALID_ARGUMENT
    assert _rows_rc(p, True) == sa.OK
    p = _rows()
    p.v.data = p.k.data
    assert _rows_rc(p, True) == sa.E_INVALID_ARGUMENT
    assert _rows_rc(p, False) == sa.OK
    for read in (False, True):
        p = _rows()
        p.kv_len = p.k.data + 512 if read else p.cache.k + 512
        assert _rows_rc(p, read) == sa.E_INVALID_ARGUMENT
    p = _rows()
    p.k.nb[3] = 0                        # streams that share rows: to be read only
    assert _rows_rc(p, False) == sa.OK
    assert _rows_rc(p, True) == sa.E_INVALID_ARGUMENT


def test_pool_attach_refusals():
    lib = _lib()
    pool = sa.KvPool(100, 2, 8)
    c = _cache8(blocks=8, n=100)
    assert lib.sixi_kv8_pool_attach(None, ctypes.byref(c)) == sa.E_INVALID_ARGUMENT
    assert lib.sixi_kv8_pool_attach(pool.h, None) == sa.E_INVALID_ARGUMENT
    for path, value, want in (("n", 99, sa.E_INVALID_ARGUMENT), ("n_blocks", 4, sa.E_INVALID_ARGUMENT), ("k", None, sa.E_INVALID_ARGUMENT),
                              ("k_nb.0", 32 * 128 + 16, sa.E_INVALID_ARGUMENT),    # pages are copied a head's blocks in one piece
                              ("v_exp_nb.0", 2, sa.E_INVALID_ARGUMENT), ("k_exp_nb.2", 33, sa.E_ALIGNMENT), ("head_dim", 96, sa.E_UNSUPPORTED)):
        c = _cache8(blocks=8, n=100)
        _set(c, path, value)
        assert lib.sixi_kv8_pool_attach(pool.h, ctypes.byref(c)) == want, path
    pool.close()


# ---- attention ----

def _attn(D=128, H=24, heads=4, n_q=16, S=2, blocks=64, kind=sa.TYPE_F16, out=sa.TYPE_F32, mode=sa.MASK_BLOCK_CAUSAL):
    p = sa.SixiKv8AttnParams()
    es, oes = (4 if t == sa.TYPE_F32 else 2 for t in (kind, out))
    p.q = _view(5, kind, es, [D, n_q, H, S])
    p.out = _view(6, out, oes, [D, H, n_q, S])
    p.cache = _cache8(D, heads, blocks, S)
    p.kv_len, p.q_len = _at(7), _at(8)
    p.mask_mode = mode
    if mode == sa.MASK_EXPLICIT:
        p.mask = sa.make_view(_at(9), sa.TYPE_F16, [blocks * 32, n_q, 1, S], [2, blocks * 64, blocks * 64 * n_q, blocks * 64 * n_q])
    p.scale = D ** -0.5
    return p


def _attn_rc(p):
    return _lib().sixi_kv8_attn_validate(ctypes.byref(p))


def _bytes(p, name="sixi_kv8_attn_workspace_bytes"):
    n = ctypes.c_size_t(0)
    assert getattr(_lib(), name)(ctypes.byref(p), ctypes.byref(n)) == sa.OK
    return n.value


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("mode", [sa.MASK_NONE, sa.MASK_BLOCK_CAUSAL, sa.MASK_EXPLICIT])
@pytest.mark.parametrize("n_q", [1, 5, 16, 200])
def test_attention_descriptions_pass_and_size_a_workspace(D, mode, n_q):
    p = _attn(D=D, mode=mode, n_q=n_q)
    assert _attn_rc(p) == sa.OK
    n = _bytes(p)
    assert n >= 256 and n % 256 == 0
    p.kv_len = _at(7) + 4          # the lengths' values do not matter to it, nor does a workspace
    p.workspace, p.workspace_bytes = _at(20), 1
    assert _bytes(p) == n


def test_workspace_is_bounded_however_long_the_cache():
    """Pieces are cut to the places there are: the scratch does not grow with the cells or the streams' tiles."""
    sizes = [_bytes(_attn(n_q=1, blocks=b)) for b in (64, 4096, 1 << 20)]
    assert sizes[0] == sizes[1] == sizes[2]
    many = _attn(n_q=4096, blocks=4096)
    assert _bytes(many) < 1 << 27
    many.q_len = None              # every row is there: tiles enough for all places, nothing to join
    assert _bytes(many) == 256


ATTN_REFUSED = [
    ({"flags": 1}, sa.E_INVALID_ARGUMENT),
    ({"q.data": None}, sa.E_INVALID_ARGUMENT),
    ({"out.data": None}, sa.E_INVALID_ARGUMENT),
    ({"q.type": sa.TYPE_Q8_0}, sa.E_UNSUPPORTED),
    ({"out.type": sa.TYPE_BF16}, sa.E_UNSUPPORTED),
    ({"q.ne.1": 0}, sa.E_INVALID_ARGUMENT),
    ({"q.ne.2": 23, "out.ne.1": 23}, sa.E_INVALID_ARGUMENT),     # heads that kv-heads do not divide
    ({"q.ne.0": 256}, sa.E_INVALID_ARGUMENT),
    ({"out.ne.2": 15}, sa.E_INVALID_ARGUMENT),
    ({"cache.n": 1}, sa.E_INVALID_ARGUMENT),
    ({"cache.head_dim": 192}, sa.E_UNSUPPORTED),
    ({"q.nb.0": 4}, sa.E_INVALID_ARGUMENT),
    ({"q.nb.1": 264}, sa.E_ALIGNMENT),
    ({"out.data": _at(6) + 8}, sa.E_ALIGNMENT),
    ({"q_len": _at(8) + 1}, sa.E_ALIGNMENT),
    ({"out.nb.2": 0}, sa.E_INVALID_ARGUMENT),
    ({"out.data": _at(5)}, sa.E_INVALID_ARGUMENT),
    ({"out.data": _at(2)}, sa.E_INVALID_ARGUMENT),
    ({"kv_len": _at(6) + 64}, sa.E_INVALID_ARGUMENT),
    ({"mask_mode": 3}, sa.E_INVALID_ARGUMENT),
    ({"mask_mode": sa.MASK_EXPLICIT}, sa.E_INVALID_ARGUMENT),    # and no mask
    ({"kv_len": None}, sa.E_INVALID_ARGUMENT),                   # block-causal without lengths
    ({"scale": math.inf}, sa.E_INVALID_ARGUMENT),
    ({"scale": math.nan}, sa.E_INVALID_ARGUMENT),
    ({"scale": 2.0 ** 41}, sa.E_INVALID_ARGUMENT),
    ({"cache.n_blocks": 0}, sa.E_INVALID_ARGUMENT),
    ({"page_table": _at(10), "page_table_stride": 2}, sa.E_INVALID_ARGUMENT),
    ({"page_table": _at(10), "page_table_stride": 1 << 40, "cache.n_blocks": 8}, sa.E_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("change,want", ATTN_REFUSED, ids=lambda c: ",".join(c) if isinstance(c, dict) else "")
def test_attention_refusals(change, want):
    p = _attn()
    for path, value in change.items():
        _set(p, path, value)
    assert _attn_rc(p) == want
    p.workspace, p.workspace_bytes = _at(20), 1 << 30
    assert _lib().sixi_kv8_attn(ctypes.byref(p)) == want


@pytest.mark.parametrize("change,want", [
    ({"mask.type": sa.TYPE_F32}, sa.E_INVALID_ARGUMENT),
    ({"mask.ne.0": 2047}, sa.E_INVALID_ARGUMENT),
    ({"mask.ne.1": 15}, sa.E_INVALID_ARGUMENT),
    ({"mask.ne.2": 24}, sa.E_INVALID_ARGUMENT),
    ({"mask.ne.3": 3}, sa.E_INVALID_ARGUMENT),
    ({"mask.nb.1": 4097}, sa.E_ALIGNMENT),
    ({"mask.data": _at(9) + 1}, sa.E_ALIGNMENT),
    ({"mask.data": _at(6)}, sa.E_INVALID_ARGUMENT),
], ids=lambda c: ",".join(c) if isinstance(c, dict) else "")
def test_mask_refusals(change, want):
    p = _attn(mode=sa.MASK_EXPLICIT)
    assert _attn_rc(p) == sa.OK
    for path, value in change.items():
        _set(p, path, value)
    assert _attn_rc(p) == want


def test_attention_limits():
    assert _attn_rc(_attn(S=512, n_q=1)) == sa.OK
    assert _attn_rc(_attn(S=513, n_q=1)) == sa.E_UNSUPPORTED
    assert _attn_rc(_attn(n_q=2048, blocks=64)) == sa.OK
    assert _attn_rc(_attn(n_q=2049, blocks=64)) == sa.E_INVALID_ARGUMENT   # more rows than cells
    assert _attn_rc(_attn(H=4096, heads=1, n_q=1 << 17, S=1, blocks=1 << 13)) == sa.E_UNSUPPORTED


def test_attention_workspace_refusals():
    """Nothing is launched: the workspace is missing, misaligned, too small, or what the call reads or writes."""
    lib = _lib()
    p = _attn()
    n = _bytes(p)
    for at, size, want in ((None, n, sa.E_INVALID_ARGUMENT), (_at(20) + 128, n, sa.E_ALIGNMENT), (_at(20), n - 1, sa.E_OUT_OF_BOUNDS),
                           (_at(5), n, sa.E_INVALID_ARGUMENT), (_at(6) + 256, n, sa.E_INVALID_ARGUMENT), (_at(1), n, sa.E_INVALID_ARGUMENT),
                           (_at(4) - 256, n, sa.E_INVALID_ARGUMENT), (_at(7) - 256, n, sa.E_INVALID_ARGUMENT)):
        p.workspace, p.workspace_bytes = at, size
        assert lib.sixi_kv8_attn(ctypes.byref(p)) == want, (at, size)
    assert lib.sixi_kv8_attn(None) == sa.E_INVALID_ARGUMENT
    assert lib.sixi_kv8_attn_workspace_bytes(ctypes.byref(p), None) == sa.E_INVALID_ARGUMENT


# ---- rotary positions ----

def _rope(D=128, H=24, heads=4, n=16, S=2, kind=sa.TYPE_F32, out=sa.TYPE_F16, rot=64):
    p = sa.SixiQkRopeParams()
    es, oes = (4 if t == sa.TYPE_F32 else 2 for t in (kind, out))
    p.q, p.k = _view(1, kind, es, [D, H, n, S]), _view(2, kind, es, [D, heads, n, S])
    p.q_out, p.k_out = _view(3, out, oes, [D, H, n, S]), _view(4, out, oes, [D, heads, n, S])
    p.freqs, p.q_norm, p.k_norm = _at(5), _at(6), _at(7)
    p.eps, p.mscale, p.n_rot, p.layout = 1e-6, 1.0, rot, sa.ROPE_HALF
    p.kv_len, p.q_len = _at(8), _at(9)
    return p


def _rope_rc(p):
    return _lib().sixi_qk_rope_validate(ctypes.byref(p))


def test_rope_descriptions_pass():
    assert _rope_rc(_rope()) == sa.OK
    p = _rope(kind=sa.TYPE_F16)
    p.q_out, p.k_out = p.q, p.k                       # in place
    assert _rope_rc(p) == sa.OK
    p.k = p.k_out = sa.make_view(None, sa.TYPE_F32, [0] * 4, [0] * 4)
    p.k_norm = None
    assert _rope_rc(p) == sa.OK                       # no K
    p.q_norm = None
    p.flags, p.n_rot = sa.ROPE_INVERSE, 128
    assert _rope_rc(p) == sa.OK
    p.n_rot, p.freqs = 0, None
    assert _rope_rc(p) == sa.OK


ROPE_REFUSED = [
    ({"flags": 2}, sa.E_INVALID_ARGUMENT),
    ({"flags": sa.ROPE_INVERSE}, sa.E_INVALID_ARGUMENT),                 # with norm weights
    ({"layout": 2}, sa.E_INVALID_ARGUMENT),
    ({"n_rot": -16}, sa.E_INVALID_ARGUMENT),
    ({"n_rot": 24}, sa.E_INVALID_ARGUMENT),
    ({"n_rot": 144}, sa.E_INVALID_ARGUMENT),
    ({"freqs": None}, sa.E_INVALID_ARGUMENT),
    ({"freqs": _at(5) + 4}, sa.E_ALIGNMENT),
    ({"q_norm": _at(6) + 4}, sa.E_ALIGNMENT),
    ({"k_norm": None}, sa.E_INVALID_ARGUMENT),
    ({"q_norm": None}, sa.E_INVALID_ARGUMENT),
    ({"eps": math.nan}, sa.E_INVALID_ARGUMENT),
    ({"eps": -1.0}, sa.E_INVALID_ARGUMENT),
    ({"mscale": math.inf}, sa.E_INVALID_ARGUMENT),
    ({"pos": _at(10), "pos_stride": -1}, sa.E_INVALID_ARGUMENT),
    ({"pos": _at(10), "pos_stride": 1 << 40}, sa.E_INTEGER_OVERFLOW),
    ({"pos": _at(10) + 2}, sa.E_ALIGNMENT),
    ({"q.type": sa.TYPE_BF16}, sa.E_INVALID_ARGUMENT),
    ({"q.data": None}, sa.E_INVALID_ARGUMENT),
    ({"k_out.data": None}, sa.E_INVALID_ARGUMENT),
    ({"q.nb.1": 520}, sa.E_ALIGNMENT),
    ({"q_out.nb.1": 0}, sa.E_INVALID_ARGUMENT),
    ({"q_out.ne.2": 15}, sa.E_INVALID_ARGUMENT),
    ({"k.ne.2": 15, "k_out.ne.2": 15}, sa.E_INVALID_ARGUMENT),
    ({"q_out.data": _at(1)}, sa.E_INVALID_ARGUMENT),                     # over the input, in another type
    ({"q_out.data": _at(2)}, sa.E_INVALID_ARGUMENT),
    ({"k_out.data": _at(3) + 4096}, sa.E_INVALID_ARGUMENT),
    ({"q_len": _at(3) + 64}, sa.E_INVALID_ARGUMENT),
    ({"freqs": _at(4) + 64}, sa.E_INVALID_ARGUMENT),
    ({"k_norm": _at(3) + 64}, sa.E_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("change,want", ROPE_REFUSED, ids=lambda c: ",".join(c) if isinstance(c, dict) else "")
def test_rope_refusals(change, want):
    p = _rope()
    for path, value in change.items():
        _set(p, path, value)
    assert _rope_rc(p) == want
    assert _lib().sixi_qk_rope(ctypes.byref(p)) == want


def test_rope_limits():
    for D in (8, 24, 272):
        assert _rope_rc(_rope(D=D, rot=0)) == sa.E_UNSUPPORTED
    assert _rope_rc(_rope(n=1 << 23, S=1, H=1, heads=1)) == sa.OK
    assert _rope_rc(_rope(n=(1 << 23) + 1, S=1, H=1, heads=1)) == sa.E_UNSUPPORTED
    assert _rope_rc(_rope(H=65536)) == sa.E_UNSUPPORTED
    assert _rope_rc(_rope(S=65536, n=1)) == sa.E_UNSUPPORTED
    assert _lib().sixi_qk_rope(None) == sa.E_INVALID_ARGUMENT
    p = _rope(n=0)
    assert _lib().sixi_qk_rope(ctypes.byref(p)) == sa.OK                 # nothing to do


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 1e7), (128, 10000.0)])
@pytest.mark.parametrize("scaling,factor,trained", [(sa.ROPE_SCALE_NONE, 3.0, 0), (sa.ROPE_SCALE_LINEAR, 3.0, 0),
                                                   (sa.ROPE_SCALE_YARN, 4.0, 4096), (sa.ROPE_SCALE_YARN, 16.0, 32768),
                                                   (sa.ROPE_SCALE_YARN, 1.0, 16)])
def test_rope_frequencies(rot, base, scaling, factor, trained):
    """The tables against their formulas: base^(-2i/rot), stretched by the share of each pair's turns over the trained
    positions.  powers of 64 bits: within 2^-48 of each."""
    f, m = sa.rope_frequencies(rot, base, scaling, factor, trained, device="cpu")
    i = np.arange(rot // 2)
    want = base ** (-2.0 * i / rot)
    if scaling == sa.ROPE_SCALE_LINEAR:
        want = want / factor
    if scaling == sa.ROPE_SCALE_YARN:
        def pair(turns):
            return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(0.0, math.floor(pair(32.0))), min(rot - 1.0, math.ceil(pair(1.0)))
        share = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        want = want * (1 - share) + want / factor * share
    assert f.dtype == torch.float64 and f.shape == (rot // 2,)
    assert np.allclose(f.numpy(), want, rtol=2.0 ** -48, atol=0)
    yarn = scaling == sa.ROPE_SCALE_YARN
    assert m == (np.float32(0.1 * math.log(factor) + 1.0) if yarn else 1.0)
    if yarn and rot == 128 and factor > 1:
        assert f[0] == 1.0 and abs(float(f[-1]) / want[-1] - 1) < 1e-12      # the fastest pair as trained


def test_rope_frequencies_refusals():
    for args in ((3, 1e4), (-2, 1e4), (64, 1.0), (64, math.nan), (64, 1e4, 3), (64, 1e4, sa.ROPE_SCALE_LINEAR, 0.5),
                 (64, 1e4, sa.ROPE_SCALE_LINEAR, math.inf), (64, 1e4, sa.ROPE_SCALE_YARN, 4.0, 0),
                 (64, 1e4, sa.ROPE_SCALE_YARN, 4.0, 4096, 1.0, 1.0), (64, 1e4, sa.ROPE_SCALE_YARN, 4.0, 4096, 32.0, 0.0)):
        with pytest.raises(sa.SixiAttnError) as e:
            sa.rope_frequencies(*args, device="cpu")
        assert e.value.code == sa.E_INVALID_ARGUMENT, args


# ---- draft verification ----

def _draft(V=1000, n=5, S=3, kind=sa.TYPE_F32, probs=True):
    p = sa.SixiDraftParams()
    es = 4 if kind == sa.TYPE_F32 else 2
    p.logits = _view(1, kind, es, [V, n, S, 1])
    if probs:
        p.draft_probs = _view(2, sa.TYPE_F32, 4, [V, n - 1, S, 1])
    p.draft, p.draft_stride, p.u, p.u_stride = _at(3), n - 1, _at(4), n - 1
    p.u_next, p.temperature, p.q_len, p.keep, p.token = _at(5), _at(6), _at(7), _at(8), _at(9)
    return p


def _draft_rc(p):
    return _lib().sixi_draft_validate(ctypes.byref(p))


@pytest.mark.parametrize("kind", [sa.TYPE_F32, sa.TYPE_F16, sa.TYPE_BF16])
@pytest.mark.parametrize("V,n,S", [(1, 1, 1), (1000, 5, 3), (248320, 17, 64)])
def test_draft_descriptions_pass_and_size_a_workspace(kind, V, n, S):
    p = _draft(V, n, S, kind, probs=n > 1)
    assert _draft_rc(p) == sa.OK
    got = _bytes(p, "sixi_draft_workspace_bytes")
    assert got >= 256 and got % 256 == 0
    p.temperature = p.q_len = None
    p.draft_probs.data = None
    if n == 1:
        p.draft = p.u = None
    assert _draft_rc(p) == sa.OK and _bytes(p, "sixi_draft_workspace_bytes") == got


DRAFT_REFUSED = [
    ({"flags": 1}, sa.E_INVALID_ARGUMENT),
    ({"logits.data": None}, sa.E_INVALID_ARGUMENT),
    ({"logits.type": sa.TYPE_Q8_0}, sa.E_INVALID_ARGUMENT),
    ({"logits.nb.0": 8}, sa.E_INVALID_ARGUMENT),
    ({"logits.ne.0": 0}, sa.E_INVALID_ARGUMENT),
    ({"logits.ne.1": 0}, sa.E_INVALID_ARGUMENT),
    ({"logits.ne.3": 2}, sa.E_INVALID_ARGUMENT),
    ({"logits.nb.1": 4002}, sa.E_ALIGNMENT),
    ({"logits.nb.2": -4}, sa.E_INVALID_ARGUMENT),
    ({"logits.nb.2": (1 << 62) + 4}, sa.E_INTEGER_OVERFLOW),
    ({"logits.data": _at(1) + 2}, sa.E_ALIGNMENT),
    ({"draft_probs.ne.0": 999}, sa.E_INVALID_ARGUMENT),
    ({"draft_probs.ne.1": 3}, sa.E_INVALID_ARGUMENT),
    ({"draft_probs.type": 99}, sa.E_INVALID_ARGUMENT),
    ({"draft": None}, sa.E_INVALID_ARGUMENT),
    ({"u": None}, sa.E_INVALID_ARGUMENT),
    ({"u_next": None}, sa.E_INVALID_ARGUMENT),
    ({"keep": None}, sa.E_INVALID_ARGUMENT),
    ({"token": None}, sa.E_INVALID_ARGUMENT),
    ({"token": _at(9) + 2}, sa.E_ALIGNMENT),
    ({"draft_stride": -1}, sa.E_INVALID_ARGUMENT),
    ({"u_stride": 1 << 40}, sa.E_INTEGER_OVERFLOW),
    ({"keep": _at(9) + 4}, sa.E_INVALID_ARGUMENT),
    ({"keep": _at(7)}, sa.E_INVALID_ARGUMENT),
    ({"token": _at(3) + 8}, sa.E_INVALID_ARGUMENT),
    ({"token": _at(2) + 400}, sa.E_INVALID_ARGUMENT),
    ({"logits.ne.1": 1025, "draft_probs.data": None}, sa.E_UNSUPPORTED),
    ({"logits.ne.2": 65536}, sa.E_UNSUPPORTED),
]


@pytest.mark.parametrize("change,want", DRAFT_REFUSED, ids=lambda c: ",".join(c) if isinstance(c, dict) else "")
def test_draft_refusals(change, want):
    p = _draft()
    for path, value in change.items():
        _set(p, path, value)
    assert _draft_rc(p) == want
    p.workspace, p.workspace_bytes = _at(20), 1 << 40
    assert _lib().sixi_draft_verify(ctypes.byref(p)) == want


def test_draft_workspace_refusals():
    lib = _lib()
    p = _draft()
    n = _bytes(p, "sixi_draft_workspace_bytes")
    for at, size, want in ((None, n, sa.E_INVALID_ARGUMENT), (_at(20) + 64, n, sa.E_ALIGNMENT), (_at(20), n - 1, sa.E_OUT_OF_BOUNDS),
                           *((_at(i), n, sa.E_INVALID_ARGUMENT) for i in range(1, 10))):
        p.workspace, p.workspace_bytes = at, size
        assert lib.sixi_draft_verify(ctypes.byref(p)) == want, (at, size)
    assert lib.sixi_draft_verify(None) == sa.E_INVALID_ARGUMENT
    p = _draft(S=0)
    p.logits.data = p.u_next = p.keep = p.token = p.draft = p.u = None
    p.draft_probs.data = None
    assert lib.sixi_draft_verify(ctypes.byref(p)) == sa.OK               # no streams: nothing to do


# ---- the Python binding ----

def test_binding_refuses_host_tensors_and_wrong_types():
    x = torch.zeros((1, 4, 2, 128))
    f = torch.zeros(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="GPU"):
        sa.qk_rope(x, x, f)
    i8 = [torch.zeros(s, dtype=torch.int8) for s in ((1, 2, 2, 8, 32, 16), (1, 2, 2), (1, 2, 2, 128, 32), (1, 2, 2))]
    with pytest.raises(ValueError, match="GPU"):
        sa.Kv8Cache(*i8)
    with pytest.raises(ValueError, match="int8"):
        sa.Kv8Cache(*[t.float() for t in i8])
    with pytest.raises(ValueError, match="expected k"):
        sa.Kv8Cache(i8[2], i8[1], i8[0], i8[3])
    with pytest.raises(ValueError, match="head dim"):
        sa.Kv8Cache(i8[0][:, :, :, :4], i8[1], i8[2][:, :, :, :64], i8[3])
    with pytest.raises(ValueError, match="contiguous"):
        sa.Kv8Cache(i8[0].transpose(3, 4).contiguous().transpose(3, 4), i8[1], i8[2], i8[3])
    with pytest.raises(ValueError, match="multiple of 32"):
        sa.Kv8Cache.empty(1, 100, 2, 128, device="cpu")


# ---- the kernels as built ----

@pytest.mark.parametrize("src", ["kv8_store.hip", "kv8_attn.hip", "rope.hip", "draft_verify.hip"])
def test_kernels_use_no_scratch_and_no_packed_f32(src, tmp_path_factory):
    asm = _asm_of(src, tmp_path_factory)
    assert asm.count(".private_segment_fixed_size:") > 0
    assert not kernels_with_scratch(asm)
    assert not re.search(r"v_pk_(add|mul|fma)_f32", asm)
