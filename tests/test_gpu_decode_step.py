"""Rotary positions, the 8-bit cache, its attention and the draft verification as a decoder runs them: step after step,
eagerly, on another stream, and as captured graphs that share their handles.

Every stage is compared with its 64-bit restatement on what the stage before it left: the cache bit for bit, rejected
tokens' cells included."""
import sys

import numpy as np
import pytest
import torch

import sixi_attn as sa
from kv8_ref import PAGE, Cells, attention
from test_gpu_draft import _rule
from test_gpu_kv8 import _cells_of
from test_gpu_rope import _check, _reference

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", file=sys.stderr, flush=True)


class Decoder:
    """One layer whose attention output is the logits (V = H * D): buffers for blocks of up to n rows, the cache, and the
    lengths, which the steps move on."""

    def __init__(self, S, n, H, heads, D, cells, paged=False, seed=0):
        self.S, self.n, self.H, self.heads, self.D, self.cells = S, n, H, heads, D, cells
        gen = self.gen = torch.Generator(device="cuda").manual_seed(seed)

        def randn(*shape, dtype=torch.float32):
            return torch.randn(shape, generator=gen, device="cuda").to(dtype)

        self.q, self.k, self.v = randn(S, n, H, D), randn(S, n, heads, D), randn(S, n, heads, D, dtype=torch.float16)
        self.q_rot, self.k_rot = torch.zeros_like(self.q, dtype=torch.float16), torch.zeros_like(self.k, dtype=torch.float16)
        self.out = torch.zeros((S, n, H, D), device="cuda")
        self.freqs, self.mscale = sa.rope_frequencies(D // 2, 1e4, sa.ROPE_SCALE_YARN, 4.0, 64)
        self.table = None
        if paged:
            per = cells // PAGE
            self.cache = sa.Kv8Cache.empty(S * per + 1, PAGE, heads, D)
            self.table = torch.randperm(S * per + 1, generator=gen, device="cuda")[:S * per].to(torch.int32).reshape(S, per)
        else:
            self.cache = sa.Kv8Cache.empty(S, cells, heads, D)
        self.kv_len = torch.zeros(S, dtype=torch.int32, device="cuda")
        self.q_len = torch.full((S,), n, dtype=torch.int32, device="cuda")
        self.keep, self.token = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(2))
        self.draft = torch.zeros((S, max(n - 1, 1)), dtype=torch.int32, device="cuda")
        self.u, self.u_next = torch.zeros((S, max(n - 1, 1)), device="cuda"), torch.zeros(S, device="cuda")
        self.heat = torch.full((S,), 0.05, device="cuda")
        self.attend, self.judge = sa.Kv8Attention(), sa.DraftVerify()

    def feed(self):
        """New inputs in the same buffers."""
        def normal(t):
            t.copy_(torch.randn(t.shape, generator=self.gen, device="cuda"))

        for t in (self.q, self.k, self.v):
            normal(t)
        self.k.mul_(torch.exp2(torch.randint(-3, 4, (1,), generator=self.gen, device="cuda").float()))
        self.q_len.copy_(torch.randint(1, self.n + 1, (self.S,), generator=self.gen, device="cuda"))
        self.draft.copy_(torch.randint(0, self.H * self.D, self.draft.shape, generator=self.gen, device="cuda"))
        self.u.copy_(torch.rand(self.u.shape, generator=self.gen, device="cuda") * 2e-3)
        self.u.mul_(torch.randint(0, 2, self.u.shape, generator=self.gen, device="cuda"))   # (every other token stays)
        self.u_next.copy_(torch.rand(self.S, generator=self.gen, device="cuda"))

    def cache_step(self, rows=None):
        """Rotation, store and attention of the first `rows` rows (all)."""
        r = slice(0, self.n if rows is None else rows)
        args = dict(kv_len=self.kv_len, q_len=self.q_len)
        sa.qk_rope(self.q[:, r], self.k[:, r], self.freqs, self.q_rot[:, r], self.k_rot[:, r], mscale=self.mscale, **args)
        sa.kv8_write(self.k_rot[:, r], self.v[:, r], self.cache, page_table=self.table, **args)
        self.attend(self.q_rot[:, r], self.cache, self.out[:, r], page_table=self.table, **args)

    def step(self, rows=None):
        n = self.n if rows is None else rows
        self.cache_step(rows)
        self.judge(self.out[:, :n].flatten(2), self.draft, self.u, self.u_next, self.keep, self.token, q_len=self.q_len,
                   temperature=self.heat)
        self.kv_len.add_(self.keep)

    def state(self):
        c = self.cache
        return [c.k, c.k_exp, c.v, c.v_exp, self.kv_len, self.out, self.keep, self.token]


@pytest.mark.parametrize("S,n,H,heads,D,paged,steps", [(3, 5, 8, 2, 128, False, 8), (2, 9, 6, 1, 256, True, 6), (1, 1, 4, 4, 128, True, 40)])
def test_steps_against_the_formulas(S, n, H, heads, D, paged, steps):
    cells = 512
    d = Decoder(S, n, H, heads, D, cells, paged, seed=S + n)
    k_ref, v_ref = Cells(S, cells, heads, D), Cells(S, cells, heads, D)
    # a prompt of different lengths in front, through the same calls
    p = Decoder(S, 200, H, heads, D, cells, seed=9)
    p.cache, p.table = d.cache, d.table
    p.q_len.copy_(torch.tensor([200, 31, 64][:S], dtype=torch.int32))
    moved = False
    for i in range(steps + 1):
        x = p if i == 0 else d
        _say(f"decode step {i}: S={S} rows={x.n} H={H} heads={heads} D={D} paged={paged}")
        if i > 0:
            d.feed()
        first, rows = d.kv_len.tolist(), x.q_len.tolist()
        x.kv_len.copy_(d.kv_len)
        if i == 0:
            x.cache_step()
        else:
            x.step()
        live = np.arange(x.n) < np.asarray(rows)[:, None]
        pos = np.asarray(first)[:, None] + np.arange(x.n)
        for got, src in ((x.q_rot, x.q), (x.k_rot, x.k)):
            want, size = _reference(src.double().cpu().numpy(), x.freqs.cpu().numpy(), pos, sa.ROPE_HALF, x.mscale, None)
            g = got.clone()
            g[~torch.from_numpy(live).cuda()] = float("nan")
            _check(g, want, size, live, f"step {i} rotation")
        k_ref.write(x.k_rot.double().cpu().numpy(), first, rows)
        v_ref.write(x.v.double().cpu().numpy(), first, rows)
        for got, want in zip(_cells_of(d.cache, d.table), (k_ref, v_ref)):
            assert np.array_equal(got.codes, want.codes) and np.array_equal(got.exps, want.exps)
        want, tol = attention(x.q_rot.double().cpu().numpy(), k_ref.values(), v_ref.values(), v_ref.exps, first, rows, D ** -0.5,
                              sa.MASK_BLOCK_CAUSAL)
        off = np.abs(x.out.double().cpu().numpy() - want)[live]
        assert (off <= tol[live] + 2.0 ** -22 * np.abs(want[live])).all()
        if i == 0:
            d.kv_len.copy_(x.q_len)
            continue
        logits = d.out.flatten(2).double().cpu().numpy()
        keep, token = zip(*[_rule(logits[s], d.draft[s].tolist(), d.u[s].tolist(), float(d.u_next[s]), rows[s], float(d.heat[s]), None)
                            for s in range(S)])
        assert d.keep.tolist() == list(keep) and d.token.tolist() == list(token)
        assert d.kv_len.tolist() == [a + b for a, b in zip(first, keep)]
        moved = moved or any(a > 1 for a in keep)
    assert moved or n == 1


def test_steps_on_another_stream():
    a, b = (Decoder(2, 6, 8, 2, 128, 256, seed=3) for _ in range(2))
    side = torch.cuda.Stream()
    for _ in range(6):
        a.feed()
        b.feed()
        a.step()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            b.step()
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a.state(), b.state()))


def _captured(fn):
    """fn as a graph, after a run of its own on the capture's kind of stream."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fn()
    return g


@pytest.mark.parametrize("D,paged", [(128, False), (256, True)])
def test_graphs_that_share_their_handles(D, paged):
    """A step of one row and one of six, captured over the same handles (the second needs a larger workspace than the first
    was captured with), replayed in turn with eager work between; the lengths move on within the graphs."""
    _say(f"decode graphs D={D} paged={paged}")
    made = [Decoder(2, 6, 8, 2, D, 768, paged, seed=5) for _ in range(2)]
    a, b = made
    graphs = {rows: _captured(lambda rows=rows: b.step(rows)) for rows in (1, 6)}
    for x, y in zip(b.state(), a.state()):   # what the warm-up runs moved
        x.copy_(y)
    start = torch.tensor([300, 11], dtype=torch.int32)
    a.kv_len.copy_(start)
    b.kv_len.copy_(start)
    for i, rows in enumerate((6, 1, 1, 6, 1, 6, 6, 1)):
        a.feed()
        b.feed()
        a.step(rows)
        torch.cuda.synchronize()
        graphs[rows].replay()
        torch.cuda.synchronize()
        for name, x, y in zip(("k", "k_exp", "v", "v_exp", "kv_len", "out", "keep", "token"), a.state(), b.state()):
            assert torch.equal(x, y), f"replay {i} of {rows} rows: {name}"
        _ = torch.ones(4096, device="cuda").sum().item()   # eager work between replays


def test_kept_rows_move_a_recurrent_state():
    """keep as the GDN's snap: the state after exactly the rows that stay, whatever else the block held."""
    S, n, G, K = 4, 5, 4, 128
    d = Decoder(S, n, 8, 2, 128, 256, seed=7)
    d.feed()
    d.u[0] = d.u[1] = 0.0
    d.step()
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((S, n, G, K), generator=gen, device="cuda") / K ** 0.5 for _ in range(3))
    al, be = (torch.rand((S, n, G), generator=gen, device="cuda") for _ in range(2))
    state = torch.randn((S, G, K, K), generator=gen, device="cuda")
    y = torch.zeros((S, n, G, K), device="cuda")
    got, want = torch.zeros_like(state), torch.zeros_like(state)
    sa.gdn_verify(q, k, v, al, be, y, state, got, d.q_len, d.keep)
    sa.gdn_verify(q, k, v, al, be, y, state, want, d.keep, d.keep)   # the block without what was rejected
    assert d.keep.tolist()[:2] == d.q_len.tolist()[:2]
    assert torch.equal(got, want)
