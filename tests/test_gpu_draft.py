"""Draft verification on the GPU (sixi_draft_verify) against the rule in 64 bits, token by token.

Tokens and row counts are whole numbers and must be equal.  The reference says when an input stands so near a border
(a running sum or an acceptance within 1e-9 of its number) that 64-bit sums of another order may fall on the other
side; the inputs here keep clear of that, which the reference asserts."""
import sys

import numpy as np
import pytest
import torch

import sixi_attn as sa

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", file=sys.stderr, flush=True)


def _softmax(x, heat):
    """The target's distribution of one row of logits (float64)."""
    x = np.where(np.isnan(x), -np.inf, x)
    p = np.zeros_like(x)
    top = x.max()
    if top == -np.inf:
        return p
    if not heat > 0:
        p[int(np.argmax(x))] = 1.0
        return p
    if top == np.inf:
        p[x == np.inf] = 1.0
    else:
        p = np.exp((x - top) / heat)
    return p / p.sum()


def _rule(logits, draft, u, u_next, rows, heat, probs):
    """(keep, token) of one stream."""
    if rows <= 0:
        return 0, -1
    V = logits.shape[1]
    j = 0
    while True:
        p = _softmax(logits[j], heat)
        w = p
        if j < rows - 1:
            d = int(draft[j])
            known = 0 <= d < V
            q = (probs[j] if probs is not None else np.eye(1, V, d)[0]) if known or probs is not None else np.zeros(V)
            left, right = float(u[j]) * (float(q[d]) if known else 1.0), float(p[d]) if known else 0.0
            # no rounding decides: apart, equal, or 0 against a weight that 64 bits hold (p > 0 however it is formed)
            assert left == right or abs(left - right) > 1e-9 or left == 0 and right > 1e-250
            if left < right:
                j += 1
                continue
            w = np.maximum(p - q, 0.0)
            if not w.sum() > 0:
                w = p
        if not w.sum() > 0:
            return j + 1, -1
        c = np.cumsum(w)
        mark = float(u_next) * c[-1]
        t = int(np.searchsorted(c, mark, side="right"))
        last = int(np.nonzero(w)[0][-1])
        near = np.abs(c[max(0, t - 1):t + 1] - mark).min()
        assert near > 1e-12 * c[-1] or u_next in (0.0, 1.0)
        return j + 1, min(t, last)


def _case(s, n, V, with_probs, seed, dtype=torch.float32, greedy=False, rows=None, noise=0.7, size=3.0):
    rng = np.random.default_rng(seed)
    logits = (size * rng.standard_normal((s, n, V))).astype(np.float32)
    guess = np.exp(logits[:, :n - 1] + noise * rng.standard_normal((s, n - 1, V)))
    guess = (guess / guess.sum(-1, keepdims=True)).astype(np.float32)
    logits[:, :, rng.random(V) < 0.1] = -np.inf
    logits = torch.from_numpy(logits).to(dtype)
    draft = np.zeros((s, n - 1), np.int32)
    for i in range(s):
        for j in range(n - 1):
            draft[i, j] = rng.choice(V, p=guess[i, j].astype(np.float64) / guess[i, j].astype(np.float64).sum()) if with_probs else int(guess[i, j].argmax())
    heat = rng.uniform(0.5, 1.5, s).astype(np.float32)
    if greedy:
        heat[::2] = 0.0
    return {"logits": logits, "draft": draft, "u": rng.random((s, n - 1)).astype(np.float32),
            "u_next": rng.random(s).astype(np.float32), "heat": heat, "probs": guess if with_probs else None,
            "rows": [n] * s if rows is None else rows}


def _run(c, handle=None, heat=True):
    s = c["logits"].shape[0]
    keep, token = (torch.full((s,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    t = {k: torch.from_numpy(c[k]).cuda() for k in ("draft", "u", "u_next", "heat")}
    (handle or sa.DraftVerify())(c["logits"].cuda(), t["draft"], t["u"], t["u_next"], keep, token,
                                 draft_probs=None if c["probs"] is None else torch.from_numpy(c["probs"]).cuda(),
                                 q_len=torch.tensor(c["rows"], dtype=torch.int32, device="cuda"),
                                 temperature=t["heat"] if heat else None)
    return keep.tolist(), token.tolist()


def _want(c, heat=True):
    n = c["logits"].shape[1]
    x = c["logits"].double().numpy()
    return [list(z) for z in zip(*[
        _rule(x[i], c["draft"][i], c["u"][i], c["u_next"][i], min(max(c["rows"][i], 0), n), c["heat"][i] if heat else 1.0,
              None if c["probs"] is None else c["probs"][i].astype(np.float64)) for i in range(len(x))])]


@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("s,n,V", [(1, 1, 1), (1, 2, 7), (3, 5, 100), (2, 16, 4096), (4, 3, 4097), (1, 17, 12001),
                                   (2, 40, 300), (2, 4, 70001)])
def test_draft_verify(s, n, V, with_probs, dtype):
    _say(f"draft s={s} n={n} V={V} probs={with_probs} dtype={dtype}")
    c = _case(s, n, V, with_probs, s * 31 + n + V, dtype)
    if V > 1:
        assert list(_run(c)) == _want(c)
    else:
        keep, token = _run(c)
        assert all(t in (0, -1) for t in token)


@pytest.mark.parametrize("with_probs", [False, True])
def test_draft_verify_ragged_and_greedy(with_probs):
    rows = [6, 1, 0, 3, -2, 9, 2]
    c = _case(7, 6, 5000, with_probs, 11, greedy=True, rows=rows)
    got = _run(c)
    assert list(got) == _want(c)
    assert got[0][2] == got[0][4] == 0 and got[1][2] == got[1][4] == -1


def test_draft_verify_every_place_of_the_first_rejection():
    """Drafts that are the target's own, but one; u decides there."""
    n, V = 9, 600
    for stop in range(n):
        c = _case(1, n, V, True, 100 + stop)
        x = c["logits"].double().numpy()[0]
        for j in range(n - 1):
            p = _softmax(x[j], c["heat"][0])
            c["probs"][0, j] = p
            c["draft"][0, j] = int(np.argmax(p))
        if stop < n - 1:
            c["draft"][0, stop] = int(np.nonzero(x[stop] == -np.inf)[0][0])   # a token that the filter struck
        got = _run(c)
        assert got[0] == [stop + 1]
        assert list(got) == _want(c)


def test_draft_verify_without_temperature_and_without_lengths():
    c = _case(3, 4, 900, True, 5)
    assert list(_run(c, heat=False)) == _want(c, heat=False)
    keep, token = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
    t = {k: torch.from_numpy(c[k]).cuda() for k in ("draft", "u", "u_next", "probs")}
    sa.DraftVerify()(c["logits"].cuda(), t["draft"], t["u"], t["u_next"], keep, token, draft_probs=t["probs"])
    assert [keep.tolist(), token.tolist()] == _want(c, heat=False)


def test_draft_verify_extremes():
    """Rows of -inf, +inf and NaN logits, ties, drafted tokens out of range, u_next at its ends, p equal to q."""
    n, V = 3, 5000
    c = _case(9, n, V, True, 8)
    x = c["logits"].numpy()
    x[0, 0] = -np.inf                                   # no weight at all
    x[1, 0, 4000] = x[1, 0, 17] = np.inf                # two that take all
    c["draft"][1, 0] = 17
    c["u"][1, 0] = 0.0
    x[2, :, ::2] = np.nan
    c["draft"][3, 0], c["draft"][4, 0], c["draft"][5, 0] = -1, V, 1 << 30
    c["u_next"][6] = 0.0
    c["u_next"][7] = 1.0
    c["heat"][8] = 0.0                                  # a tie, greedy: the lowest token
    x[8, 0] = 1.0
    c["draft"][8, 0] = 3
    c["u"][8, 0] = 0.5
    got, want = _run(c), _want(c)
    assert list(got) == want
    assert got[0][0] == 1 and got[1][0] == -1
    assert got[0][3:6] == [1, 1, 1] and got[0][8] == 1 and got[1][8] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_draft_verify_temperatures(dtype):
    """From the smallest number of the type to the largest, the logits far from 0: what differs by more than 1000 powers of
    two from the top has no weight, whatever steps f32 has there; at the largest, what is not struck weighs alike.  NaN is
    greedy, as 0."""
    heats = [1e-40, 1e-30, 1e-12, 1e-9, 2e-8, 1e-7, 3e-7, 1e-6, 1e-5, 1e-3, 30.0, 1e6, 1e20, 1e33, 3e38, float("nan"), 0.0]
    for shift in (0.0, 100.0, -5000.0):
        c = _case(len(heats), 3, 9000, False, 31, dtype=dtype)
        c["heat"] = np.array(heats, np.float32)
        c["logits"] = (c["logits"].float() + shift).to(dtype)
        c["u"][:] = np.linspace(0.001, 0.3, c["u"].size, dtype=np.float32).reshape(c["u"].shape)
        with np.errstate(over="ignore"):
            want = _want(c)
        assert list(_run(c)) == want, shift


def test_draft_verify_where_p_minus_q_leaves_nothing():
    """A drafted token that both distributions leave out, both equal elsewhere: the draw is from p."""
    V = 64
    x = np.full((1, 2, V), -np.inf, np.float32)
    x[0, :, :4] = 0.0
    probs = np.zeros((1, 1, V), np.float32)
    probs[0, 0, :4] = 0.25
    c = {"logits": torch.from_numpy(x), "draft": np.array([[9]], np.int32), "u": np.array([[0.5]], np.float32),
         "u_next": np.array([0.6], np.float32), "heat": np.ones(1, np.float32), "probs": probs, "rows": [2]}
    assert _run(c) == ([1], [2])


def test_draft_verify_strides_and_misaligned_rows():
    """Logits as a slice of a wider f16 tensor whose rows begin at odd addresses, ids and numbers as slices."""
    c = _case(2, 5, 333, True, 21, torch.float16)
    wide = torch.full((2, 7, 341), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 1:6, 3:336] = c["logits"].cuda()
    probs = torch.full((2, 9, 335), float("nan"), device="cuda")
    probs[:, ::2][:, :4, 1:334] = torch.from_numpy(c["probs"]).cuda()
    ids = torch.zeros((2, 11), dtype=torch.int32, device="cuda")
    ids[:, 2:6] = torch.from_numpy(c["draft"]).cuda()
    u = torch.zeros((2, 6), device="cuda")
    u[:, 1:5] = torch.from_numpy(c["u"]).cuda()
    keep, token = (torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2))
    sa.DraftVerify()(wide[:, 1:6, 3:336], ids[:, 2:6], u[:, 1:5], torch.from_numpy(c["u_next"]).cuda(), keep, token,
                     draft_probs=probs[:, ::2][:, :4, 1:334], temperature=torch.from_numpy(c["heat"]).cuda())
    assert [keep.tolist(), token.tolist()] == _want(c)


def test_draft_verify_rows_past_32_bits():
    """Rows of logits and of the drafter's distribution three GiB apart."""
    c = _case(1, 3, 5000, True, 44)
    step = 3 << 28                                        # in f32 elements
    want = _run(c)
    assert list(want) == _want(c)
    wide = torch.empty(2 * step + 5000, device="cuda")
    logits = wide.as_strided((1, 3, 5000), (wide.numel(), step, 1))
    logits.copy_(c["logits"])
    more = torch.empty(step + 5000, device="cuda")
    probs = more.as_strided((1, 2, 5000), (more.numel(), step, 1))
    probs.copy_(torch.from_numpy(c["probs"]))
    keep, token = (torch.full((1,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    sa.DraftVerify()(logits, torch.from_numpy(c["draft"]).cuda(), torch.from_numpy(c["u"]).cuda(), torch.from_numpy(c["u_next"]).cuda(),
                     keep, token, draft_probs=probs, temperature=torch.from_numpy(c["heat"]).cuda())
    assert (keep.tolist(), token.tolist()) == want


def test_draft_verify_draws_as_the_target_would():
    """Over 20000 draws of a two-row block the first token is distributed as p (both the kept and the drawn)."""
    V, N = 8, 20000
    rng = np.random.default_rng(3)
    logits = np.tile(rng.standard_normal((1, 2, V)), (N, 1, 1)).astype(np.float32)
    p, q = _softmax(logits[0, 0].astype(np.float64), 1.0), _softmax(rng.standard_normal(V), 1.0)
    ids = rng.choice(V, size=(N, 1), p=q).astype(np.int32)
    keep, token = (torch.zeros(N, dtype=torch.int32, device="cuda") for _ in range(2))
    sa.DraftVerify()(torch.from_numpy(logits).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(rng.random((N, 1)).astype(np.float32)).cuda(),
                     torch.from_numpy(rng.random(N).astype(np.float32)).cuda(), keep, token,
                     draft_probs=torch.from_numpy(np.tile(q, (N, 1, 1)).astype(np.float32)).cuda())
    first = np.where(keep.cpu().numpy() == 2, ids[:, 0], token.cpu().numpy())
    share = np.bincount(first, minlength=V) / N
    # five standard deviations of a share of N draws
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / N)).all()


def test_draft_verify_is_the_same_every_time():
    c = _case(3, 6, 40000, True, 14)
    h = sa.DraftVerify()
    first = _run(c, h)
    for _ in range(3):
        assert _run(c, h) == first
