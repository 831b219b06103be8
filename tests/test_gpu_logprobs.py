"""gmoe_logprobs against the 64-bit restatement: ids exactly, values to fp32.

Tolerance. ln p = (x - m) - log1p(S): x - m is rounded once (2^-24 of it), S is a sum of exponentials,
each within 2^-22 (its argument's rounding times the argument, at most 2^-24 |x - m| e^(x - m) <=
2^-24, and the exponential's own), so log1p(S) is within 2^-21 of S / (1 + S) and 2^-23 of itself, and the
difference rounds once: 2^-21 (1 + |ln p| / 4) in all, and relative to ln p itself where that
is small: S / (1 + S) <= log1p(S). The entropy has three such terms: 2^-20 of itself. Sums over a
vocabulary in fp32 add 2^-24 sqrt(V / 256) at most in a lane's chain."""
import numpy as np
import pytest

import gmoe
import serve_ref as ref

pytestmark = pytest.mark.gpu


def check(x, given, top, ld=None, shift=0, stream=None):
    n, V = x.shape
    ld = ld or V
    buf = np.full(shift + n * ld + 8, np.nan, np.float32)  # what lies between the rows is not read as logits
    for i in range(n):
        buf[shift + i * ld:shift + i * ld + V] = x[i]
    given = np.asarray(given, np.int32).reshape(n, -1)
    g = given.shape[1]
    lp = gmoe.LogProbs(n, V, top, g)
    d = ref.Arrays(x=buf, given=given, logprob=np.full((n + 1, max(g, 1)), 7, np.float32), entropy=np.full(n + 1, 7, np.float32),
                   top_id=np.full((n + 1, max(top, 1)), 7, np.int32), top_logprob=np.full((n + 1, max(top, 1)), 7, np.float32),
                   work=np.full(max(16, lp.workspace), 0xFF, np.uint8))
    out = []
    for _ in range(2):
        lp(d.p("x", 4 * shift), ld, d.p("given"), d.p("logprob"), d.p("entropy"), d.p("top_id"), d.p("top_logprob"), d.p("work"),
           lp.workspace, stream=stream)
        ref.sync()
        out.append([d.get(k) for k in ("logprob", "entropy", "top_id", "top_logprob")])
    for p, q in zip(*out):
        assert np.array_equal(p, q, equal_nan=p.dtype == np.float32)  # the same bits again
    got = [o[:n] for o in out[0]]
    assert all((o[n:] == 7).all() for o in out[0])
    want = ref.logprobs(x, given, top)
    tol = 2.0 ** -24 * (8 + np.sqrt(V / 256))
    if g:
        close(got[0], want[0], tol)
    else:
        assert (got[0] == 7).all()
    close(got[1], want[1], 2 * tol)
    if top:
        assert np.array_equal(got[2], want[2]), (np.argwhere(got[2] != want[2])[:5], got[2][got[2] != want[2]][:5], want[2][got[2] != want[2]][:5])
        close(got[3], want[3], tol)
    else:
        assert (got[2] == 7).all()
    return got


def close(got, want, tol):
    """Within tol (1 + |v|) of v, and within tol of itself where v is small."""
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    err, size = np.abs(got[fine] - want[fine]), np.abs(want[fine])
    if err.size:
        print(f"[logprobs] {np.max(err / np.maximum(np.minimum(1 + size, 8 * size), 1e-300)):.2e} of {tol:.2e}", flush=True)
        assert (err <= tol * np.minimum(1 + size, 8 * size) + 1e-37).all()


def logits(rng, n, V, spread=2.0, peaks=3):
    x = rng.standard_normal((n, V)).astype(np.float32) * np.float32(spread)
    for i in range(n):
        x[i, rng.integers(0, V, peaks)] = 10 + 3 * rng.standard_normal(peaks)
    return x


@pytest.mark.parametrize("n,V,top,g", [(1, 1, 1, 1), (1, 2, 5, 2), (3, 63, 64, 1), (2, 64, 20, 1), (5, 65, 20, 3), (1, 300, 64, 1),
                                       (7, 1000, 5, 1), (1, 4095, 20, 1), (2, 4097, 20, 0), (1, 8193, 64, 1), (3, 20001, 32, 2),
                                       (1, 154880, 20, 1), (2, 154880, 0, 1), (1, 154881, 64, 5), (300, 700, 5, 1), (600, 20011, 3, 1)])
def test_sizes(n, V, top, g):
    print(f"[case] {n} {V} {top} {g}", flush=True)
    rng = np.random.default_rng(n + V)
    check(logits(rng, n, V), rng.integers(0, V, (n, g)), top)


@pytest.mark.parametrize("extra,shift", [(1, 0), (3, 1), (4, 0), (8, 2), (0, 3)])
@pytest.mark.parametrize("n,V", [(3, 5000), (300, 515)])
def test_strides_and_alignment(n, V, extra, shift):
    rng = np.random.default_rng(extra)
    check(logits(rng, n, V), rng.integers(0, V, (n, 1)), 9, V + extra, shift)


@pytest.mark.parametrize("V", [100, 5000, 70001])
@pytest.mark.parametrize("n", [1, 400])
def test_masks(V, n):
    """-inf and the lowest value on most of a row; rows with fewer tokens left than alternatives,
    one left, none left; ties everywhere."""
    rng = np.random.default_rng(V)
    x = logits(rng, n + 8, V)
    low = np.finfo(np.float32).min
    x[0, rng.random(V) < 0.99] = -np.inf
    x[1, rng.random(V) < 0.99] = low
    x[2], x[2, V // 2] = -np.inf, 3.0
    x[3], x[3, V // 2] = low, 3.0
    x[4] = -np.inf
    x[5] = low
    x[6] = 1.5
    x[7] = np.round(x[7])
    x[7, ::2] = -0.0
    x[7, 1::4] = 0.0
    if n == 1:
        for i in range(8):
            check(x[i:i + 1], [[V // 2, 0]], 7)
    check(x, np.stack([np.full(n + 8, V // 2), rng.integers(0, V, n + 8)], 1), 7)


def test_rows_of_nothing_numbers():
    rng = np.random.default_rng(0)
    x = logits(rng, 6, 9000)
    x[0, 8999], x[1, 0], x[2, 100], x[2, 200] = np.nan, np.inf, np.inf, -np.inf
    x[3, 5], x[3, 6] = -np.nan, np.inf
    x[4, 17] = 3e38
    for i in range(6):
        check(x[i:i + 1], [[17]], 4)
    check(x, np.full((6, 1), 17), 4)
    check(np.tile(x, (90, 1)), np.full((540, 1), 17), 4)


def test_given_ids_outside_the_vocabulary():
    x = logits(np.random.default_rng(1), 2, 500)
    got = check(x, [[-1, 499, 500], [0, 1 << 30, -(1 << 31)]], 2)
    assert np.isnan(got[0]).tolist() == [[True, False, True], [False, True, True]]


@pytest.mark.parametrize("n", [1, 300])
def test_near_certain_tokens_keep_their_precision(n):
    """One token 30 to 60 above the rest: ln p of 1e-9 to 1e-21, and the entropy, to fp32's relative precision."""
    rng = np.random.default_rng(2)
    V = 6000
    x = rng.standard_normal((n, V)).astype(np.float32)
    at = rng.integers(0, V, n)
    x[np.arange(n), at] = 30 + 30 * rng.random(n)
    got = check(x, at[:, None], 3)
    assert (got[0] < 0).all() and (got[0] > -1e-8).all() and (got[1] > 0).all()


@pytest.mark.parametrize("n", [1, 280])
def test_alternatives_wherever_they_lie(n):
    """The likeliest tokens all beside each other, strided, at the ends, and all equal."""
    rng = np.random.default_rng(3)
    V, k = 40000, 64
    for place in (np.arange(64), np.arange(64) * 256, V - 64 + np.arange(64), np.arange(64) * 4, np.concatenate([[0], V - 63 + np.arange(63)]),
                  1000 + np.arange(64) * 64):
        x = rng.standard_normal((n, V)).astype(np.float32)
        x[:, place] = 20 + rng.random((n, 64)).astype(np.float32)
        got = check(x, place[:1][None].repeat(n, 0), k)
        assert (np.sort(got[2], 1) == np.sort(place)).all()
        x[:, place] = 20
        got = check(x, place[:1][None].repeat(n, 0), k)
        assert (got[2] == np.sort(place)).all()


def test_rising_and_falling_rows():
    for n in (1, 260):
        x = np.tile(np.linspace(-5, 5, 30000, dtype=np.float32), (n, 1))
        check(x, np.zeros((n, 1)), 33)
        check(x[:, ::-1].copy(), np.zeros((n, 1)), 33)


def test_replays_and_overlapping_graphs():
    """Captured calls on two streams at once, each with its own workspace, over new logits at each replay."""
    rng = np.random.default_rng(5)
    V, calls = 60000, []
    for i in range(2):
        lp, s = gmoe.LogProbs(2, V, 8, 1), gmoe.Stream()
        d = ref.Arrays(x=logits(rng, 2, V), given=np.array([[5], [9]], np.int32), logprob=np.zeros((2, 1), np.float32),
                       entropy=np.zeros(2, np.float32), top_id=np.zeros((2, 8), np.int32), top_logprob=np.zeros((2, 8), np.float32),
                       work=np.zeros(max(16, lp.workspace), np.uint8))

        def call(stream, lp=lp, d=d):
            lp(d.p("x"), V, d.p("given"), d.p("logprob"), d.p("entropy"), d.p("top_id"), d.p("top_logprob"), d.p("work"), lp.workspace,
               stream=stream)
        calls.append((d, s, ref.capture(s, lambda: call(s.h))))
    for step in range(4):
        xs = [logits(rng, 2, V) for _ in calls]
        for (d, _, _), x in zip(calls, xs):
            d.put("x", x)
        ref.sync()
        for _, s, exe in calls:
            gmoe.hip_check(gmoe.hip().hipGraphLaunch(exe, s.h), "hipGraphLaunch")
        for (d, s, _), x in zip(calls, xs):
            s.sync()
            want = ref.logprobs(x, d.host["given"], 8)
            assert np.array_equal(d.get("top_id"), want[2])
            close(d.get("logprob"), want[0], 2.0 ** -24 * 30)
            close(d.get("entropy"), want[1], 2.0 ** -24 * 60)
