"""The latent cache in 4 bits: rows written and read back against the 64-bit restatement, byte for
byte, and the attention over its pages.

Tolerance of the attention. The cache's values are exact in every form, so what is rounded is the
scores, the exponentials and the sums, in fp32 (2^-24 a rounding). A score is a sum of c = kv + rope
products whose partial sums stay within about the largest score s: c roundings of independent
signs, of standard deviation below 2^-24 s sqrt(c) together, then the split of the queries into two
fp16 parts (2^-22 of a product at most, independent signs: below 2^-22 s). An exponential carries its score's
error and 2^-22 of its own (the exponential's and the reference's roundings); a result is a mean of values weighted by
exponentials, with 2^-24 sqrt(64) for a tile's sum. Its relative error's standard deviation is then below
u = 2^-24 (s (sqrt(c) + 4) + 16); the 2-norm is held to 4 u and the largest element, of some
thousands, to 8 u of the largest value in the cache."""
import numpy as np
import pytest

import gmoe
import serve_ref as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def latent(rng, n, kv, rope):
    return (rng.standard_normal((n, kv + rope)) * np.concatenate([1 + 0.3 * rng.standard_normal(kv), np.full(rope, 2.0)])).astype(np.float32)


# ---- rows --------------------------------------------------------------------------------------

SHAPES = [(512, 64), (64, 16), (32, 2), (96, 34), (256, 32), (480, 62)]


def put(x, kv, rope, slot, n_pages, P, ld=None, shift=0, fill=0xA5):
    """Appends x's rows (entry and rope part side by side, ld floats apart, from float `shift` on)."""
    n = len(x)
    ld = ld or kv + rope
    buf = np.full(shift + n * ld + 4, 1e9, np.float32)
    for t in range(n):
        buf[shift + t * ld:shift + t * ld + kv + rope] = x[t]
    d = ref.Arrays(x=buf, slot=np.asarray(slot, np.int32), rows=np.full((n_pages * P, ref.row_bytes(kv, rope)), fill, np.uint8))
    c = gmoe.Cache4(d.p("rows"), kv, rope, n_pages, P)
    c.append(n, d.p("x", 4 * shift), ld, d.p("x", 4 * (shift + kv)), ld, d.p("slot"))
    ref.sync()
    return d, c


@pytest.mark.parametrize("kv,rope", SHAPES)
@pytest.mark.parametrize("n", [1, 5, 300])
def test_rows_byte_for_byte(kv, rope, n):
    rng = np.random.default_rng(n + kv)
    P = 16
    n_pages = n // P + 2
    slot = rng.permutation(n_pages * P)[:n]
    x = latent(rng, n, kv, rope) * np.exp2(rng.integers(-30, 20, (n, 1))).astype(np.float32)
    for ld, shift in ((kv + rope, 0), (kv + rope + 3, 1), (kv + rope + 4, 4)):
        d, c = put(x, kv, rope, slot, n_pages, P, ld, shift)
        want = np.full((n_pages * P, ref.row_bytes(kv, rope)), 0xA5, np.uint8)
        want[slot] = ref.encode(x, kv, rope)
        assert np.array_equal(d.get("rows"), want)
        back = ref.Arrays(comp=np.zeros((n, kv + 1), np.float32), pe=np.zeros((n, rope + 5), np.float32))
        c.read(n, d.p("slot"), back.p("comp"), kv + 1, back.p("pe"), rope + 5)
        ref.sync()
        v = ref.decode(ref.encode(x, kv, rope), kv, rope).astype(np.float32)
        assert np.array_equal(back.get("comp")[:, :kv], v[:, :kv]) and np.array_equal(back.get("pe")[:, :rope], v[:, kv:])
        assert not back.get("comp")[:, kv:].any() and not back.get("pe")[:, rope:].any()


def test_every_rounding_and_scale():
    """Ties, the neighbours of ties, the scales' ends, zeros of both signs, denormals."""
    kv, rope = 64, 2
    mid = (ref.MAGNITUDES[1:] + ref.MAGNITUDES[:-1]) / 2
    base = np.concatenate([ref.MAGNITUDES, mid, [6.5, 7.0]]).astype(np.float32)
    near = np.concatenate([base, np.nextafter(base, np.float32(0)), np.nextafter(base, np.float32(9))])
    near = near[near <= 7]
    rows = []
    for e in (-160, -149, -126, -24, -23, -22, 0, 12, 13, 14, 60, 120):
        for sign in (1, -1):
            v = np.zeros((2, 32), np.float32)
            v.reshape(-1)[:len(near)] = np.ldexp(near, e) * sign
            v[:, 31] = np.ldexp(np.float32(7), e)  # both blocks at this scale
            rows.append(np.concatenate([v.reshape(-1), np.ldexp(np.float32([7.001, -3]), e)]))
    rows.append(np.full(66, -0.0, np.float32))
    x = np.array(rows, np.float32)
    d, _ = put(x, kv, rope, np.arange(len(x)), len(x), 1)
    assert np.array_equal(d.get("rows"), ref.encode(x, kv, rope))


def test_infinities_and_nans_spoil_their_block_alone():
    kv, rope = 64, 32
    x = latent(np.random.default_rng(0), 3, kv, rope)
    x[0, 40], x[1, 70], x[2, 3] = np.nan, np.inf, -np.inf
    d, c = put(x, kv, rope, [0, 1, 2], 3, 1)
    assert np.array_equal(d.get("rows"), ref.encode(x, kv, rope))
    back = ref.Arrays(v=np.zeros((3, kv), np.float32))
    c.read(3, d.p("slot"), back.p("v"), kv, None, 0)
    ref.sync()
    nan = np.isnan(back.get("v"))
    assert nan[0, 32:].all() and not nan[0, :32].any() and not nan[1].any() and nan[2, :32].all() and not nan[2, 32:].any()


def test_slots_outside_the_pool():
    kv, rope = 32, 2
    x = latent(np.random.default_rng(0), 5, kv, rope)
    d, c = put(x, kv, rope, [-1, 3, 8, 0, -(1 << 31)], 2, 4)
    want = np.full((8, 48), 0xA5, np.uint8)
    want[[3, 0]] = ref.encode(x[[1, 3]], kv, rope)
    assert np.array_equal(d.get("rows"), want)
    back = ref.Arrays(comp=np.full((5, kv), 9, np.float32), pe=np.full((5, rope), 9, np.float32))
    c.read(5, d.p("slot"), back.p("comp"), kv, back.p("pe"), rope)
    ref.sync()
    assert not back.get("comp")[[0, 2, 4]].any() and not back.get("pe")[[0, 2, 4]].any() and back.get("comp")[1].any()


# ---- the attention -----------------------------------------------------------------------------


class Attention:
    """A batch on the device with its cache filled, and calls of the attention on it."""

    def __init__(self, seen, fresh, H, kv, rope, P, seed=0, spoil=None, pads=(0, 0, 0), shift=0, x=None, sigma=2.5, **kw):
        rng = np.random.default_rng(seed)
        a, rest, n_pages, T = ref.batch_arrays(seen, fresh, P, rng, **kw)
        m = ref.page_maps(a["seen"], a["fresh"], list(rest), a["table"], T, P)
        a.update({k: m[k] for k in ("table", "offsets", "context")})
        rows = ref.encode(latent(rng, n_pages * P, kv, rope) if x is None else x(n_pages * P), kv, rope)
        if spoil:
            spoil(a, rows)
        n = int(m["totals"][0])
        self.scale = 1 / 16
        s = sigma / (self.scale * np.sqrt(kv + rope))
        self.q_abs = (s * rng.standard_normal((n, H, kv))).astype(np.float32)
        self.q_pe = (s / 2 * rng.standard_normal((n, H, rope))).astype(np.float32)
        self.a, self.rows, self.n, self.shape, self.P, self.T = a, rows, n, (H, kv, rope), P, T
        self.lds = (H * kv + pads[0], H * rope + pads[1], H * kv + pads[2])
        self.shift = shift
        self.c = gmoe.Cache4(0, kv, rope, n_pages, P)
        self.load()

    def load(self):
        H, kv, rope = self.shape

        def spread(v, ld):
            buf = np.full(self.shift + len(v) * ld + 8, 3e38, np.float32)
            for t in range(len(v)):
                buf[self.shift + t * ld:][:v[t].size] = v[t].reshape(-1)
            return buf

        self.d = ref.Arrays(**self.a, rows=self.rows, q_abs=spread(self.q_abs, self.lds[0]), q_pe=spread(self.q_pe, self.lds[1]),
                            out=np.full(self.shift + (self.n + 2) * self.lds[2], 7.0, np.float32),
                            work=np.full(self.c.attend_workspace(H), 0xFF, np.uint8))
        self.c.c.rows = self.d.p("rows")
        self.batch = ref.make_batch(self.a, self.d, self.T, self.P)

    def call(self, scale=None, stream=None, work="work"):
        H, kv, rope = self.shape
        o = 4 * self.shift
        self.c.attend(self.batch, H, self.scale if scale is None else scale, self.d.p("q_abs", o), self.lds[0], self.d.p("q_pe", o),
                      self.lds[1], self.d.p("out", o), self.lds[2], self.d.p(work), self.d.host[work].nbytes, stream=stream)

    def got(self):
        """The results; everything around them must be as it was."""
        H, kv, _ = self.shape
        flat = self.d.get("out")
        assert (flat[:self.shift] == 7).all()
        rows = flat[self.shift:self.shift + self.n * self.lds[2]].reshape(self.n, self.lds[2])
        assert (rows[:, H * kv:] == 7).all() and (flat[self.shift + self.n * self.lds[2]:] == 7).all()
        return rows[:, :H * kv].reshape(self.n, H, kv)

    def want(self):
        return ref.attend(self.q_abs, self.q_pe, self.rows, self.a["table"], self.a["offsets"], self.a["context"], self.P, self.scale)

    def check(self, **kw):
        self.call(**kw)
        ref.sync()
        got, (want, s) = self.got().astype(np.float64), self.want()
        H, kv, rope = self.shape
        u = U * (s * (np.sqrt(kv + rope) + 4) + 16)
        values = ref.decode(self.rows, kv, rope)[:, :kv]
        biggest = np.nanmax(np.abs(values))
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan)
        err = np.abs(np.where(nan, 0, got) - np.where(nan, 0, want))
        norm = np.linalg.norm(want[~nan])
        print(f"[attend] rel {np.linalg.norm(err) / max(norm, 1e-300):.2e} of {4 * u:.2e}, max {err.max() / biggest:.2e} of {8 * u:.2e}", flush=True)
        assert np.linalg.norm(err) <= 4 * u * norm
        assert err.max() <= 8 * u * biggest
        return got


GLM = (20, 512, 64)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 700, 4097])
def test_one_token(length):
    print(f"[case] {length}", flush=True)
    Attention([length - 1], [1], *GLM, 16, seed=length).check()


@pytest.mark.parametrize("shape", [(1, 512, 64), (4, 64, 16), (8, 32, 2), (16, 256, 32), (20, 96, 34), (32, 512, 64), (33, 480, 62),
                                   (64, 128, 64), (128, 512, 64), (256, 32, 64), (5, 224, 2)])
def test_shapes(shape):
    print(f"[case] {shape}", flush=True)
    Attention([0, 70, 130, 5], [1, 3, 1, 40], *shape, 32, seed=sum(shape)).check()


@pytest.mark.parametrize("P", [1, 2, 8, 16, 64, 256, 4096])
def test_page_sizes(P):
    Attention([P - 1, 2 * P, 0], [2, 1, 33] if P < 4096 else [1, 1, 3], 4, 64, 16, P, seed=P).check()


@pytest.mark.parametrize("kind", ["decode", "mixed", "prompt", "short", "idle", "many"])
def test_batches(kind):
    rng = np.random.default_rng(9)
    print(f"[case] {kind}", flush=True)
    if kind == "decode":  # ragged: one far longer than the rest, which is cut, and tiny ones, which are not
        seen = np.array([8000, 0, 1, 30, 63, 64, 500, 2000])
        Attention(seen, np.ones(8), *GLM, 64, seed=1).check()
    elif kind == "mixed":
        Attention([300, 0, 17, 1200, 64], [1, 90, 0, 25, 1], *GLM, 16, seed=2).check()
    elif kind == "prompt":
        Attention([777], [201], *GLM, 128, seed=3).check()
    elif kind == "short":  # the pool is too small for the last two: zeros
        t = Attention([20, 40, 16, 0], [1, 1, 4, 3], 4, 64, 16, 16, seed=4, free=0)
        assert t.a["context"].tolist() == [21, 41, 0, 0]
        assert not t.check()[2:].any()
    elif kind == "idle":
        Attention([0, 5, 0, 9, 0], [0, 0, 2, 0, 0], 4, 64, 16, 16, seed=5).check()
    else:
        seen = rng.integers(0, 90, 700)
        Attention(seen, (rng.random(700) < 0.8).astype(int), 3, 32, 8, 16, seed=6).check()


@pytest.mark.parametrize("pads,shift", [((4, 4, 4), 0), ((1, 2, 3), 0), ((0, 0, 0), 1), ((64, 0, 4), 4)])
def test_strides_and_alignment(pads, shift):
    Attention([100, 3], [1, 30], 20, 512, 64, 16, seed=7, pads=pads, shift=shift).check()


def test_masked_positions_may_hold_anything():
    """NaN rows past the last position, and of a later token of the same tile, reach no result; an
    attended one makes its token's results NaN."""
    def spoil(a, rows):
        for r in range(2):  # past the end, in the last page
            page, at = a["table"][r, a["context"][r] // 16], a["context"][r] % 16
            rows[page * 16 + at:page * 16 + 16] = 255
        # one block of the last but one token's row (position 41 of request 1's 0..42)
        rows[a["table"][1, 41 // 16] * 16 + 41 % 16, 288 + 5] = 255
    t = Attention([20, 40], [1, 3], *GLM, 16, seed=8, spoil=spoil)
    got = t.check()
    assert np.isfinite(got[:2]).all() and np.isnan(got[2:]).all()


def test_pages_outside_the_pool_are_not_attended():
    def spoil(a, rows):
        a["table"][0, 1], a["table"][1, 0], a["table"][2, 0] = -1, len(rows) // 16, 1 << 30
    t = Attention([40, 30, 3], [2, 1, 1], *GLM, 16, seed=10, spoil=spoil)
    got = t.check()
    assert not got[3].any() and got[:3].any(axis=(1, 2)).all()  # request 2 has nothing left


def test_a_context_past_its_table():
    def spoil(a, rows):
        a["context"][0] += 100
    Attention([40], [20], 4, 64, 16, 16, seed=11, spoil=spoil).check()


def test_scales_of_queries_and_values():
    """Queries far from 1 at a scale that makes up for it, rows of very different sizes, a zero row."""
    for e in (-100, -60, 60, 90):
        t = Attention([200], [3], *GLM, 16, seed=12)
        t.scale, t.q_abs, t.q_pe = np.ldexp(t.scale, -e), np.ldexp(t.q_abs, e), np.ldexp(t.q_pe, e)
        t.load()
        t.check()
    rng = np.random.default_rng(3)

    def uneven(n):
        x = latent(rng, n, 512, 64) * np.exp2(rng.integers(-20, 3, (n, 1)))
        x[::7] = 0
        return x.astype(np.float32)
    Attention([500, 20], [1, 2], *GLM, 16, seed=13, x=uneven).check()


def test_peaked_scores():
    """Scores of standard deviation 40: one position has nearly all of the weight."""
    Attention([900, 10], [1, 70], *GLM, 16, seed=14, sigma=40).check()


def test_zero_queries_average_the_values():
    t = Attention([99], [1], *GLM, 16, seed=15)
    t.q_abs[:], t.q_pe[:] = 0, 0
    t.load()
    t.check()


def test_results_do_not_depend_on_the_batch_or_repeat():
    """The same call twice gives the same bits, whatever the workspace holds."""
    t = Attention([3000, 50, 700], [1, 9, 1], *GLM, 64, seed=16)
    first = t.check()
    t.d.put("work", np.zeros_like(t.d.host["work"]))
    t.call()
    ref.sync()
    assert np.array_equal(t.got(), first)


def test_a_long_cache_past_32_bits():
    """Rows beyond 4 GiB of one pool."""
    kv, rope, P = 512, 64, 4096
    n_pages = (5 << 30) // (320 * P)
    rng = np.random.default_rng(17)
    x = latent(rng, 300, kv, rope)
    rows = gmoe.DeviceArray(n_pages * P * 320)
    table = np.array([[n_pages - 1]], np.int32)
    slot = (n_pages - 1) * P + np.arange(300)
    d = ref.Arrays(x=x, slot=slot.astype(np.int32), table=table, offsets=np.array([0, 1], np.int32), context=np.array([300], np.int32),
                   q=rng.standard_normal((1, 20, 576)).astype(np.float32), out=np.zeros((1, 20, kv), np.float32))
    c = gmoe.Cache4(rows.ptr.value, kv, rope, n_pages, P)
    c.append(300, d.p("x"), 576, d.p("x", 4 * kv), 576, d.p("slot"))
    work = gmoe.DeviceArray(c.attend_workspace(20))
    q = d.host["q"]
    d2 = ref.Arrays(a=q[..., :kv], p=q[..., kv:])
    b = gmoe.Batch(1, 1, 1, P, table=d.p("table"), offsets=d.p("offsets"), context=d.p("context"))
    c.attend(b, 20, 0.1, d2.p("a"), 20 * kv, d2.p("p"), 20 * rope, d.p("out"), 20 * kv, work.ptr.value, work.nbytes)
    ref.sync()
    small = np.zeros((P, 320), np.uint8)
    small[:300] = ref.encode(x, kv, rope)
    want, s = ref.attend(q[..., :kv], q[..., kv:], small, np.zeros((1, 1), np.int32), [0, 1], [300], P, 0.1)
    err = np.linalg.norm(d.get("out") - want) / np.linalg.norm(want)
    assert err <= 4 * U * (s * (24 + 4) + 16)


def test_captured_and_overlapping_calls():
    """Two captured graphs with workspaces of their own, replayed on two streams at once, and each
    replay after new lengths, equal the eager results."""
    ts = [Attention([2000, 30], [1, 1], *GLM, 64, seed=20 + i, extra_pages=6, gap=2) for i in range(2)]
    ss = [gmoe.Stream() for _ in ts]
    exes = [ref.capture(s, lambda t=t, s=s: t.call(stream=s.h)) for t, s in zip(ts, ss)]
    for step in range(4):
        for t in ts:
            t.a["context"][:] = [2001 - 300 * step, 31 + step]
            t.d.put("context", t.a["context"])
            t.d.put("out", np.full_like(t.d.host["out"], 7.0))
        for t in ts:
            t.check()
        eager = [t.got() for t in ts]
        for t in ts:
            t.d.put("out", np.full_like(t.d.host["out"], 7.0))
        for _ in range(3):
            for s, e in zip(ss, exes):
                gmoe.hip_check(gmoe.hip().hipGraphLaunch(e, s.h), "hipGraphLaunch")
        for s in ss:
            s.sync()
        for t, e in zip(ts, eager):
            assert np.array_equal(t.got(), e)
