"""gmoe_page_maps against the request-by-request restatement: every array, exactly."""
import numpy as np
import pytest

import gmoe
import serve_ref as ref

pytestmark = pytest.mark.gpu


def check(seen, fresh, P, rng, **kw):
    a, rest, n_pages, T = ref.batch_arrays(seen, fresh, P, rng, **kw)
    want = ref.page_maps(a["seen"], a["fresh"], list(rest), a["table"], T, P)
    d = ref.Arrays(**a)
    b = ref.make_batch(a, d, T, P)
    for _ in range(2):  # the call may be repeated
        b.maps()
        ref.sync()
        for k, v in want.items():
            assert np.array_equal(d.get(k), v), (k, np.argwhere(d.get(k) != v)[:5])
    for k in ("seen", "fresh", "n_free", "free_pages"):
        assert np.array_equal(d.get(k), a[k]), k
    return want


CASES = {
    "one_first_token": ([0], [1], 16, {}),
    "one_page_boundary": ([16], [1], 16, {}),
    "inside_a_page": ([15], [1], 16, {}),
    "nothing_new": ([5, 0, 32], [0, 0, 0], 16, {}),
    "a_prompt_over_many_pages": ([3], [1000], 16, {}),
    "pages_of_one": ([7, 0, 2], [5, 1, 0], 1, {}),
    "wide_table": ([17, 100, 4], [3, 30, 1], 32, {"gap": 9}),
    "idle_between": ([9, 8, 7, 0, 64], [0, 3, 0, 0, 2], 8, {}),
    "pool_one_short": ([0, 0, 0, 16], [40, 17, 1, 0], 16, {"free": 5}),
    "pool_empty": ([15, 16], [1, 1], 16, {"free": 0}),
    "tokens_past_the_arrays": ([0, 5, 0, 0], [10, 7, 4, 1], 16, {"max_tokens": 16}),
    "table_too_narrow": ([0, 30, 3], [33, 3, 2], 16, {"width": 2}),
    "exactly_full": ([0, 16], [32, 16], 16, {"width": 2, "max_tokens": 48, "extra_pages": 0}),
}


@pytest.mark.parametrize("name", list(CASES))
def test_cases(name):
    seen, fresh, P, kw = CASES[name]
    print(f"[case] {name}", flush=True)
    check(seen, fresh, P, np.random.default_rng(1), **kw)


def test_negative_and_absurd_lengths_are_short():
    rng = np.random.default_rng(2)
    a, rest, _, T = ref.batch_arrays([4, 4, 4, 4, 4], [2, 2, 2, 2, 2], 16, rng)
    a["seen"][1], a["fresh"][2], a["seen"][3] = -1, -5, (1 << 31) - 1
    want = ref.page_maps(a["seen"], a["fresh"], list(rest), a["table"], T, 16)
    assert want["totals"].tolist() == [8, 0, 3]
    d = ref.Arrays(**a)
    ref.make_batch(a, d, T, 16).maps()
    ref.sync()
    for k, v in want.items():
        assert np.array_equal(d.get(k), v), k


@pytest.mark.parametrize("R", [2, 63, 64, 65, 255, 256, 257, 1000, 4096])
def test_many_requests(R):
    rng = np.random.default_rng(R)
    seen = rng.integers(0, 300, R)
    fresh = np.where(rng.random(R) < 0.1, 0, np.where(rng.random(R) < 0.1, rng.integers(2, 200, R), 1))
    check(seen, fresh, 32, rng)
    check(seen, fresh, 32, rng, free=max(1, R // 8))


def test_slots_past_31_bits_are_none():
    rng = np.random.default_rng(3)
    a, _, _, T = ref.batch_arrays([0, 0], [2, 2], 65536, rng)
    a["free_pages"][:] = [3, 9, 32767, 32768, -4][:len(a["free_pages"])]
    a["n_free"][0] = 5 if len(a["free_pages"]) == 5 else len(a["free_pages"])
    want = ref.page_maps(a["seen"], a["fresh"], list(a["free_pages"]), a["table"], T, 65536)
    d = ref.Arrays(**a)
    ref.make_batch(a, d, T, 65536).maps()
    ref.sync()
    assert np.array_equal(d.get("slot"), want["slot"]) and (want["slot"] == -1).any()


def test_replays_follow_the_lengths():
    """A captured call reads lengths, pool and count anew at each replay."""
    rng = np.random.default_rng(4)
    P, seen, fresh = 16, np.array([15, 3, 40]), np.array([1, 1, 1])
    a, rest, _, T = ref.batch_arrays(seen, fresh, P, rng, extra_pages=20, max_tokens=3, gap=4)
    d, s = ref.Arrays(**a), gmoe.Stream()
    b = ref.make_batch(a, d, T, P)
    exe = ref.capture(s, lambda: b.maps(stream=s.h))
    table, pool = a["table"], list(rest)
    for _ in range(20):
        want = ref.page_maps(seen, fresh, pool, table, T, P)
        gmoe.hip_check(gmoe.hip().hipGraphLaunch(exe, s.h), "hipGraphLaunch")
        s.sync()
        for k, v in want.items():
            assert np.array_equal(d.get(k), v), k
        table, pool, seen = want["table"], pool[:len(pool) - int(want["totals"][1])], seen + fresh
        d.put("seen", seen)
        d.put("n_free", [len(pool)])
