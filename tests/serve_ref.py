"""The serving operators (include/gmoe_serve.h) restated in 64 bits with numpy, and what their GPU
tests share: device copies of arrays, and batches of requests with their pools and tables."""
import ctypes as C

import numpy as np

import gmoe

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


# ---- the formulas ------------------------------------------------------------------------------


def page_maps(seen, fresh, free, table, max_tokens, page_size):
    """Request by request, token by token."""
    seen, fresh = [int(v) for v in seen], [int(v) for v in fresh]
    R, width = table.shape
    table = table.copy()
    offsets, context = np.zeros(R + 1, np.int32), np.zeros(R, np.int32)
    request, position, slot = (np.full(max_tokens, -1, np.int32) for _ in range(3))
    tokens = needs = taken = shorts = 0
    for r in range(R):
        begin, tokens = tokens, tokens + max(0, fresh[r])
        fits = min(seen[r], fresh[r]) >= 0 and max(seen[r], fresh[r]) <= 1 << 30 and tokens <= max_tokens
        have, want = -(-seen[r] // page_size), -(-(seen[r] + fresh[r]) // page_size)
        fits = fits and want <= width
        first = needs
        if fits:
            needs += want - have
        ok = fits and (want == have or needs <= len(free))
        if ok:
            for j in range(have, want):
                table[r, j] = free[len(free) - 1 - (first + j - have)]
            taken += want - have
            context[r] = seen[r] + fresh[r]
        else:
            shorts += 1
        for i in range(max(0, min(tokens, max_tokens) - begin)):
            request[begin + i] = r
            if ok:
                p = seen[r] + i
                position[begin + i] = p
                page = int(table[r, p // page_size])
                s = page * page_size + p % page_size
                slot[begin + i] = s if page >= 0 and s < 2 ** 31 else -1
        offsets[r + 1] = min(tokens, max_tokens)
    return {"table": table, "offsets": offsets, "context": context, "request": request, "position": position, "slot": slot,
            "totals": np.array([min(tokens, max_tokens), taken, shorts], np.int32)}


def row_bytes(kv, rope):
    return -(-17 * (kv // 32 + -(-rope // 32)) // 16) * 16


def encode(x, kv, rope):
    """Rows [n, kv + rope] as bytes of the cache."""
    n, nb = x.shape[0], kv // 32 + -(-rope // 32)
    b = np.zeros((n, nb * 32))
    b[:, :kv + rope] = x
    negative = np.zeros((n, nb * 32), np.uint8)
    negative[:, :kv + rope] = np.signbit(x)
    b, negative = b.reshape(n, nb, 32), negative.reshape(n, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    amax = np.abs(np.where(bad[..., None], 0.0, b)).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(amax > 0, np.frexp(amax)[1] - 3, -1000)  # 2^(e + 2) <= amax < 2^(e + 3)
    e = np.clip(np.where(amax > 7 * np.exp2(e.astype(float)), e + 1, e), -23, 13)
    y = np.abs(np.where(bad[..., None], 0.0, b)) / np.exp2(e.astype(float))[..., None]
    code = np.zeros(y.shape, np.uint8)
    for c in range(1, 8):
        middle = (MAGNITUDES[c - 1] + MAGNITUDES[c]) / 2
        code = np.where((y > middle) | ((y == middle) & (c % 2 == 0)), c, code).astype(np.uint8)
    code |= negative << 3
    code[bad] = 0
    code = code.reshape(n, nb * 16, 2)
    rows = np.zeros((n, row_bytes(kv, rope)), np.uint8)
    rows[:, :nb * 16] = code[..., 0] | code[..., 1] << 4
    rows[:, nb * 16:nb * 17] = np.where(bad, 255, e + 127)
    return rows


def decode(rows, kv, rope):
    nb = kv // 32 + -(-rope // 32)
    code = np.stack([rows[:, :nb * 16] & 15, rows[:, :nb * 16] >> 4], -1).reshape(len(rows), nb, 32)
    byte = rows[:, nb * 16:nb * 17].astype(float)
    v = np.where(code & 8, -1.0, 1.0) * MAGNITUDES[code & 7] * np.exp2(byte - 127)[..., None]
    v[rows[:, nb * 16:nb * 17] == 255] = np.nan
    return v.reshape(len(rows), nb * 32)[:, :kv + rope]


def attend(q_abs, q_pe, rows, table, offsets, context, page_size, scale):
    """(results [n, H, kv], largest |score|): token by token; pages outside the pool are left out."""
    n, H, kv = q_abs.shape
    rope, n_pages = q_pe.shape[2], len(rows) // page_size
    out, largest = np.zeros((n, H, kv)), 0.0
    for r in range(len(context)):
        t0, t1 = int(offsets[r]), int(offsets[r + 1])
        ctx = min(int(context[r]), table.shape[1] * page_size)
        if t1 == t0 or ctx <= 0:
            continue
        p = np.arange(ctx)
        page = table[r, p // page_size].astype(np.int64)
        on = (page >= 0) & (page < n_pages)
        v = decode(rows[np.where(on, page, 0) * page_size + p % page_size], kv, rope)
        for t in range(t0, t1):
            keep = on & (p <= int(context[r]) - (t1 - t0) + t - t0)
            if not keep.any():
                continue
            k = v[keep]
            s = scale * np.concatenate([q_abs[t], q_pe[t]], 1).astype(np.float64) @ k.T
            if np.isfinite(s).all():
                largest = max(largest, np.abs(s).max())
            e = np.exp(s - s.max(-1, keepdims=True))
            out[t] = e @ k[:, :kv] / e.sum(-1, keepdims=True)
    return out, largest


def logprobs(x, given, top):
    x = x.astype(np.float64)
    n, V = x.shape
    lp, ent = np.full(given.shape, np.nan), np.full(n, np.nan)
    ids, tlp = np.full((n, top), -1, np.int32), np.full((n, top), np.nan)
    for i in range(n):
        inside = (given[i] >= 0) & (given[i] < V)
        m = x[i].max()
        if not m < np.inf:  # a NaN, or +inf
            continue
        if m == -np.inf:
            lp[i, inside], ent[i], tlp[i] = -np.inf, 0.0, -np.inf
            continue
        e = np.exp(x[i] - m)
        im = int(x[i].argmax())
        rest = e.sum() - e[im] if e.sum() > 1.5 else np.delete(e, im).sum()
        ls = np.log1p(rest)
        lp[i, inside] = x[i][given[i][inside]] - m - ls
        on = e > 0
        ent[i] = ls + (e[on] * (m - x[i][on])).sum() / (1 + rest)
        order = np.lexsort((np.arange(V), -x[i]))[:top]
        ids[i, :len(order)] = order
        tlp[i] = -np.inf
        tlp[i, :len(order)] = x[i][order] - m - ls
    return lp, ent, ids, tlp


# ---- on the device -----------------------------------------------------------------------------


class Arrays:
    """Device copies of numpy arrays by name; .p(name) their addresses, .get(name) them back."""

    def __init__(self, **arrays):
        self.host = {k: np.ascontiguousarray(v) for k, v in arrays.items()}
        self.dev = {k: gmoe.DeviceArray.from_numpy(v) for k, v in self.host.items()}

    def p(self, name, offset=0):
        return self.dev[name].ptr.value + offset

    def get(self, name):
        return self.dev[name].download(self.host[name].shape, self.host[name].dtype)

    def put(self, name, value):
        self.dev[name].upload(np.ascontiguousarray(value, self.host[name].dtype))


OUTPUTS = ("offsets", "context", "request", "position", "slot", "totals")


def batch_arrays(seen, fresh, page_size, rng, extra_pages=3, max_tokens=None, width=None, free=None, gap=0):
    """Host arrays of a batch: a pool of pages in random order, the tables of what is cached."""
    seen, fresh = np.asarray(seen, np.int64), np.asarray(fresh, np.int64)
    R = len(seen)
    have, want = -(-seen // page_size), -(-(seen + fresh) // page_size)
    if width is None:
        width = max(1, int(want.max()) + gap)
    n_pages = int(want.sum()) + extra_pages
    ids = rng.permutation(n_pages).astype(np.int32)
    table = np.full((R, width), -1, np.int32)
    at = 0
    for r in range(R):
        table[r, :min(width, have[r])] = ids[at:at + have[r]][:width]
        at += have[r]
    rest = ids[at:] if free is None else ids[at:at + free]
    if max_tokens is None:
        max_tokens = max(1, int(fresh.sum()) + 3)
    a = {"seen": seen.astype(np.int32), "fresh": fresh.astype(np.int32),
         "free_pages": rest if len(rest) else np.zeros(1, np.int32), "n_free": np.array([len(rest)], np.int32), "table": table}
    sizes = dict(offsets=R + 1, context=R, request=max_tokens, position=max_tokens, slot=max_tokens, totals=3)
    a.update({k: np.full(v, -77, np.int32) for k, v in sizes.items()})
    return a, rest, n_pages, max_tokens


def make_batch(arrays, dev, max_tokens, page_size):
    R, width = arrays["table"].shape
    return gmoe.Batch(R, max_tokens, width, page_size, **{k: dev.p(k) for k in gmoe._BATCH_ARRAYS})


def capture(stream, call):
    """`call` captured into a graph, ready to launch."""
    hip = gmoe.hip()
    gmoe.hip_check(hip.hipStreamBeginCapture(stream.h, 0), "hipStreamBeginCapture")
    call()
    graph, exe = C.c_void_p(), C.c_void_p()
    gmoe.hip_check(hip.hipStreamEndCapture(stream.h, C.byref(graph)), "hipStreamEndCapture")
    gmoe.hip_check(hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0), "hipGraphInstantiate")
    return exe


def sync():
    gmoe.hip_check(gmoe.hip().hipDeviceSynchronize(), "hipDeviceSynchronize")
