"""The operators of a serving step over several requests, as timed cases: page tables and slot
maps from request lengths, latent rows written to a paged cache in 4 bits, MLA attention over
that cache, and log probabilities of given tokens with entropy and top alternatives.

The cache's form. A position's row is kv_lora_rank + rope_dim values (the rope part padded
with zeros to whole blocks) in blocks of 32 columns: the e2m1 codes, two a byte (the even
column in the low half), then one scale byte a block (2^(byte - 127)), padded to 16 bytes.
A block's scale is the power of two that puts its largest magnitude in (3.5, 7] steps, within
2^-23 .. 2^13, and each value is the nearest code, ties to the even code, at most 6 steps.
"""
import math
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
VOCAB = 154880  # GLM-4.7-Flash's
MAG = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # e2m1 magnitudes by code
BYTE_LO, BYTE_HI = 104, 140  # scales of 2^-23 .. 2^13

own = False


def _package():
    sys.path.insert(0, os.path.join(ROOT, "glm.c_amd"))
    import gmoe

    return gmoe


def listed():
    return [
        # one sequence's next token: the smallest call, where latency counts
        {"name": "maps_1", "op": "maps", "R": 1, "kind": "decode", "len": 4096, "P": 64},
        # a decode step of a middling batch
        {"name": "maps_64", "op": "maps", "R": 64, "kind": "decode", "len": 8192, "P": 64},
        # many requests, one in sixteen with a prompt chunk, some idle, the pool too small for all
        {"name": "maps_1000_mixed", "op": "maps", "R": 1000, "kind": "mixed", "len": 2048, "P": 16},
        # a decode batch's new latent rows, one a request
        {"name": "append_64", "op": "append", "n": 64, "kv": 512, "rope": 64, "P": 64},
        # a long prompt's rows at once, an odd number
        {"name": "append_8191", "op": "append", "n": 8191, "kv": 512, "rope": 64, "P": 64},
        # one long sequence's decode: few rows, the cache split over the GPU
        {"name": "attend_1", "op": "attend", "R": 1, "kind": "decode", "len": 4097, "H": 20, "kv": 512, "rope": 64, "P": 64},
        # a decode batch of ragged lengths, from a few positions to 8192
        {"name": "attend_64_ragged", "op": "attend", "R": 64, "kind": "decode", "len": 8192, "H": 20, "kv": 512, "rope": 64,
         "P": 64},
        # a prompt chunk beside decoding requests
        {"name": "attend_mixed", "op": "attend", "R": 17, "kind": "mixed", "len": 2048, "H": 20, "kv": 512, "rope": 64,
         "P": 16},
        # a prompt's later batch, of odd length
        {"name": "attend_prompt_1023", "op": "attend", "R": 1, "kind": "prompt", "fresh": 1023, "len": 4000, "H": 20,
         "kv": 512, "rope": 64, "P": 128},
        # one token's scores after a decode step
        {"name": "logprobs_1", "op": "logprobs", "n": 1, "V": VOCAB, "top": 20, "given": 1, "ld": VOCAB},
        # a decode batch's
        {"name": "logprobs_64", "op": "logprobs", "n": 64, "V": VOCAB, "top": 5, "given": 1, "ld": VOCAB},
        # a scored prompt's rows, an odd vocabulary in wider rows
        {"name": "logprobs_801", "op": "logprobs", "n": 801, "V": 151551, "top": 1, "given": 4, "ld": 151555},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["maps", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    P = rng.choice([16, 32, 64, 128])
    if op == "maps":
        return {"op": op, "R": _log(rng, 1, 1000), "kind": rng.choice(["decode", "mixed"]), "len": _log(rng, 16, 2048), "P": P}
    kv, rope = rng.choice([(512, 64), (512, 64), (512, 64), (256, 32), (64, 16)])
    if op == "append":
        return {"op": op, "n": _log(rng, 1, 8191), "kv": kv, "rope": rope, "P": P}
    if op == "attend":
        H = rng.choice([4, 16, 20, 20, 20, 32])
        kind = rng.choice(["decode", "decode", "mixed", "prompt"])
        if kind == "prompt":
            fresh = _log(rng, 2, 640)
            c = {"R": 1, "fresh": fresh, "len": fresh + rng.choice([0, _log(rng, 1, 3000)])}
        elif kind == "mixed":
            c = {"R": rng.randint(2, 16), "len": _log(rng, 64, 2000)}
        else:
            c = {"R": _log(rng, 1, 64), "len": _log(rng, 1, 5000)}
        return {"op": op, "kind": kind, **c, "H": H, "kv": kv, "rope": rope, "P": P}
    V = rng.choice([VOCAB, _log(rng, 300, VOCAB)])
    return {"op": op, "n": _log(rng, 1, 790), "V": V, "top": rng.choice([0, 1, 5, 20, 32]), "given": rng.choice([1, 1, 1, 3]),
            "ld": V + rng.choice([0, 0, 1, 4])}


# ---- inputs --------------------------------------------------------------------------------


def _gen(seed, *key):
    s = 29 + seed
    for k in key:
        s = (s * 1000003 + int(k) + 1) % (1 << 62)
    g = torch.Generator(device=DEV)
    g.manual_seed(s)
    return g


def _lengths(case):
    """(seen, fresh) of every request: of the case alone, so that its work is known."""
    R, L, kind = case["R"], case["len"], case["kind"]
    r = np.random.default_rng(1000 * R + L)
    if kind == "prompt":
        return np.array([L - case["fresh"]]), np.array([case["fresh"]])
    total = np.exp(r.uniform(math.log(min(8, L)), math.log(L), R)).round().astype(np.int64).clip(1, L)
    total[0] = L
    fresh = np.ones(R, np.int64)
    if kind == "mixed":
        fresh[r.permutation(R)[:max(1, R // 16)]] = 301  # a prompt's chunk
        fresh[r.random(R) < 0.05] = 0  # idle in this step
        fresh = np.minimum(fresh, total)
    return total - fresh, fresh


def _i32(a):
    return torch.from_numpy(np.asarray(a).astype(np.int32)).to(DEV)


def _row_bytes(kv, rope):
    blocks = kv // 32 + (rope + 31) // 32
    return (17 * blocks + 15) // 16 * 16


def _requests(case, seed):
    """The lengths, a pool of pages in random order and the tables of what is cached already."""
    P = case["P"]
    seen, fresh = _lengths(case)
    R = len(seen)
    have, want = -(-seen // P), -(-(seen + fresh) // P)
    width = int(want.max()) + 3
    n_pages = int(want.sum()) + 7
    ids = np.random.default_rng(seed).permutation(n_pages)
    table = np.full((R, width), -1)
    at = 0
    for r in range(R):
        table[r, :have[r]] = ids[at:at + have[r]]
        at += have[r]
    free = ids[at:]
    if case["op"] == "maps" and case["kind"] == "mixed":  # too few pages for the last requests
        free = free[:max(1, (want - have).sum() * 9 // 10)]
    return {"seen": _i32(seen), "fresh": _i32(fresh), "free": _i32(free), "n_free": _i32([len(free)]), "table": _i32(table),
            "R": R, "width": width, "P": P, "n_pages": n_pages, "max_tokens": int(fresh.sum()) + 5,
            "max_len": int((seen + fresh).max()), "max_fresh": int(fresh.max())}


def _logits(case, seed):
    """Logits of a language model's kind (a few likely tokens over a wide bulk), one row in
    eight under a mask that leaves a hundredth of the vocabulary and what is likely or given, by
    -inf or the lowest value."""
    g = _gen(seed, 5)
    n, V = case["n"], case["V"]
    x = torch.empty(n, case["ld"], device=DEV)
    x.normal_(0.0, 2.0, generator=g)
    for row in range(1, n, 8):
        low = -math.inf if row % 16 == 1 else torch.finfo(torch.float32).min
        x[row].masked_fill_(torch.rand(case["ld"], generator=g, device=DEV) > 0.01, low)
    peak = torch.randint(0, V, (n, 8), generator=g, device=DEV)
    given = torch.randint(0, V, (n, case["given"]), generator=g, device=DEV)
    x.scatter_(1, given, 2.0 * torch.randn(n, case["given"], generator=g, device=DEV))
    x.scatter_(1, peak, 12.0 + 4.0 * torch.randn(n, 8, generator=g, device=DEV))
    given[:, 0] = peak[:, 0]
    given = given.int()
    return x, given


def prepare(case, seed):
    s = {"case": case}
    if case["op"] == "maps":
        s.update(_requests(case, seed))
        R, T = s["R"], s["max_tokens"]
        for name, n in (("offsets", R + 1), ("context", R), ("request", T), ("position", T), ("slot", T), ("totals", 3)):
            s[name] = torch.zeros(n, dtype=torch.int32, device=DEV)
    elif case["op"] == "append":
        n, kv, rope, P = case["n"], case["kv"], case["rope"], case["P"]
        s["n_pages"] = n // P + 3
        # the rows as the model has them: entry and rope part side by side
        s["kv_a"] = _latent(case, n, seed)
        s["slot"] = torch.randperm(s["n_pages"] * P, generator=_gen(seed, 2), device=DEV)[:n].int()
        s["rows"] = torch.zeros(s["n_pages"] * P, _row_bytes(kv, rope), dtype=torch.uint8, device=DEV)
        s["comp"], s["pe"] = torch.empty(n, kv, device=DEV), torch.empty(n, rope, device=DEV)
    elif case["op"] == "attend":
        s.update(_attend_inputs(case, seed))
    else:
        s["x"], s["given"] = _logits(case, seed)
        n, k = case["n"], case["top"]
        s["logprob"] = torch.empty(n, case["given"], device=DEV)
        s["entropy"] = torch.empty(n, device=DEV)
        s["top_id"] = torch.empty(n, k, dtype=torch.int32, device=DEV)
        s["top_logprob"] = torch.empty(n, k, device=DEV)
    return s


def _latent(case, n, seed):
    """Latent rows: normalised entries of uneven columns, rope parts twice as large."""
    g = _gen(seed, 1)
    kv, rope = case["kv"], case["rope"]
    gain = torch.cat([1 + 0.3 * torch.randn(kv, generator=g, device=DEV), 2 * torch.ones(rope, device=DEV)])
    return torch.randn(n, kv + rope, generator=g, device=DEV) * gain


def _attend_inputs(case, seed):
    s = _requests(case, seed)
    kv, rope, H = case["kv"], case["rope"], case["H"]
    n_slots = s["n_pages"] * s["P"]
    s["rows"] = torch.cat([_encode(_latent(case, min(65536, n_slots - i), seed + i), kv, rope) for i in range(0, n_slots, 65536)])
    full = _maps_plain(s)
    s.update({k: full[k] for k in ("table", "offsets", "context")})
    n = int(full["totals"][0])
    s["n"] = n
    g = _gen(seed, 3)
    s["scale"] = 1 / math.sqrt(256)
    sigma = 2.5 / (s["scale"] * math.sqrt(kv + rope))  # scores of standard deviation 2.5
    s["q_abs"] = sigma * torch.randn(n, H, kv, generator=g, device=DEV)
    s["q_pe"] = sigma / 2 * torch.randn(n, H, rope, generator=g, device=DEV)
    s["out"] = torch.empty(n, H, kv, device=DEV)
    return s


# ---- the plain forms -----------------------------------------------------------------------


def _maps_plain(s):
    seen, fresh, P, T = s["seen"].long(), s["fresh"].long(), s["P"], s["max_tokens"]
    R, width, n_free = s["R"], s["width"], s["n_free"].long()
    have, want = (seen + P - 1) // P, (seen + fresh + P - 1) // P
    ends = fresh.cumsum(0)
    starts = ends - fresh
    fits = (ends <= T) & (want <= width)
    need = torch.where(fits, want - have, 0)
    cum = need.cumsum(0)
    ok = fits & ((need == 0) | (cum <= n_free))
    first = n_free - 1 - (cum - need)  # the request's first page in the pool
    j = torch.arange(width, device=DEV).unsqueeze(0)
    new = (j >= have[:, None]) & (j < want[:, None]) & ok[:, None]
    at = (first[:, None] - (j - have[:, None])).clamp(0, s["free"].numel() - 1)
    table = torch.where(new, s["free"][at], s["table"])
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(ends, t, right=True)
    there = r < R
    r = r.clamp_max(R - 1)
    served = there & ok[r]
    position = torch.where(served, seen[r] + t - starts[r], -1)
    page = table[r, (position // P).clamp_min(0)].long()
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), ends]).clamp_max(T)
    taken = torch.where(ok, need, 0).sum()
    totals = torch.stack([offsets[-1], taken, (~ok).sum()])
    i32 = {"table": table, "offsets": offsets, "context": torch.where(ok, seen + fresh, 0),
           "request": torch.where(there, r, -1), "position": position,
           "slot": torch.where(served, page * P + position % P, -1), "totals": totals}
    return {k: v.int() for k, v in i32.items()}


def _encode(x, kv, rope):
    """[n, kv + rope] fp32 to rows of the cache."""
    n, pad = x.shape[0], -rope % 32
    b = torch.nn.functional.pad(x, (0, pad)).view(n, -1, 32)
    amax = b.abs().amax(-1)
    byte = ((amax.view(torch.int32) + 0x1FFFFF) >> 23).sub(2).clamp(BYTE_LO, BYTE_HI)
    steps = b * torch.exp2((127 - byte).float()).unsqueeze(-1)
    mag = steps.abs()
    # codes up to 2 in halves, to 4 in ones, then in twos: round() takes ties to even
    code = torch.where(mag < 1.75, (2 * mag).round(), torch.where(mag < 3.5, 2 + mag.round(), (4 + (mag / 2).round()).clamp_max(7)))
    code = (code.int() | (steps.view(torch.int32) >> 28 & 8)).view(n, -1, 2)
    packed = code[..., 0] | code[..., 1] << 4
    rows = torch.cat([packed, byte], 1)
    return torch.nn.functional.pad(rows, (0, _row_bytes(kv, rope) - rows.shape[1])).to(torch.uint8)


def _decode(rows, kv, rope, dtype=torch.float32):
    """Rows of the cache to [.., kv + rope] values."""
    cols = kv + (rope + 31) // 32 * 32
    codes = rows[..., :cols // 2]
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    values = torch.tensor(MAG + tuple(-v for v in MAG), dtype=dtype, device=rows.device)[codes]
    scale = torch.exp2(torch.arange(256, dtype=dtype, device=rows.device) - 127)[rows[..., cols // 2:cols // 2 + cols // 32].long()]
    return (values.unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)[..., :kv + rope]


def _append_plain(s):
    kv, rope = s["case"]["kv"], s["case"]["rope"]
    slot = s["slot"].long()
    s["rows"][slot] = _encode(s["kv_a"], kv, rope)
    back = _decode(s["rows"][slot], kv, rope)
    return {"comp": back[:, :kv].contiguous(), "pe": back[:, kv:].contiguous()}


def _attend_plain(s):
    c = s["case"]
    H, kv, rope, P, R, L, F = c["H"], c["kv"], c["rope"], s["P"], s["R"], s["max_len"], s["max_fresh"]
    offsets, context = s["offsets"].long(), s["context"].long()
    starts, fresh = offsets[:-1], offsets[1:] - offsets[:-1]
    pos = torch.arange(L, device=DEV)
    page = s["table"][:, pos // P].long().clamp_min(0)
    k = _decode(s["rows"][page * P + pos % P], kv, rope)  # [R, L, kv + rope]
    i = torch.arange(F, device=DEV)
    token = (starts[:, None] + i).clamp_max(s["n"] - 1)  # [R, F]
    q = torch.cat([s["q_abs"], s["q_pe"]], -1)[token].flatten(1, 2)  # [R, F H, kv + rope]
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s["scale"]).view(R, F, H, L)
    last = context[:, None] - fresh[:, None] + i  # the token's own position
    p.masked_fill_((pos > last[..., None])[:, :, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(R, F * H, L), k[..., :kv]).view(R, F, H, kv) / total
    return out[i < fresh[:, None]]


def _keys(x):
    """Unique integers in the order of the values, the lower index first among equals."""
    b = x.view(torch.int32) if x.is_contiguous() else x.contiguous().view(torch.int32)
    b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
    return b * (1 << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))


def _logprobs_plain(s):
    c = s["case"]
    x = s["x"][:, :c["V"]]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    lse = total.log()
    d.mul_(e).masked_fill_(e == 0, 0)  # e (x - m), none where e vanishes
    entropy = (lse - d.sum(-1, keepdim=True) / total)[:, 0]
    top = _keys(x).topk(c["top"], -1).indices if c["top"] else torch.empty(c["n"], 0, dtype=torch.long, device=DEV)
    return {"logprob": x.gather(1, s["given"].long()) - m - lse, "entropy": entropy, "top_id": top.int(),
            "top_logprob": x.gather(1, top) - m - lse}


# ---- the framework's operators -------------------------------------------------------------


def _batch(s):
    gmoe = _package()
    names = ("seen", "fresh", "free", "n_free", "table", "offsets", "context", "request", "position", "slot", "totals")
    return gmoe.Batch(s["R"], s["max_tokens"], s["width"], s["P"], **{k: s[k].data_ptr() for k in names if k in s})


def _own(s):
    """The calls of a user's program; its objects are made at the first pass and kept."""
    c = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "maps":
        if "batch" not in s:
            s["batch"] = _batch(s)
        s["batch"].maps(stream=stream)
        return {k: s[k] for k in ("table", "offsets", "context", "request", "position", "slot", "totals")}
    if c["op"] in ("append", "attend") and "cache" not in s:
        s["cache"] = _package().Cache4(s["rows"].data_ptr(), c["kv"], c["rope"], s["n_pages"], c["P"])
    if c["op"] == "append":
        x, n, kv, ld = s["kv_a"].data_ptr(), c["n"], c["kv"], s["kv_a"].stride(0)
        s["cache"].append(n, x, ld, x + 4 * kv, ld, s["slot"].data_ptr(), stream=stream)
        s["cache"].read(n, s["slot"].data_ptr(), s["comp"].data_ptr(), kv, s["pe"].data_ptr(), c["rope"], stream=stream)
        return {"comp": s["comp"], "pe": s["pe"]}
    if c["op"] == "attend":
        if "batch" not in s:
            s["batch"] = _batch(s)
            s["work"] = torch.empty(s["cache"].attend_workspace(c["H"]), dtype=torch.uint8, device=DEV)
        s["cache"].attend(s["batch"], c["H"], s["scale"], s["q_abs"].data_ptr(), c["H"] * c["kv"], s["q_pe"].data_ptr(),
                          c["H"] * c["rope"], s["out"].data_ptr(), c["H"] * c["kv"], s["work"].data_ptr(), s["work"].numel(),
                          stream=stream)
        return s["out"]
    if "scorer" not in s:
        s["scorer"] = _package().LogProbs(c["n"], c["V"], c["top"], c["given"])
        s["work"] = torch.empty(s["scorer"].workspace, dtype=torch.uint8, device=DEV)
    s["scorer"](s["x"].data_ptr(), c["ld"], s["given"].data_ptr(), s["logprob"].data_ptr(), s["entropy"].data_ptr(),
                s["top_id"].data_ptr(), s["top_logprob"].data_ptr(), s["work"].data_ptr(), s["work"].numel(), stream=stream)
    return {k: s[k] for k in ("logprob", "entropy", "top_id", "top_logprob")}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "maps":
        return _maps_plain(state)
    if op == "append":
        return _append_plain(state)
    return _attend_plain(state) if op == "attend" else _logprobs_plain(state)


def work(case):
    if case["op"] == "logprobs":
        n, V = case["n"], case["V"]
        return {"bytes": 4 * n * V + 8 * n * (case["top"] + case["given"]) + 4 * n, "flops": 5 * n * V}
    if case["op"] == "append":  # the values in and back out, the rows written and read
        n, cols = case["n"], case["kv"] + case["rope"]
        return {"bytes": n * (8 * cols + 2 * _row_bytes(case["kv"], case["rope"]) + 8), "flops": 6 * n * cols}
    seen, fresh = _lengths(case)
    P = case["P"]
    have, want = -(-seen // P), -(-(seen + fresh) // P)
    n, R = int(fresh.sum()), len(seen)
    if case["op"] == "maps":  # lengths, new pages, each row's last old page; the arrays written
        return {"bytes": int(4 * (3 * R + 2 * (want - have).sum() + 2 * R + 3 * n + 4)), "flops": 10 * (R + n)}
    H, kv, rope = case["H"], case["kv"], case["rope"]
    row = 17 * (kv // 32 + (rope + 31) // 32)
    live = fresh > 0
    pairs = int((fresh * seen + fresh * (fresh + 1) // 2).sum())
    return {"bytes": int(((seen + fresh)[live]).sum()) * row + 4 * n * H * (2 * kv + rope) + 4 * int(want.sum()),
            "flops": 2 * pairs * H * (2 * kv + rope)}


# ---- the same in 64 bits -------------------------------------------------------------------


def _exact_rows(x, kv, rope):
    """The values that the cache stands for: each block's scale and each value's nearest step."""
    n, cols = x.shape
    b = torch.zeros(n, (cols + 31) // 32 * 32, dtype=torch.float64, device=x.device)
    b[:, :cols] = x.double()
    b = b.view(n, -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(amax.clamp_min(1e-300))) - 2
    e = torch.where(amax > 7 * 2.0 ** e, e + 1, e).clamp(-23, 13)
    y = b / 2.0 ** e
    steps = torch.tensor(MAG, dtype=torch.float64, device=x.device)
    best = torch.zeros_like(y)
    for code in range(1, 8):  # over the middle of two steps, or on it where the upper code is even
        middle = (steps[code - 1] + steps[code]) / 2
        best = torch.where((y.abs() > middle) | ((y.abs() == middle) & (code % 2 == 0)), steps[code], best)
    return (best * y.sign() * 2.0 ** e).view(n, -1)[:, :cols]


def exact(case, seed):
    if case["op"] == "maps":
        return None
    if case["op"] == "append":
        kv = case["kv"]
        v = _exact_rows(_latent(case, case["n"], seed), kv, case["rope"])
        return {"comp": v[:, :kv].contiguous(), "pe": v[:, kv:].contiguous()}
    if case["op"] == "logprobs":
        x, given = _logits(case, seed)
        out = {"logprob": [], "entropy": [], "top_id": None, "top_logprob": []}
        for at in range(0, case["n"], 64):
            v = x[at:at + 64, :case["V"]].double()
            lp = v - torch.logsumexp(v, -1, keepdim=True)
            out["logprob"].append(lp.gather(1, given[at:at + 64].long()))
            out["entropy"].append(torch.special.entr(lp.exp()).sum(-1))
            out["top_logprob"].append(lp.topk(case["top"], -1).values)
        return {k: None if v is None else torch.cat(v) for k, v in out.items()}
    s = _attend_inputs(case, seed)
    seen, fresh = _lengths(case)
    kv, rope, P = case["kv"], case["rope"], case["P"]
    out, t = [], 0
    for r in range(len(seen)):
        n = int(seen[r] + fresh[r])
        pages = s["table"][r, :-(-n // P)].long()
        rows = s["rows"].view(-1, P, s["rows"].shape[1])[pages].flatten(0, 1)[:n]
        k = _decode(rows, kv, rope, torch.float64)
        for a in range(0, int(fresh[r]), 128):  # a token block: the positions up to its last
            b = min(a + 128, int(fresh[r]))
            q = torch.cat([s["q_abs"][t + a:t + b], s["q_pe"][t + a:t + b]], -1).double()
            m = int(seen[r]) + b
            p = (q.flatten(0, 1) @ k[:m].T.contiguous() * s["scale"]).view(b - a, -1, m)
            later = torch.arange(m, device=DEV) > torch.arange(int(seen[r]) + a, m, device=DEV)[:, None]
            p = p.masked_fill(later[:, None], -math.inf).softmax(-1)
            out.append((p.flatten(0, 1) @ k[:m, :kv]).view(b - a, -1, kv))
        t += int(fresh[r])
    return torch.cat(out)
