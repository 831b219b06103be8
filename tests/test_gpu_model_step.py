"""Steps of several requests through a whole model (gmoe_model_step): page tables, 4-bit cache,
attention, products, MoE layers, LM head and log probabilities together, against the same model
in 64 bits with numpy (its cached rows rounded by serve_ref's encoding; its MoE layers by the oracle in
fp32).

Rounding to 4 bits is a step function: the comparison holds if no cached value is so near the middle
of two magnitudes that fp32 could round it the other way. So the 64-bit model is also run in fp32, and
16 times the largest difference of the two (numpy's sums and the kernels' round in different orders, both
by halves of 2^-23 an operation) must be less than the smallest distance from a middle, which picks the seeds
here on the CPU, and bounds what the results may be off by."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import gmoe
import oracle
import serve_ref as ref

SHAPE = gmoe.Shape(dim=256, moe_ffn_dim=256, n_routed_experts=8, n_experts_used=2)
CFG = dict(dim=256, hidden_dim=96, n_layers=3, n_heads=3, vocab_size=130, q_lora_rank=64, kv_lora_rank=64, rope_dim=8,
           qk_nope_dim=32, head_k_dim=40, v_head_dim=32, group_size=32, cache_cap=40, attn_layers=3, has_l0_ffn=1, max_batch=16)
ONE = dict(CFG, n_layers=1, attn_layers=1, has_l0_ffn=0, max_batch=80, cache_cap=96, group_size=16)
MIDDLES = (ref.MAGNITUDES[1:] + ref.MAGNITUDES[:-1]) / 2


class Plain:
    """The model with its products in `kind`; requests' rows as the cache's bytes."""

    def __init__(self, cfg, g, attn, moe, kind):
        self.c, self.kind, self.moe = cfg, kind, moe
        w = lambda d, n: (d[n + "_q"].reshape(*d[n + "_s"].shape, -1) * d[n + "_s"].astype(np.float64)[..., None]).reshape(
            d[n + "_q"].shape).astype(kind)
        self.g = {n: w(g, n) for n in ("tok", "out")}
        self.ffn = [w(g, "l0_ffn_" + n) for n in ("gate", "up", "down")] if cfg["has_l0_ffn"] else None
        self.norms = {n: v.astype(kind) for n, v in g.items() if n.endswith("norm")}
        self.attn = [dict({n: w(a, n) for n in ("q_a", "q_b", "kv_a", "k_b", "v_b", "attn_out")},
                          **{n: a[n].astype(kind) for n in ("attn_norm", "q_a_norm", "kv_a_norm")}) for a in attn]
        self.rows = {}
        self.scaled, self.margin = [], np.inf

    def norm(self, x, weight):
        return x / np.sqrt((x * x).mean(dtype=self.kind) + self.kind(1e-5)) * weight

    def turn(self, x, p):
        rope = self.c["rope_dim"]
        i = np.arange(0, rope, 2, dtype=np.float32)
        angle = np.float32(p) * np.power(np.float32(1e6), -(i / np.float32(rope)), dtype=np.float32)
        c, s = np.cos(angle.astype(np.float64)).astype(self.kind), np.sin(angle.astype(np.float64)).astype(self.kind)
        out = np.empty_like(x)
        out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
        out[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
        return out

    def store(self, entry, key):
        kv, rope = self.c["kv_lora_rank"], self.c["rope_dim"]
        row = ref.encode(entry[None].astype(np.float64), kv, rope)
        blocks = kv // 32 + 1  # rope_dim is 32 at most
        scales = np.repeat(np.exp2(row[0, blocks * 16:blocks * 17].astype(float) - 127), 32)[:kv + rope]
        y = np.abs(entry) / scales
        self.scaled.append(y)
        # from a middle of two magnitudes, and of a block's largest from where its scale changes
        self.margin = min(self.margin, np.abs(y[:, None] - MIDDLES).min(),
                          *(min(b.max() - 3.5, 7 - b.max()) for b in np.split(y, range(32, kv + 1, 32))))
        self.rows.setdefault(key, []).append(row[0])
        return ref.decode(np.array(self.rows[key]), kv, rope).astype(self.kind)

    def token(self, request, p, token):
        c = self.c
        kv, H, nope = c["kv_lora_rank"], c["n_heads"], c["qk_nope_dim"]
        x = self.g["tok"][token]
        for l, a in enumerate(self.attn):
            h = self.norm(x, a["attn_norm"])
            q = (a["q_b"] @ self.norm(a["q_a"] @ h, a["q_a_norm"])).reshape(H, -1)
            k = a["kv_a"] @ h
            v = self.store(np.concatenate([self.norm(k[:kv], a["kv_a_norm"]), self.turn(k[kv:], p)]), (request, l))
            absorbed = np.stack([a["k_b"][i * kv:(i + 1) * kv] @ q[i, :nope] for i in range(H)])
            s = self.kind(c["head_k_dim"] ** -0.5) * np.concatenate([absorbed, self.turn(q[:, nope:], p)], 1) @ v.T
            e = np.exp(s - s.max(1, keepdims=True))
            ctx = e @ v[:, :kv] / e.sum(1, keepdims=True)
            x = x + a["attn_out"] @ (a["v_b"].reshape(H, -1, kv) @ ctx[..., None]).reshape(-1)
            if l == 0 and self.ffn:
                h = self.norm(x, self.norms["l0_ffn_norm"])
                u = self.ffn[0] @ h
                x = x + self.ffn[2] @ (u / (1 + np.exp(-u)) * (self.ffn[1] @ h))
            if l > 0:
                added = oracle.Oracle("port").layer(SHAPE, self.moe[l], x.astype(np.float32)[None])
                x = x + (added["shared_out"][0].astype(self.kind) + added["routed_out"][0])
        return self.g["out"] @ self.norm(x, self.norms["output_norm"])

    def step(self, seen, fresh, tokens, every):
        """Logits of each row, in the step's order."""
        out, at = [], 0
        for r, n in enumerate(fresh):
            for i in range(n):
                logits = self.token(r, seen[r] + i, tokens[at + i])
                if every or i == n - 1:
                    out.append(logits)
            at += n
        return np.array(out)

    def release(self, request):
        for l in range(len(self.attn)):
            self.rows.pop((request, l), None)


# ("step", new tokens of each request, every token's row) or ("release", request)
MIXED = [("step", [5, 0, 3], False), ("step", [1, 9, 1], False), ("step", [1, 1, 0], True), ("release", 1), ("step", [1, 2], False),
         ("step", [0, 1, 0], False), ("step", [2, 1, 7, 3], True)]
LONG = [("step", [70, 10], True), ("step", [1, 1], False)]
CASES = {"mixed": (CFG, MIXED, 4, 4, 13), "long": (ONE, LONG, 8, 2, 12)}
SEEDS = {"mixed": 8, "long": 8}


def expected(name, seed):
    """(weights, steps [(op, tokens, given, logits)], how far they may be off)."""
    cfg, ops, _, R, _ = CASES[name]
    g, attn = gmoe.synth_model_weights(cfg, seed)
    moe = {l: gmoe.HostLayer(SHAPE, seed=seed, layer=l, norm_mode=gmoe.SYNTH_NORM_RANDOM) for l in range(1, cfg["n_layers"])}
    rng = np.random.default_rng(seed)
    models = [Plain(cfg, g, attn, moe, kind) for kind in (np.float64, np.float32)]
    seen, steps, lost = [0] * R, [], 0.0
    for op in ops:
        if op[0] == "release":
            seen[op[1]] = 0
            for m in models:
                m.release(op[1])
            steps.append((op, None, None, None))
            continue
        _, fresh, every = op
        tokens = rng.integers(0, cfg["vocab_size"], sum(fresh)).astype(np.int32)
        want, single = (m.step(seen, fresh, tokens, every) for m in models)
        lost = max(lost, np.abs(want - single).max())
        steps.append((op, tokens, rng.integers(0, cfg["vocab_size"], len(want)).astype(np.int32), want))
        for r, n in enumerate(fresh):
            seen[r] += n
    off = max(np.abs(a - b).max() for a, b in zip(models[0].scaled, models[1].scaled))
    return g, attn, moe, steps, 16 * lost, 16 * off, models[0].margin


@pytest.mark.parametrize("name", list(CASES))
def test_no_cached_value_is_near_a_middle(name):
    *_, bound, off, margin = expected(name, SEEDS[name])
    assert off < margin and bound < 1e-2, (bound, off, margin)


def open_model(name, g, attn, moe):
    cfg, _, page_size, R, n_pages = CASES[name]
    model, ctx = gmoe.Model(cfg), None
    model.upload(g)
    for l, a in enumerate(attn):
        model.upload_attn(l, a)
    if moe:
        ctx = gmoe.Context(SHAPE, n_layers=cfg["n_layers"], max_tokens=cfg["max_batch"])
        for l, w in moe.items():
            ctx.upload(l, w)
        model.set_moe(ctx, moe)
    model.open_pages(R, page_size, n_pages)
    return model, ctx


@pytest.mark.gpu
@pytest.mark.parametrize("own_stream", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_steps_match_the_model_in_64_bits(name, own_stream):
    cfg, _, P, R, n_pages = CASES[name]
    g, attn, moe, steps, bound, *_ = expected(name, SEEDS[name])
    model, ctx = open_model(name, g, attn, moe)
    stream = gmoe.Stream() if own_stream else None
    st = stream.h if stream else None
    try:
        seen = np.zeros(R, int)
        for i, (op, tokens, given, want) in enumerate(steps):
            print(f"[case] {name} {i}: {op}", flush=True)
            if op[0] == "release":
                model.release(op[1], stream=st)
                seen[op[1]] = 0
            else:
                got = model.step(op[1], tokens, every=op[2], given=given, top=3, logits=True, stream=st)
                seen[:len(op[1])] += op[1]
                assert np.abs(got["logits"] - want).max() <= bound
                lp, ent, ids, tlp = ref.logprobs(got["logits"], given[:, None], 3)
                # the operator on the step's own logits: relative 2^-20 as in its own tests' fp32 sums
                assert np.abs(got["logprob"] - lp[:, 0]).max() <= 2 ** -20 * np.abs(lp).max()
                assert np.abs(got["entropy"] - ent).max() <= 2 ** -20 * np.abs(ent).max()
                assert np.array_equal(got["top_id"], ids)
                assert np.abs(got["top_logprob"] - tlp).max() <= 2 ** -20 * np.abs(lp).max()
            assert model.free_pages() == n_pages - int((-(-seen // P)).sum())
    finally:
        model.close()
        if ctx:
            ctx.close()


@pytest.mark.gpu
def test_refused_steps_change_nothing():
    g, attn, moe, steps, bound, *_ = expected("mixed", SEEDS["mixed"])
    model, ctx = open_model("mixed", g, attn, moe)
    try:
        (op, tokens, given, want) = steps[0]
        first = model.step(op[1], tokens, every=op[2], logits=True)["logits"]
        left = model.free_pages()

        def refused(code, fresh, **k):
            n = sum(max(0, f) for f in fresh)
            b = gmoe.ModelBatch(k.get("n", len(fresh)), 0, k.get("top", 0), np.array(fresh + [0] * 8, np.int32).ctypes.data,
                                np.zeros(n + 1, np.int32).ctypes.data, k.get("given"))
            assert model.lib.gmoe_model_step(model.h, b, None) == code
            assert model.free_pages() == left

        refused(-1, [0, 0, 0])               # no token
        refused(-1, [17])                    # past max_batch
        refused(-1, [1, -1])
        refused(-1, [1], n=5)                # more requests than opened
        refused(-1, [1], n=0)
        refused(-1, [1], top=65)
        refused(-1, [1], top=1)              # no place for it
        refused(-1, [1], given=4096)
        for fill in ([0, 12], [0, 12], [0, 12]):  # request 1: 36 positions, 9 pages
            model.step(fill, np.zeros(12, np.int32))
        left = model.free_pages()
        assert left == 1
        refused(-1, [0, 5])                  # past cache_cap
        refused(-3, [4, 0, 2])               # two pages
        with pytest.raises(RuntimeError):
            model.open_pages(1, 4, 4)        # open already
        with pytest.raises(RuntimeError):
            model.release(4)
        model.release(1)
        model.release(1)                     # holds none: nothing to do
        model.release(0)
        model.release(2)
        assert model.free_pages() == 13
        again = model.step(op[1], tokens, every=op[2], logits=True)["logits"]
        assert np.array_equal(again, first)
    finally:
        model.close()
        ctx.close()


@pytest.mark.gpu
def test_a_pool_that_does_not_fit_leaves_the_model_as_it_was():
    cfg = dict(CFG, max_batch=1)
    g, attn = gmoe.synth_model_weights(cfg, 2)
    model = gmoe.Model(cfg)
    try:
        model.upload(g)
        for l, a in enumerate(attn):
            model.upload_attn(l, a)
        want = model.forward_token(5, 0).copy()
        with pytest.raises(RuntimeError, match=r"gmoe_model_open_pages failed \(-3\)"):
            model.open_pages(4, 1 << 16, (1 << 15) - 1)  # 2^31 positions of 64 bytes in three layers: 412 GB
        assert model.free_pages() == -1
        assert np.array_equal(model.forward_token(5, 0), want)
        with pytest.raises(RuntimeError, match=r"gmoe_model_step failed \(-1\)"):
            model.step([1], [5])
        model.open_pages(4, 16, 8)
        model.step([1], [5])
        assert model.free_pages() == 7
    finally:
        model.close()


@pytest.mark.gpu
def test_the_fp32_cache_is_left_alone():
    """A sequence decoded on the model's own cache gives the same bits with steps between its tokens."""
    g, attn, moe, steps, *_ = expected("mixed", SEEDS["mixed"])
    plain, ctx_p = open_model("mixed", g, attn, moe)
    model, ctx = open_model("mixed", g, attn, moe)
    try:
        sequence = [5, 17, 99, 42, 7]
        for pos, tok in enumerate(sequence):
            want = plain.forward_token(tok, pos).copy()
            op, tokens, *_ = steps[pos]
            if op[0] == "step":
                model.step(op[1], tokens)
            assert np.array_equal(model.forward_token(tok, pos), want)
    finally:
        model.close()
        ctx.close()
        plain.close()
        ctx_p.close()


def test_ctypes_struct_matches_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "gmoe_model.h"', "int main(void) {",
             'printf("%zu\\n", sizeof(gmoe_model_batch));']
    lines += [f'printf("%zu\\n", offsetof(gmoe_model_batch, {f}));' for f, _ in gmoe.ModelBatch._fields_]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "probe"), str(tmp_path / "probe.c"), f"-I{root}/include"], check=True)
    out = subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [C.sizeof(gmoe.ModelBatch)] + [getattr(gmoe.ModelBatch, f).offset for f, _ in gmoe.ModelBatch._fields_]


def test_refusals_without_a_model():
    lib = gmoe.gmoe_lib()
    assert lib.gmoe_model_open_pages(None, 1, 16, 4) == -1
    assert lib.gmoe_model_step(None, None, None) == -1
    assert lib.gmoe_model_release(None, 0, None) == -1
    assert lib.gmoe_model_free_pages(None) == -1
