"""A serving step's operators together, as a program without a model would run them: page maps, two
layers' appends and attentions, log probabilities of the second layer's results as logits, captured into
one graph at a fixed capacity and replayed step after step over lengths that change on the device. Each
replay is held to the 64-bit restatements and to the same calls made eagerly."""
import numpy as np
import pytest

import gmoe
import serve_ref as ref
from test_gpu_kv4 import U, latent
from test_gpu_logprobs import close

pytestmark = pytest.mark.gpu

H, KV, ROPE, P, T, R, WIDTH, PAGES, TOP = 5, 64, 16, 4, 40, 4, 40, 90, 4
SCALE = 1 / 16
# new tokens of each request, step by step: prompts, single tokens, idle ones, a full step, a step with none
STEPS = [[7, 0, 1, 20], [1, 1, 0, 1], [0, 33, 1, 1], [10, 10, 10, 10], [0, 0, 0, 0], [1, 1, 1, 1]]


class Step:
    def __init__(self):
        V = H * KV
        ints = dict(seen=R, fresh=R, n_free=1, offsets=R + 1, context=R, request=T, position=T, slot=T, totals=3)
        self.lp = gmoe.LogProbs(T, V, TOP, 1)
        row = ref.row_bytes(KV, ROPE)
        self.c = [gmoe.Cache4(0, KV, ROPE, PAGES, P) for _ in range(2)]
        self.d = ref.Arrays(free_pages=np.random.default_rng(1).permutation(PAGES).astype(np.int32), table=np.full((R, WIDTH), -1, np.int32),
                            **{k: np.zeros(v, np.int32) for k, v in ints.items()},
                            **{f"rows{l}": np.full((PAGES * P, row), 255, np.uint8) for l in range(2)},
                            **{f"x{l}": np.zeros((T, KV + ROPE), np.float32) for l in range(2)},
                            **{f"q{l}": np.zeros((T, H * (KV + ROPE)), np.float32) for l in range(2)},
                            **{f"out{l}": np.zeros((T, V), np.float32) for l in range(2)},
                            given=np.zeros(T, np.int32), logprob=np.zeros(T, np.float32), entropy=np.zeros(T, np.float32),
                            top_id=np.zeros((T, TOP), np.int32), top_logprob=np.zeros((T, TOP), np.float32),
                            work=np.full(self.c[0].attend_workspace(H), 0xFF, np.uint8),
                            score_work=np.full(max(16, self.lp.workspace), 0xFF, np.uint8))
        for l in range(2):
            self.c[l].c.rows = self.d.p(f"rows{l}")
        self.batch = gmoe.Batch(R, T, WIDTH, P, **{k: self.d.p(k) for k in gmoe._BATCH_ARRAYS})

    def call(self, stream=None):
        d = self.d
        self.batch.maps(stream)
        for l in range(2):
            self.c[l].append(T, d.p(f"x{l}"), KV + ROPE, d.p(f"x{l}", 4 * KV), KV + ROPE, d.p("slot"), stream)
            self.c[l].attend(self.batch, H, SCALE, d.p(f"q{l}"), H * (KV + ROPE), d.p(f"q{l}", 4 * H * KV), H * (KV + ROPE),
                             d.p(f"out{l}"), H * KV, d.p("work"), d.host["work"].nbytes, stream=stream)
        self.lp(d.p("out1"), H * KV, d.p("given"), d.p("logprob"), d.p("entropy"), d.p("top_id"), d.p("top_logprob"), d.p("score_work"),
                self.lp.workspace, stream=stream)


def test_a_captured_step_over_changing_lengths():
    eager, graph, stream = Step(), Step(), gmoe.Stream()
    exe = ref.capture(stream, lambda: graph.call(stream.h))
    rng = np.random.default_rng(3)
    seen, n_free = np.zeros(R, np.int32), PAGES
    free = eager.d.host["free_pages"]
    table, rows = eager.d.host["table"].copy(), [eager.d.host[f"rows{l}"].copy() for l in range(2)]
    for i, fresh in enumerate(STEPS):
        print(f"[case] step {i}: {fresh}", flush=True)
        new = dict(seen=seen, fresh=fresh, n_free=[n_free], given=rng.integers(0, H * KV, T))
        new.update({f"x{l}": latent(rng, T, KV, ROPE) for l in range(2)})
        new.update({f"q{l}": 4 * rng.standard_normal((T, H * (KV + ROPE))) for l in range(2)})
        for s in (eager, graph):
            for k, v in new.items():
                s.d.put(k, np.asarray(v))
        eager.call()
        ref.sync()
        gmoe.hip_check(gmoe.hip().hipGraphLaunch(exe, stream.h), "hipGraphLaunch")
        stream.sync()
        n = sum(fresh)
        want = ref.page_maps(seen, fresh, list(free[:n_free]), table, T, P)
        table = want["table"]
        for k in ref.OUTPUTS + ("table",):
            assert np.array_equal(eager.d.get(k), want[k]), k
        for l in range(2):
            x = new[f"x{l}"][:n]
            rows[l][want["slot"][:n]] = ref.encode(x, KV, ROPE)
            assert np.array_equal(eager.d.get(f"rows{l}"), rows[l])
            q = new[f"q{l}"].astype(np.float32)
            full, s = ref.attend(q[:, :H * KV].reshape(T, H, KV), q[:, H * KV:].reshape(T, H, ROPE), rows[l], table, want["offsets"],
                                 want["context"], P, SCALE)
            u = U * (s * (np.sqrt(KV + ROPE) + 4) + 16)  # (as in the attention's own tests)
            err = np.abs(eager.d.get(f"out{l}")[:n] - full.reshape(T, -1)[:n])
            if n:
                assert np.linalg.norm(err) <= 4 * u * np.linalg.norm(full[:n])
        lp, ent, ids, tlp = ref.logprobs(eager.d.get("out1")[:n], np.asarray(new["given"])[:n, None], TOP)
        tol = 2.0 ** -24 * (8 + np.sqrt(H * KV / 256))
        close(eager.d.get("logprob")[:n], lp[:, 0], tol)
        close(eager.d.get("entropy")[:n], ent, 2 * tol)
        assert np.array_equal(eager.d.get("top_id")[:n], ids)
        close(eager.d.get("top_logprob")[:n], tlp, tol)
        for k in ref.OUTPUTS + ("table", "rows0", "rows1"):
            assert np.array_equal(eager.d.get(k), graph.d.get(k)), k
        for k in ("out0", "out1", "logprob", "entropy", "top_id", "top_logprob"):
            assert np.array_equal(eager.d.get(k)[:n], graph.d.get(k)[:n]), k
        seen = (seen + fresh).astype(np.int32)
        n_free -= int(want["totals"][1])
