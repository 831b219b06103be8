"""The serving operators' host side without a GPU: gmoe_serve.h's functions are exported, the ctypes
structs match it, sizes that have no meaning are refused before any device call, and the formulas that
the GPU tests compare with (serve_ref.py) against cases worked out by hand."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import gmoe
import serve_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(ROOT, "include")
HERE = 4096  # a non-null, aligned address that no refused call reads


def test_every_declared_function_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INC, "gmoe_serve.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(gmoe_\w+)\s*\(", text))
    assert len(names) == 8
    out = subprocess.run(["nm", "-D", "--defined-only", gmoe.LIBGMOE], capture_output=True, text=True, check=True).stdout
    assert names <= {line.split()[-1] for line in out.splitlines() if " T " in line}


def test_ctypes_structs_match_the_header(tmp_path):
    mirrors = {"gmoe_batch": gmoe.GmoeBatch, "gmoe_kv4": gmoe.GmoeKv4, "gmoe_kv4_heads": gmoe.GmoeKv4Heads,
               "gmoe_logprobs_args": gmoe.GmoeLogprobsArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "gmoe_serve.h"', "int main(void) {"]
    for name, cls in mirrors.items():
        lines.append(f'printf("{name} sizeof %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "probe"), str(src), f"-I{INC}"], check=True)
    for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, val = line.split()
        cls = mirrors[name]
        assert int(val) == (C.sizeof(cls) if field == "sizeof" else getattr(cls, field).offset), line


def batch(**over):
    sizes = dict(n_requests=2, max_tokens=8, max_pages=4, page_size=16)
    sizes.update({k: v for k, v in over.items() if k in sizes})
    arrays = {k: HERE for k in gmoe._BATCH_ARRAYS}
    arrays.update({k: v for k, v in over.items() if k in arrays})
    return gmoe.Batch(*sizes.values(), **arrays)


@pytest.mark.parametrize("over", [dict(n_requests=0), dict(n_requests=4097), dict(max_tokens=0), dict(max_tokens=(1 << 19) + 1),
                                  dict(max_pages=0), dict(max_pages=(1 << 19) + 1), dict(page_size=0), dict(page_size=48),
                                  dict(page_size=-16), dict(page_size=1 << 17)] + [{k: None} for k in gmoe._BATCH_ARRAYS])
def test_page_maps_refuses(over):
    with pytest.raises(RuntimeError, match=r"gmoe_page_maps failed \(-1\)"):
        batch(**over).maps()


def cache(rows=HERE, kv=512, rope=64, n_pages=4, page_size=16):
    return gmoe.Cache4(rows, kv, rope, n_pages, page_size)


BAD_CACHES = [dict(rows=None), dict(rows=HERE + 8), dict(kv=0), dict(kv=48), dict(kv=544), dict(rope=0), dict(rope=7),
              dict(rope=66), dict(n_pages=0), dict(n_pages=-1), dict(n_pages=1 << 27), dict(page_size=24), dict(page_size=0)]


@pytest.mark.parametrize("over", BAD_CACHES)
def test_a_bad_cache_is_refused(over):
    c = cache(**over)
    with pytest.raises(RuntimeError, match=r"\(-1\)"):
        c.append(1, HERE, 512, HERE, 64, HERE)
    with pytest.raises(RuntimeError, match=r"\(-1\)"):
        c.read(1, HERE, HERE, 512, HERE, 64)
    with pytest.raises(RuntimeError, match=r"\(-1\)"):
        c.attend(batch(), 4, 1.0, HERE, 2048, HERE, 256, HERE, 2048, HERE, 1 << 40)


@pytest.mark.parametrize("args", [(-1, HERE, 512, HERE, 64, HERE), ((1 << 19) + 1, HERE, 512, HERE, 64, HERE),
                                  (1, None, 512, HERE, 64, HERE), (1, HERE, 512, None, 64, HERE), (1, HERE, 512, HERE, 64, None),
                                  (2, HERE, -512, HERE, 64, HERE), (2, HERE, 512, HERE, -1, HERE), (2, HERE + 2, 512, HERE, 64, HERE)])
def test_append_refuses(args):
    with pytest.raises(RuntimeError, match=r"gmoe_kv4_append failed \(-1\)"):
        cache().append(*args)


@pytest.mark.parametrize("args", [(-1, HERE, HERE, 512, HERE, 64), (1, None, HERE, 512, HERE, 64), (1, HERE, None, 512, None, 64),
                                  (2, HERE, HERE, 511, HERE, 64), (2, HERE, HERE, 512, HERE, 62), (2, HERE, HERE + 1, 512, HERE, 64)])
def test_read_refuses(args):
    with pytest.raises(RuntimeError, match=r"gmoe_kv4_read failed \(-1\)"):
        cache().read(*args)


def test_no_tokens_is_nothing_to_do():
    cache().append(0, None, 0, None, 0, None)
    cache().read(0, None, None, 0, None, 0)
    gmoe.LogProbs(0, 100, 5, 1)(None, 100, None, None, None, None, None, None, 0)


@pytest.mark.parametrize("over", [dict(n_heads=0), dict(n_heads=257), dict(q_abs=None), dict(q_pe=None), dict(out=None), dict(ld_q_abs=-1),
                                  dict(ld_q_pe=-1), dict(ld_out=4 * 512 - 1), dict(q_abs=HERE + 1), dict(work=None), dict(work=HERE + 4),
                                  dict(work_bytes=-1), dict(page_size=32), dict(table=None), dict(offsets=None), dict(context=None)])
def test_attend_refuses(over):
    c = cache()
    a = dict(n_heads=4, scale=0.1, q_abs=HERE, ld_q_abs=2048, q_pe=HERE, ld_q_pe=256, out=HERE, ld_out=2048, work=HERE,
             work_bytes=c.attend_workspace(4))
    a.update({k: v for k, v in over.items() if k in a})
    if over.get("work_bytes") == -1:
        a["work_bytes"] = c.attend_workspace(4) - 1
    with pytest.raises(RuntimeError, match=r"gmoe_kv4_attend failed \(-1\)"):
        c.attend(batch(**{k: v for k, v in over.items() if k not in a}), **a)


@pytest.mark.parametrize("over", [dict(n=-1), dict(n=(1 << 24) + 1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(top=-1), dict(top=65), dict(n_given=-1),
                                  dict(ld=99), dict(logits=None), dict(logits=HERE + 2), dict(given=None), dict(logprob=None),
                                  dict(top_id=None), dict(top_logprob=None)])
def test_logprobs_refuses(over):
    s = dict(n=2, vocab=100, top=5, n_given=1)
    a = dict(logits=HERE, ld=100, given=HERE, logprob=HERE, entropy=None, top_id=HERE, top_logprob=HERE, work=HERE, work_bytes=1 << 40)
    s.update({k: v for k, v in over.items() if k in s})
    a.update({k: v for k, v in over.items() if k in a})
    with pytest.raises(RuntimeError, match=r"gmoe_logprobs failed \(-1\)"):
        gmoe.LogProbs(**s)(**a)


def test_a_short_workspace_is_refused():
    lp = gmoe.LogProbs(1, 154880, 20, 1)  # one row over the whole GPU
    assert lp.workspace > 0
    for work, size in ((HERE, lp.workspace - 1), (None, lp.workspace), (HERE + 8, lp.workspace)):
        with pytest.raises(RuntimeError, match="workspace"):
            lp(HERE, 154880, HERE, HERE, None, HERE, HERE, work, size)


def test_sizes():
    assert gmoe.Cache4.row_bytes(512, 64) == 320 == ref.row_bytes(512, 64)
    for kv in (32, 64, 96, 512):
        for rope in (2, 16, 32, 34, 64):
            assert gmoe.Cache4.row_bytes(kv, rope) == ref.row_bytes(kv, rope)
    assert gmoe.Cache4.row_bytes(40, 64) == 0 and gmoe.Cache4.row_bytes(512, 65) == 0
    assert cache().attend_workspace(0) == 0 and cache().attend_workspace(300) == 0


def test_the_reference_encoding_by_hand():
    x = np.zeros((1, 34))
    x[0, :8] = [7.0, -0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]  # amax 7: steps of 1; every tie goes to the even code
    x[0, 32:] = [7.01, 0.5]  # over 7 steps of 1: steps of 2
    r = ref.encode(x, 32, 2)
    assert r.shape == (1, 48) and r[0, 32] == 127 and r[0, 33] == 128
    assert list(ref.decode(r, 32, 2)[0, :8]) == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    assert list(ref.decode(r, 32, 2)[0, 32:]) == [8.0, 0.0] and r[0, 0] == 0x80 | 7
    assert ref.encode(np.full((1, 34), 1e30), 32, 2)[0, 32] == 140 and ref.encode(np.full((1, 34), 1e-30), 32, 2)[0, 32] == 104
    assert ref.encode(np.full((1, 34), np.nan), 32, 2)[0, 32] == 255


def test_the_reference_maps_by_hand():
    table = np.array([[5, -1, -1], [7, 8, -1], [-1, -1, -1]], np.int32)
    m = ref.page_maps([3, 8, 0], [2, 1, 3], [10, 11, 12], table, 8, 4)
    # request 0 ends in its second page, 1 begins a third, 2 begins its first
    assert m["table"].tolist() == [[5, 12, -1], [7, 8, 11], [10, -1, -1]]
    assert m["slot"][:6].tolist() == [23, 48, 44, 40, 41, 42] and m["slot"][6:].tolist() == [-1, -1]
    assert m["totals"].tolist() == [6, 3, 0]
    m = ref.page_maps([3, 8, 0], [2, 1, 3], [10, 11], table, 8, 4)  # a page too few: the last is short
    assert m["totals"].tolist() == [6, 2, 1] and m["context"].tolist() == [5, 9, 0] and m["position"][3:6].tolist() == [-1, -1, -1]
