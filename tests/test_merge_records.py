"""The records that the decode kernel of shared rows leaves for its merge. A run whose wait ran out leaves its items' records as the
workspace held them, so the merge judges a record before it follows it. Such a run-out cannot be produced on demand: the judgement is
plain C++ and is tried here on the host, against the indices that the merge kernel forms, and that the kernel asks it first is
checked where it is written."""
import ctypes
import itertools
import os
import re
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend-moe-engine_b200", "csrc")
RUNS, PARTS = 74, 128


@pytest.fixture(scope="module")
def holds(tmp_path_factory):
    at = tmp_path_factory.mktemp("records")
    (at / "holds.cpp").write_text('#include "shared_merge_record.h"\n'
                                  'extern "C" int holds(int q0, int q1, int first, int last, int entry, int by_query, int batch, int runs) {\n'
                                  '  return b200kv::MergeHolds({q0, q1, first, last}, entry, by_query != 0, batch, runs);\n}\n'
                                  'extern "C" int parts() { return b200kv::kMergeParts; }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, str(at / "holds.cpp"), "-o", str(at / "holds.so")], check=True)
    lib = ctypes.CDLL(str(at / "holds.so"))
    assert lib.parts() == PARTS >= RUNS
    return lambda *args: bool(lib.holds(*args))


@pytest.mark.parametrize("batch,by_query", [(1, 1), (2, 1), (5, 1), (74, 1), (75, 0), (3000, 0)])
def test_no_record_leads_out_of_the_arrays(holds, batch, by_query):
    rng = np.random.default_rng(batch)
    some = [-2 ** 31, -2, -1, 0, 1, 2, 72, 73, 74, 75, 127, 128, 147, 148, batch - 2, batch - 1, batch, batch + 1, 0x3F800000, 2 ** 31 - 1]
    entries = range(min(batch, RUNS))
    taken = 0
    records = [(*r, e) for r in itertools.product(some, some, (-1, 0, 3, 73, 74, 2 ** 31 - 1), (-1, 0, 4, 73, 74, 127, 2 ** 31 - 1)) for e in (0, entries[-1])]
    records += [tuple(int(v) for v in rng.integers(-2 ** 31, 2 ** 31, 4)) + (0,) for _ in range(2000)]
    for q0, q1, first, last, entry in records:
        if not holds(q0, q1, first, last, entry, by_query, batch, RUNS):
            continue
        taken += 1
        assert 0 <= q0 < batch and (q1 < 0 or q1 < batch)          # rows of out and lse
        assert 0 <= first and 2 * last + 1 < 2 * RUNS              # slots of the partials
        assert 1 <= last - first + 1 <= PARTS                      # weights in shared memory
        assert q1 < 0 or q1 == q0 + 1
        assert entry == (q0 if by_query else last)                 # no two CTAs write one query
    assert taken > 0


@pytest.mark.parametrize("batch,by_query", [(1, 1), (2, 1), (74, 1), (75, 0)])
def test_every_record_that_a_run_writes_is_taken(holds, batch, by_query):
    for q0 in range(batch):
        for q1 in (-1, q0 + 1):
            if q1 >= batch:
                continue
            for first, last in ((0, 1), (0, RUNS - 1), (5, 9), (RUNS - 2, RUNS - 1)):
                assert holds(q0, q1, first, last, q0 if by_query else last, by_query, batch, RUNS)
    assert not holds(-1, -1, 0, 0, 0, by_query, batch, RUNS)       # nothing to merge


def test_the_merge_judges_a_record_before_it_uses_it():
    with open(os.path.join(CSRC, "mla_decode_shared.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    kernel = text[text.index("MlaSharedMergeKernel(const"):]
    loaded = kernel.index("= p.merges[")
    judged = kernel.index("if (!MergeHolds(merge", loaded)
    assert re.match(r"if \(!MergeHolds\(merge, [^;]*\)\) return;", kernel[judged:])
    assert "merge." not in kernel[loaded:judged]
