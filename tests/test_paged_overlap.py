"""Tensors of one paged call that share memory, without a GPU: the C entries
refuse them before anything is launched, and the rule itself is compared with
the bytes one by one."""
import os
import random
import subprocess

import pytest

from tests.test_paged_host import A, INVALID, call

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROW = 8 * 128 * 2                                 # bytes of a row of `call`'s queries


@pytest.mark.parametrize("bad,ops", [
    # a view of q some rows, one head or 16 bytes further
    (dict(out=A + ROW), ("append", "attend")), (dict(out=A - ROW), ("append", "attend")),
    (dict(out=A + 256), ("append", "attend")), (dict(out=A + 16), ("append", "attend")),
    (dict(out=A + 5 * ROW + 7 * 256 + 240), ("append", "attend")),
    # rows or heads of the result on top of each other
    (dict(row_stride=0), ("append", "attend")), (dict(q_head=0), ("append", "attend")),
    (dict(row_stride=8 * 128 - 8), ("append", "attend")), (dict(q_head=120), ("append", "attend")),
    # queries out over the new keys or values
    (dict(kr=2 * A), ("append",)), (dict(vr=2 * A + 5 * ROW), ("append",)), (dict(kr=2 * A - 256), ("append",)),
])
def test_refusals(bad, ops):
    _, fn = call(**bad)
    for op in ops:
        assert fn[op]() == INVALID, op


PROGRAM = r"""
#include <cstdio>
#include "paged_overlap.h"
int main()
{
    okv::RowSpan a, b;
    long long v[11];
    while (scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld %lld %lld", v, v + 1, v + 2, v + 3, v + 4, v + 5,
                 v + 6, v + 7, v + 8, v + 9, v + 10) == 11) {
        const orchkv_rows_t x = {(void *)v[0], v[1], v[2]}, y = {(void *)v[5], v[6], v[7]};
        a = okv::row_span(x, v[3], v[4], v[10], 1);
        b = okv::row_span(y, v[8], v[9], v[10], 1);
        printf("%d %d\n", okv::overlap(a, b), okv::overlaps_itself(a));
    }
}
"""


def touched(p, row, head, rows, heads, block):
    return [p + r * row + h * head + x for r in range(rows) for h in range(heads) for x in range(block)]


def test_the_rule_is_the_bytes(tmp_path):
    """3000 pairs of small tensors of equal row strides, interleaved in every
    way: exact; others may only be called overlapping when their spans are."""
    src, exe = tmp_path / "o.cpp", tmp_path / "o"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "orchkv_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = random.Random(0)
    cases = []
    for k in range(3000):
        block = r.choice([1, 2, 4])
        row, head = r.randrange(0, 40), r.randrange(0, 40)
        a = (100 + r.randrange(60), row, head, r.randrange(0, 5), r.randrange(1, 5))
        b = (100 + r.randrange(60), row if k % 4 else r.randrange(0, 40), head if k % 3 else r.randrange(0, 40),
             r.randrange(0, 5), r.randrange(1, 5))
        cases.append((a, b, block))
    text = "\n".join(" ".join(map(str, a + b + (block,))) for a, b, block in cases)
    out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
    seen = set()
    for (a, b, block), line in zip(cases, out):
        over, itself = map(int, line.split())
        ta, tb = touched(*a, block), touched(*b, block)
        assert itself == (len(set(ta)) < len(ta)), (a, block)
        share = bool(set(ta) & set(tb))
        if min(a[3], b[3]) < 2 or a[1] == b[1]:
            assert over == share, (a, b, block)
        else:
            assert over >= share and (not over or (min(ta) <= max(tb) and min(tb) <= max(ta)))
        seen.add((over, share, itself))
    assert {(0, 0, 0), (1, 1, 0), (1, 1, 1), (0, 0, 1)} <= seen


@pytest.mark.parametrize("bad,op", [
    # several places of the pages in one memory
    (dict(page_stride=0), "append"), (dict(token_stride=0), "append"), (dict(head_stride=0), "append"),
    # masses over q or lse (which `call` has at the same address)
    (dict(out=A), "mass"), (dict(out=A + 5 * ROW), "mass"), (dict(out=A - 4 * 4096 * 4), "mass"),
])
def test_broadcast_pages_and_masses_over_inputs(bad, op):
    assert call(**bad)[1][op]() == INVALID
