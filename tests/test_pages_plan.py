"""Order and cutting of page moves, on the host: what the launches do in turn is what the list says, with a last page that is shorter."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest
import torch

from tests.helpers import dev
from tests.test_pages import _filled, _same, _want

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "worldattention_b200", "csrc")
SOURCE = """
#include "wa_pages_plan.cuh"
extern "C" int launches(const int *dst, const int *src, int n, int pages, int whole, int most, int *moves, int *sizes, int *parts, int *part_of) {
    const wa::PagePlan plan = wa::plan_moves(dst, src, n, pages, whole);
    std::vector<wa::PageMove> move(most);
    std::vector<int> part(most + 1);
    int k = 0, at = 0, q = 0;
    for (wa::PageCut cut; cut.at < (int)plan.move.size(); ++k) {
        const int before = cut.at;
        parts[k] = wa::next_moves(plan, whole, most, cut, move.data(), part.data());
        if (cut.at <= before) return -1;
        sizes[k] = part[parts[k]];
        for (int i = 0; i < sizes[k]; ++i) moves[2 * (at + i)] = move[i].to, moves[2 * (at + i) + 1] = move[i].from;
        for (int i = 0; i <= parts[k]; ++i) part_of[q++] = part[i];
        at += sizes[k];
    }
    return k;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = os.environ.get("CXX") or shutil.which("g++")
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, str(where / "plan.cpp"), "-o", str(where / "plan.so")], check=True)
    f = ctypes.CDLL(str(where / "plan.so")).launches

    def launches(dst, src, pages, whole, most):
        n = len(dst)
        ints = lambda v: (ctypes.c_int * len(v))(*v)  # noqa: E731
        moves, sizes, parts, part_of = ((ctypes.c_int * (8 * n + 64))() for _ in range(4))
        k = f(ints(dst), ints([-1 if s is None else s for s in src]), n, pages, whole, most, moves, sizes, parts, part_of)
        assert k >= 0
        got, at, q = [], 0, 0
        for i in range(k):
            assert sizes[i] <= most
            got.append([[(moves[2 * (at + j)], moves[2 * (at + j) + 1]) for j in range(part_of[q + p], part_of[q + p + 1])] for p in range(parts[i])])
            at, q = at + sizes[i], q + parts[i] + 1
        return got
    return launches


def _check(plan, dst, src, rows, page, most):
    """`rows` token rows in pages of `page`; a part runs as a thread of its own, in any order among the parts of a launch."""
    pages = -(-rows // page)
    cache = list(range(rows))
    rows_of = lambda p: min(page, rows - p * page)  # noqa: E731
    want = list(cache)
    for d, s in zip(dst, src):
        for r in range(rows_of(d) if s is None else min(rows_of(d), rows_of(s))):
            want[d * page + r] = -1 if s is None else cache[s * page + r]
    for launch in plan(dst, src, max([*dst, *(s for s in src if s is not None)]) + 1, rows // page, most):
        written, read = [], []
        for part in launch:
            kept, w, rd = [], set(), set()
            for to, frm in part:
                if frm == -3:
                    kept = cache[to * page:to * page + rows_of(to)]
                    rd.add(to)
                    continue
                w.add(to)
                new = kept if frm == -2 else [-1] * rows_of(to) if frm == -1 else cache[frm * page:frm * page + rows_of(frm)]
                if frm >= 0:
                    rd.add(frm)
                n = min(len(new), rows_of(to))
                cache[to * page:to * page + n] = new[:n]
            written.append(w)
            read.append(rd)
        for i, w in enumerate(written):
            assert not any(w & (written[j] | read[j]) for j in range(len(launch)) if j != i)
    assert cache == want, (pages, most)


def _ring(order):
    return order, order[1:] + order[:1]


@pytest.mark.parametrize("pages", [1022, 1023, 1024, 1025, 1026, 1100, 2044, 2045, 2046, 2047, 2048])
@pytest.mark.parametrize("short", [False, True])
def test_rings_longer_than_a_launch(plan, pages, short):
    up = list(range(pages))
    for order in (up, up[::-1], up[1:] + up[:1], up[-2:] + up[:-2], up[pages // 2:] + up[:pages // 2], up[:1] + up[:0:-1], random.Random(pages).sample(up, pages)):
        _check(plan, *_ring(order), pages * 2 - short, 2, 1024)
    dst, src = _ring(up)
    _check(plan, dst[::-1], src[::-1], pages * 2 - short, 2, 1024)


@pytest.mark.parametrize("most", [8, 32])
def test_every_place_of_the_short_page(plan, most):
    """Rings of every length around one, two and three launches, with the short page at every place and the list begun at every place."""
    for pages in range(2, 3 * most + 3):
        for at in range(pages):
            order = list(range(pages - 1))
            order.insert(at, pages - 1)
            for first in {0, at, max(at - 1, 0), (at + 1) % pages, pages // 2}:
                dst, src = _ring(order)
                _check(plan, dst[first:] + dst[:first], src[first:] + src[:first], pages * 3 - 1, 3, most)


def test_rings_trees_and_clears(plan):
    rng = random.Random(5)
    for _ in range(1500):
        pages, page = rng.randrange(2, 120), rng.randrange(1, 4)
        dst = rng.sample(range(pages), rng.randrange(1, pages + 1))
        if rng.random() < 0.5:            # only rings
            src = rng.sample(dst, len(dst))
        else:
            src = [None if rng.random() < 0.1 else rng.randrange(pages) for _ in dst]
        _check(plan, dst, src, pages * page - rng.randrange(page), page, rng.choice([8, 9, 32]))


@pytest.mark.gpu
@pytest.mark.parametrize("pages,how", [(1024, "up"), (2046, "up"), (1100, "down"), (2048, "down"), (1100, "from the short page")])
def test_rings_through_a_short_page(pages, how):
    from worldattention_b200.hkv import move_pages
    up = list(range(pages))
    dst, src = _ring({"up": up, "down": up[::-1], "from the short page": up[-1:] + up[:-1]}[how])
    caches = [_filled((b, tokens, width), torch.bfloat16, b) for b, tokens, width in ((1, 2 * pages - 1, 8), (2, 2 * pages + 6, 24))]
    want = [_want(c, dst, src, 2) for c in caches]
    move_pages(caches, dst, src, 2)
    assert all(_same(c, w) for c, w in zip(caches, want))
    assert caches[0].device == dev()
