// Order of simultaneous moves of pages and their distribution over launches.  Plain C++, without a word of CUDA: tests run it on the host.
//
// The moves of a list are put into an order in which no page is overwritten before it has been read for the last time: a page that is
// read by several comes after them, a ring of pages keeps one page's piece in registers.  They are split into parts that share no page that is both
// read and written.  A list that is longer than a launch takes is cut; within a ring the kept piece goes back to memory at the cut, to
// the page that is free there, and the next launch keeps it from there.
//
// One page number may stand for a page that is shorter than others, the last one.  A move between it and a whole page moves the rows that both have, so it can
// neither take a whole page's kept piece nor free a whole page: rings are not begun at it, nor cut where it is the free page or the next to be read.
#pragma once
#include <algorithm>
#include <numeric>
#include <vector>

namespace wa {

constexpr int PM_CLEAR = -1, PM_SAVED = -2, PM_SAVE = -3;      // sources that are no page: zeros, the kept piece; keep a piece of `to`

struct alignas(8) PageMove {
    int to, from;
};

struct PagePlan {
    std::vector<PageMove> move;
    std::vector<int> part, hole;       // of each move: its part, and the page that the kept piece may be put back to behind it (-1: none is kept)
    explicit PagePlan(size_t most) { move.reserve(most), part.reserve(most), hole.reserve(most); }
};

// `pages`: one more than the largest page number.  Pages from `whole` on, at most one, may be shorter.
inline PagePlan plan_moves(const int *dst, const int *src, int n, int pages, int whole) {
    std::vector<int> op(pages, -1), readers(pages, 0), root(pages);
    std::iota(root.begin(), root.end(), 0);
    auto find = [&](int a) {
        while (root[a] != a) a = root[a] = root[root[a]];
        return a;
    };
    for (int i = 0; i < n; ++i)
        if (dst[i] != src[i]) op[dst[i]] = i;
    for (int i = 0; i < n; ++i)
        if (dst[i] != src[i] && src[i] >= 0) {
            ++readers[src[i]];
            if (op[src[i]] >= 0) root[find(dst[i])] = find(src[i]);
        }
    PagePlan plan(n + n / 2);                  // (a ring of two or more is a move longer)
    std::vector<char> done(n, 0);
    auto emit = [&](int d, int s, int hole) {
        plan.move.push_back(PageMove{d, s});
        plan.part.push_back(find(d));
        plan.hole.push_back(hole);
    };
    for (int i = 0; i < n; ++i) {              // from pages that nothing reads
        int j = i;
        while (j >= 0 && dst[j] != src[j] && !done[j] && readers[dst[j]] == 0) {
            done[j] = 1;
            emit(dst[j], src[j] < 0 ? PM_CLEAR : src[j], -1);
            const int s = src[j];
            j = s >= 0 && --readers[s] == 0 ? op[s] : -1;
        }
    }
    for (int i = 0; i < n; ++i) {              // what is left are rings
        if (done[i] || dst[i] == src[i]) continue;
        const int start = dst[i] < whole ? i : op[src[i]];
        emit(dst[start], PM_SAVE, dst[start]);
        for (int j = start; !done[j]; j = op[src[j]]) {
            done[j] = 1;
            const bool closes = src[j] == dst[start];
            emit(dst[j], closes ? PM_SAVED : src[j], closes ? -1 : src[j]);
        }
    }
    // part by part, in the order above within each
    std::vector<int> by(plan.move.size());
    std::iota(by.begin(), by.end(), 0);
    std::stable_sort(by.begin(), by.end(), [&](int a, int b) { return plan.part[a] < plan.part[b]; });
    PagePlan sorted(by.size());
    for (int i : by) {
        sorted.move.push_back(plan.move[i]);
        sorted.part.push_back(plan.part[i]);
        sorted.hole.push_back(plan.hole[i]);
    }
    return sorted;
}

// Where the next launch begins: its first move, and the page that holds the kept piece of a ring that the launch before cut (-1: none).
struct PageCut {
    int at = 0, reopen = -1;
};

// The next launch's moves, at most `most` of them (eight or more), to `move`; the first of each part, and the end behind the last, to `part`.  -> parts
inline int next_moves(const PagePlan &plan, int whole, int most, PageCut &cut, PageMove *move, int *part) {
    const int total = (int)plan.move.size(), begin = cut.at;
    int n = 0, parts = 0;
    if (cut.reopen >= 0) move[n++] = PageMove{cut.reopen, PM_SAVE};
    int stop = std::min(total, begin + most - n);
    const auto open = [&] { return stop < total && plan.hole[stop - 1] >= 0; };
    if (open()) {
        --stop;            // room for the kept piece
        while (open() && (plan.hole[stop - 1] >= whole || plan.move[stop].from >= whole)) --stop;
    }
    for (int m = begin; m < stop; ++m) {
        if (m == begin || plan.part[m] != plan.part[m - 1]) part[parts++] = m == begin ? 0 : n;
        move[n++] = plan.move[m];
    }
    cut.reopen = open() ? plan.hole[stop - 1] : -1;
    if (cut.reopen >= 0) move[n++] = PageMove{cut.reopen, PM_SAVED};
    cut.at = stop;
    part[parts] = n;
    return parts;
}

}  // namespace wa
