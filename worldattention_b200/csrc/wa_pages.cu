// Moves of cache pages in place: new[d_i] = old[s_i] for all i at once, or zeros, in all tensors of a call.
//
// Copying, forking, moving together and clearing pages are all of this form; the roll of a key/value window (wan/modules/
// causal_model.py:331-360) is the one that moves every page to the front.  No scratch and no order between thread blocks is needed:
// whatever happens to one 16-byte piece of a page happens to the same piece of every page, independently of all other pieces.  So
// a thread takes a piece (its place within a page) and runs a short list of page numbers over it: load from the source pages,
// store to the destinations.  The host puts a list into an order in which that can be done and splits it into parts that run side by side
// (wa_pages_plan.cuh).
//
// Bound: HBM, every moved page is read once and written once.  A thread has four pieces of one move in flight and makes the moves of a part one
// after the other: the loads of several moves at a time touch as many more pages, which DRAM takes badly (60 tensors of 21 pages of 4.8 MB,
// 12 moved together and 9 cleared, 9.5 GB: loads of four moves 2440 us, of two 1597, of one 1451 = 6.5 TB/s, what a plain copy reaches; a window of two
// tensors rolled by 3 of 21 frames: 78, 64 and 66).
// Page numbers and tensors travel as launch parameters: nothing is copied to the device, and the call can be captured.
#include <algorithm>
#include <new>
#include <vector>

#include "wa_common.cuh"
#include "wa_pages_plan.cuh"

namespace wa {

constexpr int PM_THREADS = 256, PM_PIECES = 4;                   // pieces of a thread, whose loads are in flight together

struct PageTensor {
    char *ptr;
    long long batch_stride, row_stride, page_stride;            // bytes
    long long rows;                                             // tokens of a sample
    int page_rows, row_pieces;                                  // tokens of a page, pieces of a token
};

template <int TENSORS, int MOVES>
struct PageMoves {
    PageTensor tensor[TENSORS];
    PageMove move[MOVES];
    int part[MOVES + 1];               // first move of each part
    int tensors, last_of[TENSORS];     // last_of: first launch row behind each tensor's (samples of all tensors are the grid's z)
};

template <typename Piece, int TENSORS, int MOVES>
__global__ void __launch_bounds__(PM_THREADS)
move_pages_kernel(const __grid_constant__ PageMoves<TENSORS, MOVES> p) {
    pdl_wait();
    int t = 0;
    while ((int)blockIdx.z >= p.last_of[t]) ++t;
    const PageTensor &x = p.tensor[t];
    const unsigned pieces = (unsigned)x.page_rows * (unsigned)x.row_pieces;      // below 2^31
    const unsigned first = blockIdx.x * (unsigned)(PM_THREADS * PM_PIECES) + threadIdx.x;
    if (first >= pieces) return;
    char *base = x.ptr + (blockIdx.z - (t ? p.last_of[t - 1] : 0)) * x.batch_stride;
    long long at[PM_PIECES];
    int row[PM_PIECES];
#pragma unroll
    for (int u = 0; u < PM_PIECES; ++u) {
        const unsigned e = first + u * PM_THREADS, r = e / (unsigned)x.row_pieces;
        row[u] = e < pieces ? (int)r : INT32_MAX;
        at[u] = (long long)r * x.row_stride + (long long)(e - r * (unsigned)x.row_pieces) * (long long)sizeof(Piece);
    }
    const auto rows_of = [&](int page) {        // the last page may be shorter
        const long long left = x.rows - (long long)page * x.page_rows;
        return (int)(left < x.page_rows ? left : x.page_rows);
    };
    Piece kept[PM_PIECES] = {};
    int kept_rows = 0;
    const int end = p.part[blockIdx.y + 1];
    for (int i = p.part[blockIdx.y]; i < end; ++i) {
        const PageMove m = p.move[i];
        const int page = m.from >= 0 ? m.from : m.to, mine = rows_of(page);
        const bool load = m.from >= 0 || m.from == PM_SAVE;
        const char *src = base + (long long)page * x.page_stride;
        Piece v[PM_PIECES];
#pragma unroll
        for (int u = 0; u < PM_PIECES; ++u) {
            v[u] = m.from == PM_SAVED ? kept[u] : Piece{};
            if (load && row[u] < mine) v[u] = *reinterpret_cast<const Piece *>(src + at[u]);
        }
        if (m.from == PM_SAVE) {
#pragma unroll
            for (int u = 0; u < PM_PIECES; ++u) kept[u] = v[u];
            kept_rows = mine;
            continue;
        }
        const int rows = min(m.from == PM_SAVED ? kept_rows : mine, rows_of(m.to));
        char *dst = base + (long long)m.to * x.page_stride;
#pragma unroll
        for (int u = 0; u < PM_PIECES; ++u)
            if (row[u] < rows) *reinterpret_cast<Piece *>(dst + at[u]) = v[u];
    }
}

template <typename Piece, int TENSORS, int MOVES>
static int launch_moves(const wa_page_tensor *tensors, int n_tensors, const PagePlan &plan, int whole_pages, cudaStream_t stream, const char *what) {
    const int total = (int)plan.move.size();
    // a tensor at a time is added as long as there is room; all lists run over a group of tensors before the next group
    for (int t0 = 0; t0 < n_tensors;) {
        PageMoves<TENSORS, MOVES> p{};
        long long widest = 0, rows = 0;
        int t = t0;
        for (; t < n_tensors && p.tensors < TENSORS; ++t) {
            const wa_page_tensor &x = tensors[t];
            if (rows + x.batch > 65535 && p.tensors > 0) break;
            WA_REQUIRE(x.batch <= 65535, WA_ERR_UNSUPPORTED, "%s: more than 65535 samples", what);
            PageTensor &y = p.tensor[p.tensors];
            y.ptr = (char *)x.ptr; y.batch_stride = x.batch_stride; y.row_stride = x.token_stride; y.page_stride = x.token_stride * x.page_tokens;
            y.rows = x.tokens; y.page_rows = x.page_tokens; y.row_pieces = (int)(x.row_bytes / (int64_t)sizeof(Piece));
            rows += x.batch;
            p.last_of[p.tensors++] = (int)rows;
            widest = std::max(widest, (long long)y.page_rows * y.row_pieces);
        }
        t0 = t;
        if (widest == 0 || rows == 0) continue;
        WA_REQUIRE(widest < (1ll << 31) - PM_THREADS * PM_PIECES, WA_ERR_UNSUPPORTED, "%s: pages of more than 2^31 pieces", what);
        const long long gx = (widest + PM_THREADS * PM_PIECES - 1) / (PM_THREADS * PM_PIECES);
        for (PageCut cut; cut.at < total;) {
            const int parts = next_moves(plan, whole_pages, MOVES, cut, p.move, p.part);
            const cudaError_t e = launch_dependent(move_pages_kernel<Piece, TENSORS, MOVES>, dim3((unsigned)gx, parts, (unsigned)rows), dim3(PM_THREADS), 0, stream, p);
            if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
            const int rc = check_launch(what);
            if (rc) return rc;
        }
    }
    return 0;
}

template <typename Piece>
static int launch_moves(const wa_page_tensor *tensors, int n_tensors, const PagePlan &plan, int whole_pages, cudaStream_t stream, const char *what) {
    // parameters are copied with every launch: a small call has small ones
    if (n_tensors <= 8 && plan.move.size() <= 32) return launch_moves<Piece, 8, 32>(tensors, n_tensors, plan, whole_pages, stream, what);
    return launch_moves<Piece, 128, 1024>(tensors, n_tensors, plan, whole_pages, stream, what);
}

// Token rows of a tensor do not overlap: of its two axes the one with the larger stride steps over all of the other.
static bool rows_apart(const wa_page_tensor &x) {
    int64_t inner = x.token_stride, n_inner = x.tokens, outer = x.batch_stride, n_outer = x.batch;
    if (n_inner <= 1 || (n_outer > 1 && outer < inner)) std::swap(inner, outer), std::swap(n_inner, n_outer);
    if (n_inner > 1 && inner < x.row_bytes) return false;
    return n_outer <= 1 || outer >= (n_inner > 1 ? (n_inner - 1) * inner : 0) + x.row_bytes;
}

// Tensors that lie apart, or whose rows alternate (keys and values of a token side by side, two samples of one cache).  `most` > 1: looked at
// sample by sample where a tensor has no more (keys and values of a sample one behind the other).
static bool tensors_apart(const wa_page_tensor *tensors, int n, int most) {
    struct Span {
        uintptr_t from, to;
        int64_t row, step[2], count[2];
    };
    std::vector<Span> spans;
    for (int t = 0; t < n; ++t) {
        const wa_page_tensor &x = tensors[t];
        if (x.tokens * x.row_bytes * x.batch == 0) continue;
        int64_t step[2] = {x.token_stride, x.batch_stride}, count[2] = {x.tokens, x.batch};
        if (count[0] <= 1 || (count[1] > 1 && step[1] < step[0])) std::swap(step[0], step[1]), std::swap(count[0], count[1]);
        // slices of the outer axis one by one (they do not overlap, see above), or all at once
        const int64_t slices = count[1] <= most ? count[1] : 1, each = count[1] / slices;
        for (int64_t i = 0; i < slices; ++i) {
            const uintptr_t from = (uintptr_t)x.ptr + (uintptr_t)(slices > 1 ? i * step[1] : 0);
            const uintptr_t bytes = (uintptr_t)((count[0] - 1) * step[0] + (each > 1 ? (each - 1) * step[1] : 0) + x.row_bytes);
            spans.push_back({from, from + bytes, x.row_bytes, {step[0], step[1]}, {count[0], each}});
        }
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.from < b.from; });
    for (size_t i = 0; i < spans.size(); ++i)
        for (size_t j = i + 1; j < spans.size() && spans[j].from < spans[i].to; ++j) {
            const Span &a = spans[i], &b = spans[j];
            int64_t step = 0;                       // the smallest that is taken; all others are multiples of it, or the two count as one
            for (const Span *x : {&a, &b})
                for (int k = 0; k < 2; ++k)
                    if (x->count[k] > 1 && (step == 0 || x->step[k] < step)) step = x->step[k];
            if (step <= 0) return false;
            for (const Span *x : {&a, &b})
                for (int k = 0; k < 2; ++k)
                    if (x->count[k] > 1 && x->step[k] % step) return false;
            const int64_t off = (int64_t)((b.from - a.from) % (uintptr_t)step);
            if (off < a.row || off + b.row > step) return false;
        }
    return true;
}

static int move_pages(const wa_page_tensor *tensors, int n_tensors, const int32_t *dst, const int32_t *src, int n, cudaStream_t stream) {
    const char *what = "wa_hkv_move_pages";
    WA_REQUIRE(n_tensors >= 0 && n >= 0, WA_ERR_ARG, "%s: sizes must not be negative", what);
    if (n == 0 || n_tensors == 0) return 0;
    WA_REQUIRE(tensors && dst && src, WA_ERR_ARG, "%s: null pointer", what);
    int64_t pages = INT32_MAX, whole = INT32_MAX;
    uintptr_t bits = 0;
    for (int t = 0; t < n_tensors; ++t) {
        const wa_page_tensor &x = tensors[t];
        WA_REQUIRE(x.batch >= 0 && x.tokens >= 0 && x.row_bytes >= 0 && x.page_tokens > 0, WA_ERR_ARG, "%s: sizes must be positive", what);
        WA_REQUIRE(x.ptr || x.tokens * x.row_bytes * x.batch == 0, WA_ERR_ARG, "%s: null pointer", what);
        WA_REQUIRE(x.row_bytes < (1ll << 31), WA_ERR_UNSUPPORTED, "%s: rows of more than 2^31 bytes", what);
        WA_REQUIRE(rows_apart(x), WA_ERR_ARG, "%s: the tokens of a tensor must not overlap", what);
        pages = std::min(pages, (x.tokens + x.page_tokens - 1) / x.page_tokens);
        whole = std::min(whole, x.tokens / x.page_tokens);
        bits |= (uintptr_t)x.ptr | (uintptr_t)x.batch_stride | (uintptr_t)x.token_stride | (uintptr_t)x.row_bytes;
    }
    WA_REQUIRE(tensors_apart(tensors, n_tensors, 1) || tensors_apart(tensors, n_tensors, 4096), WA_ERR_ARG, "%s: two tensors share memory", what);
    int most = 0;
    for (int i = 0; i < n; ++i) {
        WA_REQUIRE(dst[i] >= 0 && dst[i] < pages && src[i] >= -1 && src[i] < pages, WA_ERR_ARG, "%s: move %d of page %d to page %d leaves the %lld pages of a tensor",
                   what, i, src[i], dst[i], (long long)pages);
        most = std::max(most, std::max(dst[i], src[i]) + 1);
    }
    std::vector<char> taken(most, 0);
    for (int i = 0; i < n; ++i) {
        WA_REQUIRE(!taken[dst[i]], WA_ERR_ARG, "%s: page %d is the destination of two moves", what, dst[i]);
        taken[dst[i]] = 1;
    }
    const int whole_pages = (int)std::min<int64_t>(whole, INT32_MAX);      // (`pages` or one less: whole in every tensor)
    const PagePlan plan = plan_moves(dst, src, n, most, whole_pages);
    if (plan.move.empty()) return 0;
    if (bits % 16 == 0) return launch_moves<uint4>(tensors, n_tensors, plan, whole_pages, stream, what);
    if (bits % 4 == 0) return launch_moves<uint32_t>(tensors, n_tensors, plan, whole_pages, stream, what);
    return launch_moves<unsigned char>(tensors, n_tensors, plan, whole_pages, stream, what);
}

}  // namespace wa

extern "C" int wa_hkv_move_pages(const wa_page_tensor *tensors, int n_tensors, const int32_t *dst, const int32_t *src, int n, void *stream) {
    try {
        return wa::move_pages(tensors, n_tensors, dst, src, n, (cudaStream_t)stream);
    } catch (const std::bad_alloc &) {
        return wa::fail(WA_ERR_ARG, "wa_hkv_move_pages: out of host memory");
    }
}
