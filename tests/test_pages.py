"""Moves of cache pages in place, against a copy of the caches indexed all at once."""
import ctypes
import random

import pytest
import torch

from tests.helpers import dev


def _refused(tensors, dst, src):
    from worldattention_b200 import _lib
    arr = (_lib.PageTensor * max(1, len(tensors)))(*tensors)
    ints = lambda v: (ctypes.c_int32 * max(1, len(v)))(*v)  # noqa: E731
    rc = _lib.lib().wa_hkv_move_pages(arr, len(tensors), ints(dst), ints(src), len(dst), None)
    return rc, _lib.lib().wa_last_error().decode()


def test_moves_that_cannot_be_made_are_refused_before_any_launch():
    from worldattention_b200 import _lib
    # ptr, batch stride, token stride, tokens, row bytes, batch, page tokens: nothing of these is touched
    x = _lib.PageTensor(4096, 64000, 64, 1000, 64, 1, 100)
    far = _lib.PageTensor(1 << 30, 64000, 64, 950, 64, 1, 100)
    assert _refused([], [0], [1])[0] == 0 and _refused([x], [], [])[0] == 0      # nothing to do
    for dst, src, tensors, word in [([10], [0], [x], "leaves"), ([0], [10], [x], "leaves"), ([-1], [0], [x], "leaves"), ([0], [-2], [x], "leaves"),
                                    ([3, 3], [1, 2], [x], "two moves"), ([0], [1], [x, x], "share memory"), ([9], [0], [far, x][:1] + [_lib.PageTensor(1 << 32, 6400, 64, 850, 64, 1, 100)], "leaves"),
                                    ([0], [1], [x, _lib.PageTensor(4096 + 640, 64000, 64, 1000, 64, 1, 100)], "share memory"),
                                    ([0], [1], [_lib.PageTensor(4096, 0, 32, 1000, 64, 1, 100)], "overlap"),
                                    ([0], [1], [_lib.PageTensor(4096, 640, 64, 1000, 64, 2, 100)], "overlap"),
                                    ([0], [1], [_lib.PageTensor(None, 0, 64, 1000, 64, 1, 100)], "null"),
                                    ([0], [1], [_lib.PageTensor(4096, 0, 64, 1000, 64, 1, 0)], "positive")]:
        rc, said = _refused(tensors, dst, src)
        assert rc == _lib.WA_ERR_ARG and word in said, (dst, src, rc, said)


def test_caches_packed_into_one_tensor_are_apart():
    """By a brute-force look at every byte, on moves of a page to itself: nothing is launched."""
    from worldattention_b200 import _lib
    rng = random.Random(3)

    def views(t, shape, names):             # [B, tokens] views of rows of 16 bytes within one contiguous tensor of these axes
        strides, at = {}, 16
        for n, size in reversed(list(zip(names, shape))):
            strides[n] = at
            at *= size
        size = dict(zip(names, shape))
        return [_lib.PageTensor(4096 + i * strides["n"], strides["b"], strides["t"], size["t"], 16, size["b"], 1) for i in range(size["n"])]
    for names in (("b", "n", "t"), ("n", "b", "t"), ("b", "t", "n"), ("t", "b", "n"), ("t", "n", "b"), ("n", "t", "b")):
        for shape in ((2, 2, 8), (3, 4, 1), (1, 2, 5), (70, 2, 3), (2, 1, 1), (5, 2, 80)):
            rc, said = _refused(views(None, shape, names), [0], [0])
            assert rc == 0, (names, shape, said)
    agreed = 0
    for _ in range(3000):
        one = lambda: _lib.PageTensor(4096 + 16 * rng.randrange(40), 16 * rng.randrange(0, 25), 16 * rng.randrange(0, 25), rng.randrange(1, 4), 16 * rng.randrange(1, 4),  # noqa: E731
                                      rng.randrange(1, 4), 1)
        pair = [one(), one()]
        taken = [sorted(x.ptr + b * x.batch_stride + t * x.token_stride + r for b in range(x.batch) for t in range(x.tokens) for r in range(x.row_bytes)) for x in pair]
        whole = all(len(set(y)) == len(y) for y in taken)
        rc, said = _refused(pair, [0], [0])
        if not whole or set(taken[0]) & set(taken[1]):
            assert rc == _lib.WA_ERR_ARG, [(x.ptr, x.batch_stride, x.token_stride, x.tokens, x.row_bytes, x.batch) for x in pair]
        else:
            agreed += rc == 0
    assert agreed > 100


def test_python_refuses_what_is_no_cuda_cache():
    from worldattention_b200.hkv import move_pages
    with pytest.raises(RuntimeError, match="CUDA"):
        move_pages([torch.zeros(1, 8, 4)], [0], [1], 2)
    with pytest.raises(ValueError, match="equally long"):
        move_pages([], [0], [], 2)
    with pytest.raises(ValueError, match="negative"):
        move_pages([], [0], [-1], 2)
    with pytest.raises((ValueError, OverflowError)):
        move_pages([], [0], [1 << 40], 2)
    with pytest.raises(TypeError):
        move_pages([], 3, [1], 2)


def _want(cache, dst, src, page):
    old, new = cache.clone(), cache.clone()
    tokens = cache.shape[1]
    for d, s in zip(dst, src):
        n = min(page, tokens - d * page)
        if s is None:
            new[:, d * page:d * page + n] = 0
        else:
            n = min(n, tokens - s * page)
            new[:, d * page:d * page + n] = old[:, s * page:s * page + n]
    return new


def _filled(shape, dtype, seed):
    g = torch.Generator(device=dev()).manual_seed(seed)
    x = torch.randint(0, 256, (*shape[:-1], shape[-1] * dtype.itemsize), generator=g, device=dev(), dtype=torch.uint8)      # any bits, NaNs too
    return x.view(dtype)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,page,shape,dtype", [(64, 8, (4, 16), torch.bfloat16), (61, 8, (3, 5), torch.float32), (64, 1, (128,), torch.bfloat16),
                                                     (100, 13, (7,), torch.bfloat16), (33, 4, (3,), torch.uint8), (40, 5, (), torch.float64),
                                                     (4096, 2, (8,), torch.bfloat16), (2000, 1, (24,), torch.float32)])
@pytest.mark.parametrize("how", ["roll", "fork", "compact", "ring", "reverse", "random", "into the short page"])
def test_moves(tokens, page, shape, dtype, how):
    from worldattention_b200.hkv import move_pages
    n = -(-tokens // page)
    rng = random.Random(tokens * 31 + page)
    if how == "roll":
        dst, src = list(range(n - 3)), list(range(3, n))
    elif how == "fork":
        dst, src = list(range(1, n - 1)), [0 if i % 2 else n - 1 for i in range(1, n - 1)]
    elif how == "compact":
        keep = sorted(rng.sample(range(n), n // 2))
        dst, src = list(range(n)), keep + [None] * (n - len(keep))
    elif how == "ring":                     # one ring through every page: longer than the moves of a launch for the long cases
        dst, src = list(range(n)), [(i * 1 + 1) % n for i in range(n)]
    elif how == "reverse":                  # rings of two, and a page that stays
        dst, src = list(range(n)), list(reversed(range(n)))
    elif how == "random":                   # trees that hang on rings, clears, pages that stay
        dst = rng.sample(range(n), max(1, n - n // 5))
        src = [None if rng.random() < 0.1 else rng.randrange(n) for _ in dst]
    else:
        dst, src = [n - 1, 0], [0, n - 1]
    caches = [_filled((b, tokens) + shape if shape else (b, tokens), dtype, i) for i, b in enumerate((1, 2, 3))]
    want = [_want(c, dst, src, page) for c in caches]
    move_pages(caches, dst, src, page)
    for c, w in zip(caches, want):
        assert _same(c, w)


@pytest.mark.gpu
def test_views_lengths_of_their_own_and_many_tensors():
    from worldattention_b200.hkv import move_pages
    big = _filled((2, 50, 2, 3, 8), torch.bfloat16, 1)                      # keys and values side by side, inside a larger cache
    kept = big.clone()
    k, v = big[:, 2:46, 0], big[:, 2:46, 1]
    coarse = _filled((2, 12, 3, 8), torch.bfloat16, 2)
    dst, src = [0, 1, 2], [1, 2, 3]
    want = [_want(k, dst, src, 11), _want(v, dst, src, 11), _want(coarse, dst, src, 3)]
    move_pages((k, v, coarse), dst, src, (11, 11, 3))
    assert all(_same(a, b) for a, b in zip((k, v, coarse), want))
    assert _same(big[:, :2], kept[:, :2]) and _same(big[:, 46:], kept[:, 46:])
    time_first = _filled((40, 2, 24), torch.float32, 3).transpose(0, 1)      # [B, tokens, C] with samples inside tokens
    want = _want(time_first, dst, src, 10)
    move_pages([time_first], dst, src, 10)
    assert _same(time_first, want)
    many = [_filled((1, 20, 8), torch.float32, 10 + i) for i in range(300)]  # more than the tensors of a launch
    want = [_want(c, [0, 3, 1], [3, 0, None], 5) for c in many]
    move_pages(many, [0, 3, 1], [3, 0, None], 5)
    assert all(_same(a, b) for a, b in zip(many, want))
    empty = torch.empty(0, 20, 8, device=dev())
    move_pages([empty], [0], [1], 5)
    move_pages([many[0], empty], [0], [1], 5)
    odd = _filled((1, 41), torch.uint8, 5)[:, 1:]                            # no 16-byte rows, an odd address
    want = _want(odd, [0, 1], [1, 0], 20)
    move_pages([odd], [0, 1], [1, 0], 20)
    assert _same(odd, want)


@pytest.mark.gpu
def test_behind_two_to_the_31_bytes():
    from worldattention_b200.hkv import move_pages
    cache = torch.zeros(1, 5 << 20, 512, dtype=torch.bfloat16, device=dev())      # 5 GiB
    page = 1 << 20
    cache[0, 4 * page:] = 3.0
    cache[0, :page] = 1.0
    move_pages([cache], [0, 4, 2], [4, 0, 4], page)
    assert [float(cache[0, i * page + page - 1, 511]) for i in range(5)] == [3.0, 0.0, 3.0, 0.0, 1.0]
    assert bool((cache[0, 4 * page:] == 1).all()) and bool((cache[0, 2 * page:3 * page] == 3).all())


@pytest.mark.gpu
def test_streams_graphs_gradients_and_refusals():
    from worldattention_b200.hkv import move_pages
    c = _filled((1, 64, 16), torch.float32, 1)
    want = _want(_want(c, [0, 1], [1, 2], 16), [0, 1], [1, 2], 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        move_pages([c], [0, 1], [1, 2], 16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            move_pages([c], [0, 1], [1, 2], 16)
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert _same(c, want)
    x = torch.randn(1, 8, 4, device=dev(), requires_grad=True)
    with pytest.raises(RuntimeError, match="in place"):
        move_pages([x], [0], [1], 2)
    with torch.no_grad():
        move_pages([x], [0], [1], 2)
    y = torch.randn(1, 8, 4, device=dev())
    z = (y * x).sum()
    move_pages([y], [0], [1], 2)                 # y was saved for x's gradient
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    for bad, word in [(lambda: move_pages([c], [0, 0], [1, 2], 16), "two moves"), (lambda: move_pages([c], [4], [0], 16), "leaves"),
                      (lambda: move_pages([c, c], [0], [1], 16), "share memory"), (lambda: move_pages([c[:, :, ::2]], [0], [1], 16), "contiguous"),
                      (lambda: move_pages([c[0, 0]], [0], [1], 16), "tokens"), (lambda: move_pages([c], [0], [1], 0), "positive"),
                      (lambda: move_pages([c], [0], [1], [16, 16]), "each tensor"), (lambda: move_pages([c[:, :1].expand(1, 64, 16)], [0], [1], 16), "overlap")]:
        with pytest.raises(ValueError, match=word):
            bad()
    assert _same(c, want)


@pytest.mark.gpu
@pytest.mark.parametrize("frame,block,window,dropped", [(130, 64, 7, 3), (130, 64, 6, 3), (390, 128, 21, 3), (65, 64, 5, 1), (40, 64, 4, 2), (64, 64, 3, 2), (130, 128, 5, 4)])
def test_the_window_rolls_as_through_clones(frame, block, window, dropped):
    from worldattention_b200.causal_dit import roll_window
    from worldattention_b200.hsa import HSAAttention
    hsa = HSAAttention(2, 128, block_size=block, proj_segment_len=frame)
    for size in (window * frame, window * frame - frame // 3):          # a whole window, and one whose last frame is cut short: refused
        coarse = hsa.coarse_cache_size(window * frame)
        cache = {n: _filled((1, rows, 2, 128), torch.bfloat16, i) for i, (n, rows) in enumerate((("k", window * frame), ("v", window * frame), ("k_coarse", coarse), ("v_coarse", coarse)))}
        evict, keep = dropped * frame, size - dropped * frame
        want = {n: t.clone() for n, t in cache.items()}
        if size % frame:
            with pytest.raises(ValueError, match="segment-aligned"):
                roll_window(cache, hsa, evict, keep)
        else:
            c0, c1 = hsa.token_range_to_coarse(evict, evict + keep)
            for name, a, n in (("k", evict, keep), ("v", evict, keep), ("k_coarse", c0, c1 - c0), ("v_coarse", c0, c1 - c0)):
                want[name][:, :n] = cache[name][:, a:a + n].clone()
            roll_window(cache, hsa, evict, keep)
        for n in cache:
            assert _same(cache[n], want[n]), n


@pytest.mark.gpu
def test_keys_and_values_of_a_sample_one_behind_the_other():
    from worldattention_b200.hkv import move_pages
    both = _filled((2, 2, 40, 3, 8), torch.bfloat16, 9)                       # [B, keys and values, tokens, H, D]
    k, v = both[:, 0], both[:, 1]
    want = [_want(x, [0, 1, 2], [1, 3, None], 10) for x in (k, v)]
    move_pages((k, v), [0, 1, 2], [1, 3, None], 10)
    assert all(_same(a, b) for a, b in zip((k, v), want))
