"""The operators between two steps on the device, against their plain 64-bit forms: attention that keeps its weights,
eviction of cached positions, verification of drafted tokens."""
import math
import random

import pytest
import torch

import plain_between as pb

pytestmark = pytest.mark.gpu
PAGE = 64


def _rounding(dtype):
    return torch.finfo(dtype).eps / 2


def _tables(rng, lengths, extra_pages, spare=0):
    """(table rows with -1 behind a sequence's pages, number of pages, ids not used)"""
    used = [(n + PAGE - 1) // PAGE for n in lengths]
    n_pages = max(1, sum(used) + extra_pages)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    width, rows, at = max(used + [1]) + spare, [], 0
    for u in used:
        rows.append(ids[at:at + u] + [-1] * (width - u))
        at += u
    return rows, n_pages, ids[at:]


# ---- attention that keeps its weights --------------------------------------------------------------------------------
def _attention(cuda, starts, news, heads, kv_heads, dim, dtype, with_out=True, v_dim=None, seed=0, in_place=True, spoil=None, q_pad=0,
               loose=False, scale=None):
    from camelid_b200.csrc import ops
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    lengths = [s + n for s, n in zip(starts, news)]
    table, n_pages, _ = _tables(rng, lengths, 2, spare=1)
    v_dim = v_dim or dim
    k = torch.randn(n_pages, kv_heads, PAGE, dim, generator=gen).to(dtype)
    v = torch.randn(n_pages, kv_heads, PAGE, v_dim, generator=gen).to(dtype)
    scores = torch.rand(n_pages, kv_heads, PAGE, generator=gen) * 3
    rows = sum(news)
    q = (1.5 * torch.randn(rows + 2, heads * dim + q_pad, generator=gen)).to(dtype)
    row0 = [sum(news[:i]) for i in range(len(news))]
    k_dev, v_dev, s_dev = k.clone(), v.clone(), scores.clone()
    if spoil is not None:                     # what lies behind a sequence's last place must not matter
        for i, n in enumerate(lengths):
            for p in range(n, (n + PAGE - 1) // PAGE * PAGE):
                k_dev[table[i][p // PAGE], :, p % PAGE] = spoil
                v_dev[table[i][p // PAGE], :, p % PAGE] = spoil
            for p in range(starts[i], n):     # nor what a new place's score was
                s_dev[table[i][p // PAGE], :, p % PAGE] = spoil
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    out = torch.full((rows + 2, heads * v_dim), 7.0, dtype=dtype, device=cuda)
    q_dev = q.to(cuda)[:, :heads * dim]
    k_dev, v_dev, s_dev = k_dev.to(cuda), v_dev.to(cuda), s_dev.to(cuda)
    s_out = s_dev if in_place else s_dev.clone()
    max_new, max_len = max(news + [1]), max(lengths + [1])
    if loose:
        max_new, max_len = max_new + 3, max_len + 200
    scratch = torch.empty(ops.attn_weights_floats(len(news), heads, kv_heads, dim, dtype, max_new, max_len, with_out, v_dim), device=cuda)
    scratch.fill_(float("nan"))
    scale = 1 / math.sqrt(dim) if scale is None else scale
    ops.attn_paged_weights(q_dev, out if with_out else None, k_dev, v_dev if with_out else None, s_dev, ints(table), ints(row0), ints(starts),
                           ints(news), heads, max_new, max_len, scale, scratch, None if in_place else s_out)
    torch.cuda.synchronize()
    ref, ref_scores, tol, tol_scores = pb.weights(q[:, :heads * dim], k, v if with_out else None, scores, table, row0, starts, news, heads, scale)
    if with_out:
        got = out.cpu().double()
        assert bool((got[rows:] == 7.0).all()), "rows behind the last sequence were written"
        mma = dtype == torch.bfloat16
        # bfloat16 probabilities times values: half a step of each, of the sum of the products' sizes
        absolute = torch.zeros_like(ref)
        if mma:
            absolute = pb.weights(q[:, :heads * dim], k, v.abs(), scores, table, row0, starts, news, heads, scale)[0] * _rounding(dtype)
        bound = tol + absolute + _rounding(dtype) * (ref.abs() + tol + absolute) + 1e-30
        assert bool(((got - ref)[:rows].abs() <= bound[:rows]).all()), float(((got - ref)[:rows].abs() / bound[:rows]).max())
    new_scores = s_out.cpu().double()
    live = torch.zeros(ref_scores.shape, dtype=torch.bool)
    for i, n in enumerate(lengths):
        for p in range(n if news[i] else 0):
            live[table[i][p // PAGE], :, p % PAGE] = True
    assert bool(((new_scores - ref_scores).abs() <= tol_scores + 1e-30)[live].all()), float(
        ((new_scores - ref_scores).abs() / (tol_scores + 1e-30))[live].max())
    untouched = s_dev if not in_place else None
    if untouched is not None:
        assert torch.equal(torch.nan_to_num(s_out.cpu()[~live]), torch.nan_to_num(s_dev.cpu()[~live]))
    elif spoil is None:
        assert torch.equal(s_out.cpu()[~live], scores[~live])
    return out, s_out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 128), (6, 1, 96), (8, 1, 16), (3, 1, 256), (16, 1, 64)])
def test_weights_of_single_tokens(cuda, dtype, heads, kv_heads, dim):
    _attention(cuda, [0, 1, 62, 63, 64, 200, 517], [1] * 7, heads, kv_heads, dim, dtype, seed=heads + dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 48])
def test_weights_of_drafted_steps(cuda, dtype, dim):
    """Unequal numbers of new tokens, a sequence without any, places that later rows alone see."""
    _attention(cuda, [0, 130, 61, 7, 300], [5, 1, 8, 0, 3], 8, 2, dim, dtype, seed=dim)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 80), (torch.float32, 64)])
def test_weights_of_a_prompts_last_rows(cuda, dtype, dim):
    _attention(cuda, [0, 500, 129], [33, 64, 2], 8, 2, dim, dtype, with_out=False, seed=3)
    _attention(cuda, [70, 300], [64, 40], 8, 1, dim, dtype, with_out=False, seed=4)
    _attention(cuda, [70, 0, 5], [20, 3, 1], 4, 2, dim, dtype, with_out=False, seed=5)
    _attention(cuda, [700], [2], 4, 2, dim, dtype, with_out=False, seed=6)


@pytest.mark.parametrize("dim", [64, 128])
def test_weights_of_many_rows_with_output(cuda, dim):
    _attention(cuda, [70, 300, 0], [9, 4, 12], 16, 2, dim, torch.bfloat16, seed=7)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 112), (torch.float32, 32)])
def test_weights_do_not_read_behind_the_end(cuda, dtype, dim):
    for spoil in (float("nan"), float("inf"), -float("inf")):
        _attention(cuda, [10, 64, 190], [3, 1, 2], 4, 2, dim, dtype, spoil=spoil, in_place=False)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 128)])
def test_weights_with_strided_rows_and_loose_bounds(cuda, dtype, dim):
    _attention(cuda, [10, 333], [2, 1], 8, 4, dim, dtype, q_pad=40, loose=True, in_place=False)
    _attention(cuda, [10, 333], [2, 1], 8, 4, dim, dtype, q_pad=3, loose=True)


@pytest.mark.parametrize("with_out", [True, False])
def test_weights_keep_within_their_scratch(cuda, monkeypatch, with_out):
    """Every form of the kernels, also of rows that begin off 16 bytes, leaves alone what lies behind the scratch it asks for."""
    from camelid_b200.csrc import ops
    given = ops.attn_paged_weights
    checked = []

    def guarded(*args):
        args = list(args)
        room = torch.full((args[13].numel() + 4096,), 7.0, device=cuda)
        args[13] = room[:args[13].numel()].fill_(float("nan"))
        given(*args)
        checked.append(bool((room[-4096:] == 7.0).all()))
    monkeypatch.setattr(ops, "attn_paged_weights", guarded)
    for dtype, dim, v_dim in ((torch.bfloat16, 64, 64), (torch.bfloat16, 128, 128), (torch.float32, 64, 64), (torch.bfloat16, 48, 80)):
        for heads, kv_heads, news in ((4, 2, [1, 1, 1]), (8, 2, [5, 1, 2]), (4, 1, [8, 3, 0]), (8, 2, [3, 9, 1])):
            for q_pad in (0, 3):
                _attention(cuda, [700, 0, 129], news, heads, kv_heads, dim, dtype, with_out=with_out, v_dim=v_dim if with_out else None, q_pad=q_pad,
                           seed=dim + heads, loose=news[1] == 9)
    assert len(checked) == 32 and all(checked)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 48)])
def test_products_of_unequal_sequences_take_the_caches_pages(cuda, monkeypatch, dtype, dim):
    """One long sequence among short ones: the scratch of the cache's pages is smaller than a rectangle, and enough. Cached places,
    single tokens, drafted steps, rows that see nothing of a page, a sequence without new tokens."""
    from camelid_b200.csrc import ops
    given = ops.attn_paged_weights
    used = []

    def exact(q, out, k, v, scores, table, row0, start, new, heads, max_new, max_len, scale, scratch, *more):
        small = ops.attn_weights_floats(table.shape[0], heads, k.shape[1], k.shape[3], q.dtype, max_new, max_len, out is not None,
                                        n_pages=k.shape[0])
        room = torch.full((small + 4096,), 7.0, device=cuda)
        given(q, out, k, v, scores, table, row0, start, new, heads, max_new, max_len, scale, room[:small].fill_(float("nan")), *more)
        assert bool((room[small:] == 7.0).all())
        used.append((small, scratch.numel()))
    monkeypatch.setattr(ops, "attn_paged_weights", exact)
    group = 2 if dtype == torch.float32 or dim == 48 else 4
    for news in ([1] * 6, [4, 1, 0, 2, 3, 1]):
        for with_out in (True, False):
            _attention(cuda, [3000, 5, 64, 0, 130, 63], news, 2 * group, 2, dim, dtype, with_out=with_out, seed=dim + news[0], in_place=news[0] == 1)
    # (of 9 rows and more the room holds the other form's parts as well: 12 pairs * 16 rows * (2 + splits * (2 + dim)))
    assert all(small < rectangle for small, rectangle in used) and len(used) == 4


def test_weights_with_values_of_another_size(cuda):
    _attention(cuda, [100, 3], [1, 2], 4, 2, 64, torch.bfloat16, v_dim=32)
    _attention(cuda, [100, 3], [1, 2], 4, 2, 32, torch.float32, v_dim=128)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 128)])
def test_a_later_rows_value_does_not_reach_an_earlier_row(cuda, dtype, dim):
    """Infinite keys and values at a place that only the last row sees."""
    from camelid_b200.csrc import ops
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(4, 1, PAGE, dim, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(3, 2 * dim, generator=gen).to(dtype)
    k[1, 0, 10], v[1, 0, 10] = float("inf"), float("nan")         # place 74: the third row's own
    scores = torch.zeros(4, 1, PAGE)
    out = torch.zeros(3, 2 * dim, dtype=dtype, device=cuda)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    scratch = torch.empty(ops.attn_weights_floats(1, 2, 1, dim, dtype, 3, 75, True), device=cuda)
    s_dev = scores.to(cuda)
    ops.attn_paged_weights(q.to(cuda), out, k.to(cuda), v.to(cuda), s_dev, ints([[0, 1]]), ints([0]), ints([72]), ints([3]), 2, 3, 75,
                           dim ** -0.5, scratch)
    ref = pb.weights(q[:2], k, v, scores, [[0, 1]], [0], [72], [2], 2, dim ** -0.5)[0]
    got = out.cpu().double()[:2]
    assert bool(torch.isfinite(got).all())
    assert float((got - ref).abs().max()) <= 4 * _rounding(dtype) * float(ref.abs().max()) + 1e-5


def test_weights_with_missing_pages(cuda):
    """A page that the table does not name holds nothing to see; a row without any place gives zeros."""
    from camelid_b200.csrc import ops
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 32), (torch.bfloat16, 128)):
        gen = torch.Generator().manual_seed(6)
        k, v = (torch.randn(3, 1, PAGE, dim, generator=gen).to(dtype) for _ in range(2))
        q = torch.randn(2, 2 * dim, generator=gen).to(dtype)
        table, start = [[-1, 1, 3], [-1, 99, -1]], [130, 70]
        scores = torch.rand(3, 1, PAGE, generator=gen)
        out = torch.ones(2, 2 * dim, dtype=dtype, device=cuda)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)    # noqa: E731
        scratch = torch.empty(ops.attn_weights_floats(2, 2, 1, dim, dtype, 1, 131, True), device=cuda)
        s_dev = scores.to(cuda)
        ops.attn_paged_weights(q.to(cuda), out, k.to(cuda), v.to(cuda), s_dev, ints(table), ints([0, 1]), ints(start), ints([1, 1]), 2, 1,
                               131, dim ** -0.5, scratch)
        ref, ref_scores, tol, tol_scores = pb.weights(q, k, v, scores, table, [0, 1], start, [1, 1], 2, dim ** -0.5)
        got = out.cpu().double()
        assert bool((got[1] == 0).all())
        assert float((got - ref).abs().max()) <= 4 * _rounding(dtype) * float(ref.abs().max()) + 1e-5
        assert bool(((s_dev.cpu().double() - ref_scores).abs() <= tol_scores + 1e-30).all())


def test_weights_refuse_an_error_word_elsewhere(cuda):
    """The kernels would write it: on the host, or as another type."""
    from camelid_b200 import KernelError
    from camelid_b200.csrc import ops
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    k, s = torch.zeros(1, 1, PAGE, 64, dtype=torch.bfloat16, device=cuda), torch.zeros(1, 1, PAGE, device=cuda)
    q = torch.zeros(2, 64, dtype=torch.bfloat16, device=cuda)
    scratch = torch.empty(ops.attn_weights_floats(1, 1, 1, 64, torch.bfloat16, 2, 64, False), device=cuda)
    args = (q, None, k, None, s, ints([[0]]), ints([0]), ints([0]), ints([2]), 1, 2, 64, 0.125, scratch)
    with pytest.raises(KernelError):
        ops.attn_paged_weights(*args, err=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(AssertionError):
        ops.attn_paged_weights(*args, err=torch.zeros(1, device=cuda))
    ops.attn_paged_weights(*args, err=ints([0]))


@pytest.mark.parametrize("dim", [64, 128])
def test_window_at_the_limits_of_its_kernels(cuda, dim):
    """Rows just below, at and beyond what the tensor-memory kernels take, and stretches that end inside a tile."""
    for heads, new in ((16, 4), (16, 3), (21, 3), (16, 32), (16, 33), (9, 30), (16, 8), (16, 16)):
        _attention(cuda, [200, 5], [new, min(new, 2)], heads, 1, dim, torch.bfloat16, with_out=False, seed=heads + new)
    _attention(cuda, [2100, 1279, 0], [20, 1, 20], 8, 2, dim, torch.bfloat16, with_out=False, seed=8, in_place=False, spoil=float("nan"))
    _attention(cuda, [300, 40], [16, 9], 8, 2, dim, torch.bfloat16, with_out=False, loose=True, q_pad=8)


@pytest.mark.parametrize("dim", [64, 128])
def test_window_of_many_unequal_sequences(cuda, dim):
    """More sequences than lanes, than blocks of a kv head, some without new tokens, and rows in several passes."""
    rng = random.Random(dim)
    starts = [rng.choice((0, 3, 64, 127, 128, 300, 900)) for _ in range(40)]
    news = [rng.choice((0, 1, 9, 17, 20)) for _ in range(40)]
    _attention(cuda, starts, news, 8, 1, dim, torch.bfloat16, with_out=False, seed=dim)
    _attention(cuda, starts[:21], news[:20] + [20], 32, 8, dim, torch.bfloat16, with_out=False, seed=dim + 1, in_place=False)
    _attention(cuda, [500, 70, 0, 33], [70, 10, 33, 0], 16, 1, dim, torch.bfloat16, with_out=False, seed=3, spoil=float("nan"), in_place=False)
    _attention(cuda, [4000, 0, 130], [9, 9, 9], 4, 1, dim, torch.bfloat16, with_out=False, seed=4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,v_dim", [(256, 16), (16, 256), (240, 112), (48, 240)])
def test_float_path_with_keys_and_values_of_many_sizes(cuda, dtype, dim, v_dim):
    for heads, kv_heads, starts, news in ((2, 1, [150, 64], [1, 2]), (8, 1, [500, 0, 63], [1, 1, 1]), (6, 2, [130, 7], [5, 3])):
        _attention(cuda, starts, news, heads, kv_heads, dim, dtype, v_dim=v_dim, seed=heads)
    _attention(cuda, [100, 5], [11, 4], 4, 2, dim, dtype, with_out=False, seed=9, spoil=float("inf"), in_place=False)


def test_window_with_missing_pages(cuda):
    from camelid_b200.csrc import ops
    for dim in (64, 128):
        gen = torch.Generator().manual_seed(6)
        k = torch.randn(5, 1, PAGE, dim, generator=gen).to(torch.bfloat16)
        q = torch.randn(40, 4 * dim, generator=gen).to(torch.bfloat16)
        table = [[-1, 1, 3, 99, 0], [2, -1, -1, -1, -1]]
        start, new, row0 = [260, 100], [20, 20], [0, 20]
        scores = torch.rand(5, 1, PAGE, generator=gen)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)    # noqa: E731
        scratch = torch.empty(ops.attn_weights_floats(2, 4, 1, dim, torch.bfloat16, 20, 280, False), device=cuda)
        s_dev = scores.to(cuda)
        ops.attn_paged_weights(q.to(cuda), None, k.to(cuda), None, s_dev, ints(table), ints(row0), ints(start), ints(new), 4, 20, 280, dim ** -0.5,
                               scratch)
        _, ref, _, tol = pb.weights(q, k, None, scores, table, row0, start, new, 4, dim ** -0.5)
        assert bool(((s_dev.cpu().double() - ref).abs() <= tol + 1e-30).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [5, 9, 17, 20, 33, 70])
def test_window_with_an_infinite_key(cuda, dim, new):
    """A key of minus infinity weighs nothing: its score stays a number, whatever rows fill up a tile."""
    from camelid_b200.csrc import ops
    gen = torch.Generator().manual_seed(new)
    k = torch.randn(9, 1, PAGE, dim, generator=gen).to(torch.bfloat16)
    q = torch.randn(new, 8 * dim, generator=gen).to(torch.bfloat16)
    q[:, ::dim] = q[:, ::dim].abs() + 0.1                      # the channel of every head that meets the infinite one
    k[4, 0, 7, 0] = -math.inf
    start, scores = 9 * PAGE - new - 3, torch.rand(9, 1, PAGE, generator=gen)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    scratch = torch.empty(ops.attn_weights_floats(1, 8, 1, dim, torch.bfloat16, new, start + new, False), device=cuda)
    s_dev = scores.to(cuda)
    ops.attn_paged_weights(q.to(cuda), None, k.to(cuda), None, s_dev, ints([list(range(9))]), ints([0]), ints([start]), ints([new]), 8, new,
                           start + new, dim ** -0.5, scratch)
    without = k.clone()
    without[4, 0, 7] = 0.0                                     # the tolerances of the other places
    _, _, _, tol = pb.weights(q, without, None, scores, [list(range(9))], [0], [start], [new], 8, dim ** -0.5)
    _, ref, _, _ = pb.weights(q, k, None, scores, [list(range(9))], [0], [start], [new], 8, dim ** -0.5)
    assert bool(torch.isfinite(ref).all()) and float(s_dev[4, 0, 7]) == float(scores[4, 0, 7])
    assert bool(((s_dev.cpu().double() - ref).abs() <= 2 * tol + 1e-30).all())


@pytest.mark.parametrize("dtype,dim,new", [(torch.bfloat16, 64, 1), (torch.bfloat16, 128, 6), (torch.bfloat16, 64, 40), (torch.float32, 48, 1),
                                           (torch.float32, 64, 9)])
def test_places_that_the_same_step_brought_start_from_zero(cuda, dtype, dim, new):
    """``seq_cached``: the places between it and the rows' own were written by this step, whatever score their page held."""
    from camelid_b200.csrc import ops
    gen = torch.Generator().manual_seed(new)
    with_out = new < 30
    k, v = (torch.randn(4, 2, PAGE, dim, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(2 * new, 8 * dim, generator=gen).to(dtype)
    scores = torch.rand(4, 2, PAGE, generator=gen)
    table, start, cached = [[0, 2], [3, 1]], [80, 70], [30, 70]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    scratch = torch.empty(ops.attn_weights_floats(2, 8, 2, dim, dtype, new, 120, with_out), device=cuda)
    s_dev, out = scores.to(cuda), torch.empty(2 * new, 8 * dim, dtype=dtype, device=cuda)
    ops.attn_paged_weights(q.to(cuda), out if with_out else None, k.to(cuda), v.to(cuda) if with_out else None, s_dev, ints(table), ints([0, new]),
                           ints(start), ints([new, new]), 8, new, 120, dim ** -0.5, scratch, seq_cached=ints(cached))
    for p in range(30, 80):
        scores[table[0][p // PAGE], :, p % PAGE] = 0
    _, ref, _, tol = pb.weights(q, k, v if with_out else None, scores, table, [0, new], start, [new, new], 8, dim ** -0.5)
    assert bool(((s_dev.cpu().double() - ref).abs() <= tol + 1e-30).all())


def test_weights_of_large_scores(cuda):
    """Scores of hundreds: nothing overflows, one place takes everything."""
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 128)):
        _attention(cuda, [150, 40], [1, 2], 4, 2, dim, dtype, scale=20.0)


# ---- eviction ---------------------------------------------------------------------------------------------------------
def _evict(cuda, lengths, keeps, first, recent, dtype=torch.bfloat16, entries=2, heads=2, dim=64, v_dim=64, in_place=False, rotary=0,
           interleaved=False, seed=0, scores=None, room=None):
    from camelid_b200.csrc import ops
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    kept_n = [min(n, m) for n, m in zip(lengths, keeps)]
    out_used = [(m + PAGE - 1) // PAGE for m in kept_n]
    table, n_pages, ids = _tables(rng, lengths, 1 if in_place else sum(out_used) + 1, spare=1)
    if in_place:
        out_table = table
    else:
        width, out_table, at = max(out_used + [1]), [], 0
        for u in out_used:
            out_table.append(ids[at:at + u] + [-1] * (width - u))
            at += u
    k = torch.randn(entries, n_pages, heads, PAGE, dim, generator=gen).to(dtype)
    v = torch.randn(entries, n_pages, heads, PAGE, v_dim, generator=gen).to(dtype) if v_dim else None
    s = torch.randint(0, 40, (entries, n_pages, heads, PAGE), generator=gen).float() / 8 if scores is None else scores(entries, n_pages, heads)
    inv_freq = (10000.0 ** (-torch.arange(rotary // 2).double() / max(rotary // 2, 1))).float() if rotary else None
    room = max(kept_n + [1]) if room is None else room
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    k_dev, s_dev = k.to(cuda), s.to(cuda)
    v_dev = v.to(cuda) if v_dim else None
    kept = torch.full((entries, len(lengths), heads, room), -7, dtype=torch.int32, device=cuda)
    t_dev = ints(table)
    ops.evict_positions(k_dev, v_dev, s_dev, t_dev, t_dev if in_place else ints(out_table), ints(lengths), ints(keeps), kept, first, recent,
                        inv_freq=inv_freq.to(cuda) if rotary else None, interleaved=interleaved)
    torch.cuda.synchronize()
    want_k, want_v, want_s = k.double(), v.double() if v_dim else None, s.clone()
    turned = torch.zeros(k.shape[:-1], dtype=torch.bool)
    for e in range(entries):
        for i, n in enumerate(lengths):
            for h in range(heads):
                line = [float(s[e, table[i][p // PAGE], h, p % PAGE]) for p in range(n)]
                places = pb.choose(line, n, min(keeps[i], room), first, recent)
                assert kept[e, i, h].tolist() == places + [-7] * (room - len(places)), (e, i, h)
                rows = []
                for j, p in enumerate(places):
                    src = (e, table[i][p // PAGE], h, p % PAGE)
                    key = k[src].double()
                    rows.append((pb.turn(key, j - p, inv_freq, interleaved) if rotary and j != p else key, v[src].double() if v_dim else None, s[src]))
                for j, (key, val, score) in enumerate(rows):
                    dst = (e, out_table[i][j // PAGE], h, j % PAGE)
                    want_k[dst], want_s[dst] = key, score
                    turned[dst] = bool(rotary) and j != places[j]
                    if v_dim:
                        want_v[dst] = val
    got_k = k_dev.cpu().double()
    assert torch.equal(got_k[~turned], want_k[~turned])
    if bool(turned.any()):
        # float turn: the angle is off by 2^-23 of a turn's half at most, sine, cosine, two products and a sum by a rounding each
        size = want_k[turned].abs().amax(-1, keepdim=True) * 1.5
        assert bool(((got_k - want_k)[turned].abs() <= size * 16 * 2.0 ** -24 + _rounding(dtype) * want_k[turned].abs() * 1.01 + 1e-30).all())
    if v_dim:
        assert torch.equal(v_dev.cpu().double(), want_v)
    assert torch.equal(torch.nan_to_num(s_dev.cpu(), nan=-1.0), torch.nan_to_num(want_s, nan=-1.0))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("first,recent", [(0, 0), (4, 16), (3, 500), (200, 9)])
def test_evict_ragged_sequences(cuda, in_place, first, recent):
    _evict(cuda, [1, 63, 64, 65, 200, 450, 7], [1, 10, 64, 64, 77, 130, 0], first, recent, in_place=in_place, seed=first + recent)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,dim,v_dim,rotary,interleaved", [
    (torch.bfloat16, 64, 64, 64, False), (torch.float32, 128, 128, 128, False), (torch.bfloat16, 96, 32, 32, True),
    (torch.float32, 256, 256, 64, True), (torch.bfloat16, 80, 0, 80, False), (torch.bfloat16, 256, 256, 0, False)])
def test_evict_turns_keys(cuda, in_place, dtype, dim, v_dim, rotary, interleaved):
    _evict(cuda, [300, 129, 640], [200, 128, 65], 2, 20, dtype=dtype, entries=1, heads=1, dim=dim, v_dim=v_dim, rotary=rotary,
           interleaved=interleaved, in_place=in_place, seed=dim)


def test_evict_scores_that_are_equal_infinite_or_no_numbers(cuda):
    def odd(entries, n_pages, heads):
        gen = torch.Generator().manual_seed(1)
        s = torch.randint(0, 3, (entries, n_pages, heads, PAGE), generator=gen).float()
        pick = torch.randint(0, 8, s.shape, generator=gen)
        for value, at in ((float("nan"), 0), (float("inf"), 1), (-float("inf"), 2), (-0.0, 3), (-3.4e38, 4)):
            s[pick == at] = value
        return s
    for keeps in ([70, 100], [190, 5], [130, 250]):
        _evict(cuda, [200, 300], keeps, 1, 3, scores=odd)
    _evict(cuda, [200, 300], [64, 100], 0, 0, scores=lambda e, p, h: torch.full((e, p, h, PAGE), 2.5))


def test_evict_keeps_no_more_than_there_is_room_for(cuda):
    _evict(cuda, [300, 100], [200, 100], 2, 5, room=90)


def test_evict_many_pages_in_place_by_few_units(cuda):
    """Clusters of blocks that share a unit, over many rounds."""
    for seed in range(3):
        _evict(cuda, [6000], [5000 - 700 * seed], 4, 64, entries=1, heads=1, dim=16, v_dim=16, in_place=True, rotary=16, seed=seed)


def test_evict_twice_and_one_entry(cuda):
    """A cache without the axis of entries; a second eviction of what the first left."""
    from camelid_b200.csrc import ops
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(6, 2, PAGE, 32, generator=gen).to(cuda) for _ in range(2))
    s = torch.rand(6, 2, PAGE, generator=gen).to(cuda)
    before = k.clone()
    table = torch.tensor([[5, 0, 3, 1]], dtype=torch.int32, device=cuda)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    first = torch.zeros(1, 2, 150, dtype=torch.int32, device=cuda)
    second = torch.zeros(1, 2, 80, dtype=torch.int32, device=cuda)
    ops.evict_positions(k, v, s, table, table, ints([250]), ints([150]), first, 2, 10)
    ops.evict_positions(k, v, s, table, table, ints([150]), ints([80]), second, 2, 10)
    for h in range(2):
        for j in (0, 1, 2, 40, 79):
            p = int(first[0, h, int(second[0, h, j])])
            assert torch.equal(k[int(table[0, j // PAGE]), h, j % PAGE], before[int(table[0, p // PAGE]), h, p % PAGE])


# ---- verification of drafts ---------------------------------------------------------------------------------------------
def _verify(cuda, vocab, lens, temperature, with_probs, seed=0, room=None, pad=0, spread=3.0, logits=None, drafts=None, probs=None, **filters):
    from camelid_b200.csrc import ops
    gen = torch.Generator().manual_seed(seed)
    n, room = len(lens), max(lens + [0]) if room is None else room
    row0 = [sum(lens[:i]) + i for i in range(n)]
    rows = sum(lens) + n
    if logits is None:
        logits = spread * torch.randn(rows, vocab, generator=gen)
    if probs is None and with_probs:
        probs = torch.zeros(n, room, vocab)
    given = drafts is not None
    if not given:
        drafts = torch.zeros(n, room, dtype=torch.int32)
    for i in range(n):
        for j in range(0 if given else lens[i]):
            row = logits[row0[i] + j]
            q = torch.softmax((row + 0.7 * torch.randn(vocab, generator=gen)) / (temperature or 1.0), 0)
            drafts[i, j] = int(torch.multinomial(q, 1, generator=gen)) if with_probs else int(row.argmax())
            if with_probs:
                probs[i, j] = q
    accept, draw = torch.rand(n, room, generator=gen), torch.rand(n, generator=gen)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    padded = torch.full((rows, vocab + pad), float("nan"))
    padded[:, :vocab] = logits
    counts = torch.full((n,), -9, dtype=torch.int32, device=cuda)
    tokens = torch.full((n, room + 1), -9, dtype=torch.int32, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    scratch = torch.full((ops.verify_bytes(rows, n, vocab),), 255, dtype=torch.uint8, device=cuda)
    ops.verify_drafts(padded.to(cuda)[:, :vocab], ints(row0), ints(lens), drafts.to(cuda), probs.to(cuda) if with_probs else None,
                      accept.to(cuda), draw.to(cuda), temperature, filters.get("top_k", 0), filters.get("top_p", 1.0),
                      filters.get("min_p", 0.0), counts, tokens, err, scratch)
    for i in range(n):
        count, token = pb.verify(logits, row0[i], lens[i], drafts[i], probs[i] if with_probs else None, accept[i], draw[i], temperature,
                                 **filters)
        want = drafts[i, :count].tolist() + [token] + [-1] * (room - count)
        assert int(counts[i]) == count and tokens[i].tolist() == want, (i, int(counts[i]), tokens[i].tolist(), count, token)
    return counts, tokens, int(err)


@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 2.0])
@pytest.mark.parametrize("vocab", [1, 5, 97, 1531, 8192, 8193, 50257])
def test_verify_matches_plain(cuda, vocab, temperature, with_probs):
    for seed in range(3):
        assert _verify(cuda, vocab, [4, 0, 2, 7, 1], temperature, with_probs, seed=seed)[2] == 0


@pytest.mark.parametrize("filters", [{"top_k": 1}, {"top_k": 40}, {"top_k": 1000}, {"top_p": 0.5}, {"top_p": 0.95, "min_p": 0.02},
                                     {"min_p": 0.2}, {"top_k": 50, "top_p": 0.9, "min_p": 0.01}])
@pytest.mark.parametrize("vocab", [97, 1531, 40000])
def test_verify_with_the_samplers_filters(cuda, vocab, filters):
    for with_probs in (True, False):
        assert _verify(cuda, vocab, [3, 0, 5], 0.8, with_probs, seed=vocab, **filters)[2] == 0


@pytest.mark.parametrize("n", [1, 4, 5, 15, 16, 40])
def test_verify_large_vocabularies(cuda, n):
    """Every way a sequence's row is shared: sixteen, eight and four blocks, alone on a multiprocessor or not, groups of one tile and of several."""
    lens = [(3 * i) % 5 for i in range(n)]
    for vocab in (16400, 65536, 70001, 140003):
        if n * vocab <= 1_200_000:
            assert _verify(cuda, vocab, lens, 0.9, n * vocab <= 300_000, seed=n)[2] == 0
            assert _verify(cuda, vocab, lens[::-1], 1.3, False, seed=n + 1, top_p=0.97)[2] == 0


def test_verify_without_room_for_drafts(cuda):
    """No drafts at all: the next token of every sequence."""
    for vocab in (500, 40000):
        for filters in ({}, {"top_p": 0.8}):
            _verify(cuda, vocab, [0, 0, 0], 0.9, False, room=0, **filters)
            _verify(cuda, vocab, [0, 0, 0], 0.0, True, room=0)


def test_verify_strided_rows(cuda):
    for pad in (1, 3, 4):
        _verify(cuda, 1000, [3, 2], 0.9, True, pad=pad, room=6)
        _verify(cuda, 1001, [3, 2], 0.9, False, pad=pad, top_p=0.9)
        _verify(cuda, 9001, [3, 2], 0.0, False, pad=pad)


def test_verify_logits_at_the_types_lowest(cuda):
    """Tokens that a mask of the lowest value excludes are never drawn, at any temperature."""
    gen = torch.Generator().manual_seed(2)
    for temperature in (0.1, 1.0, 0.0):
        for filters in ({}, {"top_p": 0.9}, {"top_k": 20}):
            logits = torch.randn(8, 3000, generator=gen)
            logits[:, ::2] = torch.finfo(torch.float32).min
            _, tokens, err = _verify(cuda, 3000, [3, 3], temperature, False, logits=logits, **filters)
            assert err == 0 and all(t == -1 or t % 2 == 1 for t in tokens.flatten().tolist())


def test_verify_rows_whose_mask_leaves_nothing(cuda):
    """Rows of nothing but the lowest value: every token is as likely as the others, in vocabularies that end inside a part too."""
    for vocab in (700, 1024, 1500, 9001):
        logits = torch.full((9, vocab), torch.finfo(torch.float32).min)
        drafts = torch.full((3, 2), vocab - 1, dtype=torch.int32)
        probs = torch.full((3, 2, vocab), 1.0 / vocab)
        for temperature in (0.5, 1.0):
            for seed in (0, 1):
                assert _verify(cuda, vocab, [2, 2, 2], temperature, True, seed=seed, logits=logits, drafts=drafts, probs=probs)[2] == 0
        assert _verify(cuda, vocab, [2, 2, 2], 0.0, False, logits=logits)[2] == 0
    # drafts that a row's share decides: 1 / vocabulary lies just above what the draw asks for
    from camelid_b200.csrc import ops
    vocab, n = 1025, 4096
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=cuda)        # noqa: E731
    counts, tokens, err = ints(n), ints(n, 2), ints(1)
    logits = torch.full((2 * n, vocab), torch.finfo(torch.float32).min, device=cuda)
    scratch = torch.empty(ops.verify_bytes(2 * n, n, vocab), dtype=torch.uint8, device=cuda)
    accept = (torch.arange(n, device=cuda)[:, None].float() + 0.5) / n                # accepted while below 1 / vocabulary
    ops.verify_drafts(logits, 2 * torch.arange(n, device=cuda).int(), ints(n) + 1, ints(n, 1) + 7, None, accept, accept[:, 0].contiguous(), 1.0, 0, 1.0,
                      0.0, counts, tokens, err, scratch)
    assert int(err) == 0 and torch.equal(counts, (accept[:, 0].double() < 1.0 / vocab).int())


@pytest.mark.parametrize("filters", [{}, {"top_p": 0.9}, {"top_k": 5}])
def test_verify_temperatures_at_the_edge(cuda, filters):
    """Temperatures far below the logits' own rounding, logits far above the temperature, and temperatures that level everything."""
    gen = torch.Generator().manual_seed(12)
    base = torch.randn(6, 5000, generator=gen) * 4
    base[:, 40] = base[:, 4000] = base.amax(1) + 0.25                 # two largest of one value
    for temperature in (1e-30, 1e-10, 3e-10, 1e-9, 3e-9, 1e-8, 1e-6):
        assert _verify(cuda, 5000, [2, 2], temperature, False, logits=base, **filters)[2] == 0
    for top in (1e6, 3e7, 1e10, 1e30):
        logits = base.clone()
        logits[:, 17] = logits[:, 4500] = top
        assert _verify(cuda, 5000, [2, 2], 1.0, False, logits=logits, **filters)[2] == 0
    if not filters:
        for temperature in (1e6, 1e30, 1e38):
            assert _verify(cuda, 5000, [2, 2], temperature, True, logits=base)[2] == 0


def test_verify_equal_logits(cuda):
    """Ties: the lowest id at temperature 0, the draw's share of the ids otherwise."""
    logits = torch.zeros(2, 40000)
    _, tokens, _ = _verify(cuda, 40000, [0, 0], 0.0, False, logits=logits, room=1)
    assert tokens.tolist() == [[0, -1], [0, -1]]
    _verify(cuda, 40000, [0, 0], 1.0, False, logits=logits, room=1, top_p=0.7001)
    _verify(cuda, 40000, [0, 0], 1.0, False, logits=logits, room=1, top_k=12345)


@pytest.mark.parametrize("vocab", [1531, 9001, 40000])
def test_verify_equal_logits_at_the_border_of_top_k(cuda, vocab):
    """Of equal logits the lower ids stay, whether they fit the candidates' list or not."""
    gen = torch.Generator().manual_seed(vocab)
    logits = torch.randn(5, vocab, generator=gen) - 8.0
    for row in range(5):
        places = torch.randperm(vocab, generator=gen)
        logits[row, places[:1100]] = 1.0
        logits[row, places[:100]] = 3.0 + torch.rand(100, generator=gen)
    for top_k in (1, 99, 100, 101, 300, 1099, 1100, 1400):
        for more in ({}, {"top_p": 0.7}, {"min_p": 0.1}):
            assert _verify(cuda, vocab, [2, 1], 0.8, False, seed=top_k, logits=logits, top_k=top_k, **more)[2] == 0
    flat = torch.zeros(5, vocab)
    for top_k in (1, 40, 2048, 2049):
        assert _verify(cuda, vocab, [2, 1], 1.0, False, seed=top_k, logits=flat, top_k=top_k)[2] == 0


def test_verify_drafters_own_distribution_is_the_targets(cuda):
    """q = p: every draft stays, and where the draw of a rejection would be from nothing, p is drawn from."""
    gen = torch.Generator().manual_seed(4)
    logits = torch.randn(5, 700, generator=gen)
    probs = torch.softmax(logits[:4].double(), -1).float()[None] * 0.999
    drafts = torch.multinomial(probs[0], 1, generator=gen).T.int()
    counts, _, err = _verify(cuda, 700, [4], 1.0, True, logits=logits, drafts=drafts, probs=probs)
    assert int(counts) == 4 and err == 0
    over = probs * 3.0                          # no probabilities: more than p everywhere, a draft of which is rejected
    _verify(cuda, 700, [4], 1.0, True, logits=logits, drafts=drafts, probs=over)


def test_verify_reports_what_it_cannot_use(cuda):
    gen = torch.Generator().manual_seed(8)
    for value in (float("nan"), float("inf"), -float("inf")):
        from camelid_b200.csrc import ops
        for top_p in (1.0, 0.9):
            logits = torch.randn(4, 9000, generator=gen)
            logits[2, 8500] = value             # the second sequence's first row
            ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
            counts, tokens, err = ints([-9, -9, -9]), ints([[-9, -9]] * 3), ints([0])
            scratch = torch.empty(ops.verify_bytes(4, 3, 9000), dtype=torch.uint8, device=cuda)
            ops.verify_drafts(logits.to(cuda), ints([0, 2, 3]), ints([1, 1, 1]), ints([[int(logits[0].argmax())], [9000], [4]]), None,
                              torch.zeros(3, 1, device=cuda), torch.full((3,), 0.5, device=cuda), 1.0, 0, top_p, 0.0, counts, tokens, err,
                              scratch)
            assert counts.tolist() == [1, 0, 0] and tokens[1].tolist() == [0, -1]
            assert tokens[2].tolist() == [-1, -1]          # rows 3 and 4: there is no row 4
            assert int(err) == 1 | 4 | 8
    drafts = torch.tensor([[-1, 3]], dtype=torch.int32)
    counts, tokens, err = _verify(cuda, 500, [2], 1.0, False, drafts=drafts)
    assert int(counts) == 0 and err == 4
    probs = torch.full((1, 2, 500), -1.0)
    counts, tokens, err = _verify(cuda, 500, [2], 1.0, True, drafts=torch.tensor([[1, 3]], dtype=torch.int32), probs=probs)
    assert err == 4


def test_verify_reports_an_infinite_probability_of_another_token(cuda):
    """The probabilities of the row that the next token is drawn from are all looked at."""
    probs = torch.full((1, 1, 500), 0.0)
    probs[0, 0, 3], probs[0, 0, 77] = 1e6, float("inf")        # the draft, token 3, is rejected
    counts, tokens, err = _verify(cuda, 500, [1], 1.0, True, drafts=torch.tensor([[3]], dtype=torch.int32), probs=probs)
    assert int(counts) == 0 and int(tokens[0, 0]) not in (3, 77) and err == 4


def test_verify_keeps_the_targets_distribution(cuda):
    """Over many sequences with one draft each, the first token is distributed as the target's own."""
    from camelid_b200.csrc import ops
    n, vocab = 20000, 16
    gen = torch.Generator().manual_seed(3)
    p_logits, q = torch.randn(vocab, generator=gen), torch.softmax(torch.randn(vocab, generator=gen), 0)
    drafts = torch.multinomial(q, n, replacement=True, generator=gen).int()[:, None]
    ints = lambda x: x.to(torch.int32).to(cuda)        # noqa: E731
    counts, tokens = torch.zeros(n, dtype=torch.int32, device=cuda), torch.zeros(n, 2, dtype=torch.int32, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    scratch = torch.empty(ops.verify_bytes(2 * n, n, vocab), dtype=torch.uint8, device=cuda)
    ops.verify_drafts(p_logits.expand(2 * n, vocab).contiguous().to(cuda), ints(torch.arange(n) * 2), ints(torch.ones(n)), drafts.to(cuda),
                      q.expand(n, 1, vocab).contiguous().to(cuda), torch.rand(n, 1, generator=gen).to(cuda), torch.rand(n, generator=gen).to(cuda),
                      1.0, 0, 1.0, 0.0, counts, tokens, err, scratch)
    share = torch.bincount(tokens[:, 0].cpu().long(), minlength=vocab).double() / n
    p = torch.softmax(p_logits.double(), 0)
    assert bool(((share - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all())       # five standard deviations


# ---- captured, replayed, on other streams -------------------------------------------------------------------------------
def _calls(cuda):
    """(names, what each call changes, the calls) on buffers of their own, of all kernels of the three operators."""
    from camelid_b200.csrc import ops
    gen = torch.Generator().manual_seed(1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    calls = []
    for dtype, dim, new, with_out in ((torch.bfloat16, 64, 1, True), (torch.bfloat16, 128, 6, True), (torch.bfloat16, 128, 20, True),
                                      (torch.bfloat16, 64, 6, False), (torch.bfloat16, 64, 40, False), (torch.float32, 32, 1, True),
                                      (torch.float32, 32, 5, True)):
        k, v = (torch.randn(9, 2, PAGE, dim, generator=gen).to(dtype).to(cuda) for _ in range(2))
        q = torch.randn(2 * new, 8 * dim, generator=gen).to(dtype).to(cuda)
        old, s, out = torch.rand(9, 2, PAGE, generator=gen).to(cuda), torch.zeros(9, 2, PAGE, device=cuda), torch.zeros_like(q)
        scratch = torch.empty(ops.attn_weights_floats(2, 8, 2, dim, dtype, new, 300, with_out), device=cuda)
        args = (q, out if with_out else None, k, v if with_out else None, old, ints([[0, 1, 2, 3, 4], [5, 6, 7, 8, -1]]), ints([0, new]),
                ints([250, 200]), ints([new, new]), 8, new, 300, 0.1, scratch)
        calls.append(([s, out], lambda args=args, s=s: ops.attn_paged_weights(*args, scores_out=s)))
    for dtype in (torch.bfloat16, torch.float32):
        k, v = (torch.randn(2, 12, 2, PAGE, 32, generator=gen).to(dtype).to(cuda) for _ in range(2))
        s = torch.rand(2, 12, 2, PAGE, generator=gen).to(cuda)
        kept = torch.zeros(2, 2, 2, 100, dtype=torch.int32, device=cuda)
        args = (k, v, s, ints([[0, 1, 2, 3], [4, 5, 6, -1]]), ints([[7, 8], [9, 10]]), ints([250, 180]), ints([100, 70]), kept, 2, 10)
        freq = torch.full((16,), 0.3, device=cuda)
        calls.append(([k, v, s, kept], lambda args=args, freq=freq: ops.evict_positions(*args, inv_freq=freq)))
    for filters in ((0, 1.0, 0.0), (20, 0.9, 0.0), (0, 0.8, 0.01), (0, 0.7, 0.0)):
        logits = (3 * torch.randn(7, 9000, generator=gen)).to(cuda)
        counts, tokens, err = ints([0, 0]), torch.zeros(2, 4, dtype=torch.int32, device=cuda), ints([0])
        scratch = torch.empty(ops.verify_bytes(7, 2, 9000), dtype=torch.uint8, device=cuda)
        args = (logits, ints([0, 4]), ints([3, 2]), logits.argmax(-1).int()[torch.tensor([[0, 1, 2], [4, 5, 6]], device=cuda)], None,
                torch.rand(2, 3, generator=gen).to(cuda), torch.rand(2, generator=gen).to(cuda), 0.8, *filters, counts, tokens, err, scratch)
        calls.append(([counts, tokens, err], lambda args=args: ops.verify_drafts(*args)))
    return calls


def test_captured_and_replayed_and_on_another_stream(cuda):
    want = []
    for changed, call in _calls(cuda):
        call()
        want.append([t.clone() for t in changed])
    for i, (changed, call) in enumerate(_calls(cuda)):      # buffers of their own: made anew from the same numbers
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            call()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(changed, want[i])), i
    for i, (changed, call) in enumerate(_calls(cuda)):
        start = [t.clone() for t in changed]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()                                          # kernels are loaded and their limits set before a capture
        torch.cuda.current_stream().wait_stream(side)
        for t, s in zip(changed, start):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for _ in range(3):
            for t, s in zip(changed, start):
                t.copy_(s)
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(changed, want[i])), i


def test_the_same_call_twice_gives_the_same_bits(cuda):
    calls = _calls(cuda)
    for i, (changed, call) in enumerate(calls):
        call()
        first = [t.clone() for t in changed]
        for _ in range(5):
            call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(changed, first)), i


def test_launches_are_counted_as_they_are_captured(cuda):
    """What the count of launches gains is the number of kernels in a captured call's graph, for every form."""
    import ctypes
    from camelid_b200.csrc import ops
    nodes_of = ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    err = ints([0])
    calls = []
    for dtype, dim, heads, new, with_out, pad, want in (
            (torch.bfloat16, 64, 4, 1, True, 0, 1), (torch.bfloat16, 128, 4, 8, True, 0, 1), (torch.bfloat16, 64, 4, 9, True, 0, 3),
            (torch.bfloat16, 64, 4, 8, False, 0, 1), (torch.bfloat16, 64, 4, 9, False, 0, 2), (torch.bfloat16, 64, 4, 200, False, 0, 4),
            (torch.bfloat16, 64, 4, 3, True, 3, 3), (torch.float32, 64, 4, 2, True, 0, 1), (torch.float32, 64, 4, 3, False, 0, 3)):
        k = torch.zeros(4, 1, PAGE, dim, dtype=dtype, device=cuda)
        q = torch.zeros(new, heads * dim + pad, dtype=dtype, device=cuda)[:, :heads * dim]
        out = torch.zeros(new, heads * dim, dtype=dtype, device=cuda) if with_out else None
        scratch = torch.empty(ops.attn_weights_floats(1, heads, 1, dim, dtype, new, 256, with_out), device=cuda)
        args = (q, out, k, k if with_out else None, torch.zeros(4, 1, PAGE, device=cuda), ints([[0, 1, 2, 3]]), ints([0]), ints([0]), ints([new]), heads,
                new, 256, 0.1, scratch)
        calls.append((lambda args=args: ops.attn_paged_weights(*args, err=err), want))
    table = ints([[0, 1, 2, 3]])
    evict = (k, k.clone(), torch.zeros(4, 1, PAGE, device=cuda), table, table, ints([200]), ints([100]), ints([[[0] * 100]]), 1, 2)
    calls.append((lambda: ops.evict_positions(*evict), 2))
    for temperature, top_p in ((0.0, 1.0), (0.7, 1.0), (0.7, 0.9)):
        args = (torch.zeros(2, 90, device=cuda), ints([0]), ints([1]), ints([[3]]), None, torch.zeros(1, 1, device=cuda), torch.zeros(1, device=cuda),
                temperature, 0, top_p, 0.0, ints([0]), ints([[0, 0]]), err, torch.empty(ops.verify_bytes(2, 1, 90), dtype=torch.uint8, device=cuda))
        calls.append((lambda args=args: ops.verify_drafts(*args), 2))
    side = torch.cuda.Stream()
    for i, (call, want) in enumerate(calls):
        with torch.cuda.stream(side):
            call()                                          # kernels are loaded and their limits set before a capture
        side.synchronize()
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        before = ops.launch_count()
        with torch.cuda.graph(graph):
            call()
        assert ops.launch_count() - before == want, i
        n = ctypes.c_size_t(0)
        assert nodes_of(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
        assert n.value == want, i


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_from_tables_wider_than_the_kept_scores(cuda, in_place):
    """Scores beyond place 49,152 are read again for every digit; the border lies in either part."""
    _evict(cuda, [50_300, 49_153], [900, 49_100], 4, 64, entries=1, heads=1, dim=16, v_dim=0, in_place=in_place, rotary=0, seed=11)
    _evict(cuda, [50_300], [700], 0, 0, entries=1, heads=1, dim=16, v_dim=0, in_place=in_place, rotary=16, seed=12,
           scores=lambda e, p, h: torch.randint(0, 30000, (e, p, h, PAGE), generator=torch.Generator().manual_seed(5)).float() - 15000.0)


def test_evict_with_missing_pages(cuda):
    """Places of a page that the table does not name stay last of all, even behind infinitely low scores; where they have to stay, what
    stands at their new places is left alone."""
    from camelid_b200.csrc import ops
    gen = torch.Generator().manual_seed(2)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)        # noqa: E731
    for missing in (-1, 6, 2 ** 31 - 1):
        k, s = torch.randn(6, 1, PAGE, 32, generator=gen), torch.full((6, 1, PAGE), -float("inf"))
        table = [[5, missing, 2, 4]]
        for out_table, keep, first in ((table, 128, 0), (table, 256, 0), ([[0, 1, 3]], 130, 70)):
            k_dev, s_dev, kept = k.to(cuda), s.to(cuda), torch.full((1, 1, 256), -7, dtype=torch.int32, device=cuda)
            t = ints(table)
            ops.evict_positions(k_dev, None, s_dev, t, t if out_table is table else ints(out_table), ints([256]), ints([keep]), kept, first, 0)
            there = [p for p in range(256) if p // PAGE != 1]
            want = [p for p in range(256) if p < first or p in there[max(0, min(first, 64)):]][:keep] if first else sorted(
                there[:keep] + [p for p in range(64, 128)][:max(0, keep - 192)])
            assert kept[0, 0].tolist() == want + [-7] * (256 - len(want)), (missing, keep, first)
            ref = k.clone()
            for j, p in enumerate(want):
                dst = out_table[0][j // PAGE]
                if p in there and 0 <= dst < 6:
                    ref[dst, 0, j % PAGE] = k[table[0][p // PAGE], 0, p % PAGE]
            assert torch.equal(k_dev.cpu(), ref), (missing, keep, first)
