"""Attention of a batch whose sequences share pages, against softmax(q k / sqrt(d)) v in 64 bits over the tokens that the cache gives back.

Tolerance, per number: half a step of bf16 of the result, 2^-8 of it; the weights are rounded to bf16 before their product, 2^-8 of each, so 2^-8 of
E = sum p |v| / sum p; and a score is off by its f32 sum, (d / 16 + 2) 2^-22 of S = |q| |k| / sqrt(d), and by its exponent's argument and the
exponential, 2^-20 together for |scores| up to 16 or S: a weight and the sum by twice that, relative.

On 8-bit pages a weight, times its page's V scale over the largest of a run of pages, is rounded to f16, whose numbers below 2^-14 are 2^-24 apart: what is
small is off by up to 2^-25 instead, of the row's largest weight in the part, which is 1 or more, as is therefore the part's sum.  It multiplies the
code and that largest scale, so the part is off by 2^-25 max(scale) sum |code| at most, and what parts are joined to by no more than the worst of them
(their shares add up to 1).  Where the token that has nearly all the weight holds a zero, this is more than all the above."""
import ctypes as C
import math

import pytest
import torch


def _random(*shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16().cuda()


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _append(cache, counts, seed, layers=1):
    """counts: {slot: tokens} behind what the slots hold."""
    c = cache.cfg
    desc = [[slot, n, cache.seq_len(slot), 0] for slot, n in counts.items()]
    rows = sum(counts.values())
    cache.reserve(torch.tensor(desc, dtype=torch.int32, device="cuda"))
    for layer in range(layers):
        cache.append(layer, _random(rows, c.n_kv_heads, c.head_dim, seed=seed + layer), _random(rows, c.n_kv_heads, c.head_dim, seed=seed + 50 + layer))
    assert cache.error_word() == 0


def _held(cache, layer, slots):
    """Keys and values of the slots' tokens in 64 bits.  (gather() rounds what 8-bit pages hold to bf16; a page's codes times its scale are exact.)"""
    if cache.cfg.kv_dtype == 0:
        return {s: tuple(x.double() for x in cache.gather(layer, s)) for s in slots}
    pages, held = {}, {}
    for s in slots:
        table = cache.block_table(s)
        for p in table:
            if p not in pages:
                k, v, ks, vs = (torch.from_numpy(x) for x in cache.page_raw(layer, p))
                pages[p] = [(x.view(torch.float8_e4m3fn).double() * sc.double()[:, None, None]).permute(1, 0, 2) for x, sc in ((k, ks), (v, vs))]
        held[s] = tuple(torch.cat([pages[p][i] for p in table] or [torch.zeros((0, cache.cfg.n_kv_heads, cache.cfg.head_dim))]).cuda() for i in range(2))
    return held


def _value_codes(cache, layer, slot):
    """|code| [tokens, heads, dims] of a slot's values on 8-bit pages, and their scales [tokens, heads]."""
    raw = [[torch.from_numpy(x) for x in cache.page_raw(layer, p)] for p in cache.block_table(slot)]
    codes = [v.view(torch.float8_e4m3fn).double().abs().permute(1, 0, 2) for _, v, _, _ in raw]
    scales = [vs.double()[None].expand(v.shape[1], -1) for _, v, _, vs in raw]
    return torch.cat(codes or [torch.zeros((0, cache.cfg.n_kv_heads, cache.cfg.head_dim))]).cuda(), torch.cat(scales or [torch.zeros((0, cache.cfg.n_kv_heads))]).cuda()


def _want(cache, layer, q, row_seq, row_ctx):
    held = _held(cache, layer, {s for s in row_seq if 0 <= s < cache.cfg.max_seqs})
    small = {s: _value_codes(cache, layer, s) for s in held} if cache.cfg.kv_dtype != 0 else {}
    t, hq, d = q.shape
    group = hq // cache.cfg.n_kv_heads
    want, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for r, (s, n) in enumerate(zip(row_seq, row_ctx)):
        if s not in held or n <= 0:
            continue
        k, v = (x[:n].repeat_interleave(group, 1) for x in held[s])
        scores = torch.einsum("hd,thd->ht", q[r].double(), k) / math.sqrt(d)
        top = torch.einsum("hd,thd->ht", q[r].double().abs(), k.abs()).amax(1) / math.sqrt(d)
        p = torch.softmax(scores, 1)
        want[r] = torch.einsum("ht,thd->hd", p, v)
        e = torch.einsum("ht,thd->hd", p, v.abs())
        if cache.cfg.kv_dtype != 0:
            codes, scales = (x[:n] for x in small[s])
            tol[r] += (2.0 ** -25 * scales.amax(0)[:, None] * codes.sum(0)).repeat_interleave(group, 0)
        tol[r] += 2.0 ** -8 * want[r].abs() + (2.0 ** -8 + 2 * ((d / 16 + 2) * 2.0 ** -22 * top[:, None] + 2.0 ** -20 * (top[:, None] / 16).clamp(min=1))) * e
    return want, tol


def _check(got, want, tol):
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


def _run(cache, q, row_seq, row_ctx, layer=0, handle=None, **how):
    from dmlx_b200 import device as dev

    handle = handle or dev.SharedPrefixAttention(cache, max(len(row_seq), 1))
    handle.plan(_ints(*row_seq), _ints(*row_ctx))
    got = handle.run(layer, q, **how)
    assert cache.error_word() == 0
    return got


def _tree(dev, rows, system, docs, doc, own, hq, hkv, d, fp8=False, layers=1, seed=0):
    """`rows` sequences behind a common text and one of `docs` texts behind that, each with tokens of its own; (cache, slots, contexts)."""
    parents = 1 + docs
    longest = system + doc + max(own) + 64
    pages = -(-longest // 32)
    cache = dev.PagedKVCache(layers, hkv, d, pages * (parents + 1) + rows * (max(own) // 32 + 4), parents + rows, pages, hq, max_rows=max(longest, rows * max(own), 64),
                             kv_dtype=dev.KV_FP8_E4M3 if fp8 else dev.KV_BF16)
    if system:
        _append(cache, {0: system}, seed, layers)
    for i in range(docs):
        cache.fork(0, 1 + i, system)
        _append(cache, {1 + i: doc}, seed + 100 + i, layers)
    slots = [parents + i for i in range(rows)]
    for i, s in enumerate(slots):
        parent = 1 + i % docs if docs else 0
        if system + doc:
            cache.fork(parent, s, system + doc)
    mine = {s: own[i % len(own)] for i, s in enumerate(slots) if own[i % len(own)]}
    if mine:
        _append(cache, mine, seed + 200, layers)
    return cache, slots, [cache.seq_len(s) for s in slots]


class _Device:
    """`count` 32-bit words of device memory from `address` on."""

    def __init__(self, address, count):
        self.__cuda_array_interface__ = dict(shape=(count,), typestr="<i4", data=(address, False), version=3)


def _plan_of(handle):
    """What the handle's last plan made of the large nodes, {items per kv head, other items, blocks that work on them} and the items {slot, first member, members,
    first page, last page + 1, part, tiles of rows, -}, read behind the handle's pointers: pool, {rows, rows}, memory, header, five arrays, items."""
    words = (C.c_uint64 * 12).from_address(handle._h)
    torch.cuda.synchronize()
    header = torch.as_tensor(_Device(words[3], 5), device="cuda").tolist()
    items = torch.as_tensor(_Device(words[10], 8 * max(header[0], 1)), device="cuda").view(-1, 8)[:header[0]].tolist()
    return dict(large=header[0], other=header[1], workers=header[4], items=items)


def _forest(dev, docs, hq, hkv, d, fp8, seed=0):
    """Documents of their own, (rows, pages) each, every row with one token more.  Keys grow along a document, so that the largest score comes late, and values differ
    by 4^4 between pages; (cache, slots, contexts)."""
    pages, rows = max(p for _, p in docs) + 1, sum(r for r, _ in docs)
    cache = dev.PagedKVCache(1, hkv, d, sum(p for _, p in docs) + rows + 8, len(docs) + rows, pages, hq, max_rows=max(32 * pages, rows), kv_dtype=dev.KV_FP8_E4M3 if fp8 else dev.KV_BF16)
    slots = []
    for i, (count, of_doc) in enumerate(docs):
        tokens = 32 * of_doc
        cache.reserve(torch.tensor([[i, tokens, 0, 0]], dtype=torch.int32, device="cuda"))
        k, v = _random(tokens, hkv, d, seed=seed + i), _random(tokens, hkv, d, seed=seed + 1000 + i)
        k *= torch.linspace(0.02, 2.5, tokens, device="cuda").bfloat16()[:, None, None]
        v *= (4.0 ** ((torch.arange(tokens, device="cuda") // 32 * 7 + i) % 5 - 2)).bfloat16()[:, None, None]
        cache.append(0, k, v)
        for _ in range(count):
            slots.append(len(docs) + len(slots))
            cache.fork(i, slots[-1], tokens)
    _append(cache, {s: 1 for s in slots}, seed + 2000)
    return cache, slots, [cache.seq_len(s) for s in slots]


CASES = [  # rows, system, docs, doc, own tokens, hq, hkv, d, fp8
    (1, 0, 0, 0, [1], 4, 1, 64, False),
    (1, 0, 0, 0, [1000], 8, 2, 128, False),
    (2, 64, 0, 0, [1, 33], 8, 8, 128, False),
    (4, 500, 0, 0, [1, 20, 40], 32, 8, 128, False),
    (5, 96, 0, 0, [0, 1], 16, 1, 64, False),           # a context that is the shared pages alone; 16 query heads per kv head
    (7, 1100, 0, 0, [5, 64, 100], 12, 4, 128, False),  # 3 query heads per kv head
    (33, 300, 3, 1001, [1, 31, 32, 200], 16, 4, 64, False),
    (70, 2048, 0, 0, [3, 40], 32, 4, 128, False),      # more rows than two tiles hold
    (140, 129, 2, 64, [1, 70], 4, 2, 64, False),
    (40, 31, 4, 40, [1], 8, 2, 128, False),            # a prefix of less than a page, small nodes
    (3, 260, 0, 0, [9, 1], 8, 2, 128, True),
    (6, 1300, 0, 0, [33, 2], 16, 4, 128, True),
    (50, 700, 2, 333, [1, 64, 90], 32, 4, 128, True),
    (9, 40, 0, 0, [1], 6, 1, 128, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,system,docs,doc,own,hq,hkv,d,fp8", CASES)
def test_rows_of_a_tree(rows, system, docs, doc, own, hq, hkv, d, fp8):
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, rows, system, docs, doc, own, hq, hkv, d, fp8)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(rows)).tolist()
    slots, ctx = [slots[i] for i in order], [ctx[i] for i in order]
    q = _random(rows, hq, d, seed=9, scale=2.0)
    want, tol = _want(cache, 0, q, slots, ctx)
    _check(_run(cache, q, slots, ctx), want, tol)
    shorter = [max(1, n - 1 - 37 * i % n) for i, n in enumerate(ctx)]  # rows that see less than their slots hold
    _check(_run(cache, q, slots, shorter), *_want(cache, 0, q, slots, shorter))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_rows_of_any_kind_together(fp8):
    """A portion of a prompt (rows of one slot), the same row twice, rows without a context, slots that are none, and sequences that share nothing."""
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 12, 200, 0, 0, [5, 70, 1], 16, 4, 128, fp8)
    row_seq = [slots[0]] * 40 + [slots[3], -1, slots[3], 0, 13, slots[5], slots[6], slots[7], slots[8]]
    row_ctx = list(range(ctx[0] - 39, ctx[0] + 1)) + [ctx[3], 50, ctx[3], 32, 7, 0, 31, -4, 1]
    q = _random(len(row_seq), 16, 128, seed=3, scale=2.0)
    q[42] = q[40]
    got = _run(cache, q, row_seq, row_ctx)
    _check(got, *_want(cache, 0, q, row_seq, row_ctx))
    assert torch.equal(got[40], got[42])
    assert not bool(got[41].any()) and not bool(got[45].any()) and not bool(got[47].any())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_as_the_decode_step_s_attention_has_it(d):
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 24, 515, 2, 190, [1, 45], 8, 2, d, layers=3)
    handle = dev.SharedPrefixAttention(cache, 64)
    handle.plan(_ints(*slots), _ints(*ctx))
    for layer in range(3):
        q = _random(24, 8, d, seed=layer, scale=2.0)
        got = handle.run(layer, q)
        want, tol = _want(cache, layer, q, slots, ctx)
        _check(got, want, tol)
        _check(cache.attention(layer, q, _ints(*slots), _ints(*ctx)), want, tol)
        assert torch.equal(got, handle.run(layer, q))
    assert cache.error_word() == 0


@pytest.mark.gpu
def test_a_prefix_of_many_pages_and_rows_of_several_tiles():
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 100, 9000, 0, 0, [1, 40, 300], 16, 2, 128)
    q = _random(100, 16, 128, seed=1, scale=3.0)
    _check(_run(cache, q, slots, ctx), *_want(cache, 0, q, slots, ctx))


@pytest.mark.gpu
def test_scores_that_grow_and_scores_that_are_large():
    """Rows whose largest score comes late, again and again, and far above the others."""
    from dmlx_b200 import device as dev

    cache = dev.PagedKVCache(1, 1, 128, 128, 40, 60, 8, max_rows=2048)
    cache.reserve(torch.tensor([[0, 1600, 0, 0]], dtype=torch.int32, device="cuda"))
    k, v = _random(1600, 1, 128, seed=1), _random(1600, 1, 128, seed=2)
    k *= torch.linspace(0.01, 4.0, 1600, device="cuda").bfloat16()[:, None, None]
    cache.append(0, k, v)
    slots = list(range(1, 21))
    for s in slots:
        cache.fork(0, s, 1600)
    q = _random(20, 8, 128, seed=3, scale=2.0)
    ctx = [1600 - 3 * i for i in range(20)]
    _check(_run(cache, q, slots, ctx), *_want(cache, 0, q, slots, ctx))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_what_lies_behind_a_context_has_no_part_in_it(fp8):
    """Keys and values that are no numbers behind the tokens of a row's last page, from a sequence that had the page before."""
    from dmlx_b200 import device as dev

    cache = dev.PagedKVCache(1, 2, 128, 8, 6, 4, 8, max_rows=64, kv_dtype=dev.KV_FP8_E4M3 if fp8 else dev.KV_BF16)
    for page in range(8):
        k, v, ks, vs = cache.page_raw(0, page)
        k[:], v[:] = (0x7F, 0x7F) if fp8 else (0x7FC0, 0x7F80)  # NaN, infinity
        cache.page_load(0, page, k, v, ks + 1, vs + 1)
    _append(cache, {0: 32}, 1)
    for s in (1, 2, 3):
        cache.fork(0, s, 32)
    _append(cache, {1: 1, 2: 5, 3: 31}, 2)
    q = _random(4, 8, 128, seed=3)
    row_seq, row_ctx = [1, 2, 3, 0], [33, 37, 63, 7]
    got = _run(cache, q, row_seq, row_ctx)
    want, tol = _want(cache, 0, q, row_seq, row_ctx)
    assert bool(want.isfinite().all())
    _check(got, want, tol)


@pytest.mark.gpu
def test_numbers_that_are_not_finite_stay_in_their_row():
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 20, 400, 0, 0, [3, 40], 8, 2, 128)
    q = _random(20, 8, 128, seed=5, scale=2.0)
    want, tol = _want(cache, 0, q, slots, ctx)
    q[4, 3, 7] = float("nan")
    q[11, 6, 0] = float("inf")
    got = _run(cache, q, slots, ctx)
    fine = torch.ones(20, 8, dtype=torch.bool, device="cuda")
    fine[4, 3] = fine[11, 6] = False
    assert bool(((got.double() - want).abs() <= tol)[fine].all())
    assert not bool(got[4, 3].any())  # scores that are no numbers weigh nothing


@pytest.mark.gpu
def test_strided_rows_and_what_lies_around_them():
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 18, 130, 0, 0, [2, 50], 8, 2, 64)
    qkv = _random(18, 8 * 64 + 256, seed=6, scale=2.0)
    q = qkv[:, :512].unflatten(1, (8, 64))
    out = torch.full((20, 512 + 24), 5.0, dtype=torch.bfloat16, device="cuda")
    _run(cache, q, slots, ctx, out=out[:18, 8:520].unflatten(1, (8, 64)))
    _check(out[:18, 8:520].unflatten(1, (8, 64)), *_want(cache, 0, q, slots, ctx))
    assert bool((out[18:] == 5).all()) and bool((out[:, :8] == 5).all()) and bool((out[:, 520:] == 5).all())


@pytest.mark.gpu
def test_graphs_with_handles_of_their_own_on_two_streams():
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 30, 333, 0, 0, [1, 64], 8, 2, 128)
    sides = []
    for rows in (30, 11):
        row_seq, row_ctx, q = _ints(*slots[:rows]), _ints(*ctx[:rows]), torch.zeros((rows, 8, 128), dtype=torch.bfloat16, device="cuda")
        handle, out = dev.SharedPrefixAttention(cache, 32), torch.zeros_like(q)
        handle.plan(row_seq, row_ctx)
        handle.run(0, q, out=out)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            handle.plan(row_seq, row_ctx)
            handle.run(0, q, out=out)
        sides.append((row_seq, row_ctx, q, out, handle, graph, stream))
    for turn in range(3):
        for i, (row_seq, row_ctx, q, *_) in enumerate(sides):
            rows = q.shape[0]
            pick = torch.randperm(30, generator=torch.Generator().manual_seed(10 * turn + i))[:rows].tolist()
            row_seq.copy_(_ints(*[slots[p] for p in pick]))
            row_ctx.copy_(_ints(*[max(0, ctx[p] - turn * 50 * (p % 3)) for p in pick]))
            q.copy_(_random(rows, 8, 128, seed=turn + i, scale=2.0))
        torch.cuda.synchronize()
        for *_, graph, stream in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for row_seq, row_ctx, q, out, *_ in sides:
            _check(out, *_want(cache, 0, q, row_seq.tolist(), row_ctx.tolist()))
    assert cache.error_word() == 0


@pytest.mark.gpu
def test_plans_follow_the_pages():
    """A handle through a life: rows join, write into shared pages (copied first), leave, and their pages go to others."""
    from dmlx_b200 import device as dev

    cache = dev.PagedKVCache(1, 2, 128, 64, 8, 16, 8, max_rows=256)
    handle = dev.SharedPrefixAttention(cache, 8)
    _append(cache, {0: 150}, 1)
    for s in (1, 2, 3):
        cache.fork(0, s, 150)  # (a page is shared that is not full)
    steps = [lambda: None, lambda: _append(cache, {1: 1, 2: 1, 0: 1}, 2), lambda: _append(cache, {1: 60, 3: 40}, 3), lambda: cache.rollback(1, 70),
             lambda: _append(cache, {1: 90}, 4), lambda: cache.release([0, 2]), lambda: _append(cache, {0: 100, 4: 20}, 5), lambda: cache.fork(1, 5, 96),
             lambda: _append(cache, {5: 3, 1: 2}, 6)]
    for n, step in enumerate(steps):
        step()
        slots = [s for s in range(6) if cache.seq_len(s)]
        ctx = [cache.seq_len(s) for s in slots]
        q = _random(len(slots), 8, 128, seed=20 + n, scale=2.0)
        _check(_run(cache, q, slots, ctx, handle=handle), *_want(cache, 0, q, slots, ctx))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_a_handle_through_batches_of_many_and_few_rows(fp8):
    """16 query rows at most and more than that take other kernels; one handle, plans and layers in turn, captured and replayed too."""
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 36, 700, 0, 0, [1, 64, 130], 8, 2, 128, fp8, layers=2)
    handle = dev.SharedPrefixAttention(cache, 40)
    for n, rows in enumerate((36, 4, 1, 5, 36, 3)):
        row_seq, row_ctx = _ints(*slots[:rows]), _ints(*ctx[:rows])
        q = [_random(rows, 8, 128, seed=10 * n + layer, scale=2.0) for layer in range(2)]
        handle.plan(row_seq, row_ctx)
        got = [handle.run(layer, q[layer]) for layer in range(2)]
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            handle.plan(row_seq, row_ctx)
            again = [handle.run(layer, q[layer]) for layer in range(2)]
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            want, tol = _want(cache, layer, q[layer], slots[:rows], ctx[:rows])
            _check(got[layer], want, tol)
            _check(again[layer], want, tol)
    assert cache.error_word() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hq,hkv,d,fp8", [(70, 32, 4, 128, False), (70, 32, 4, 128, True), (33, 8, 2, 64, False), (65, 64, 4, 64, False), (9, 8, 2, 128, False)])
def test_a_row_s_bits_do_not_depend_on_its_place(rows, hq, hkv, d, fp8):
    """Plans made again, and of the rows in another order: which rows share a tile differs, no result does."""
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, rows, 650, 0, 0, [1, 40, 90], hq, hkv, d, fp8)
    q = _random(rows, hq, d, seed=4, scale=2.0)
    handle = dev.SharedPrefixAttention(cache, rows)
    first = _run(cache, q, slots, ctx, handle=handle)
    for turn in range(6):
        order = torch.randperm(rows, generator=torch.Generator().manual_seed(turn)).tolist() if turn % 2 else list(range(rows))
        again = _run(cache, q[order], [slots[i] for i in order], [ctx[i] for i in order], handle=handle)
        assert torch.equal(again, first[order])


@pytest.mark.gpu
def test_a_closed_pool_is_refused():
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 2, 64, 0, 0, [1], 4, 1, 64)
    handle = dev.SharedPrefixAttention(cache, 4)
    handle.plan(_ints(*slots), _ints(*ctx))
    cache.close()
    with pytest.raises(ValueError):
        handle.run(0, _random(2, 4, 64, seed=1))
    with pytest.raises(ValueError):
        handle.plan(_ints(*slots), _ints(*ctx))
    handle.close()


@pytest.mark.gpu
def test_as_many_rows_as_a_handle_holds():
    from dmlx_b200 import device as dev

    cache = dev.PagedKVCache(1, 1, 64, 4100, 4096, 3, 2, max_rows=4096)
    _append(cache, {0: 64}, 1)
    for s in range(1, 4096):
        cache.fork(0, s, 64)
    for lo in (1, 2049):
        _append(cache, {s: 1 for s in range(lo, min(lo + 2048, 4096))}, lo)
    slots = list(range(4096))
    ctx = [64] + [65] * 4095
    q = _random(4096, 2, 64, seed=2, scale=2.0)
    handle = dev.SharedPrefixAttention(cache, 4096)
    got = _run(cache, q, slots, ctx, handle=handle)
    some = list(range(0, 4096, 97))
    _check(got[some], *_want(cache, 0, q[some], [slots[i] for i in some], [ctx[i] for i in some]))
    alone = [0] * 4096  # no two rows share a page
    _check(_run(cache, q, slots, alone, handle=handle), torch.zeros_like(q).double(), torch.zeros_like(q).double())


@pytest.mark.gpu
def test_a_step_s_attention_half():
    """Projection, adapters, norms and rotation into pages, attention over the shared prefix, output projection with adapters: as a step calls them."""
    from dmlx_b200 import device as dev

    rows, hidden, hq, hkv, d = 21, 512, 8, 2, 64
    cache, slots, ctx = _tree(dev, rows, 333, 0, 0, [4, 40], hq, hkv, d)
    n = (hq + 2 * hkv) * d
    x = _random(rows, hidden, seed=1)
    w_qkv, w_o = _random(n, hidden, seed=2, scale=hidden ** -0.5), _random(hidden, hq * d, seed=3, scale=(hq * d) ** -0.5)
    adapters = [dev.LoraAdapters(3, n, hidden, 16), dev.LoraAdapters(3, hidden, hq * d, 16)]
    pairs = []
    for which, (w, (rows_out, cols)) in enumerate(zip(adapters, ((n, hidden), (hidden, hq * d)))):
        pairs.append({})
        for slot, rank in ((0, 16), (2, 5)):
            a, b = _random(rank, cols, seed=10 + slot + which, scale=cols ** -0.5), _random(rows_out, rank, seed=20 + slot + which, scale=rank ** -0.5)
            w.set(slot, a, b, 0.5)
            pairs[-1][slot] = (a.double(), b.double())
    row_adapter = [i % 4 - 1 for i in range(rows)]
    batch = dev.LoraBatch(32, 3, 16)
    batch.plan(_ints(*row_adapter))
    handle = dev.SharedPrefixAttention(cache, 32)
    cache.reserve(torch.tensor([[s, 1, c, 0] for s, c in zip(slots, ctx)], dtype=torch.int32, device="cuda"))
    after = [c + 1 for c in ctx]
    handle.plan(_ints(*slots), _ints(*after))
    wq, wk = _random(d, seed=30), _random(d, seed=31)
    # here the projections are plain products; in a step they are b200_qmm
    qkv = (x.float() @ w_qkv.float().T).bfloat16()
    adapters[0].apply(batch, x, qkv, out=qkv)
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((hq * d, hkv * d, hkv * d), 1))
    turned = cache.norm_rope_append(0, q, k, v, _ints(*ctx), _ints(*slots), wq, wk)
    got = handle.run(0, turned)
    want, tol = _want(cache, 0, turned, slots, after)
    _check(got, want, tol)
    flat = got.flatten(1)
    y = (flat.float() @ w_o.float().T).bfloat16()
    out = adapters[1].apply(batch, flat, y)
    for r, slot in enumerate(row_adapter):
        if slot in pairs[1]:
            a, b = pairs[1][slot]
            delta = 0.5 * b @ (a @ flat[r].double())
            assert bool(((out[r].double() - y[r].double() - delta).abs() <= 2.0 ** -8 * (y[r].double() + delta).abs() + 1e-5).all())
            a, b = pairs[0][slot]
        else:
            assert torch.equal(out[r], y[r])
    # the new key of a row is what the cache holds at its last place
    rows_q, rows_k = dev.qk_norm_rope(q, k, _ints(*ctx), wq, wk)
    assert torch.equal(rows_q, turned)
    for r, s in enumerate(slots):
        held_k, held_v = cache.gather(0, s)
        assert torch.equal(held_k[-1], rows_k[r]) and torch.equal(held_v[-1], v[r])


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [(9, 13, 22, 41, 5), (37, 40, 33, 35)])
@pytest.mark.parametrize("d,fp8", [(128, False), (128, True), (64, False)])
def test_blocks_that_take_items_of_both_kinds_in_turn(pages, d, fp8):
    """More items of large nodes than SMs, whatever lengths the plan picks (25 nodes of 8 kv heads): of one tile of rows (4 of 8 query heads) and of two (17)."""
    from dmlx_b200 import device as dev

    cache, slots, ctx = _forest(dev, [((4, 17)[i % 2], pages[i % len(pages)]) for i in range(25)], 64, 8, d, fp8)
    q = _random(len(slots), 64, d, seed=9)
    handle = dev.SharedPrefixAttention(cache, len(slots))
    got = _run(cache, q, slots, ctx, handle=handle)
    plan = _plan_of(handle)
    assert plan["large"] * 8 > plan["workers"] > 0 and {it[6] for it in plan["items"]} == {1, 2}
    for tiles in (1, 2):  # pages that end inside a block of four, and more blocks than there are places for keys and values
        lengths = [it[4] - it[3] for it in plan["items"] if it[6] == tiles]
        assert max(lengths) > (32 if min(pages) > 32 else 16) and any(n % 4 for n in lengths)
    _check(got, *_want(cache, 0, q, slots, ctx))
    assert torch.equal(got, handle.run(0, q))


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,fp8", [(128, 32, 8, False), (128, 48, 3, True), (64, 8, 8, False)])
def test_warps_that_take_many_items_in_turn(d, hq, hkv, fp8):
    """Rows that share nothing, of one page to several: more items than the chip has warps for them, so that each takes the pages of several through its ring."""
    from dmlx_b200 import device as dev

    rows = 1300
    cache = dev.PagedKVCache(1, hkv, d, 4 * rows, rows, 6, hq, max_rows=2048, kv_dtype=dev.KV_FP8_E4M3 if fp8 else dev.KV_BF16)
    counts = [(1, 40, 32, 65, 7, 129)[i % 6] for i in range(rows)]
    for lo in range(0, rows, 40):
        _append(cache, {s: counts[s] for s in range(lo, min(lo + 40, rows))}, lo)
    q = _random(rows, hq, d, seed=3, scale=2.0)
    slots = list(range(rows))
    handle = dev.SharedPrefixAttention(cache, rows)
    got = _run(cache, q, slots, counts, handle=handle)
    plan = _plan_of(handle)
    assert plan["large"] == 0 and plan["other"] * hkv > 12 * torch.cuda.get_device_properties(0).multi_processor_count
    some = list(range(0, rows, 7))
    _check(got[some], *_want(cache, 0, q[some], [slots[i] for i in some], [counts[i] for i in some]))
    assert torch.equal(got, handle.run(0, q))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [20, 3])
@pytest.mark.parametrize("fp8", [False, True])
def test_scores_that_are_no_numbers_weigh_nothing(rows, fp8):
    """A query that is no number, and keys: all of the first four pages for one kv head and some of later ones, of a node of many rows and of one of few."""
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, rows, 700, 0, 0, [3, 40], 8, 2, 128, fp8)
    q = _random(rows, 8, 128, seed=5, scale=2.0)
    want, tol = _want(cache, 0, q, slots, ctx)
    bad = q.clone()
    bad[1, 3, 7], bad[2, 6] = float("nan"), float("nan")
    got = _run(cache, bad, slots, ctx)
    fine = torch.ones(rows, 8, dtype=torch.bool, device="cuda")
    fine[1, 3] = fine[2, 6] = False
    assert bool(((got.double() - want).abs() <= tol)[fine].all())
    assert not bool(got[1, 3].any()) and not bool(got[2, 6].any())
    # keys of the second kv head
    table, hidden = cache.block_table(slots[0]), torch.zeros(700, dtype=torch.bool)
    for at, tokens in [(i, range(32)) for i in range(4)] + [(6, (0, 9, 31)), (20, (5,))]:
        k, v, ks, vs = cache.page_raw(0, table[at])
        for t in tokens:
            k[1, t, t % 128] = 0x7F if fp8 else 0x7FC0
            hidden[32 * at + t] = True
        cache.page_load(0, table[at], k, v, ks, vs)
    held = _held(cache, 0, set(slots))
    got = _run(cache, q, slots, ctx)
    assert bool(((got.double() - want).abs() <= tol)[:, :4].all())
    for r, s in enumerate(slots):
        k, v = (x[:ctx[r], 1] for x in held[s])
        there = torch.ones(ctx[r], dtype=torch.bool, device="cuda")
        there[:700] = ~hidden.cuda()
        assert bool(k[~there].isnan().any(1).all()) and bool(k[there].isfinite().all())
        scores = q[r, 4:].double() @ k[there].T / math.sqrt(128)
        top = (q[r, 4:].double().abs() @ k[there].abs().T).amax(1, keepdim=True) / math.sqrt(128)
        p = torch.softmax(scores, 1)
        of_row = 2.0 ** -8 * (p @ v[there]).abs() + (2.0 ** -8 + 2 * (10 * 2.0 ** -22 * top + 2.0 ** -20 * (top / 16).clamp(min=1))) * (p @ v[there].abs())
        if fp8:
            codes, scales = (x[:ctx[r], 1] for x in _value_codes(cache, 0, s))
            of_row += 2.0 ** -25 * scales.amax() * codes.sum(0)
        assert bool(((got[r, 4:].double() - p @ v[there]).abs() <= of_row).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_captured_layers_behind_plans_of_other_rows(fp8):
    """Layers in a graph without their plan: of more rows, of fewer, of rows for which a launch more would be needed, and of a plan that has not run."""
    from dmlx_b200 import _lib
    from dmlx_b200 import device as dev

    cache, slots, ctx = _tree(dev, 40, 400, 0, 0, [1, 64, 130], 8, 2, 128, fp8)
    q = _random(40, 8, 128, seed=2, scale=2.0)
    handle, out = dev.SharedPrefixAttention(cache, 64), torch.zeros((40, 8, 128), dtype=torch.bfloat16, device="cuda")
    plan = lambda rows: handle.plan(_ints(*slots[:rows]), _ints(*ctx[:rows]))  # noqa: E731
    unplanned, row_seq, row_ctx = torch.cuda.CUDAGraph(), _ints(*slots[:20]), _ints(*ctx[:20])
    with torch.cuda.graph(unplanned):
        handle.plan(row_seq, row_ctx)
        handle.run(0, q[:20], out=out[:20])
    out.fill_(7)
    handle.run(0, q[:20], out=out[:20])  # the plan was captured, and has not run
    assert cache.error_word() == 0 and bool((out == 7).all())
    graphs = {}
    for rows in (20, 4):
        plan(rows)
        handle.run(0, q[:rows], out=out[:rows])
        torch.cuda.synchronize()
        graphs[rows] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[rows]):
            handle.run(0, q[:rows], out=out[:rows])
    want, tol = _want(cache, 0, q, slots, ctx)
    for captured, planned in ((20, 40), (20, 8), (20, 0), (20, 20), (4, 2), (4, 0), (4, 3), (4, 40), (4, 4)):
        plan(planned)
        out.fill_(7)
        graphs[captured].replay()
        both = min(captured, planned)
        if (captured, planned) == (4, 40):
            assert cache.error_word() == _lib.ERR_INVALID_ARGUMENT
            both = 0
        assert cache.error_word() == 0
        if both:
            _check(out[:both], want[:both], tol[:both])
        assert bool((out[both:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("group", [2, 16])
def test_a_context_beyond_a_slot_s_pages_is_that_row_s_matter_alone(group):
    """A slot whose table still names pages that it has given up, and a row (of padding, say) that asks for them, ahead of rows that share what the slot still has."""
    from dmlx_b200 import device as dev

    cache = dev.PagedKVCache(1, 2, 128, 64, 8, 12, 2 * group, max_rows=512)
    _append(cache, {0: 320}, 1)
    for s in (1, 2, 3):
        cache.fork(0, s, 320)
    cache.rollback(1, 64)
    _append(cache, {1: 96}, 2)
    cache.rollback(3, 0)
    row_seq, row_ctx, held = [1, 0, 2, 3, 0], [320, 320, 320, 320, 319], [160, 320, 320, 0, 319]
    q = _random(5, 2 * group, 128, seed=3, scale=2.0)
    _check(_run(cache, q, row_seq, row_ctx), *_want(cache, 0, q, row_seq, held))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("each", [1, 6])
def test_trees_deeper_than_the_plan_goes(each, fp8):
    """Texts that go on from one another seven times, `each` rows behind every one; some go on by a page, which is too little for a node of its own."""
    from dmlx_b200 import device as dev

    lengths = [70, 130, 33, 96, 200, 32, 64]
    cache = dev.PagedKVCache(1, 2, 128, 400, 8 + 7 * each, 32, 8, max_rows=1024, kv_dtype=dev.KV_FP8_E4M3 if fp8 else dev.KV_BF16)
    slots, texts = [], 0
    for level, n in enumerate(lengths):
        if level:
            cache.fork(level - 1, level, texts)
        _append(cache, {level: n}, level)
        texts += n
        for i in range(each):
            slots.append(8 + len(slots))
            cache.fork(level, slots[-1], texts)
            if i % 3 != 2:
                _append(cache, {slots[-1]: 1 + 40 * i}, 100 + len(slots))
    order = torch.randperm(len(slots), generator=torch.Generator().manual_seed(1)).tolist()
    slots = [slots[i] for i in order] + [6, 0]
    ctx = [cache.seq_len(s) for s in slots]
    q = _random(len(slots), 8, 128, seed=4, scale=2.0)
    _check(_run(cache, q, slots, ctx), *_want(cache, 0, q, slots, ctx))


def test_what_is_refused():
    from dmlx_b200 import _lib

    lib, h = _lib.lib, C.c_void_p()
    bad = _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_prefix_attn_create(None, 8, C.byref(h)) == bad and h.value is None
    assert lib.b200_prefix_attn_create(None, 8, None) == bad
    assert lib.b200_prefix_attn_plan(None, None, None, 0, None) == bad
    assert lib.b200_prefix_attn_run(None, 0, None, 8, None, 8, None) == bad
    lib.b200_prefix_attn_destroy(None)


@pytest.mark.gpu
def test_what_is_refused_of_a_handle():
    from dmlx_b200 import _lib
    from dmlx_b200 import device as dev

    lib, bad, h = _lib.lib, _lib.ERR_INVALID_ARGUMENT, C.c_void_p()
    cache = dev.PagedKVCache(2, 2, 64, 8, 4, 4, 8, max_rows=16)
    for rows in (0, -1, 4097):
        assert lib.b200_prefix_attn_create(cache._h, rows, C.byref(h)) == bad and h.value is None
    for other in (dev.PagedKVCache(1, 1, 64, 8, 4, 4, 32, max_rows=16), dev.PagedKVCache(1, 2, 64, 8, 4, 4, 8, max_rows=16, kv_dtype=dev.KV_FP8_E4M3),
                  dev.LayeredKVCache([(2, 64, 64)], 8, 4, 4, 8, max_rows=16)):
        assert lib.b200_prefix_attn_create(other._h, 4, C.byref(h)) == _lib.ERR_UNSUPPORTED and h.value is None
    handle = dev.SharedPrefixAttention(cache, 8)
    x = torch.zeros((9, 1024), dtype=torch.bfloat16, device="cuda")
    p, ints = x.data_ptr(), torch.zeros(9, dtype=torch.int32, device="cuda")
    assert lib.b200_prefix_attn_run(handle._h, 0, p, 512, p, 512, None) == bad  # no plan yet
    assert lib.b200_prefix_attn_plan(handle._h, ints.data_ptr(), ints.data_ptr(), 9, None) == _lib.ERR_CAPACITY
    assert lib.b200_prefix_attn_plan(handle._h, None, ints.data_ptr(), 2, None) == bad
    assert lib.b200_prefix_attn_plan(handle._h, ints.data_ptr(), None, 2, None) == bad
    assert lib.b200_prefix_attn_plan(handle._h, ints.data_ptr(), ints.data_ptr(), -1, None) == bad
    handle.plan(ints[:2], ints[:2])
    for args in ((2, p, 512, p, 512), (-1, p, 512, p, 512), (0, None, 512, p, 512), (0, p, 512, None, 512), (0, p + 2, 512, p, 512), (0, p, 504, p, 512), (0, p, 516, p, 512),
                 (0, p, 512, p + 8, 512), (0, p, 512, p, 448)):
        assert lib.b200_prefix_attn_run(handle._h, *args, None) == bad, args
    q = x[:2, :512].unflatten(1, (8, 64))
    assert not bool(handle.run(0, q).any())
    with pytest.raises(ValueError):
        handle.run(0, x[:3, :512].unflatten(1, (8, 64)))
    with pytest.raises(ValueError):
        handle.run(0, q.float())
    with pytest.raises(ValueError):
        handle.plan(ints[:2].long(), ints[:2])
    handle.plan(ints[:0], ints[:0])
    assert handle.run(0, q[:0]).shape == (0, 8, 64)
