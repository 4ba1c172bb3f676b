"""Norms of query and key heads with the rotation in the same pass, against a plain form in 64 bits.

Tolerance, per number: half a step of bf16 (2^-8 of it), and 2^-18 of the pair's amplitude |n1| + |n2| for what is computed in f32: the sum of up to 256
squares (13 additions deep), rsqrtf, three products, a turn rounded to 2^-25 of itself (2 pi 2^-25 < 2^-22) and sincospif's and the rotation's own
roundings are below 2^-19 together."""
import ctypes as C

import pytest
import torch


def _plain(x, w, positions, eps, theta, rot, interleaved):
    x = x.double()
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        n = n * w.double()
    i = torch.arange(rot // 2, dtype=torch.float64)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    first, second = first.long(), second.long()
    angle = positions.double()[:, None, None] * theta ** (-2 * i / max(rot, 1))
    want, amp = n.clone(), n.abs()
    a, b = n[..., first], n[..., second]
    want[..., first] = a * angle.cos() - b * angle.sin()
    want[..., second] = a * angle.sin() + b * angle.cos()
    amp[..., first] = amp[..., second] = a.abs() + b.abs()
    return want, 2.0 ** -8 * want.abs() + 2.0 ** -18 * amp


def _check(got, want, tol):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


def _random(*shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16()


CASES = [  # rows, hq, hkv, d, rot, interleaved, first position
    (1, 32, 8, 128, 128, False, 0),
    (1, 1, 1, 64, 64, True, 2 ** 31 - 2),
    (3, 5, 1, 64, 16, False, 2 ** 24),
    (7, 3, 3, 256, 256, True, 1000003),
    (2, 8, 2, 256, 64, False, 131072),
    (33, 16, 4, 64, 32, True, 77),
    (129, 7, 1, 128, 48, False, 999999),
    (1000, 12, 3, 128, 128, False, 0),
    (5000, 4, 2, 64, 64, False, 32000),
    (4, 40, 0, 128, 128, False, 9),
    (4, 0, 6, 128, 0, False, 9),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hq,hkv,d,rot,interleaved,start", CASES)
@pytest.mark.parametrize("weights", [True, False])
def test_rows_to_rows(rows, hq, hkv, d, rot, interleaved, start, weights):
    from dmlx_b200 import device as dev

    qkv = _random(rows, (hq + 2 * hkv) * d, seed=rows, scale=3.0)
    positions = (start + torch.arange(rows)).clamp(max=2 ** 31 - 1).to(torch.int32)
    wq, wk = (_random(d, seed=s) if weights else None for s in (1, 2))
    dqkv = qkv.cuda()
    q, k = dqkv[:, :hq * d].unflatten(1, (hq, d)), dqkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    args = dict(eps=1e-5, theta=500000.0, rot_dim=rot, interleaved=interleaved)
    got_q, got_k = dev.qk_norm_rope(q, k, positions.cuda(), cuda(wq), cuda(wk), **args)
    want = [_plain(x.cpu(), w, positions, 1e-5, 500000.0, rot, interleaved) for x, w in ((q, wq), (k, wk))]
    _check(got_q, *want[0])
    _check(got_k, *want[1])
    assert torch.equal(dqkv.cpu(), qkv)
    # in place, in the projection's rows: the same bits, and the values beside them as they were
    dev.qk_norm_rope(q, k, positions.cuda(), cuda(wq), cuda(wk), q_out=q, k_out=k, **args)
    assert torch.equal(q, got_q) and torch.equal(k, got_k) and torch.equal(dqkv[:, (hq + hkv) * d:].cpu(), qkv[:, (hq + hkv) * d:])


@pytest.mark.gpu
def test_positions_before_zero_turn_back_and_zero_rows_are_zero():
    from dmlx_b200 import device as dev

    q, k = _random(4, 2, 64, seed=3), _random(4, 1, 64, seed=4)
    q[1], k[2] = 0, 0
    positions = torch.tensor([-1, -70000, 5, 6], dtype=torch.int32)
    got = dev.qk_norm_rope(q.cuda(), k.cuda(), positions.cuda())
    for x, y in zip((q, k), got):
        _check(y, *_plain(x, None, positions, 1e-5, 10000.0, 64, False))
    assert not bool(got[0][1].any()) and not bool(got[1][2].any())


@pytest.mark.gpu
def test_numbers_that_are_not_finite_stay_in_their_head():
    from dmlx_b200 import device as dev

    q, k = _random(5, 4, 128, seed=5), _random(5, 2, 128, seed=6)
    positions = torch.arange(5, dtype=torch.int32)
    clean = [_plain(x, None, positions, 1e-5, 10000.0, 64, False) for x in (q, k)]
    q[2, 1, 3], k[0, 1, 127] = float("nan"), float("inf")
    got_q, got_k = dev.qk_norm_rope(q.cuda(), k.cuda(), positions.cuda(), rot_dim=64)
    assert bool(got_q[2, 1].isnan().all()) and bool(got_k[0, 1, 127].isnan())
    ok_q, ok_k = torch.ones(5, 4, dtype=torch.bool), torch.ones(5, 2, dtype=torch.bool)
    ok_q[2, 1] = ok_k[0, 1] = False
    for got, ok, (want, tol) in ((got_q, ok_q, clean[0]), (got_k, ok_k, clean[1])):
        assert bool(((got.double().cpu() - want).abs() <= tol)[ok].all())
    assert not bool(got_k[0, 1, :127].any())  # a number over an infinite root mean square


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_into_pages_it_is_the_two_steps_in_one(fp8, d):
    """Sequences that start inside a page, a prompt over several pages, and a row whose slot holds no page."""
    from dmlx_b200 import device as dev

    hq, hkv = 8, 2
    kind = dev.KV_FP8_E4M3 if fp8 else dev.KV_BF16
    wq, wk = _random(d, seed=1).cuda(), _random(d, seed=2).cuda()
    caches = [dev.PagedKVCache(2, hkv, d, 32, 4, 8, hq, max_rows=256, kv_dtype=kind) for _ in range(2)]
    for step, counts in enumerate(([70, 1, 31], [1, 1, 1], [5, 40, 2])):
        rows = sum(counts)
        lens = [c0.seq_len(s) for c0 in caches[:1] for s in range(3)]
        desc = torch.tensor([[s, n, lens[s], 0] for s, n in enumerate(counts)], dtype=torch.int32, device="cuda")
        row_seq = torch.cat([torch.full((n,), s) for s, n in enumerate(counts)]).to(torch.int32).cuda()
        positions = torch.cat([lens[s] + torch.arange(n) for s, n in enumerate(counts)]).to(torch.int32).cuda()
        qkv = _random(rows, (hq + 2 * hkv) * d, seed=10 + step).cuda()
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((hq * d, hkv * d, hkv * d), 1))
        for layer in range(2):
            rows_q, rows_k = dev.qk_norm_rope(q, k, positions, wq, wk, rot_dim=d // 2, interleaved=layer == 1)
            for cache, fused in zip(caches, (False, True)):
                if layer == 0:
                    cache.reserve(desc)
                if fused:
                    got = cache.norm_rope_append(layer, q, k.clone(), v, positions, row_seq, wq, wk, rot_dim=d // 2, interleaved=layer == 1)
                    assert torch.equal(got, rows_q)
                else:
                    cache.append(layer, rows_k, v.contiguous())
        for s in range(3):
            for layer in range(2):
                for a, b in zip(caches[0].gather(layer, s), caches[1].gather(layer, s)):
                    assert torch.equal(a, b)
    assert caches[1].error_word() == 0


@pytest.mark.gpu
def test_rows_without_a_page_are_not_written():
    from dmlx_b200 import device as dev

    d, cache = 64, dev.PagedKVCache(1, 1, 64, 4, 2, 2, 1, max_rows=8)
    cache.reserve(torch.tensor([[0, 3, 0, 0]], dtype=torch.int32, device="cuda"))
    before = [cache.page_raw(0, p)[0].copy() for p in range(4)]
    q, k = _random(3, 1, d, seed=1).cuda(), _random(3, 1, d, seed=2).cuda()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out = cache.norm_rope_append(0, q, k, k, ints(32, -5, 2), ints(0, 0, 1))  # behind the pages held, before the first, a slot that holds none
    assert torch.equal(out, dev.qk_norm_rope(q, k, ints(32, -5, 2))[0])
    cache.norm_rope_append(0, q, k, k, ints(0, 0, 0), ints(-1, 2, 1 << 30))
    assert all((cache.page_raw(0, p)[0] == b).all() for p, b in enumerate(before))


@pytest.mark.gpu
def test_captured_and_replayed_on_another_stream():
    from dmlx_b200 import device as dev

    q, k = torch.zeros((19, 8, 128), dtype=torch.bfloat16, device="cuda"), torch.zeros((19, 2, 128), dtype=torch.bfloat16, device="cuda")
    positions = torch.zeros(19, dtype=torch.int32, device="cuda")
    out = dev.qk_norm_rope(q, k, positions)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        dev.qk_norm_rope(q, k, positions, q_out=out[0], k_out=out[1])
    for seed in (1, 2):
        hq, hk, pos = _random(19, 8, 128, seed=seed), _random(19, 2, 128, seed=seed + 5), torch.arange(19, dtype=torch.int32) * 1000 * seed
        q.copy_(hq); k.copy_(hk); positions.copy_(pos)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for got, x in zip(out, (hq, hk)):
            _check(got, *_plain(x, None, pos, 1e-5, 10000.0, 128, False))


def test_what_is_refused():
    """(Nothing of it reaches a device.)"""
    from dmlx_b200 import _lib

    lib, buf = _lib.lib, (C.c_uint16 * 4096)()
    p = (C.addressof(buf) + 15) // 16 * 16

    def call(head_dim=64, rot=64, hq=2, hkv=1, eps=1e-5, theta=1e4, rows=2, q=p, k=p, qs=128, ks=64, w=None, pos=p, qo=p, ko=p, qos=128, kos=64):
        s = _lib.NormRope(hq, hkv, head_dim, rot, 0, eps, theta)
        return lib.b200_qk_norm_rope(C.byref(s), q, k, qs, ks, w, w, pos, rows, qo, ko, qos, kos, None)

    bad, unsupported = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED
    assert lib.b200_qk_norm_rope(None, p, p, 128, 64, None, None, p, 1, p, p, 128, 64, None) == bad
    for how in (dict(head_dim=32), dict(head_dim=96), dict(rot=8), dict(rot=80), dict(rot=-16), dict(rot=24)):
        assert call(**how) == unsupported, how
    for how in (dict(rows=-1), dict(hq=-1), dict(hkv=5000), dict(theta=0.0), dict(theta=float("inf")), dict(theta=float("nan")), dict(eps=-1.0), dict(eps=float("nan")),
                dict(q=None), dict(k=None), dict(pos=None), dict(qo=None), dict(ko=None), dict(qs=120), dict(ks=68), dict(qos=64), dict(kos=60), dict(q=p + 2), dict(k=p + 8),
                dict(qo=p + 4), dict(ko=p + 8), dict(w=p + 2)):
        assert call(**how) == bad, how
    s = _lib.NormRope(2, 1, 64, 64, 0, 1e-5, 1e4)
    assert lib.b200_kv_norm_rope_append(None, 0, C.byref(s), p, p, p, 128, 64, 64, None, None, p, p, 1, p, 128, None) == bad


@pytest.mark.gpu
def test_what_is_refused_of_a_pool():
    from dmlx_b200 import _lib
    from dmlx_b200 import device as dev

    cache = dev.PagedKVCache(1, 2, 64, 4, 2, 2, 4, max_rows=8)
    x = torch.zeros((4, 512), dtype=torch.bfloat16, device="cuda")
    ints = torch.zeros(4, dtype=torch.int32, device="cuda")

    def call(layer=0, hkv=2, d=64, v=x.data_ptr(), vs=128, seq=ints.data_ptr(), kv=cache._h):
        s = _lib.NormRope(4, hkv, d, 64, 0, 1e-5, 1e4)
        return _lib.lib.b200_kv_norm_rope_append(kv, layer, C.byref(s), x.data_ptr(), x.data_ptr(), v, 512, 512, vs, None, None, ints.data_ptr(), seq, 4, x.data_ptr(), 512, None)

    for how in (dict(layer=1), dict(layer=-1), dict(hkv=1), dict(d=128), dict(v=None), dict(v=x.data_ptr() + 2), dict(vs=64), dict(vs=132), dict(seq=None)):
        assert call(**how) == _lib.ERR_INVALID_ARGUMENT, how
    layered = dev.LayeredKVCache([(2, 64, 64)], 4, 2, 2, 4, max_rows=8)
    assert call(kv=layered._h) == _lib.ERR_UNSUPPORTED
    with pytest.raises(ValueError):
        dev.qk_norm_rope(x.view(4, 8, 64).float(), x.view(4, 8, 64), ints)
    with pytest.raises(ValueError):
        dev.qk_norm_rope(x.view(4, 8, 64), x.view(4, 8, 64), ints[:3])
