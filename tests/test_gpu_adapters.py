"""Low-rank adapters of many requests beside a shared projection, against a plain form in 64 bits.

Tolerance, per number: half a step of bf16 of the result (2^-8 of it), and what f32 sums may lose on the way.  u = A x is summed over K by MMAs whose
additions may drop everything below 2^-22 of the largest term (k / 16 of them at most in a row) and 64 + 16 f32 additions; hi + lo leaves 2^-17 of u;
the second product adds rank / 16 * 2 MMAs.  With U = |A| |x| that is |s| |B| ((k / 16 + 80) 2^-22 U + 2^-17 |u|) + |s| (rank / 8 + 16) 2^-22 |B| |u|,
and 2^-22 of the last sum's terms."""
import ctypes as C

import pytest
import torch


def _adapters(dev, slots, n, k, max_rank, ranks, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = dev.LoraAdapters(slots, n, k, max_rank)
    host = {}
    for slot, rank in enumerate(ranks):
        if rank == 0:
            continue
        a = (torch.randn((rank, k), generator=g) * k ** -0.5).bfloat16()
        b = (torch.randn((n, rank), generator=g) * rank ** -0.5).bfloat16()
        scale = float(torch.rand(1, generator=g)) * 2 - 0.5
        w.set(slot, a, b, scale)
        host[slot] = (a.double(), b.double(), float(torch.tensor(scale, dtype=torch.float32)))
    return w, host


def _want(host, row_adapter, x, y):
    want, tol = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    for r, slot in enumerate(row_adapter):
        if slot not in host:
            continue
        a, b, s = host[slot]
        xr = x[r].double()
        u, big = a @ xr, a.abs() @ xr.abs()
        delta = s * (b @ u)
        want[r] += delta
        tol[r] = abs(s) * (b.abs() @ ((x.shape[1] / 16 + 80) * 2.0 ** -22 * big + (2.0 ** -17 + (a.shape[0] / 8 + 16) * 2.0 ** -22) * u.abs()))
        tol[r] += 2.0 ** -22 * (y[r].double().abs() + delta.abs())
    return want, tol + 2.0 ** -8 * want.abs()


def _check(got, want, tol):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


def _rows(rows, width, seed):
    return torch.randn((rows, width), generator=torch.Generator().manual_seed(seed)).bfloat16()


CASES = [  # rows, adapters' ranks, max_rank, n, k
    (1, [16], 16, 128, 64),
    (1, [0, 7], 8, 8, 8),
    (3, [1, 16, 5], 16, 24, 40),
    (17, [16] * 4, 16, 4096, 4096),
    (64, [8, 0, 32, 17], 32, 1032, 520),
    (129, [64, 33, 0, 48], 64, 264, 2056),
    (300, [128, 65, 80, 1], 128, 520, 1000),
    (500, [128], 128, 40, 4104),
    (700, [16, 3], 16, 5000, 72),
    (2000, [30, 32], 32, 96, 640),
    (256, [16] * 255 + [0], 16, 64, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,ranks,max_rank,n,k", CASES)
@pytest.mark.parametrize("inplace", [False, True])
def test_every_row_gets_its_adapter(rows, ranks, max_rank, n, k, inplace):
    from dmlx_b200 import device as dev

    w, host = _adapters(dev, len(ranks), n, k, max_rank, ranks)
    g = torch.Generator().manual_seed(rows)
    row_adapter = torch.randint(-1, len(ranks) + 1, (rows,), generator=g).to(torch.int32)  # (one past the last is no adapter either)
    row_adapter[0] = len(ranks) - 1
    x, y = _rows(rows, k, 1), _rows(rows, n, 2)
    batch = dev.LoraBatch(max(rows, 32), len(ranks), max_rank)
    batch.plan(row_adapter.cuda())
    dy = y.cuda()
    got = w.apply(batch, x.cuda(), dy, out=dy if inplace else None)
    assert inplace == (got.data_ptr() == dy.data_ptr())
    _check(got, *_want(host, row_adapter.tolist(), x, y))
    none = torch.tensor([s not in host for s in row_adapter.tolist()])
    assert torch.equal(got.cpu()[none], y[none])


@pytest.mark.gpu
def test_strided_rows_and_what_lies_around_them():
    from dmlx_b200 import device as dev

    rows, n, k = 37, 72, 200
    w, host = _adapters(dev, 3, n, k, 24, [24, 0, 9])
    row_adapter = torch.arange(rows, dtype=torch.int32) % 4 - 1
    x, y = _rows(rows, k + 48, 3), _rows(rows, n + 16, 4)
    out = torch.full((rows + 5, n + 40), 7.0).bfloat16().cuda()
    batch = dev.LoraBatch(64, 3, 32)
    batch.plan(row_adapter.cuda())
    dx, dy = x.cuda(), y.cuda()
    w.apply(batch, dx[:, 16:16 + k], dy[:, 8:8 + n], out=out[:rows, 24:24 + n])
    _check(out[:rows, 24:24 + n], *_want(host, row_adapter.tolist(), x[:, 16:16 + k], y[:, 8:8 + n]))
    assert bool((out[rows:] == 7).all()) and bool((out[:, :24] == 7).all()) and bool((out[:, 24 + n:] == 7).all())
    assert torch.equal(dx.cpu(), x) and torch.equal(dy.cpu(), y)


@pytest.mark.gpu
def test_a_row_s_bits_do_not_depend_on_its_batch():
    from dmlx_b200 import device as dev

    n, k, rows = 1288, 4104, 400
    w, _ = _adapters(dev, 5, n, k, 64, [64, 16, 40, 8, 33])
    g = torch.Generator().manual_seed(5)
    row_adapter = torch.randint(0, 5, (rows,), generator=g).to(torch.int32)
    row_adapter[100:350] = 2
    x, y = _rows(rows, k, 6).cuda(), _rows(rows, n, 7).cuda()
    batch = dev.LoraBatch(rows, 5, 64)
    batch.plan(row_adapter.cuda())
    whole = w.apply(batch, x, y)
    batch.plan(row_adapter.cuda())
    assert torch.equal(whole, w.apply(batch, x, y))
    for part in (slice(0, 1), slice(5, 6), slice(90, 140), slice(100, 350)):
        batch.plan(row_adapter[part].cuda().contiguous())
        assert torch.equal(w.apply(batch, x[part], y[part]), whole[part])


@pytest.mark.gpu
def test_numbers_that_are_not_finite_stay_in_their_row():
    from dmlx_b200 import device as dev

    n, k, rows = 64, 256, 20
    w, host = _adapters(dev, 2, n, k, 16, [5, 16])  # (a rank of 5 is padded to 16: the padding has no part in an infinite row)
    row_adapter = torch.tensor([0, 1] * 10, dtype=torch.int32)
    x, y = _rows(rows, k, 8), _rows(rows, n, 9)
    clean, tol = _want(host, row_adapter.tolist(), x, y)
    x[3, 17], x[4, 9], y[7, 5] = float("nan"), float("inf"), float("-inf")
    batch = dev.LoraBatch(rows, 2, 16)
    batch.plan(row_adapter.cuda())
    got = w.apply(batch, x.cuda(), y.cuda()).double().cpu()
    fine = torch.ones(rows, dtype=torch.bool)
    fine[[3, 4, 7]] = False
    assert bool(((got - clean).abs() <= tol)[fine].all())
    assert bool(got[3].isnan().all())
    a, b, s = host[0]
    want = y[4].double() + s * (b @ (a @ x[4].double()))
    assert torch.equal(got[4].isnan(), want.isnan()) and torch.equal(got[4][~want.isnan()], want[~want.isnan()])
    assert float(got[7, 5]) == float("-inf") and bool(got[7, 6:].isfinite().all())


@pytest.mark.gpu
def test_set_again_clear_and_no_rows():
    from dmlx_b200 import device as dev

    n, k, rows = 136, 96, 9
    w, host = _adapters(dev, 2, n, k, 48, [48, 48])
    x, y = _rows(rows, k, 10), _rows(rows, n, 11)
    row_adapter = [0, 1, 0, 1, 1, 0, 0, 1, -1]
    batch = dev.LoraBatch(rows, 2, 48)
    batch.plan(torch.tensor(row_adapter, dtype=torch.int32, device="cuda"))
    a, b = torch.randn((3, k)).bfloat16(), torch.randn((n, 3)).bfloat16()
    w.set(0, a, b, 0.25)  # (a smaller rank where a larger one was)
    host[0] = (a.double(), b.double(), 0.25)
    _check(w.apply(batch, x.cuda(), y.cuda()), *_want(host, row_adapter, x, y))
    w.clear(1)
    del host[1]
    _check(w.apply(batch, x.cuda(), y.cuda()), *_want(host, row_adapter, x, y))
    batch.plan(torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert w.apply(batch, x.cuda()[:0], y.cuda()[:0]).shape == (0, n)


@pytest.mark.gpu
def test_graphs_with_batches_of_their_own_on_two_streams():
    from dmlx_b200 import device as dev

    n, k, rows = 520, 1032, 90
    w, host = _adapters(dev, 4, n, k, 32, [32, 8, 20, 16])
    sides = []
    for seed in (20, 30):
        row_adapter = torch.zeros(rows, dtype=torch.int32, device="cuda")
        x, y, out = (torch.zeros((rows, width), dtype=torch.bfloat16, device="cuda") for width in (k, n, n))
        batch, stream, graph = dev.LoraBatch(rows, 4, 32), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        batch.plan(row_adapter)
        w.apply(batch, x, y, out=out)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            batch.plan(row_adapter)
            w.apply(batch, x, y, out=out)
        sides.append((seed, row_adapter, x, y, out, batch, stream, graph))
    for turn in range(3):
        hosts = []
        for seed, row_adapter, x, y, *_ in sides:
            g = torch.Generator().manual_seed(seed + turn)
            ids, hx, hy = torch.randint(-1, 4, (rows,), generator=g).to(torch.int32), _rows(rows, k, seed + turn), _rows(rows, n, seed - turn)
            row_adapter.copy_(ids); x.copy_(hx); y.copy_(hy)
            hosts.append((ids.tolist(), hx, hy))
        torch.cuda.synchronize()
        for *_, stream, graph in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for side, of in zip(sides, hosts):
            _check(side[4], *_want(host, *of))


@pytest.mark.gpu
@pytest.mark.parametrize("captured,few,many", [(40, 7, 60), (1600, 900, 2000)])
def test_captured_layers_behind_plans_of_other_rows(captured, few, many):
    """Layers in a graph without their plan work on the rows that both have, and leave what lies behind as it was."""
    from dmlx_b200 import device as dev

    n, k = 264, 640
    w, host = _adapters(dev, 2, n, k, 32, [30, 32])
    row_adapter = (torch.arange(many, dtype=torch.int32) * 7 % 5 - 1).clamp(max=1)
    x, y = _rows(many, k, 1), _rows(many, n, 2)
    ids, dx, dy, out = row_adapter.cuda(), x.cuda(), y.cuda(), torch.zeros((many, n), dtype=torch.bfloat16, device="cuda")
    dx[captured:], dy[captured:] = float("nan"), float("nan")
    batch, graph = dev.LoraBatch(many, 2, 32), torch.cuda.CUDAGraph()
    batch.plan(ids[:captured])
    w.apply(batch, dx[:captured], dy[:captured], out=out[:captured])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        w.apply(batch, dx[:captured], dy[:captured], out=out[:captured])
    want, tol = _want(host, row_adapter.tolist(), x, y)
    for planned in (many, few, 0, captured):
        batch.plan(ids[:planned])
        out.fill_(7)
        graph.replay()
        both = min(planned, captured)
        if both:
            _check(out[:both], want[:both], tol[:both])
        assert bool((out[both:] == 7).all())


class _Device:
    """`count` 32-bit words of device memory from `address` on."""

    def __init__(self, address, count):
        self.__cuda_array_interface__ = dict(shape=(count,), typestr="<i4", data=(address, False), version=3)


def _tiles_of(batch):
    """Rows of the tiles that the batch's last plan made, those of many rows and those of few, read behind the handle's pointers: five numbers, order, tiles, header."""
    words, numbers = (C.c_uint64 * 6).from_address(batch._h), (C.c_int32 * 4).from_address(batch._h)
    torch.cuda.synchronize()
    many, _, few = torch.as_tensor(_Device(words[5], 3), device="cuda").tolist()
    tiles = torch.as_tensor(_Device(words[4], 4 * numbers[3]), device="cuda").view(-1, 4).tolist()
    return [t[2] for t in tiles[:many]], [t[2] for t in tiles[numbers[3] - few:]]


def _want_of_many(host, row_adapter, x, y):
    """_want, an adapter's rows at once."""
    want, tol = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    for slot, (a, b, s) in host.items():
        at = (row_adapter == slot).nonzero()[:, 0]
        xr = x[at].double()
        u, big = xr @ a.T, xr.abs() @ a.T.abs()
        delta = s * (u @ b.T)
        tol[at] = abs(s) * (((x.shape[1] / 16 + 80) * 2.0 ** -22 * big + (2.0 ** -17 + (a.shape[0] / 8 + 16) * 2.0 ** -22) * u.abs()) @ b.T.abs())
        tol[at] += 2.0 ** -22 * (y[at].double().abs() + delta.abs())
        want[at] += delta
    return want, tol + 2.0 ** -8 * want.abs()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,ranks,max_rank,n,k,tile", [
    (3000, [16, 9], 16, 1032, 4104, 64),
    (3000, [32, 20], 32, 72, 4104, 64),
    (3000, [64, 40], 64, 72, 2120, 64),
    (2000, [128, 80], 128, 72, 2120, 64),
    (9700, [16, 16, 5], 16, 72, 2120, 128),
    (9700, [30, 17], 32, 40, 4104, 128),
    (9900, [64, 33, 48], 64, 264, 4104, 128),
    (5300, [128, 65, 100], 128, 136, 4104, 128),
])
def test_tiles_of_many_rows(rows, ranks, max_rank, n, k, tile):
    """Tiles of 64 and 128 rows, the last one of an adapter ragged, K of several steps a 64th that ends inside one; of 128 rows more shares of tiles than blocks run at
    once, so that a block's loads go on into its next one."""
    from dmlx_b200 import device as dev

    w, host = _adapters(dev, len(ranks), n, k, max_rank, ranks)
    row_adapter = torch.randint(0, len(ranks), (rows,), generator=torch.Generator().manual_seed(rows)).to(torch.int32)
    row_adapter[5:rows:97] = -1
    x, y = _rows(rows, k, 1), _rows(rows, n, 2)
    batch = dev.LoraBatch(rows, len(ranks), max_rank)
    batch.plan(row_adapter.cuda())
    many, _ = _tiles_of(batch)
    assert max(many) == tile and any(t % 16 for t in many)
    if tile == 128:
        assert 4 * len(many) > torch.cuda.get_device_properties(0).multi_processor_count * (1 if max_rank > 64 else 2)
    got = w.apply(batch, x.cuda(), y.cuda())
    _check(got, *_want_of_many(host, row_adapter, x, y))
    assert torch.equal(got.cpu()[row_adapter < 0], y[row_adapter < 0])


@pytest.mark.gpu
@pytest.mark.parametrize("ranks,max_rank", [([64, 16, 40, 8, 33], 64), ([16, 3], 16), ([20, 32], 32), ([128, 65], 128)])
def test_a_row_s_bits_do_not_depend_on_the_size_of_its_tile(ranks, max_rank):
    """The same rows in tiles of 128, of 64, and of up to 16 rows, whose operands come another way."""
    from dmlx_b200 import device as dev

    n, k, rows = 136, 4104, 6000
    w, _ = _adapters(dev, len(ranks), n, k, max_rank, ranks)
    g = torch.Generator().manual_seed(5)
    row_adapter = torch.randint(0, len(ranks), (rows,), generator=g).to(torch.int32).cuda()
    x, y = _rows(rows, k, 6).cuda(), _rows(rows, n, 7).cuda()
    batch = dev.LoraBatch(rows, len(ranks), max_rank)
    batch.plan(row_adapter)
    assert max(_tiles_of(batch)[0]) == 128
    whole = w.apply(batch, x, y)
    for count, largest in ((2000 if max_rank > 64 else 3000, 64), (300, 16), (17, 16), (1, 1)):
        some = torch.randperm(rows, generator=g)[:count].cuda()
        batch.plan(row_adapter[some].contiguous())
        many, few = _tiles_of(batch)
        assert max(many + few) <= largest and (largest <= 16) == (not many)
        assert torch.equal(w.apply(batch, x[some], y[some]), whole[some]), count


def test_what_is_refused():
    from dmlx_b200 import _lib

    lib, h = _lib.lib, C.c_void_p()
    bad = _lib.ERR_INVALID_ARGUMENT
    for args in ((0, 64, 64, 16), (4097, 64, 64, 16), (4, 64, 64, 0), (4, 64, 64, 129), (4, 60, 64, 16), (4, 64, 4, 16), (4, 0, 64, 16), (4, 64, -8, 16)):
        assert lib.b200_lora_create(*args, C.byref(h)) == bad and h.value is None, args
    for args in ((0, 4, 16), (8, 0, 16), (8, 4097, 16), (8, 4, 0), (8, 4, 200), (-1, 4, 16), (1 << 30, 4, 16)):
        assert lib.b200_lora_batch_create(*args, C.byref(h)) == bad and h.value is None, args
    assert lib.b200_lora_create(4, 64, 64, 16, None) == bad and lib.b200_lora_batch_create(8, 4, 16, None) == bad
    assert lib.b200_lora_set(None, 0, 4, 1.0, None, None) == bad
    assert lib.b200_lora_plan(None, None, 0, None) == bad
    assert lib.b200_lora_apply(None, None, None, 8, None, 8, None, 8, None) == bad
    lib.b200_lora_destroy(None)
    lib.b200_lora_batch_destroy(None)


@pytest.mark.gpu
def test_what_is_refused_of_a_handle():
    from dmlx_b200 import _lib
    from dmlx_b200 import device as dev

    lib, bad = _lib.lib, _lib.ERR_INVALID_ARGUMENT
    w, _ = _adapters(dev, 2, 64, 64, 16, [16, 0])
    batch = dev.LoraBatch(8, 2, 16)
    x = torch.zeros((9, 128), dtype=torch.bfloat16, device="cuda")
    p = x.data_ptr()
    assert lib.b200_lora_apply(w._h, batch._h, p, 64, p, 64, p, 64, None) == bad  # no plan yet
    ids = torch.zeros(9, dtype=torch.int32, device="cuda")
    assert lib.b200_lora_plan(batch._h, ids.data_ptr(), 9, None) == _lib.ERR_CAPACITY
    assert lib.b200_lora_plan(batch._h, None, 3, None) == bad and lib.b200_lora_plan(batch._h, ids.data_ptr(), -1, None) == bad
    batch.plan(ids[:3])
    for args in ((p, 56, p, 64, p, 64), (p, 68, p, 64, p, 64), (p + 2, 64, p, 64, p, 64), (p, 64, None, 64, p, 64), (p, 64, p, 64, p + 8, 64), (p, 64, p, 64, p, 72),
                 (None, 64, p, 64, p, 64), (p, 64, p, 32, p, 64)):
        assert lib.b200_lora_apply(w._h, batch._h, *args, None) == bad, args
    for other in (dev.LoraBatch(8, 3, 16), dev.LoraBatch(8, 2, 8)):  # for other adapters, or smaller ranks
        other.plan(ids[:3])
        assert lib.b200_lora_apply(w._h, other._h, p, 64, p, 64, p, 64, None) == bad
    buf = (C.c_uint16 * (64 * 17))()
    for args in ((2, 4, 1.0, buf, buf), (-1, 4, 1.0, buf, buf), (0, 17, 1.0, buf, buf), (0, -1, 1.0, buf, buf), (0, 4, 1.0, None, buf), (0, 4, 1.0, buf, None)):
        assert lib.b200_lora_set(w._h, *args) == bad, args
    with pytest.raises(ValueError):
        w.apply(batch, x[:4, :64], x[:4, :64])
    with pytest.raises(ValueError):
        w.apply(batch, x[:3, :64].float(), x[:3, :64])
    with pytest.raises(ValueError):
        w.apply(batch, x[:3, :64].cpu(), x[:3, :64])
    with pytest.raises(ValueError):
        w.apply(batch, x[:3, ::2], x[:3, :64])
    with pytest.raises(ValueError):
        batch.plan(ids.long())
    torch.cuda.synchronize()


def test_the_struct_of_the_norm_is_the_header_s(tmp_path):
    import os
    import shutil
    import subprocess

    from dmlx_b200 import _lib

    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    fields = [f for f, _ in _lib.NormRope._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dmlx_b200.h"\nint main(void) { printf("%zu", sizeof(b200_norm_rope));'
                   + "".join(f' printf(" %zu", offsetof(b200_norm_rope, {f}));' for f in fields) + " return 0; }\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    seen = [int(v) for v in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert seen == [C.sizeof(_lib.NormRope)] + [getattr(_lib.NormRope, f).offset for f in fields]
