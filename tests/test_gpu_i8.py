"""Products in 8-bit integers and the gated feed-forward block of them, against plain forms in 64 bits.

Rows in 8 bits are held to the bit: 127 x of a bf16 x is exact, and so is the nearest whole number of the quotient in 64 bits (no quotient of such numbers
that is not a half is nearer than 2^-18 to one).  A product's sum is exact; its conversion to f32, the two factors, the step's own rounding and the
bias add five roundings of f32, 5 * 2^-24 of |product| + |bias|, and bf16 half a step, 2^-8 of the result."""
import ctypes as C

import pytest
import torch



def _weight(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int16).to(torch.int8)
    return q, torch.rand(n, generator=g) * 0.01 + 1e-4


def _x(rows, k, seed):
    return (torch.randn((rows, k), generator=torch.Generator().manual_seed(seed)) * 3).bfloat16()


def _quantized(x):
    """The definition: (whole numbers, steps) in 64 bits."""
    x = x.double()
    most = x.abs().amax(1, keepdim=True)
    q = torch.where(most > 0, torch.round(127 * x / most), torch.zeros_like(x))
    return q, most / 127


def _product(q, steps, w, scales):
    return q @ w.double().T * scales.double() * steps


def _off(got, want, tol):
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (float((off - tol).max()), int((off > tol).sum()))


def _check_mm(got, want, bias, f32):
    b = torch.zeros(1, dtype=torch.float64) if bias is None else bias.double()
    tol = 5 * 2.0 ** -24 * (want.abs() + b.abs())
    want = want + b
    _off(got.cpu(), want, tol if f32 else tol + 2.0 ** -8 * want.abs())


SHAPES = [  # rows, k, n
    (1, 1, 1), (1, 128, 128), (1, 4096, 512), (2, 130, 129), (7, 100, 300), (16, 256, 128), (17, 1000, 257), (33, 127, 1000), (64, 2048, 96), (65, 384, 640),
    (100, 5000, 130), (128, 512, 256), (129, 640, 384), (200, 4097, 72), (255, 136, 515), (256, 1024, 256), (257, 1152, 256), (300, 72, 2050), (513, 896, 1100),
    (1000, 264, 520), (1537, 2176, 384),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", SHAPES)
@pytest.mark.parametrize("f32,with_bias", [(False, False), (True, True)])
def test_product(rows, k, n, f32, with_bias):
    from dmlx_b200 import device as dev

    w, scales = _weight(n, k, 1)
    x = _x(rows, k, 2)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3)) if with_bias else None
    held = dev.I8Rows(rows, k)
    got = dev.i8_mm(dev.I8Weight(w, scales), held, x.cuda(), bias=None if bias is None else bias.cuda(), f32=f32)
    assert got.dtype == (torch.float32 if f32 else torch.bfloat16)
    q, steps = _quantized(x)
    _check_mm(got, _product(q, steps, w, scales), bias, f32)
    got_q, got_steps = held.get()
    assert torch.equal(got_q.cpu().double(), q) and torch.equal(got_steps.cpu(), x.abs().float().amax(1) / 127)
    assert dev.qmm_error_word() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 8), (5, 127), (700, 256), (1300, 513), (2, 8192), (400, 9000), (3, 16384), (310, 16500), (2, 32768), (2, 32769), (3, 70001)])
def test_rows_in_8_bits_to_the_bit(rows, k):
    """Halves of a step among them: a largest of 127 * 2^e makes every odd multiple of 2^(e-1) one."""
    from dmlx_b200 import device as dev

    x = _x(rows, k, 5)
    x[0] = (torch.randint(-254, 255, (k,), generator=torch.Generator().manual_seed(6)).float() * 0.25).bfloat16()
    x[0, k // 2] = 63.5
    if rows > 1:
        x[1] = (torch.randn(k, generator=torch.Generator().manual_seed(7)) * 2).round().bfloat16()  # few numbers, many halves
        x[1, 0] = 4.0
    held = dev.I8Rows(rows, k)
    held.quantize(x.cuda())
    q, steps = held.get()
    assert torch.equal(q.cpu().double(), _quantized(x)[0])
    assert torch.equal(steps.cpu(), x.abs().float().amax(1) / 127)


@pytest.mark.gpu
def test_rows_of_the_smallest_and_largest_numbers():
    from dmlx_b200 import device as dev

    x = _x(6, 300, 8)
    x[1] = 0
    x[2] = (x[2].float() * 2.0 ** -130).bfloat16()  # 127 / largest is no f32
    x[3] = (x[3].float() * 2.0 ** 124).bfloat16()
    x[4] = 0
    x[4, 17] = 2.0 ** -133  # the smallest bf16
    w, scales = _weight(200, 300, 9)
    held = dev.I8Rows(8, 300)
    got = dev.i8_mm(dev.I8Weight(w, scales), held, x.cuda(), f32=True).cpu()
    q, _ = held.get()
    q = q.cpu().double()
    assert torch.equal(q, _quantized(x)[0])
    assert bool((q[1] == 0).all()) and q[4].abs().sum() == 127
    # the product with the step that f32 holds (subnormal for the smallest), and subnormal results half of 2^-149 off
    steps = (x.abs().float().amax(1) / 127).double()[:, None]
    want = _product(q, steps, w, scales)
    fits = want.abs() < 3.4e38
    _off(torch.where(fits, got.double(), 0.0), torch.where(fits, want, 0.0), 5 * 2.0 ** -24 * want.abs() + 2.0 ** -149)
    assert bool((got[1] == 0).all())


LARGER = [  # rows, k, n: shares of K of a few rows, tiles of rows, pairs that share K, pairs that walk many items, a weight of more tiles than there are SMs
    (1, 14336, 4096), (4, 4096, 6144), (33, 2048, 2048), (130, 4096, 1024), (200, 4096, 4096), (300, 2048, 1024), (300, 14336, 256), (512, 4096, 4096), (700, 1000, 9000),
    (1100, 4096, 6144), (2500, 520, 3000), (20, 300, 30001), (260, 200, 20000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", LARGER)
@pytest.mark.parametrize("f32", [False, True])
def test_product_larger(rows, k, n, f32):
    from dmlx_b200 import device as dev

    w, scales = (t.cuda() for t in _weight(n, k, 15))
    x, bias = _x(rows, k, 16).cuda(), torch.randn(n, generator=torch.Generator().manual_seed(17)).cuda()
    got = dev.i8_mm(dev.I8Weight(w, scales), dev.I8Rows(rows, k), x, bias=bias, f32=f32)
    want = _product(*_quantized(x), w, scales)
    tol = 5 * 2.0 ** -24 * (want.abs() + bias.double().abs())
    want = want + bias.double()
    _off(got, want, tol if f32 else tol + 2.0 ** -8 * want.abs())
    assert dev.qmm_error_word() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,f", [(1, 4096, 14336), (3, 5000, 1000), (96, 4096, 8192), (128, 1024, 14336), (333, 2222, 5777), (600, 512, 9000), (1500, 300, 3000)])
def test_feed_forward_larger(rows, k, f):
    from dmlx_b200 import device as dev

    def scaled(n, k, seed):
        q, s = _weight(n, k, seed)
        return q.cuda(), (s * 0.7 * k ** -0.5).cuda()

    gate, up, down = scaled(f, k, 4), scaled(f, k, 5), scaled(k, f, 6)
    x = _x(rows, k, 7).cuda()
    got = dev.i8_ffn(dev.I8Weight.gated(*gate, *up), dev.I8Weight(*down), dev.I8Rows(rows, k, f), x)
    _check_ffn(got, x, gate, up, down, "silu")
    assert dev.qmm_error_word() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 5, 300])
def test_rows_that_hold_no_number(rows):
    """Such a row is NaN in every column; the others keep their bits."""
    from dmlx_b200 import device as dev

    n, k, f = 200, 700, 260
    x = _x(rows, k, 10)
    w = dev.I8Weight(*_weight(n, k, 11))
    gate_up, down = dev.I8Weight.gated(*_weight(f, k, 12), *_weight(f, k, 13)), dev.I8Weight(*_weight(n, f, 14))
    held = dev.I8Rows(rows, k, f)
    good = dev.i8_mm(w, held, x.cuda()), dev.i8_ffn(gate_up, down, held, x.cuda())
    bad = x.clone()
    bad[0, 3] = float("nan")
    bad[2, 699] = float("inf")
    bad[3, 0], bad[3, 1] = -float("inf"), float("nan")
    rest = [r for r in range(rows) if r not in (0, 2, 3)]  # (of four, one)
    for got, want in zip((dev.i8_mm(w, held, bad.cuda()), dev.i8_ffn(gate_up, down, held, bad.cuda())), good):
        assert bool(got[[0, 2, 3]].isnan().all())
        assert torch.equal(got[rest], want[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("k", [131072, 131071])
def test_the_largest_sums(k):
    from dmlx_b200 import device as dev

    w = torch.full((3, k), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 127
    x = torch.full((2, k), 1.5).bfloat16()
    x[1, 1::2] = -1.5
    got = dev.i8_mm(dev.I8Weight(w, torch.full((3,), 2.0 ** -20)), dev.I8Rows(2, k), x.cuda(), f32=True)
    q, steps = _quantized(x)
    _check_mm(got, _product(q, steps, w, torch.full((3,), 2.0 ** -20)), None, True)
    with pytest.raises(Exception, match="131072"):
        dev.I8Weight(torch.zeros((1, 131073), dtype=torch.int8), torch.ones(1))


def _act(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    return torch.nn.functional.gelu(g, approximate="tanh" if name == "gelu_tanh" else "none")


def _check_ffn(got, x, gate, up, down, act):
    """The inner rows are known to 2^-17 of a number (five roundings each of gate and up; an exponential of numbers up to 30) plus 2^-20 of |gate up| (the gate's
    roundings through the activation's slope, erf to two of its last places).  A number that is nearer than that to the border between two of the
    255 may be the other one; the step is off by as much as the largest number."""
    q, s = _quantized(x)
    g, u = _product(q, s, *gate), _product(q, s, *up)
    h = _act(g, act) * u
    slack = 2.0 ** -17 * h.abs() + 2.0 ** -20 * (u * g).abs()
    at = h.abs().argmax(1, keepdim=True)
    loose = (slack.gather(1, at) / h.abs().gather(1, at)).clamp(max=1)  # of the step
    q, s = _quantized(h)
    near = (127 * h / (127 * s)).abs()
    open_ = ((near - near.floor() - 0.5).abs() <= slack / s + near * loose).double()
    w = down[0].double().abs() * down[1].double()[:, None]
    want = _product(q, s, *down)
    tol = s * (open_ @ w.T) + loose * s * (q.abs() @ w.T)
    _off(got.double().to(want.device), want, tol + (2.0 ** -8 + 2.0 ** -21) * want.abs())
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows,k,f,n", [(1, 256, 384, 256), (3, 77, 130, 55), (16, 512, 1024, 512), (40, 1000, 1500, 999), (129, 256, 640, 130), (300, 333, 257, 333),
                                        (700, 512, 896, 512)])
def test_feed_forward(act, rows, k, f, n):
    from dmlx_b200 import device as dev

    def scaled(n, k, seed):
        q, s = _weight(n, k, seed)
        return q, s * 0.7 * k ** -0.5

    gate, up, down = scaled(f, k, 1), scaled(f, k, 2), scaled(n, f, 3)
    x = _x(rows, k, 4)
    held = dev.I8Rows(rows, k, f)
    got = dev.i8_ffn(dev.I8Weight.gated(*gate, *up), dev.I8Weight(*down), held, x.cuda(), activation=act)
    _check_ffn(got, x, gate, up, down, act)
    # the handle's own rows stay
    assert torch.equal(held.get()[0].cpu().double(), _quantized(x)[0])
    again = dev.i8_ffn(dev.I8Weight.gated(*gate, *up), dev.I8Weight(*down), held, activation=act)
    assert torch.equal(got, again)
    assert dev.qmm_error_word() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,f", [(1, 512, 700), (3, 77, 130), (4, 4096, 1024), (30, 1000, 300), (200, 256, 640), (700, 333, 515)])
def test_feed_forward_into_f32(rows, k, f):
    """Rounded, it is the block's result in bf16."""
    from dmlx_b200 import device as dev

    def scaled(n, k, seed):
        q, s = _weight(n, k, seed)
        return q, s * 0.7 * k ** -0.5

    gate, up, down = scaled(f, k, 4), scaled(f, k, 5), scaled(k, f, 6)
    gate_up, down_w, held, x = dev.I8Weight.gated(*gate, *up), dev.I8Weight(*down), dev.I8Rows(rows, k, f), _x(rows, k, 7).cuda()
    got = dev.i8_ffn(gate_up, down_w, held, x, f32=True)
    assert got.dtype == torch.float32 and torch.equal(got.bfloat16(), dev.i8_ffn(gate_up, down_w, held, x))
    _check_ffn(got, x.cpu(), gate, up, down, "silu")
    wide = torch.full((rows + 1, k + 5), 7.0, device="cuda")  # on no 16-byte boundary
    dev.i8_ffn(gate_up, down_w, held, out=wide[:rows, 3:3 + k], f32=True)
    assert torch.equal(wide[:rows, 3:3 + k], got) and bool((wide[rows:] == 7).all()) and bool((wide[:, :3] == 7).all()) and bool((wide[:, 3 + k:] == 7).all())
    with pytest.raises(ValueError):
        dev.i8_ffn(gate_up, down_w, held, x, out=torch.empty((rows, k), dtype=torch.bfloat16, device="cuda"), f32=True)
    from dmlx_b200 import _lib
    assert _lib.lib.b200_i8_ffn_f32(gate_up._h, down_w._h, held._h, None, 0, rows, 0, wide.data_ptr() + 2, k + 5, None) == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.gpu
def test_a_row_s_bits_do_not_depend_on_its_batch():
    from dmlx_b200 import device as dev

    k, f, n = 1400, 1300, 650
    x = _x(1200, k, 20).cuda()
    w = dev.I8Weight(*_weight(n, k, 21))
    gate_up, down = dev.I8Weight.gated(*_weight(f, k, 22), *_weight(f, k, 23)), dev.I8Weight(*_weight(n, f, 24))
    held = dev.I8Rows(1200, k, f)
    whole = dev.i8_mm(w, held, x, f32=True), dev.i8_ffn(gate_up, down, held, x)
    for first, rows in ((0, 1), (3, 2), (9, 4), (20, 5), (100, 16), (7, 31), (500, 64), (250, 128), (40, 200), (11, 300), (600, 513)):
        part = x[first:first + rows]
        assert torch.equal(dev.i8_mm(w, held, part, f32=True), whole[0][first:first + rows]), rows
        assert torch.equal(dev.i8_ffn(gate_up, down, held, part), whole[1][first:first + rows]), rows


@pytest.mark.gpu
@pytest.mark.parametrize("k,n,sizes", [(14336, 512, (1, 2, 4, 5, 40, 130)), (4096, 1024, (1, 3, 33, 130, 250)), (14336, 256, (300, 500)), (2048, 2048, (1, 64, 96))])
def test_sums_that_a_cluster_shares_out_meet_every_time(k, n, sizes):
    """Few tiles of a long K: shares of it in every cluster, one call behind the other, against the calls of many rows."""
    from dmlx_b200 import device as dev

    rows = 4000
    w, x = dev.I8Weight(*_weight(n, k, 35)), _x(rows, k, 36).cuda()
    want, held = dev.i8_mm(w, dev.I8Rows(rows, k), x, f32=True), dev.I8Rows(rows, k)
    for size in sizes:
        got = torch.empty_like(want)
        count = min(rows, 300 * size) // size * size
        for first in range(0, count, size):
            dev.i8_mm(w, held, x[first:first + size], out=got[first:first + size], f32=True)
        assert torch.equal(got[:count], want[:count]), size
    assert dev.qmm_error_word() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_a_row_s_bits_do_not_depend_on_its_batch_with_a_bias_and_any_activation(act):
    """Each kernel brings its sums to the output by itself."""
    from dmlx_b200 import device as dev

    k, f, n = 1400, 1300, 650
    x = _x(1200, k, 25).cuda()
    w, bias = dev.I8Weight(*_weight(n, k, 26)), torch.randn(n, generator=torch.Generator().manual_seed(27)).cuda() * 30

    def scaled(n, k, seed, by):
        q, s = _weight(n, k, seed)
        return q, s * by * k ** -0.5

    gate_up, down = dev.I8Weight.gated(*scaled(f, k, 28, 0.7), *scaled(f, k, 29, 0.7)), dev.I8Weight(*scaled(n, f, 30, 0.7))
    held = dev.I8Rows(1200, k, f)
    whole = dev.i8_mm(w, held, x, bias=bias, f32=True), dev.i8_mm(w, held, x, bias=bias), dev.i8_ffn(gate_up, down, held, x, activation=act)
    for first, rows in ((0, 1), (3, 2), (9, 4), (20, 5), (100, 16), (7, 31), (500, 64), (250, 128), (40, 200), (11, 300), (600, 513)):
        part = x[first:first + rows]
        got = dev.i8_mm(w, held, part, bias=bias, f32=True), dev.i8_mm(w, held, part, bias=bias), dev.i8_ffn(gate_up, down, held, part, activation=act)
        for a, b in zip(got, whole):
            assert torch.equal(a, b[first:first + rows]), rows


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [10, 300])
def test_activations_far_out(act, rows):
    """Rows of gates around 1e-6, 1, 5 and 12 (where a GELU cancels), 90 (where an exponential is no f32), 1e4 and 1e13 (where a cube is none)."""
    from dmlx_b200 import device as dev

    k, f, n = 256, 640, 130

    def scaled(n, k, seed):
        q, s = _weight(n, k, seed)
        return q, torch.full((n,), (3 * 74 * k ** 0.5) ** -1.0)

    gate, up, down = scaled(f, k, 1), scaled(f, k, 2), scaled(n, f, 3)
    x = (_x(rows, k, 4).float() * torch.tensor([1e-6, 1.0, 5.0, 12.0, 90.0, 1e4, 1e13]).repeat(rows)[:rows, None]).bfloat16()
    got = dev.i8_ffn(dev.I8Weight.gated(*gate, *up), dev.I8Weight(*down), dev.I8Rows(rows, k, f), x.cuda(), activation=act)
    assert bool(got.isfinite().all())
    _check_ffn(got, x, gate, up, down, act)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 5, 70, 600])
def test_a_block_s_result_over_its_rows(rows):
    """They are in 8 bits before the first number of it is there."""
    from dmlx_b200 import device as dev

    k, f = 520, 700
    gate_up, down = dev.I8Weight.gated(*_weight(f, k, 31), *_weight(f, k, 32)), dev.I8Weight(*_weight(k, f, 33))
    x, held = _x(rows, k, 34).cuda(), dev.I8Rows(rows, k, f)
    want = dev.i8_ffn(gate_up, down, held, x)
    assert torch.equal(dev.i8_ffn(gate_up, down, held, x, out=x), want) and torch.equal(x, want)


@pytest.mark.gpu
def test_an_activation_that_is_none_is_refused():
    from dmlx_b200 import device as dev

    gate_up, down = dev.I8Weight.gated(*_weight(48, 64, 2), *_weight(48, 64, 3)), dev.I8Weight(*_weight(64, 48, 4))
    held = dev.I8Rows(4, 64, 48)
    held.quantize(_x(3, 64, 6).cuda())
    want = held.get()
    for name in ("relu", "SiLU", None):
        with pytest.raises(ValueError, match="activation"):
            dev.i8_ffn(gate_up, down, held, _x(4, 64, 5).cuda(), activation=name)
    assert held.rows == 3 and all(torch.equal(a, b) for a, b in zip(held.get(), want))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 70, 400])
@pytest.mark.parametrize("at,x_more,y_at,y_more", [(8, 24, 16, 40), (1, 4, 3, 6), (5, 8, 0, 1)])
def test_strided_rows_and_what_lies_around_them(rows, at, x_more, y_at, y_more):
    from dmlx_b200 import device as dev

    k, n = 523, 200
    q, scales = _weight(n, k, 30)
    w = dev.I8Weight(q, scales)
    x = _x(rows, k + x_more, 31)
    dx = x.cuda()
    for f32 in (False, True):
        out = torch.full((rows + 2, n + y_more), 7.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
        dev.i8_mm(w, dev.I8Rows(rows + 3, k + 9), dx[:, at:at + k], out=out[:rows, y_at:y_at + n], f32=f32)
        inner = x[:, at:at + k]
        _check_mm(out[:rows, y_at:y_at + n], _product(*_quantized(inner), q, scales), None, f32)
        assert bool((out[rows:] == 7).all()) and bool((out[:, :y_at] == 7).all()) and bool((out[:, y_at + n:] == 7).all())
    assert torch.equal(dx.cpu(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 300])
def test_offsets_past_32_bits(rows):
    from dmlx_b200 import device as dev

    k, n = 256, 136
    stride = (2 ** 31 // (rows - 1) + 63) // 64 * 64
    q, scales = _weight(n, k, 40)
    x = _x(rows, k, 41)
    far = torch.empty(stride * (rows - 1) + k, dtype=torch.bfloat16, device="cuda").as_strided((rows, k), (stride, 1))
    far.copy_(x)
    out = torch.empty(stride * (rows - 1) + n, dtype=torch.bfloat16, device="cuda").as_strided((rows, n), (stride, 1))
    dev.i8_mm(dev.I8Weight(q, scales), dev.I8Rows(rows, k), far, out=out)
    _check_mm(out.contiguous(), _product(*_quantized(x), q, scales), None, False)


@pytest.mark.gpu
def test_weights_from_the_device_are_the_same():
    from dmlx_b200 import device as dev

    q, scales = _weight(300, 500, 50)
    x = _x(9, 500, 51).cuda()
    held = dev.I8Rows(16, 500)
    assert torch.equal(dev.i8_mm(dev.I8Weight(q, scales), held, x), dev.i8_mm(dev.I8Weight(q.cuda(), scales.cuda()), held, x))
    assert torch.equal(dev.i8_mm(dev.I8Weight(q.cuda(), scales), held), dev.i8_mm(dev.I8Weight(q, scales.cuda()), held))


@pytest.mark.gpu
def test_no_rows():
    from dmlx_b200 import device as dev

    held = dev.I8Rows(4, 64, 64)
    w, gate_up = dev.I8Weight(*_weight(32, 64, 60)), dev.I8Weight.gated(*_weight(64, 64, 61), *_weight(64, 64, 62))
    none = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    assert dev.i8_mm(w, held, none).shape == (0, 32) and dev.i8_mm(w, held).shape == (0, 32)
    assert dev.i8_ffn(gate_up, w, held, none).shape == (0, 32)
    assert held.get()[0].shape == (0, 64)


@pytest.mark.gpu
def test_a_handle_through_calls_of_many_and_few_rows():
    """Blocks of other widths and batches of other sizes one after the other: nothing of an earlier call is seen by a later one."""
    from dmlx_b200 import device as dev

    blocks = [(dev.I8Weight.gated(*_weight(f, k, f), *_weight(f, k, f + 1)), dev.I8Weight(*_weight(k, f, f + 2)), k) for k, f in ((256, 1500), (512, 130), (384, 700))]
    held = dev.I8Rows(400, 512, 1500)
    for seed, (rows, which) in enumerate(((400, 0), (3, 1), (17, 2), (400, 1), (1, 0), (260, 2), (4, 0), (90, 1))):
        gate_up, down, k = blocks[which]
        x = _x(rows, k, 200 + seed).cuda()
        assert torch.equal(dev.i8_ffn(gate_up, down, held, x), dev.i8_ffn(gate_up, down, dev.I8Rows(rows, k, 1500), x)), (rows, which)
        assert torch.equal(held.get()[0].cpu().double(), _quantized(x.cpu())[0])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 48, 600])
def test_two_graphs_at_a_time_with_a_handle_each(rows):
    from dmlx_b200 import device as dev

    k, f = 512, 768
    gate, up, down = _weight(f, k, 70), _weight(f, k, 71), _weight(k, f, 72)
    gate_up, down_w = dev.I8Weight.gated(*gate, *up), dev.I8Weight(*down)
    graphs = []
    for i in range(2):
        held, x = dev.I8Rows(rows, k, f), torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            dev.i8_ffn(gate_up, down_w, held, x)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                y = dev.i8_ffn(gate_up, down_w, held, x)
        graphs.append((graph, stream, x, y, held))
    torch.cuda.synchronize()
    inputs = [[_x(rows, k, 80 + 10 * i + j).cuda() for j in range(3)] for i in range(2)]
    held = dev.I8Rows(rows, k, f)
    want = [[dev.i8_ffn(gate_up, down_w, held, x) for x in xs] for xs in inputs]
    torch.cuda.synchronize()
    for j in range(3):
        for (graph, stream, x, y, _), xs in zip(graphs, inputs):
            with torch.cuda.stream(stream):
                x.copy_(xs[j])
                for _ in range(4):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, y, _), w in zip(graphs, want):
            assert torch.equal(y, w[j])
    assert dev.qmm_error_word() == 0


@pytest.mark.gpu
def test_the_first_calls_of_a_process_may_be_captured():
    """Nothing is allocated, and nothing waited for, once the handles are there."""
    import os
    import subprocess
    import sys

    code = """
import torch
from dmlx_b200 import device as dev
g = torch.Generator().manual_seed(1)
w = lambda n, k: (torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int16).to(torch.int8), torch.rand(n, generator=g) * 0.001)
gate_up, down = dev.I8Weight.gated(*w(700, 300), *w(700, 300)), dev.I8Weight(*w(300, 700))
graphs = []
for rows in (2, 40, 900):
    held, x = dev.I8Rows(rows, 300, 700), torch.randn((rows, 300), generator=g).bfloat16().cuda()
    norm = torch.ones(300, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, _ = dev.residual_norm(x, x, norm, rows=held)
        y = dev.i8_ffn(gate_up, down, held)
    graph.replay()
    torch.cuda.synchronize()
    h2, _ = dev.residual_norm(x, x, norm, rows=held)
    assert torch.equal(y, dev.i8_ffn(gate_up, down, held)) and torch.equal(h, h2)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_a_handle_s_rows_in_a_graph_without_what_made_them():
    """A product in a graph takes what the handle holds when it runs."""
    from dmlx_b200 import device as dev

    rows, k, n = 20, 300, 140
    w = dev.I8Weight(*_weight(n, k, 90))
    held = dev.I8Rows(64, k)
    xs = [_x(rows, k, s).cuda() for s in (91, 92)]
    held.quantize(xs[0])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = dev.i8_mm(w, held)
    for x in xs:
        held.quantize(x)
        graph.replay()
        torch.cuda.synchronize()
        other = dev.I8Rows(rows, k)
        assert torch.equal(y, dev.i8_mm(w, other, x))


@pytest.mark.gpu
def test_refusals():
    from dmlx_b200 import _lib
    from dmlx_b200 import device as dev

    w, gate_up, down = dev.I8Weight(*_weight(32, 64, 1)), dev.I8Weight.gated(*_weight(48, 64, 2), *_weight(48, 64, 3)), dev.I8Weight(*_weight(64, 48, 4))
    held = dev.I8Rows(4, 64, 40)
    x = _x(4, 64, 5).cuda()
    for call in (lambda: dev.i8_mm(w, held), lambda: dev.i8_mm(w, held, x.float()), lambda: dev.i8_mm(w, held, x[:, :32]), lambda: dev.i8_mm(w, held, x.T),
                 lambda: dev.i8_mm(w, held, x, bias=torch.zeros(31, device="cuda")), lambda: dev.i8_mm(w, held, x, bias=torch.zeros(32, device="cuda").bfloat16()),
                 lambda: dev.i8_mm(w, held, x, out=torch.empty((4, 32), device="cuda")), lambda: dev.i8_mm(w, held, x.cpu()),
                 lambda: dev.I8Weight(torch.zeros((4, 4)), torch.ones(4)), lambda: dev.I8Weight(torch.zeros((4, 4), dtype=torch.int8), torch.ones(3)),
                 lambda: dev.I8Weight(torch.zeros((4, 4), dtype=torch.int8), torch.ones(4).double())):
        with pytest.raises(ValueError):
            call()

    def refused(status, call):
        with pytest.raises(_lib.B200Error) as e:
            call()
        assert e.value.status == status, e.value

    refused(_lib.ERR_INVALID_ARGUMENT, lambda: dev.i8_mm(gate_up, held, x))
    refused(_lib.ERR_INVALID_ARGUMENT, lambda: dev.i8_ffn(w, down, held, x))
    refused(_lib.ERR_INVALID_ARGUMENT, lambda: dev.i8_ffn(gate_up, w, held, x))
    refused(_lib.ERR_CAPACITY, lambda: dev.i8_ffn(gate_up, down, held, x))  # 48 channels, a handle for 40
    refused(_lib.ERR_CAPACITY, lambda: dev.i8_mm(w, held, _x(5, 64, 5).cuda()))
    refused(_lib.ERR_CAPACITY, lambda: held.quantize(_x(4, 65, 5).cuda()))
    held.quantize(x)
    lib, stream = _lib.lib, None
    out = torch.empty((4, 32), dtype=torch.bfloat16, device="cuda")
    assert lib.b200_i8_mm(w._h, held._h, None, 0, 3, None, out.data_ptr(), 32, 0, stream) == _lib.ERR_INVALID_ARGUMENT  # it holds four
    assert lib.b200_i8_mm(w._h, held._h, x.data_ptr(), 63, 4, None, out.data_ptr(), 32, 0, stream) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_mm(w._h, held._h, x.data_ptr() + 1, 64, 2, None, out.data_ptr(), 32, 0, stream) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_mm(w._h, held._h, x.data_ptr(), 64, 4, None, out.data_ptr(), 31, 0, stream) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_mm(w._h, held._h, x.data_ptr(), 64, 4, None, out.data_ptr() + 2, 32, 1, stream) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_mm(w._h, held._h, x.data_ptr(), 64, 4, None, None, 32, 0, stream) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_mm(w._h, held._h, x.data_ptr(), 64, -1, None, out.data_ptr(), 32, 0, stream) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_ffn(gate_up._h, down._h, held._h, x.data_ptr(), 64, 4, 3, out.data_ptr(), 64, stream) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_mm(w._h, held._h, x.data_ptr(), 64, 4, x.data_ptr() + 2, out.data_ptr(), 32, 0, stream) == _lib.ERR_INVALID_ARGUMENT
    square = dev.I8Weight(*_weight(64, 64, 6))
    for over in (lambda: dev.i8_mm(square, held, x, out=x), lambda: dev.i8_mm(square, held, x[:3], out=x[1:]), lambda: dev.i8_mm(square, held, x[:1], out=x.view(torch.float32)[:2].view(1, 64), f32=True)):
        refused(_lib.ERR_INVALID_ARGUMENT, over)
    assert lib.b200_i8_rows_get(held._h, None, out.data_ptr() + 2, stream) == _lib.ERR_INVALID_ARGUMENT
    # what was refused changed nothing
    q, _ = held.get()
    assert torch.equal(q.cpu().double(), _quantized(x.cpu())[0])


def test_refusals_without_handles():
    from dmlx_b200 import _lib

    lib, h = _lib.lib, C.c_void_p()
    q, s = (C.c_int8 * 4)(), (C.c_float * 4)()
    bad = _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_i8_weight_create(2, 2, C.addressof(q), C.addressof(s), None) == bad
    for n, k in ((0, 2), (2, 0), (-1, 2), (2, 131073), (2 ** 24 + 1, 2)):
        assert lib.b200_i8_weight_create(n, k, C.addressof(q), C.addressof(s), C.byref(h)) == bad and not h.value
    assert lib.b200_i8_weight_create(2, 2, None, C.addressof(s), C.byref(h)) == bad
    assert lib.b200_i8_weight_create(2, 2, C.addressof(q), None, C.byref(h)) == bad
    assert lib.b200_i8_weight_create(1, 2, C.addressof(q), C.addressof(s) + 2, C.byref(h)) == bad
    assert lib.b200_i8_weight_create_gated(2, 2, C.addressof(q), C.addressof(s), None, C.addressof(s), C.byref(h)) == bad
    for rows, k, hidden in ((0, 8, 0), (8, 0, 0), (8, 8, -1), (2 ** 24 + 1, 8, 0), (8, 131073, 0), (8, 8, 131073)):
        assert lib.b200_i8_rows_create(rows, k, hidden, C.byref(h)) == bad and not h.value
    assert lib.b200_i8_rows_create(8, 8, 0, None) == bad
    assert lib.b200_i8_quantize(None, None, 8, 1, 8, None) == bad
    assert lib.b200_i8_rows_get(None, None, None, None) == bad
    assert lib.b200_i8_mm(None, None, None, 0, 1, None, None, 0, 0, None) == bad
    assert lib.b200_i8_ffn(None, None, None, None, 0, 1, 0, None, 0, None) == bad
    lib.b200_i8_weight_destroy(None)
    lib.b200_i8_rows_destroy(None)
