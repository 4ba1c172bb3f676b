"""The norms behind and before a block with its gate and its factor on the residual, against a plain form in 64 bits.

u = 2^-24.  A sum of squares is 32 additions of a thread and ten of warps, 45 u of it with the squares', so 23 u of its root; rsqrt 4 u, mean and eps 2 u; the products with
the weight and with the gate 3 u; the gate's sigmoid 2^-20 (its exponential is off by 2 + 1.16 |z| of its last place, |z| up to 9 here, its reciprocal by
two).  So scale * p is off by 2^-18 of itself at most, h' by that and u of |h| + |scale p|.  The second norm adds 2^-18 of its own, and what h' is off by:
through the root no more than the norm of its errors over its own.  Rounding: half a step of bf16, 2^-8."""
import pytest
import torch


def _make(rows, n, seed, h_f32=False, y_f32=False):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    as_ = lambda t, f32: t if f32 else t.bfloat16()  # noqa: E731
    return dict(h=as_(3 * rnd(rows, n), h_f32), y=as_(rnd(rows, n), y_f32), post=(1 + 0.2 * rnd(n)).bfloat16(), norm=(1 + 0.2 * rnd(n)).bfloat16(),
                gate_row=(rnd(rows, n)).bfloat16(), gate=(0.5 + 0.3 * rnd(n)).bfloat16())


def _want(h, y, post, norm, gate, sigmoid, scale, eps):
    """(h', its tolerance, x, its tolerance) before any rounding of the results."""
    r = lambda v: (v.square().mean(-1, keepdim=True) + eps).rsqrt()  # noqa: E731
    p = y.double()
    if post is not None:
        p = p * r(p) * post.double()
    if gate is not None:
        p = p * (torch.sigmoid(gate.double()) if sigmoid else gate.double())
    p = scale * p
    out = h.double() + p
    h_tol = 2.0 ** -18 * p.abs() + 2.0 ** -23 * (h.double().abs() + p.abs())
    if norm is None:
        return out, h_tol, out, h_tol
    w = norm.double() * r(out)
    x = out * w
    size = out.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-300)
    return out, h_tol, x, w.abs() * h_tol + x.abs() * (2.0 ** -18 + h_tol.square().sum(-1, keepdim=True).sqrt() / size)


def _check(got, want, tol):
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * want.abs()
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


def _cuda(t):
    return None if t is None else t.cuda()


SHAPES = [(1, 1), (1, 4096), (2, 7), (3, 128), (5, 129), (64, 256), (33, 512), (1300, 512), (40, 513), (400, 1000), (7, 2880), (300, 4096), (320, 5003), (2, 8192), (310, 8200),
          (3, 16384), (300, 16384), (2, 16392), (5, 20001), (2, 32768), (3, 32767), (3, 32761), (5, 1023), (300, 255), (1300, 129), (4, 511), (230, 8191)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("h_f32,y_f32,post,gate,sigmoid", [(False, False, True, None, False), (True, False, True, "gate", False), (False, True, False, "gate_row", True),
                                                           (True, True, True, "gate_row", False), (False, False, False, None, False)])
def test_norms(rows, n, h_f32, y_f32, post, gate, sigmoid):
    from dmlx_b200 import device as dev

    c = _make(rows, n, rows + n, h_f32, y_f32)
    post_w, gate_w, scale, eps = c["post"] if post else None, c[gate] if gate else None, 0.22, 1e-5
    want = _want(c["h"], c["y"], post_w, c["norm"], gate_w, sigmoid, scale, eps)
    h, x = dev.residual_norm(c["h"].cuda(), c["y"].cuda(), c["norm"].cuda(), post_weight=_cuda(post_w), gate=_cuda(gate_w), gate_sigmoid=sigmoid, scale=scale, eps=eps)
    assert h.dtype == c["h"].dtype and x.dtype == torch.bfloat16
    _check(h, want[0], want[1])
    _check(x, want[2], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, 4096), (5, 130), (700, 256), (1300, 500), (300, 4096), (320, 5003), (3, 17000)])
@pytest.mark.parametrize("normed", [True, False])
def test_into_8_bits(rows, n, normed):
    """A number is half a step off at most, and the step is what the row's largest over 127 says, to two more roundings."""
    from dmlx_b200 import device as dev

    c = _make(rows, n, n)
    norm = c["norm"] if normed else None
    h_want, h_tol, x, tol = _want(c["h"], c["y"], c["post"], norm, None, False, 0.5, 1e-6)
    held = dev.I8Rows(rows + 1, n + 5)
    h, none = dev.residual_norm(c["h"].cuda(), c["y"].cuda(), _cuda(norm), post_weight=c["post"].cuda(), scale=0.5, eps=1e-6, rows=held)
    assert none is None
    _check(h, h_want, h_tol)
    q, steps = held.get()
    q, steps = q.cpu().double(), steps.cpu().double()[:, None]
    most = x.abs().amax(1, keepdim=True)
    off = (steps * 127 - most).abs()
    assert bool((off <= tol.amax(1, keepdim=True) + 2.0 ** -22 * most).all())
    assert bool(((q * steps - x).abs() <= 0.5 * steps + tol + 2.0 ** -20 * most).all()) and bool((q.abs().amax(1) == 127).all())
    # both forms at once are the same
    other = dev.I8Rows(rows, n)
    h2, x2 = dev.residual_norm(c["h"].cuda(), c["y"].cuda(), _cuda(norm), post_weight=c["post"].cuda(), scale=0.5, eps=1e-6, rows=other,
                               x_out=torch.empty((rows, n), dtype=torch.bfloat16, device="cuda"))
    _check(x2, x, tol)
    assert torch.equal(h, h2) and torch.equal(other.get()[0].cpu().double(), q)


@pytest.mark.gpu
@pytest.mark.parametrize("at", [0, 8, 1, 3])
@pytest.mark.parametrize("h_f32", [False, True])
def test_strides_places_and_what_lies_around(at, h_f32):
    from dmlx_b200 import device as dev

    rows, n, more = 37, 520, 24
    c = _make(rows, n + more, 3, h_f32)
    cut = lambda t: t[..., at:at + n]  # noqa: E731
    want = _want(cut(c["h"]), cut(c["y"]), cut(c["post"]), cut(c["norm"]), cut(c["gate_row"]), False, -1.5, 1e-5)
    h, y, gate = c["h"].cuda(), c["y"].cuda(), c["gate_row"].cuda()
    out, x_out = torch.full((rows + 2, n + more), 7.0, dtype=h.dtype, device="cuda"), torch.full((rows + 2, n + more), 7.0, dtype=torch.bfloat16, device="cuda")
    dev.residual_norm(cut(h), cut(y), cut(c["norm"].cuda()), post_weight=cut(c["post"].cuda()), gate=cut(gate), scale=-1.5, h_out=cut(out[:rows]), x_out=cut(x_out[:rows]))
    _check(cut(out[:rows]), want[0], want[1])
    _check(cut(x_out[:rows]), want[2], want[3])
    for t in (out, x_out):
        assert bool((t[rows:] == 7).all()) and bool((t[:, :at] == 7).all()) and bool((t[:, at + n:] == 7).all())
    assert torch.equal(h.cpu(), c["h"]) and torch.equal(y.cpu(), c["y"]) and torch.equal(gate.cpu(), c["gate_row"])
    # into h itself, the same bits
    dev.residual_norm(cut(h), cut(y), cut(c["norm"].cuda()), post_weight=cut(c["post"].cuda()), gate=cut(gate), scale=-1.5, h_out=cut(h), x_out=cut(x_out[:rows]))
    assert torch.equal(cut(h), cut(out[:rows]))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [200, 4096])
def test_rows_that_hold_no_number_and_rows_of_nothing(n):
    from dmlx_b200 import device as dev

    rows = 9
    c = _make(rows, n, 5)
    run = lambda h, y, held=None: dev.residual_norm(h.cuda(), y.cuda(), c["norm"].cuda(), post_weight=c["post"].cuda(), scale=0.3, rows=held)  # noqa: E731
    good = run(c["h"], c["y"])
    h, y = c["h"].clone(), c["y"].clone()
    y[1, 3], h[4, 0], y[6, n - 1] = float("nan"), float("inf"), -float("inf")
    h[7], y[7] = 0, 0
    bad = run(h, y)
    rest = [0, 2, 3, 5, 8]
    for g, b in zip(good, bad):
        assert torch.equal(g[rest], b[rest])
        assert bool(b[1].isnan().all()) and bool((b[7] == 0).all())
    assert bool(bad[1][4].isnan().any()) and bool(bad[1][6].isnan().all())
    held = dev.I8Rows(rows, n)
    run(h, y, held)
    q, steps = held.get()
    assert bool((q[[1, 4, 6, 7]] == 0).all()) and float(steps[7]) == 0 and not bool(steps[[1, 4, 6]].isfinite().any())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    from dmlx_b200 import device as dev

    rows, n, stride = 2, 136, 2 ** 31 + 64
    c = _make(rows, n, 6)
    far = lambda: torch.empty(stride + n, dtype=torch.bfloat16, device="cuda").as_strided((rows, n), (stride, 1))  # noqa: E731
    h, y, out, x = far(), far(), far(), far()
    h.copy_(c["h"])
    y.copy_(c["y"])
    dev.residual_norm(h, y, c["norm"].cuda(), scale=0.3, h_out=out, x_out=x)
    want = _want(c["h"], c["y"], None, c["norm"], None, False, 0.3, 1e-5)
    _check(out.contiguous(), want[0], want[1])
    _check(x.contiguous(), want[2], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 500])
def test_the_half_of_a_layer_in_a_graph(rows):
    """Norms into 8 bits, the feed-forward block, norms for the next block: replayed, the bits of the calls one by one; and against a layer in 64 bits that quantises
    nothing, whose products' errors are then those of 8 bits (half a step of 127 of a largest of five deviations, three times over, spread over a row: a cosine of
    0.999 leaves four times that)."""
    from dmlx_b200 import device as dev

    n, f = 768, 1280
    g = torch.Generator().manual_seed(rows)

    def weight(n, k):
        w = torch.randn((n, k), generator=g) * k ** -0.5
        s = w.abs().amax(1) / 127
        return torch.round(w / s[:, None]).to(torch.int8), s

    gate, up, down = weight(f, n), weight(f, n), weight(n, f)
    gate_up, down_w = dev.I8Weight.gated(*gate, *up), dev.I8Weight(*down)
    c = _make(rows, n, 7)
    held = dev.I8Rows(rows, n, f)
    h, y, post, norm = c["h"].cuda(), c["y"].cuda(), c["post"].cuda(), c["norm"].cuda()

    def half():
        h1, _ = dev.residual_norm(h, y, norm, post_weight=post, scale=0.4, rows=held)
        return dev.residual_norm(h1, dev.i8_ffn(gate_up, down_w, held), norm, post_weight=post, scale=0.4)

    half()
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        replayed = half()
    c2 = _make(rows, n, 8)
    h.copy_(c2["h"])
    y.copy_(c2["y"])
    graph.replay()
    torch.cuda.synchronize()
    once = half()
    for a, b in zip(replayed, once):
        assert torch.equal(a, b)
    w64 = [q.double() * s.double()[:, None] for q, s in (gate, up, down)]
    h1, _, x, _ = _want(c2["h"], c2["y"], c["post"], c["norm"], None, False, 0.4, 1e-5)
    inner = torch.nn.functional.silu(x @ w64[0].T) * (x @ w64[1].T)
    h2, _, x2, _ = _want(h1, inner @ w64[2].T, c["post"], c["norm"], None, False, 0.4, 1e-5)
    for got, want in zip(once, (h2, x2)):
        assert float(torch.nn.functional.cosine_similarity(got.double().cpu().flatten(), want.flatten(), 0)) > 0.999


@pytest.mark.gpu
@pytest.mark.parametrize("n", [136, 504, 1000, 2056, 4096, 8192, 8200, 16384, 20008, 32768])
@pytest.mark.parametrize("h_f32,y_f32", [(False, False), (True, False), (True, True)])
def test_a_row_s_bits_do_not_depend_on_its_batch(n, h_f32, y_f32):
    """Its sums of squares are made in an order that its columns alone set, where rows are whole 16-byte pieces.  (An f32 h' shows the first sum's last bit, x and 8-bit
    rows the second's.)"""
    from dmlx_b200 import device as dev

    rows = 1300 if n < 600 else 700 if n < 9000 else 200
    c = _make(rows, n, n, h_f32, y_f32)
    post, norm, gate = c["post"].cuda(), c["norm"].cuda(), c["gate"].cuda()

    def run(h, y, h_out=None, x_out=None):
        held = dev.I8Rows(len(h), n)
        alone = dev.residual_norm(h, y, norm, post_weight=post, gate=gate, scale=0.37, h_out=h_out, x_out=x_out)
        both = dev.residual_norm(h, y, norm, post_weight=post, gate=gate, scale=0.37, x_out=torch.empty((len(h), n), dtype=torch.bfloat16, device="cuda"), rows=held)
        assert all(torch.equal(a, b) for a, b in zip(alone, both))
        return *both, *held.get()

    h, y = c["h"].cuda(), c["y"].cuda()
    whole = run(h, y)
    for first, count in ((0, 1), (1, 1), (5, 2), (6, 3), (11, 7), (40, 64), (37, 150)):
        for got, want in zip(run(h[first:first + count], y[first:first + count]), whole):
            assert torch.equal(got, want[first:first + count]), (first, count)
    for at in (0, 8, 24):  # anywhere in wider rows
        cut = [torch.zeros((20, n + 24), dtype=t, device="cuda")[:, at:at + n] for t in (h.dtype, y.dtype, h.dtype, torch.bfloat16)]
        cut[0].copy_(h[:20])
        cut[1].copy_(y[:20])
        for got, want in zip(run(*cut), whole):
            assert torch.equal(got, want[:20]), at


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(5, 5003), (600, 1030), (3, 8195), (1300, 300)])
@pytest.mark.parametrize("at", [0, 1, 3])
@pytest.mark.parametrize("h_f32", [False, True])
def test_into_h_itself_without_a_norm_behind_the_block(rows, n, at, h_f32):
    """No sum stands between the loads and the stores then: rows of several warps, on no 16-byte boundary."""
    from dmlx_b200 import device as dev

    c = _make(rows, n + 5, 12, h_f32)
    cut = lambda t: t[..., at:at + n]  # noqa: E731
    h, y, norm = c["h"].cuda(), cut(c["y"].cuda()), cut(c["norm"].cuda())
    for post in (False, True):
        weight = cut(c["post"].cuda()) if post else None
        want = dev.residual_norm(cut(h), y, norm, post_weight=weight, scale=0.7, h_out=cut(torch.empty_like(h)))
        mine = h.clone()
        got = dev.residual_norm(cut(mine), y, norm, post_weight=weight, scale=0.7, h_out=cut(mine))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(mine[:, :at], h[:, :at]) and torch.equal(mine[:, at + n:], h[:, at + n:])


@pytest.mark.gpu
def test_a_gate_s_sigmoid_in_f32():
    """2^t with t exact is off by two of its last places, 4 u, its factor's second order by 88^2 (4.9e-6)^2 / 2 = 1.6 u at the most, the reciprocal by 2 u; that factor, the sum,
    the products with y and with the scale and the sum with h by u each: 2^-20 in all.  Behind a divisor past 2^126 the quotient is
    nothing, where the sigmoid is under 2^-126."""
    from dmlx_b200 import device as dev

    gate = torch.cat([torch.linspace(-60, 60, 2000), torch.tensor([-87.0, -87.5, -88.5, -89.0, -1e4, -3e38, 0.0, 89.0, 1e4, 3e38, -float("inf"), float("inf")])]).bfloat16()
    n = len(gate)
    y = torch.randn((3, n), generator=torch.Generator().manual_seed(2))
    h, none = dev.residual_norm(torch.zeros((3, n), device="cuda"), y.cuda(), gate=gate.cuda(), gate_sigmoid=True, scale=1000.0, x_out=torch.empty((3, n), dtype=torch.bfloat16, device="cuda"))
    want = 1000 * y.double() * torch.sigmoid(gate.double())
    off = (h.cpu().double() - want).abs()
    tol = 2.0 ** -20 * want.abs() + 1000 * y.double().abs() * 2.0 ** -126 + 2.0 ** -149
    assert bool((off <= tol).all()), float((off / want.abs().clamp(min=1e-30)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, 4096), (700, 1000), (3, 16384), (300, 504), (64, 8192), (320, 5003), (5, 131), (2, 32761)])
@pytest.mark.parametrize("h_f32,y_f32", [(False, False), (False, True), (True, False), (True, True)])
def test_an_h_that_leaves_as_another_type(rows, n, h_f32, y_f32):
    from dmlx_b200 import device as dev

    c = _make(rows, n, rows + n, h_f32, y_f32)
    to = torch.bfloat16 if h_f32 else torch.float32
    args = dict(post_weight=c["post"].cuda(), gate=c["gate"].cuda(), scale=0.22)
    h, y, norm = c["h"].cuda(), c["y"].cuda(), c["norm"].cuda()
    got = dev.residual_norm(h, y, norm, h_dtype=to, **args)
    assert got[0].dtype == to and got[1].dtype == torch.bfloat16
    want = _want(c["h"], c["y"], c["post"], c["norm"], c["gate"], False, 0.22, 1e-5)
    _check(got[0], want[0], want[1])
    _check(got[1], want[2], want[3])
    if n % 8 == 0:  # (a row's sums are the same then) what f32 rows give, rounded where it is bf16
        wide = dev.residual_norm(h.float(), y, norm, **args)
        assert torch.equal(got[0], wide[0].to(to)) and torch.equal(got[1], wide[1])
    out = torch.full((rows + 1, n + 5), 7.0, dtype=to, device="cuda")
    dev.residual_norm(h, y, norm, h_dtype=to, h_out=out[:rows, 3:3 + n], x_out=got[1], **args)
    _check(out[:rows, 3:3 + n], want[0], want[1])
    assert bool((out[rows:] == 7).all()) and bool((out[:, :3] == 7).all()) and bool((out[:, 3 + n:] == 7).all())


@pytest.mark.gpu
def test_refusals_of_an_h_of_another_type():
    from dmlx_b200 import _lib
    from dmlx_b200 import device as dev

    c = {k: v.cuda() for k, v in _make(4, 64, 14).items()}
    h, y, norm = c["h"], c["y"], c["norm"]
    for call in (lambda: dev.residual_norm(h, y, norm, h_dtype=torch.float16), lambda: dev.residual_norm(h, y, norm, h_dtype=torch.float32, h_out=torch.empty_like(h)),
                 lambda: dev.residual_norm(h.float(), y, norm, h_dtype=torch.bfloat16, h_out=h.float())):
        with pytest.raises(ValueError):
            call()
    both = torch.zeros((8, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.B200Error) as e:  # over itself, in other strides
        dev.residual_norm(both[:4], y, norm, h_dtype=torch.float32, h_out=both.view(-1).view(torch.float32).view(4, 64))
    assert e.value.status == _lib.ERR_INVALID_ARGUMENT


def test_a_type_of_h_that_there_is_none_of_is_refused_without_a_device():
    import ctypes as C

    from dmlx_b200 import _lib

    run = lambda h_f32, h_out, out: _lib.lib.b200_residual_norm(C.byref(_lib.ResidualNormShape(8, h_f32, 0, 0, 1.0, 1e-5, h_out)), 0x1000, 8, 0x2000, 8, None, 0, None, None, 1, out, 8,  # noqa: E731
                                                               None, 0, None, None)
    bad = _lib.ERR_INVALID_ARGUMENT
    assert run(0, 3, 0x3000) == bad and run(0, -1, 0x3000) == bad
    assert run(0, 2, 0x3002) == bad and run(0, 2, 0x1000) == bad and run(1, 1, 0x1000) == bad  # on no number's boundary, over h of another type
    if not torch.cuda.is_available():  # these are not run: the addresses are made up
        for h_f32, h_out, out in ((0, 1, 0x1000), (1, 2, 0x1000), (1, 0, 0x1000), (1, 1, 0x3002), (0, 2, 0x3004)):
            assert run(h_f32, h_out, out) not in (_lib.OK, bad), (h_f32, h_out)


@pytest.mark.gpu
def test_8_bit_rows_that_are_closed_are_refused():
    from dmlx_b200 import device as dev

    c = {k: v.cuda() for k, v in _make(4, 64, 13).items()}
    held = dev.I8Rows(4, 64)
    held.close()
    h = c["h"].clone()
    with pytest.raises(ValueError, match="closed"):
        dev.residual_norm(c["h"], c["y"], c["norm"], h_out=c["h"], rows=held)
    assert torch.equal(h, c["h"])


@pytest.mark.gpu
def test_refusals():
    from dmlx_b200 import _lib
    from dmlx_b200 import device as dev

    c = {k: v.cuda() for k, v in _make(4, 64, 9).items()}
    h, y, norm = c["h"], c["y"], c["norm"]
    for call in (lambda: dev.residual_norm(h, y[:3], norm), lambda: dev.residual_norm(h, y, norm[:32]), lambda: dev.residual_norm(h.half(), y, norm),
                 lambda: dev.residual_norm(h, y, norm.float()), lambda: dev.residual_norm(h, y, norm, gate=c["gate"][:3]),
                 lambda: dev.residual_norm(h, y, norm, gate=c["gate_row"].float()), lambda: dev.residual_norm(h, y, norm, h_out=h.float()), lambda: dev.residual_norm(h.cpu(), y, norm)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.B200Error) as e:
        dev.residual_norm(h, y, norm, rows=dev.I8Rows(3, 64))
    assert e.value.status == _lib.ERR_CAPACITY
    with pytest.raises(_lib.B200Error):
        dev.residual_norm(h, y, norm, eps=-1.0)
    for call in (lambda: dev.residual_norm(h, y, norm, h_out=y), lambda: dev.residual_norm(h, y, norm, x_out=h), lambda: dev.residual_norm(h, y, norm, x_out=y)):
        with pytest.raises(_lib.B200Error) as e:
            call()
        assert e.value.status == _lib.ERR_INVALID_ARGUMENT
    both = torch.zeros((5, 128), dtype=torch.bfloat16, device="cuda")
    side = both[:4, :64].copy_(h), both[:4, 64:]
    for call in (lambda: dev.residual_norm(h, y, norm, gate=c["gate_row"], h_out=c["gate_row"]), lambda: dev.residual_norm(h, y, norm, x_out=c["gate_row"], gate=c["gate_row"]),
                 lambda: dev.residual_norm(side[0], y, norm, h_out=both[1:, :64]), lambda: dev.residual_norm(side[0], y, norm, x_out=both[1:, 32:96]),
                 lambda: dev.residual_norm(h[:1], y[:1], norm, x_out=norm[None]), lambda: dev.residual_norm(h[:1], y[:1], post_weight=norm, h_out=norm[None])):
        with pytest.raises(_lib.B200Error) as e:
            call()
        assert e.value.status == _lib.ERR_INVALID_ARGUMENT
    # columns side by side are apart
    want = dev.residual_norm(h, y, norm, scale=0.5)
    got = dev.residual_norm(side[0], y, norm, scale=0.5, h_out=side[0], x_out=side[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = torch.zeros((1, 32769), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.B200Error) as e:
        dev.residual_norm(wide, wide)
    assert e.value.status == _lib.ERR_UNSUPPORTED
    none = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    assert dev.residual_norm(none, none, norm)[0].shape == (0, 64)


@pytest.mark.gpu
def test_a_factor_that_is_a_tensor_is_read_at_each_call():
    from dmlx_b200 import device as dev

    c = {k: v.cuda() for k, v in _make(2, 64, 11).items()}
    factor = torch.tensor(0.25)
    for value in (0.25, -3.0):
        factor.fill_(value)
        got, want = dev.residual_norm(c["h"], c["y"], c["norm"], scale=factor), dev.residual_norm(c["h"], c["y"], c["norm"], scale=value)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_outputs_over_inputs_are_refused_without_a_device():
    import ctypes as C

    from dmlx_b200 import _lib

    shape = _lib.ResidualNormShape(8, 0, 0, 0, 1.0, 1e-5)
    at = dict(h=0x10000, h_stride=32, y=0x20000, y_stride=32, gate=0x30000, gate_stride=32, post=0x40000, norm=0x50000, rows=3, out=0x60000, out_stride=32, x=0x70000, x_stride=32)

    def run(**other):
        a = dict(at, **other)
        return _lib.lib.b200_residual_norm(C.byref(shape), a["h"], a["h_stride"], a["y"], a["y_stride"], a["gate"], a["gate_stride"], a["post"], a["norm"], a["rows"], a["out"],
                                           a["out_stride"], a["x"], a["x_stride"], None, None)

    # a row is 16 bytes, rows are 64 apart
    over = [dict(out=at["y"]), dict(out=at["y"] + 14), dict(out=at["y"] + 2 * 64 + 14), dict(x=at["y"] - 2 * 64 - 14), dict(x=at["h"]), dict(out=at["h"] + 64), dict(out=at["h"], out_stride=40),
            dict(out=at["gate"]), dict(x=at["gate"] + 8), dict(gate_stride=0, out=at["gate"] - 2 * 64), dict(out=at["post"] + 14), dict(x=at["norm"] - 64 - 14), dict(x=at["out"] + 2),
            dict(x=at["out"] + 16, x_stride=40), dict(rows=1, out=at["y"] + 14)]
    for other in over:
        assert run(**other) == _lib.ERR_INVALID_ARGUMENT, other
    if not torch.cuda.is_available():  # these are not run: the addresses are made up
        for other in (dict(), dict(out=at["h"]), dict(out=at["y"] + 16), dict(out=at["y"] + 48), dict(x=at["out"] + 16), dict(x=at["y"] - 2 * 64 - 16), dict(rows=1, out=at["y"] + 16),
                      dict(gate=None, out=at["gate"]), dict(gate_stride=0, out=at["gate"] + 16), dict(x=None)):
            assert run(**other) not in (_lib.OK, _lib.ERR_INVALID_ARGUMENT), other


def test_refusals_without_a_device():
    import ctypes as C

    from dmlx_b200 import _lib

    run = lambda shape, rows=1, p=64, stride=8: _lib.lib.b200_residual_norm(shape and C.byref(shape), p, stride, p, stride, None, 0, None, None, rows, p, stride, None, 0, None, None)  # noqa: E731
    bad = _lib.ERR_INVALID_ARGUMENT
    assert run(None) == bad
    assert run(_lib.ResidualNormShape(8, 0, 0, 0, 1.0, 1e-5), rows=-1) == bad
    assert run(_lib.ResidualNormShape(0, 0, 0, 0, 1.0, 1e-5)) == _lib.ERR_UNSUPPORTED
    assert run(_lib.ResidualNormShape(32769, 0, 0, 0, 1.0, 1e-5)) == _lib.ERR_UNSUPPORTED
    assert run(_lib.ResidualNormShape(8, 0, 0, 0, 1.0, float("nan"))) == bad
    assert run(_lib.ResidualNormShape(8, 0, 0, 0, 1.0, 1e-5), p=None) == bad
    assert run(_lib.ResidualNormShape(8, 1, 0, 0, 1.0, 1e-5), p=66) == bad
    assert run(_lib.ResidualNormShape(8, 0, 0, 0, 1.0, 1e-5), rows=2, stride=7) == bad


def test_the_shape_has_the_header_s_layout(tmp_path):
    import ctypes as C
    import os
    import shutil
    import subprocess

    from dmlx_b200 import _lib

    if shutil.which("gcc") is None:
        return
    shape = _lib.ResidualNormShape
    lines = "".join(f'printf("%zu ", offsetof(b200_residual_norm_shape, {name}));' for name, _ in shape._fields_)
    (tmp_path / "l.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dmlx_b200.h"\nint main(void) {' + lines + 'printf("%zu", sizeof(b200_residual_norm_shape)); return 0; }')
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c99", "-I", include, str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(shape, name).offset for name, _ in shape._fields_] + [C.sizeof(shape)]
