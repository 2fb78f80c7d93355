"""Dense products with bias, activation and residual, and their gradients: against 64-bit formulas and differences, refusals, streams, graphs."""
import math

import pytest
import torch

from nvfp4_gemm import _C, TokenOrder, linear, route_tokens, sort_tokens, unsort_tokens

gpu = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ACTIVATIONS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
# Largest |slope| and |curvature| of the activations (those of gelu are 1.13 and 0.80, of silu 1.10 and 0.50)
SLOPE, CURVATURE = 1.2, 0.9


def gen(seed):
    return torch.Generator().manual_seed(seed)


def act64(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if name == "silu" else z


def sum_error(a, b):
    """Bound on an FP32 sum of products: K roundings (2^-23 each: the tensor core may cut instead of rounding) of partial sums no
    larger than the sum of magnitudes."""
    return (a.double().abs() @ b.double().abs()) * (a.shape[1] + 4) * 2.0 ** -23


def make(m, n, k, dtype, seed, out=None):
    g = gen(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype)
    return x, w, torch.randn(n, generator=g).to(dtype), torch.randn(m, n, generator=g).to(out or dtype)


def check_forward(got, x, w, bias, residual, activation, out):
    z = x.double() @ w.double().t()
    if bias is not None:
        z = z + bias.double()
    want = act64(z, activation)
    # activation: its argument's error times the slope; 16 roundings of its own, and those of the exponential's argument (three, and one more
    # in the hardware's base 2), which count as that argument's size
    argument = {"gelu": z * z / 2 + 2, "gelu_tanh": 1.6 * (z.abs() + 0.044715 * z.abs() ** 3)}.get(activation, z.abs()).clamp(max=200)
    error = SLOPE * (sum_error(x, w.t()) + z.abs() * 2.0 ** -23) + want.abs() * (16 + 4 * argument) * 2.0 ** -23
    if residual is not None:
        want = want + residual.double()
        error = error + want.abs() * 2.0 ** -23
    floor = 2.0 ** -25 if out == torch.float16 else 1e-40
    assert got.dtype == out and got.shape == want.shape
    worst = ((got.cpu().double() - want).abs() - (error + (want.abs() + error) * 1.01 * HALF_STEP[out] + floor)).max()
    assert worst <= 0, float(worst)


# ---- refusals --------------------------------------------------------------------------------------------------------


def error_of(rc):
    assert rc == 1
    return _C.lib().nvfp4_last_error().decode()


def call(x=1024, ldx=64, w=1024, ldw=64, bias=None, residual=None, ldr=0, d=1024, ldd=32, slopes=None, lds=0, m=4, n=32, k=64, dtype=0, out=0, act=0):
    return _C.lib().nvfp4_linear(x, ldx, w, ldw, bias, residual, ldr, d, ldd, slopes, lds, m, n, k, dtype, out, act, None, None)


@pytest.mark.parametrize("change, text", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(d=None), "null output"), (dict(x=1032), "16-byte"), (dict(w=1026), "16-byte"),
    (dict(ldx=68), "multiple of 8"), (dict(ldx=56), "cover the row"), (dict(ldw=60), "multiple of 8"), (dict(k=60), "K must be"), (dict(k=0), "K must be"),
    (dict(m=-1), "negative"), (dict(dtype=1), "BF16 or FP16"), (dict(dtype=3), "BF16 or FP16"), (dict(out=2), "operands' type"), (dict(act=5), "activation"),
    (dict(act=-1), "activation"), (dict(ldd=31), "smaller than the row"), (dict(residual=1024, ldr=8), "smaller than the row"), (dict(d=1025), "aligned"),
    (dict(bias=1025), "aligned"), (dict(out=1, d=1026), "aligned"), (dict(slopes=1024, lds=31), "smaller than the row")])
def test_products_refuse(change, text):
    assert text in error_of(call(**change))


def test_gradients_refuse():
    lib = _C.lib()
    assert "K must be" in error_of(lib.nvfp4_linear_dx(1024, 32, 1024, 64, 1024, 64, 4, 32, 60, 0, None, None))
    assert "dz must" in error_of(lib.nvfp4_linear_dx(1026, 32, 1024, 64, 1024, 64, 4, 32, 64, 0, None, None))
    assert "empty contraction" in error_of(lib.nvfp4_linear_dx(1024, 32, 1024, 64, 1024, 64, 4, 0, 64, 0, None, None))
    assert "empty contraction" in error_of(lib.nvfp4_linear_dw(1024, 32, 1024, 64, 1024, 64, 0, 32, 64, 0, None, None))
    assert "rows overlap" in error_of(lib.nvfp4_linear_dw(1024, 32, 1024, 64, 1024, 56, 4, 32, 64, 0, None, None))
    assert "stride of slopes" in error_of(lib.nvfp4_linear_dz(1024, 33, 1024, 32, 1024, 40, None, 4, 33, 0, 0, None))
    assert "stride of dz" in error_of(lib.nvfp4_linear_dz(1024, 33, 1024, 40, 1024, 32, None, 4, 33, 0, 0, None))
    assert "operands' type" in error_of(lib.nvfp4_linear_dz(1024, 32, 1024, 32, 1024, 32, None, 4, 32, 0, 2, None))
    assert lib.nvfp4_linear_dz(1024, 32, 1024, 32, None, 32, None, 4, 32, 0, 0, None) == 0


def test_empty_products_are_nothing():
    assert call(m=0, x=None) == 0 and call(n=0, d=None) == 0


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="x is a 2-D"):
        linear(torch.zeros(2, 8), torch.zeros(2, 8))


# ---- forward ---------------------------------------------------------------------------------------------------------

# tokens to the tiles of the few-row form (16, 32, 64, 128), contractions that split over clusters or not, narrow, odd and wide outputs,
# left-over pieces of every tile, enough tiles for the pairs
SIZES = [(1, 1, 8), (1, 4096, 4096), (2, 4096, 2048), (1, 700, 4104), (2, 513, 2048), (1, 130, 20000), (2, 9, 1000), (3, 25, 3768), (16, 128, 64), (17, 513, 2048), (33, 1411, 2048), (64, 96, 520), (65, 31, 72), (128, 1000, 1024),
         (129, 64, 200), (300, 33, 1032), (257, 129, 8), (500, 256, 4096), (1000, 65, 136), (2049, 128, 4096), (777, 3001, 264), (4099, 2050, 72), (2500, 4104, 392)]


@gpu
@pytest.mark.parametrize("m, n, k", SIZES)
def test_products_against_64_bits(m, n, k):
    for i, dtype in enumerate((torch.bfloat16, torch.float16)):
        x, w, bias, residual = make(m, n, k, dtype, m + n + k)
        act = ACTIVATIONS[(m + i) % 5]
        check_forward(linear(x.cuda(), w.cuda()), x, w, None, None, "none", dtype)
        check_forward(linear(x.cuda(), w.cuda(), bias.cuda(), residual.cuda(), activation=act), x, w, bias, residual, act, dtype)
        check_forward(linear(x.cuda(), w.cuda(), bias.cuda(), out_dtype=torch.float32, activation=act), x, w, bias, None, act, torch.float32)


# One wave of wide tiles and several waves of them, columns and rows left over, rows that are whole 16 bytes and rows that are not
@gpu
@pytest.mark.parametrize("m, n, k", [(16283, 128, 264), (4000, 500, 392), (3900, 500, 64), (2500, 4104, 392), (1000, 1001, 72), (9000, 36, 8)])
def test_fp32_outputs_with_a_residual(m, n, k):
    x, w, bias, residual = make(m, n, k, torch.bfloat16, m + n, torch.float32)
    check_forward(linear(x.cuda(), w.cuda(), bias.cuda(), residual.cuda(), activation="gelu", out_dtype=torch.float32), x, w, bias, residual, "gelu",
                  torch.float32)
    wide = torch.full((m, n + 4), 7.0, device="cuda")                       # a residual of longer rows
    wide[:, :n] = residual.cuda()
    check_forward(linear(x.cuda(), w.cuda(), None, wide[:, :n], out_dtype=torch.float32), x, w, None, residual, "none", torch.float32)


@gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("m, n, k", [(5, 200, 512), (200, 200, 64), (3000, 1536, 128)])
def test_every_activation(m, n, k, activation):
    for dtype in (torch.bfloat16, torch.float16):
        x, w, bias, residual = make(m, n, k, dtype, 7, torch.float32)
        w = w * 3                                                          # far into both tails
        check_forward(linear(x.cuda(), w.cuda(), bias.cuda(), residual.cuda(), activation=activation, out_dtype=torch.float32), x, w, bias, residual,
                      activation, torch.float32)
        check_forward(linear(x.cuda(), w.cuda(), None, residual.to(dtype).cuda(), activation=activation), x, w, None, residual.to(dtype), activation, dtype)


@gpu
def test_strided_operands_and_residuals():
    for m, n, k in ((9, 77, 128), (300, 77, 128), (2600, 2056, 64)):
        for dtype in (torch.bfloat16, torch.float16):
            x, w, bias, residual = make(m, n, k, dtype, 3)
            wide_x = torch.full((m, k + 24), float("nan"), dtype=dtype, device="cuda")
            wide_w = torch.full((2 * n, k), float("nan"), dtype=dtype, device="cuda")
            wide_r = torch.full((m, n + 5), float("nan"), dtype=dtype, device="cuda")
            vx, vw, vr = wide_x[:, 8:8 + k], wide_w[::2], wide_r[:, 3:3 + n]
            vx.copy_(x), vw.copy_(w), vr.copy_(residual)
            vb = torch.full((n + 1,), float("nan"), dtype=dtype, device="cuda")[1:]
            vb.copy_(bias)
            check_forward(linear(vx, vw, vb, vr, activation="silu"), x, w, bias, residual, "silu", dtype)
            for bad in (wide_x[:, 1:1 + k], wide_x[:, :k].t()[:k, :m] if m >= k else wide_x[:, 4:4 + k]):
                with pytest.raises(RuntimeError):
                    linear(bad, vw)


@gpu
def test_infinities_and_nan_stay_in_their_rows():
    for m in (40, 400, 2600):
        x, w, bias, residual = make(m, 2056, 64, torch.bfloat16, 5)
        x[3, 0], x[7, 1], x[m - 1, 5] = float("inf"), float("nan"), -float("inf")
        got = linear(x.cuda(), w.cuda(), bias.cuda(), residual.cuda(), activation="relu").cpu()
        clean = torch.ones(m, dtype=torch.bool)
        clean[[3, 7, m - 1]] = False
        check_forward(got[clean], x[clean], w, bias, residual[clean], "relu", torch.bfloat16)
        assert torch.isnan(got[7]).all()
        inf = torch.where(w[:, 0] > 0, float("inf"), torch.where(w[:, 0] < 0, 0.0, float("nan")))
        assert torch.equal((inf + residual[3].float()).to(torch.bfloat16), got[3])


@gpu
def test_python_refusals():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    for args, kw in (((x, w.half()), {}), ((x, w[:, :32]), {}), ((x.float(), w.float()), {}), ((x[:, :60], w[:, :60]), {}), ((x, w, torch.zeros(7).cuda().bfloat16()), {}),
                     ((x, w, torch.zeros(8).cuda()), {}), ((x, w, None, x), {}), ((x, w), dict(activation="tanh")), ((x, w), dict(out_dtype=torch.float16)),
                     ((x, w, None, torch.zeros(4, 8, device="cuda")), {}), ((x, w.cpu()), {})):
        with pytest.raises(RuntimeError):
            linear(*args, **kw)
    assert linear(x[:0], w).shape == (0, 8) and linear(x, w[:0]).shape == (4, 0)


# ---- backward --------------------------------------------------------------------------------------------------------

TRAIN_SIZES = [(1, 1, 8), (1, 300, 64), (2, 41, 264), (7, 33, 72), (130, 64, 200), (33, 1411, 520), (300, 129, 1032), (1000, 128, 2048), (513, 2050, 264), (2600, 2056, 3080)]


@gpu
@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m, n, k", TRAIN_SIZES)
def test_gradients_against_the_formulas(m, n, k, activation):
    for dtype, out in ((torch.bfloat16, None), (torch.float16, torch.float32)):
        x, w, bias, residual = make(m, n, k, dtype, 11, out)
        dd = torch.randn(m, n, generator=gen(12)).to(out or dtype)
        leaves = [t.cuda().requires_grad_() for t in (x, w, bias, residual)]
        y = linear(*leaves, activation=activation, out_dtype=out)
        check_forward(y.detach(), x, w, bias, residual, activation, out or dtype)
        dx, dw, db, dr = torch.autograd.grad(y, leaves, dd.cuda())
        assert torch.equal(dr.cpu(), dd)
        z = (x.double() @ w.double().t() + bias.double()).requires_grad_()
        (dz,) = torch.autograd.grad(act64(z, activation), z, dd.double())
        z = z.detach()
        # the slope is kept in steps of 2^-14; it is taken at the z that the forward sum gave, curvature times that sum's error away, and
        # costs some 64 roundings itself; a sign that the sum's error can flip costs relu the whole slope
        z_error = sum_error(x, w.t()) + z.abs() * 2.0 ** -23
        if activation == "none":
            dz_error = torch.zeros_like(z)
        elif activation == "relu":
            dz_error = torch.where(z.abs() <= z_error, dd.double().abs(), 0.0)
        else:
            dz_error = dd.double().abs() * (2.0 ** -15 + CURVATURE * z_error + 64 * 2.0 ** -23)
        tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-40
        db_error = dz_error.sum(dim=0) + dz.abs().sum(dim=0) * (m + 4) * 2.0 ** -24
        assert (db.cpu().double() - dz.sum(dim=0)).abs().le(db_error + (dz.sum(dim=0).abs() + db_error) * 1.01 * HALF_STEP[dtype] + tiny).all()
        rounded = dz_error + (dz.abs() + dz_error) * 1.01 * HALF_STEP[dtype] + tiny      # dz rounded for the tensor cores
        for got, want, size in ((dx, dz @ w.double(), (dz.abs() + rounded) @ w.double().abs()), (dw, dz.t() @ x.double(), (dz.abs() + rounded).t() @ x.double().abs())):
            other, terms = (w, n) if got is dx else (x, m)
            spread = (rounded if got is dx else rounded.t()) @ other.double().abs()
            error = spread + size * (terms + 4) * 2.0 ** -23
            assert got.dtype == dtype
            assert (got.cpu().double() - want).abs().le(error + (want.abs() + error) * 1.01 * HALF_STEP[dtype] + tiny).all()


@gpu
def test_gradients_against_differences():
    m, n, k = 6, 10, 16
    g = gen(2)
    x, w = torch.randn(m, k, generator=g).half(), (torch.randn(n, k, generator=g) * 0.3).half()
    bias, dd = torch.randn(n, generator=g).half(), torch.randn(m, n, generator=g)
    for activation in ("gelu", "gelu_tanh", "silu"):
        leaves = [t.cuda().requires_grad_() for t in (x, w, bias)]
        grads = torch.autograd.grad(linear(*leaves, activation=activation, out_dtype=torch.float32), leaves, dd.cuda())
        f = lambda a, b, c: float((act64(a @ b.t() + c, activation) * dd.double()).sum())
        base = [x.double(), w.double(), bias.double()]
        for which, grad in enumerate(grads):
            for at in range(0, base[which].numel(), 7):
                h = 1e-5
                moved = []
                for sign in (h, -h):
                    args = [t.clone() for t in base]
                    args[which].view(-1)[at] += sign
                    moved.append(f(*args))
                slope = (moved[0] - moved[1]) / (2 * h)
                # dz rounded to FP16 (2^-11, values of a few) in sums of up to 16 terms, the result rounded once
                assert abs(slope - float(grad.reshape(-1)[at])) < 16 * 4 * 2 * 2.0 ** -11


@gpu
def test_gradients_wanted_alone_strided_and_of_nothing():
    m, n, k = 70, 33, 136
    x, w, bias, residual = (t.cuda() for t in make(m, n, k, torch.bfloat16, 3))
    full = [t.clone().requires_grad_() for t in (x, w, bias, residual)]
    dd = torch.randn(m, n + 3, generator=gen(1)).bfloat16().cuda()[:, 1:1 + n]
    want = torch.autograd.grad(linear(*full, activation="silu"), full, dd)
    for i in range(4):
        args = [x, w, bias, residual]
        args[i] = args[i].clone().requires_grad_()
        (got,) = torch.autograd.grad(linear(*args, activation="silu"), [args[i]], dd)
        assert torch.equal(got, want[i]), i
    # one value for every element: an expanded gradient, with and without an activation
    for act in ("none", "silu"):
        a = torch.autograd.grad(linear(*full, activation=act).sum(), full)
        b = torch.autograd.grad(linear(*full, activation=act), full, torch.ones(m, n, dtype=torch.bfloat16, device="cuda"))
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    empty = [t.clone().requires_grad_() for t in (x[:0], w, bias)]
    dx, dw, db = torch.autograd.grad(linear(*empty, activation="gelu").sum(), empty)
    assert dx.shape == (0, k) and (dw == 0).all() and (db == 0).all()


# ---- streams, graphs, repeated calls ---------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("m, n, k", [(1, 4096, 4096), (40, 520, 2048), (400, 200, 1024), (3000, 2056, 128)])
def test_repeated_calls_streams_and_graphs_give_the_same_bits(m, n, k):
    x, w, bias, residual = (t.cuda() for t in make(m, n, k, torch.bfloat16, 9))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = linear(x, w, bias, residual, activation="gelu", device_status=status)
    outs = [linear(x, w, bias, residual, activation="gelu", device_status=status) for _ in range(20)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs.append(linear(x, w, bias, residual, activation="gelu", device_status=status))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = linear(x, w, bias, residual, activation="gelu", device_status=status)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in outs + [held])
    x.copy_(torch.randn(m, k, generator=gen(10)))
    graph.replay()
    assert torch.equal(held, linear(x, w, bias, residual, activation="gelu"))
    assert _C.read_status(status) == 0


@gpu
@pytest.mark.parametrize("sms", [1, 2, 3, 296])
def test_any_number_of_sms(sms):
    """set_num_sms sizes the persistent grids, and the choice of the form goes by it."""
    before = _C.get_num_sms()
    try:
        _C.set_num_sms(sms)
        for m, n, k in ((1, 300, 512), (130, 200, 1024), (700, 600, 64), (1300, 1288, 128)):
            x, w, bias, residual = make(m, n, k, torch.bfloat16, 2)
            check_forward(linear(x.cuda(), w.cuda(), bias.cuda(), residual.cuda(), activation="silu"), x, w, bias, residual, "silu", torch.bfloat16)
    finally:
        _C.set_num_sms(before)


@gpu
def test_slopes_are_left_alone_without_an_activation():
    for n in (40, 41):
        x, w, _, _ = make(600, n, 64, torch.float16, 1)
        x, w = x.cuda(), w.cuda()
        d, slopes = torch.empty(600, n, dtype=torch.float16, device="cuda"), torch.full((600, 48), 7, dtype=torch.int16, device="cuda")
        rc = _C.lib().nvfp4_linear(x.data_ptr(), 64, w.data_ptr(), 64, None, None, 0, d.data_ptr(), n, slopes.data_ptr(), 48, 600, n, 64, 2, 2, 0, None,
                                   torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0 and (slopes == 7).all()
        rc = _C.lib().nvfp4_linear(x.data_ptr(), 64, w.data_ptr(), 64, None, None, 0, d.data_ptr(), n, slopes.data_ptr(), 48, 600, n, 64, 2, 2, 1, None,
                                   torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        want = ((x.double() @ w.double().t() > 0).to(torch.int16) << 14) + 8192
        sure = (x.double() @ w.double().t()).abs() > 1e-4
        assert rc == 0 and (slopes[:, :n] == want)[sure].all() and (slopes[:, n:] == 7).all()


@gpu
@pytest.mark.parametrize("activation", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activations_and_slopes_of_extreme_values(activation):
    """z from a sweep over all of FP16, infinities and NaN, in each of the epilogue's ways: K = 8 with one nonzero product gives z exactly."""
    z = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.float16)
    z = torch.cat([z, torch.tensor([-0.0, 65504.0, -65504.0], dtype=torch.float16)])
    finite = torch.isfinite(z)
    n = 8
    w = torch.zeros(n, 8, dtype=torch.float16)
    w[:, 0] = 1
    for rows in (z[-9000:], z, z[20000:20100]):                            # tiles, pairs, few rows
        x = torch.zeros(rows.numel(), 8, dtype=torch.float16)
        x[:, 0] = rows
        for columns in (8, 7):
            for out in (torch.float16, torch.float32):
                leaf = x.cuda().requires_grad_()
                y = linear(leaf, w[:columns].cuda(), activation=activation, out_dtype=out)
                d = torch.zeros(rows.numel(), columns, dtype=out)
                d[:, 0] = 1
                (dx,) = torch.autograd.grad(y, leaf, d.cuda())
                v = rows.double()
                real = torch.isfinite(rows)
                want = act64(v, activation)[:, None].expand(-1, columns)
                got = y.detach().cpu().double()
                argument = {"gelu": v * v / 2 + 2, "gelu_tanh": 1.6 * (v.abs() + 0.044715 * v.abs() ** 3)}.get(activation, v.abs()).clamp(max=200)[:, None]
                floor = 2.0 ** -24 if out == torch.float16 else 1e-37
                assert (got - want)[real].abs().le((want.abs() * ((16 + 4 * argument) * 2.0 ** -23 + 1.01 * HALF_STEP[out]) + floor)[real]).all()
                assert torch.isnan(got[torch.isnan(rows)]).all() and (got[rows == math.inf] == math.inf).all()
                leaf64 = torch.where(real, v, 0.0).requires_grad_()
                (slope,) = torch.autograd.grad(act64(leaf64, activation).sum(), leaf64)
                slope = torch.where(torch.isnan(slope), 0.0, slope) if activation == "gelu_tanh" else slope     # 0 * inf of the formula far out
                far = v.abs() > 30                                         # there the formulas meet their limits
                slope = torch.where(far, (v > 0).double(), slope)
                sx = dx[:, 0].cpu().double()
                assert (sx - slope)[real].abs().le(2.0 ** -15 + 64 * 2.0 ** -23 + 1.1 * 2.0 ** -11).all()
                assert torch.isnan(sx[torch.isnan(rows)]).all() and (sx[rows == math.inf] == 1).all()


@gpu
def test_outputs_beyond_32_bits():
    """More output elements than 32 bits count; the last rows and columns against 64-bit products, and the gradient of the weight's last rows."""
    m, n, k = 530000, 8200, 16
    x = torch.randn(m, k, generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    w = (torch.randn(n, k, generator=torch.Generator("cuda").manual_seed(2), device="cuda") * 0.25).bfloat16()
    for columns in (n, n - 1):                                            # through TMA, and the odd stride's way
        d = linear(x, w[:columns], activation="silu")
        at = torch.tensor([0, 1, 200000, 262143, 262144, m - 130, m - 2, m - 1], device="cuda")
        check_forward(d[at], x[at].cpu(), w[:columns].cpu(), None, None, "silu", torch.bfloat16)
        del d


@gpu
def test_a_captured_training_step():
    x, w, bias, residual = (t.cuda() for t in make(200, 136, 264, torch.bfloat16, 4))
    leaves = [t.requires_grad_() for t in (x, w, bias, residual)]
    dd = torch.randn(200, 136, generator=gen(5)).bfloat16().cuda()
    step = lambda: torch.autograd.grad(linear(*leaves, activation="gelu"), leaves, dd)
    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
def test_router_sorted_experts_and_shared_expert_train_together():
    """logits = linear -> route -> sort -> a dense expert per group -> back, plus a shared expert whose last product adds the routed
    sum as its residual: the gradients of the whole against the same layer in 64 bits."""
    tokens, experts, k, hidden, inter = 96, 4, 2, 64, 128
    g = gen(8)
    half = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(torch.float16)
    x, gate = half(tokens, hidden), half(experts, hidden, scale=0.3)
    expert_w = half(experts, hidden, hidden, scale=0.125)
    w1, w2 = half(inter, hidden, scale=0.125), half(hidden, inter, scale=0.09)
    dy = torch.randn(tokens, hidden, generator=g).to(torch.float16)

    leaves = [t.cuda().requires_grad_() for t in (x, gate, expert_w, w1, w2)]
    lx, lg, le, l1, l2 = leaves
    ids, weights = route_tokens(linear(lx, lg, out_dtype=torch.float32), k)
    rows, order = sort_tokens(lx, ids, experts, alignment=16)
    bounds = [int((order.m_indices == e).sum()) for e in range(experts)] + [int((order.m_indices < 0).sum())]
    outs = [linear(part, le[e]) if e < experts else part for e, part in enumerate(torch.split(rows, bounds))]
    routed = unsort_tokens(torch.cat(outs), order, weights)
    y = linear(linear(lx, l1, activation="silu"), l2, residual=routed)
    got = torch.autograd.grad(y, leaves, dy.cuda())

    exact = [t.double().requires_grad_() for t in (x, gate, expert_w, w1, w2)]
    ex, eg, ee, e1, e2 = exact
    probs = torch.softmax(ex @ eg.t(), dim=1)
    top = ids.cpu()
    wt = probs.gather(1, top)
    wt = wt / wt.sum(dim=1, keepdim=True)
    routed = sum(wt[:, j, None] * torch.einsum("th,toh->to", ex, ee[top[:, j]]) for j in range(k))
    want_y = act64(ex @ e1.t(), "silu") @ e2.t() + routed
    want = torch.autograd.grad(want_y, exact, dy.double())
    # every value passes at most six roundings to FP16 on its way (rows, hidden products, dz, sums): relative to the largest of its kind
    for a, b in zip([y.detach(), *got], [want_y.detach(), *want]):
        assert (a.cpu().double() - b).abs().max() <= 6 * 2.0 ** -11 * 4 * b.abs().max()


@gpu
@pytest.mark.parametrize("activation, lo, hi", [("silu", -20.0, -5.0), ("gelu", -7.0, -3.5), ("gelu_tanh", -6.0, -3.5)])
def test_gradients_keep_their_digits_where_slopes_are_small(activation, lo, hi):
    """Units deep in the negative tail: z is the bias, exact in its type, and one row's bias gradient is dz."""
    for dtype in (torch.bfloat16, torch.float16):
        for m, n in ((1, 513), (1, 512), (70, 512), (300, 2048), (2600, 4096), (2600, 4097)):      # token kernel, few rows, tiles, pairs, odd widths
            for out in (dtype, torch.float32):
                x, w = torch.zeros(m, 8, dtype=dtype), torch.zeros(n, 8, dtype=dtype)
                x[:, 0], w[:, 0] = 1, 1
                bias = torch.linspace(lo, hi, n).to(dtype)
                z = bias.double() + 1
                at = (torch.arange(n) * 7) % m                            # a row of its own to every column, or few: the others are zero
                scale = 2.0 ** (torch.floor(-torch.log2(z.abs() * torch.exp(-0.5 * z * z if activation != "silu" else z))).clamp(max=14))
                dd = torch.zeros(m, n, dtype=out)
                dd[at, torch.arange(n)] = scale.to(out)                   # brings what FP16 could not hold into its range
                leaves = [t.cuda().requires_grad_() for t in (x, w, bias)]
                y = linear(*leaves, activation=activation, out_dtype=out)
                dw, db = torch.autograd.grad(y, leaves[1:], dd.cuda())
                leaf = z.clone().requires_grad_()
                (slope,) = torch.autograd.grad(act64(leaf, activation).sum(), leaf)
                want = slope * scale
                # the slope's code is off by 2^-11 of it; exp of an argument of up to 30 with three roundings, twice over where slope and
                # value nearly cancel; then the rounding of db, or of dz and dw
                argument = {"gelu": z * z / 2 + 2, "gelu_tanh": 1.6 * (z.abs() + 0.044715 * z.abs() ** 3)}.get(activation, z.abs())
                error = want.abs() * (2.0 ** -11 + 2 * (16 + 4 * argument) * 2.0 ** -23)
                tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-40
                for got, roundings in ((db, 1), (dw[:, 0], 2)):
                    off = (got.cpu().double() - want).abs()
                    assert off.le(error * 1.01 + roundings * (want.abs() * 1.02 * HALF_STEP[dtype] + tiny)).all(), float((off / want.abs()).max())


# ---- waits that run out ----------------------------------------------------------------------------------------------


def test_expired_waits_need_a_bound():
    for budget in (0, -1, 2000000001):
        assert "budget" in error_of(_C.lib().nvfp4_debug_linear_expired(1024, 64, 1024, 64, None, None, 0, 1024, 32, None, 0, 4, 32, 64, 0, 0, 0, 0, budget, None, None))


# the swapped tiles, split over clusters and not, the other ones, pairs; rows that TMA addresses and rows that it does not
@gpu
@pytest.mark.parametrize("m, n, k", [(1, 4096, 4096), (33, 1411, 2048), (256, 4096, 1024), (400, 200, 1024), (200, 2049, 64), (3000, 2056, 128), (3000, 2057, 128), (3000, 128, 4096),
                                     (2500, 4104, 392), (16384, 128, 264)])
def test_what_an_expired_wait_leaves_is_nan(m, n, k):
    """Products that are never issued, residuals that are never fetched: the kernels end after half a millisecond, with the status bit and NaN
    in place of results, also for callers without a status word, and the next call is an ordinary one."""
    seen = 0
    for out in (torch.bfloat16, torch.float32):
        x, w, bias, residual = (t.cuda() for t in make(m, n, k, torch.bfloat16, 3, out))
        want, _ = _C.linear(x, w, bias, residual, "gelu", out, keep=True)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        for word in (status, None):
            for r in (residual, None):
                d, slopes = _C.debug_linear_expired(x, w, bias, r, "gelu", out, 1_000_000, word)
                assert torch.isnan(d).all() and (slopes[:, :n] == -1).all() and (slopes[:, n:] == 0).all()
        with pytest.raises(RuntimeError, match="error 4"):
            _C.read_status(status)
        d, _ = _C.debug_linear_expired(x, w, bias, residual, "gelu", out, 1_000_000, status, withhold_residuals=True)
        expired = int(status.item())
        assert torch.isnan(d).all() if expired else torch.equal(d, want)     # forms that read it themselves finish
        seen += expired
        assert torch.equal(_C.linear(x, w, bias, residual, "gelu", out, keep=True)[0], want)
    assert seen or (m, n, k) != (3000, 2056, 128)


@gpu
def test_gradients_that_nobody_asks_for_are_not_computed():
    """x from a layer before needs a gradient, this call of autograd.grad does not: no memory is taken for it."""
    m, n, k = 4096, 64, 4096

    def memory(y, wanted, dd):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        grads = torch.autograd.grad(y, wanted, dd, retain_graph=True)
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before, grads

    x, w, bias, residual = (t.cuda().requires_grad_() for t in make(m, n, k, torch.bfloat16, 1))
    dd = torch.randn(m, n, generator=gen(2)).bfloat16().cuda()
    leaves = [x, w, bias, residual]
    for activation in ("none", "silu"):
        y = linear(*leaves, activation=activation)
        _, full = memory(y, leaves, dd)
        for i, most in ((1, 4 << 20), (2, 4 << 20), (3, 1 << 20)):       # dx alone is 32 MB
            taken, (grad,) = memory(y, [leaves[i]], dd)
            assert taken < most and torch.equal(grad, full[i]), (activation, i, taken)
    rows = torch.randn(4096, 4096, generator=gen(3)).bfloat16().cuda().requires_grad_()
    place = torch.randperm(4096, generator=gen(4)).view(2048, 2).cuda()
    order = TokenOrder(place, torch.zeros(4096, dtype=torch.int32, device="cuda"), torch.zeros(4096, dtype=torch.int32, device="cuda"))
    weights = torch.rand(2048, 2, generator=gen(5)).cuda().requires_grad_()
    y = unsort_tokens(rows, order, weights)
    dy = torch.randn(2048, 4096, generator=gen(6)).bfloat16().cuda()
    _, full = memory(y, [rows, weights], dy)
    taken, (grad,) = memory(y, [weights], dy)
    assert taken < 4 << 20 and torch.equal(grad, full[1])
    assert torch.equal(memory(y, [rows], dy)[1][0], full[0])


@gpu
@pytest.mark.parametrize("dtype, tokens, n, k", [(torch.float16, 70001, 1300, 1032), (torch.float16, 150000, 40, 64), (torch.float16, 500000, 300, 264),
                                                 (torch.bfloat16, 1100000, 40, 64), (torch.bfloat16, 2300001, 9, 8), (torch.bfloat16, 300000, 1100, 2056)])
def test_sums_over_very_many_tokens(dtype, tokens, n, k):
    """Operands of one sign: a cut at every step of the sum shows, and in FP16 it would be more than the rounding of the result."""
    g = torch.Generator("cuda").manual_seed(5)
    x = (torch.rand(tokens, k, generator=g, device="cuda") + 0.5).to(dtype)
    dd = ((torch.rand(tokens, n, generator=g, device="cuda") + 0.5) * (8.0 / tokens)).to(dtype)
    w = torch.zeros(n, k, dtype=dtype, device="cuda").requires_grad_()
    (dw,) = torch.autograd.grad(linear(x, w), w, dd)
    want = sum(dd[i:i + 100000].double().t() @ x[i:i + 100000].double() for i in range(0, tokens, 100000))
    # sums of 1024 products leave the tensor core, which may cut at each of its 64 steps (2^-22 of the sum so far, on average half of the
    # last), and are added in FP32, where a rounding is of the sum so far, too
    error = want * ((tokens / 1024 / 2 + 4) * 2.0 ** -24 + 32 * 2.0 ** -22)
    step = 2.0 ** (torch.floor(torch.log2(want)) - {torch.float16: 10, torch.bfloat16: 7}[dtype])
    worst = ((dw.double() - want).abs() - (0.5 * step + error))
    assert worst.max() <= 0


@gpu
@pytest.mark.parametrize("m, n, k", [(1, 300, 4096), (2, 64, 20000), (1, 1000, 20000), (5, 200, 4096), (40, 500, 20000), (300, 128, 4096), (700, 1024, 4096), (3000, 128, 20000),
                                     (3000, 3001, 4096), (16384, 128, 4096)])
def test_fp32_outputs_are_sums_of_short_sums(m, n, k):
    """Operands of one sign: nothing cancels, and a sum that stayed in the tensor core's accumulator, or lost a part, would show (BF16 products are
    cut by 1.9e-9 of the sum each, FP16 ones by 6e-9: 8e-6 and more for K = 4096)."""
    g = torch.Generator("cuda").manual_seed(m)
    few = m <= 2 and n * k <= 5 << 20                                     # without tensor cores: a lane's chain of K / 32 products at most
    error = (k / 64 + 16) * 2.0 ** -24 if few else 8 * 2.0 ** -22 + (k / 512 + 12) * 2.0 ** -24      # 16 steps of 16, K / 256 sums, up to eight CTAs' sums
    for dtype in (torch.bfloat16, torch.float16):
        x = (torch.rand(m, k, generator=g, device="cuda") + 0.5).to(dtype)
        w = (torch.rand(n, k, generator=g, device="cuda") + 0.5).to(dtype)
        want = x.double() @ w.double().t()
        assert ((linear(x, w, out_dtype=torch.float32).double() - want).abs() / want).max() <= error


@gpu
@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("scale", [1e-9, 3e-20, 0.1, 1.0, 1e6, 1e9])
@pytest.mark.parametrize("m, n, k", [(5, 24, 16), (300, 40, 64), (3000, 33, 72), (2700, 2056, 264)])
def test_fp32_gradients_outside_of_fp16(m, n, k, scale, binding, monkeypatch):
    """FP16 operands, an FP32 output and FP32 gradients that FP16 does not hold, while their sums times x or w are ordinary numbers."""
    _C.lib()
    if not binding:
        monkeypatch.setattr(_C, "_binding", None)
    g = gen(9)
    dd = torch.randn(m, n, generator=g) * scale
    big = min(max(2.0 / scale, 2.0 ** -10), 2.0 ** 9)                       # brings the terms of a sum towards 1
    for activation in ("none", "silu"):
        for which in ("dx", "dw"):
            # the operand that the gradient meets is large (or small), the other one makes up for it in z
            x, w = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g)
            x, w = (x / (big * k ** 0.5), w * big) if which == "dx" else (x * big, w / (big * k ** 0.5))
            x, w, bias = x.half(), w.half(), torch.randn(n, generator=g).half()
            leaves = [t.cuda().requires_grad_() for t in (x, w, bias)]
            y = linear(*leaves, activation=activation, out_dtype=torch.float32)
            dx, dw, db = torch.autograd.grad(y, leaves, dd.cuda())
            z = (x.double() @ w.double().t() + bias.double()).requires_grad_()
            (dz,) = torch.autograd.grad(act64(z, activation), z, dd.double())
            z = z.detach()
            slope = 0.0 if activation == "none" else 2.0 ** -15 + CURVATURE * (sum_error(x, w.t()) + z.abs() * 2.0 ** -23) + 64 * 2.0 ** -23
            dz_error = dd.double().abs() * slope
            # dz rounded to FP16 of a multiple whose largest is 1/4 at least: smaller than 2^-14 of that it loses up to 2^-25
            rounded = dz_error + (dz.abs() + dz_error) * 1.01 * 2.0 ** -11 + 4 * 2.0 ** -25 * float(dz.abs().max())
            for name, got, want, size, spread, terms in (("db", db, dz.sum(dim=0), dz.abs().sum(dim=0), dz_error.sum(dim=0), m),
                                                         ("dx", dx, dz @ w.double(), dz.abs() @ w.double().abs(), rounded @ w.double().abs(), n),
                                                         ("dw", dw, dz.t() @ x.double(), dz.abs().t() @ x.double().abs(), rounded.t() @ x.double().abs(), m)):
                error = spread + size * (terms + 4) * 2.0 ** -23
                ok = (got.cpu().double() - want).abs().le(error + (want.abs() + error) * 1.01 * 2.0 ** -11 + 2.0 ** -25)
                held = want.abs() + error < 65000                         # a result beyond FP16 is an infinity, or its largest number
                assert ok[held].all(), (name, activation, which)
                assert (got.cpu().abs()[want.abs() - error > 65536] == math.inf).all()


@gpu
def test_infinite_gradients_stay_in_their_rows():
    x, w, bias, _ = make(40, 24, 64, torch.float16, 3)
    for scale in (1e-9, 1.0):
        dd = torch.randn(40, 24, generator=gen(1)) * scale
        clean = dd.clone()
        dd[3, 5], dd[7, 2] = math.inf, math.nan
        clean[3, 5] = clean[7, 2] = 0
        leaves = [t.cuda().requires_grad_() for t in (x, w)]
        y = linear(*leaves, out_dtype=torch.float32)
        dx, dw = torch.autograd.grad(y, leaves, dd.cuda(), retain_graph=True)
        want_x, want_w = torch.autograd.grad(y, leaves, clean.cuda())
        rows, columns = torch.ones(40, dtype=torch.bool), torch.ones(24, dtype=torch.bool)
        rows[[3, 7]] = False
        columns[[5, 2]] = False
        assert torch.equal(dx[rows], want_x[rows]) and torch.equal(dw[columns], want_w[columns])
        assert torch.isnan(dx[7]).all() and not torch.isfinite(dx[3]).any() and not torch.isfinite(dw[2]).any()


def test_scales_refuse():
    lib = _C.lib()
    assert "FP16 operands" in error_of(lib.nvfp4_linear_dz_scaled(1024, 32, 1024, 32, 1024, 32, None, 4, 32, 0, 1, 1024, None))
    assert "FP16 operands" in error_of(lib.nvfp4_linear_dz_scaled(1024, 32, 1024, 32, 1024, 32, None, 4, 32, 2, 2, 1024, None))
    assert "goes with dz" in error_of(lib.nvfp4_linear_dz_scaled(1024, 32, 1024, 32, None, 32, 1024, 4, 32, 2, 1, 1024, None))
    assert "scale is not aligned" in error_of(lib.nvfp4_linear_dz_scaled(1024, 32, 1024, 32, 1024, 32, None, 4, 32, 2, 1, 1026, None))


@gpu
def test_long_sums_with_everything_in_the_epilogue():
    """FP16 sums of 20000 products of one sign that no cluster shares: forward with bias, activation, kept slopes and residual, and dx."""
    g = torch.Generator("cuda").manual_seed(6)
    some = lambda *s, scale=1.0: ((torch.rand(*s, generator=g, device="cuda") + 0.5) * scale).half()
    dtype, k = torch.float16, 20000
    cut = (k / 1024 / 2 + 4) * 2.0 ** -24 + 32 * 2.0 ** -22                  # sums of 1024 with 64 steps each, added in FP32
    for n in (2056, 2057):                                                # through TMA, and the odd stride's way
        x, w, bias, residual = some(2600, k), some(n, k, scale=1 / k), some(n), some(2600, n)
        leaves = [t.requires_grad_() for t in (bias, residual)]
        y = linear(x, w, *leaves, activation="silu")
        z = x.double() @ w.double().t() + bias.detach().double()
        want = act64(z, "silu") + residual.detach().double()
        error = SLOPE * z * cut + want * 40 * 2.0 ** -23                  # z, silu and the sum, each with a few roundings
        assert (y.detach().double() - want).abs().le(error + (want + error) * 1.01 * HALF_STEP[dtype]).all()
        dd = some(2600, n, scale=1 / 2600)
        db, dr = torch.autograd.grad(y, leaves, dd)
        slope = torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))
        want = (dd.double() * slope).sum(dim=0)
        assert torch.equal(dr, dd) and (db.double() - want).abs().le(want * (2.0 ** -13 + 1.01 * HALF_STEP[dtype])).all()      # slopes near 1.09: 2^-15 of them
    x, w = torch.zeros(2600, 2056, dtype=dtype, device="cuda").requires_grad_(), some(k, 2056, scale=1 / k)
    dd = some(2600, k)
    (dx,) = torch.autograd.grad(linear(x, w), x, dd)
    want = dd.double() @ w.double()
    step = 2.0 ** (torch.floor(torch.log2(want)) - 10)
    assert ((dx.double() - want).abs() <= 0.5 * step + want * cut).all()


@gpu
def test_captured_training_steps_side_by_side_see_new_data():
    """Two captures of one step, replayed at the same time on streams of their own: lists of pairs, peaks of gradients and sums of columns live in
    workspaces of each capture."""
    tokens, experts, k, hidden = 700, 16, 4, 128
    g = gen(7)
    half = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).half().cuda().requires_grad_()
    leaves = [half(tokens, hidden), half(experts, hidden, scale=0.2), half(264, hidden, scale=0.1), half(264, scale=0.1), half(hidden, 264, scale=0.06)]
    dy = torch.randn(tokens, hidden, generator=g).cuda()

    def step():
        x, gate, w1, bias, w2 = leaves
        ids, weights = route_tokens(linear(x, gate, out_dtype=torch.float32), k, renormalize=False)
        rows, order = sort_tokens(x, ids, experts, alignment=16)
        late = order._replace(place=order.place.masked_fill(weights.detach() < 0.05, -1))                    # pairs dropped afterwards
        y = linear(linear(unsort_tokens(rows, late, weights), w1, bias, activation="gelu"), w2, out_dtype=torch.float32)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for scale in (1.0, 1e-7, 1e6):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(tokens, hidden, generator=g))
            dy.copy_(torch.randn(tokens, hidden, generator=g) * scale)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a.nan_to_num(1.0, 2.0, 3.0), b.nan_to_num(1.0, 2.0, 3.0)) for a, b in zip(want, out))
