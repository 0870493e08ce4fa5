"""Row codes, dense layers in 8-bit integers and 8-bit activation checkpoints against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHORT = np.arange(4, 9) / 8.0   # mantissas of a short scale in [1/2, 1]


def _codes64(x, bits=24):
    """Codes and scales by the definition: float32 roundings, each of one value that float64 holds well enough."""
    x = x.detach().cpu().to(torch.float32).double().numpy()
    a = np.abs(x).max(1)
    f = lambda v: v.astype(np.float32).astype(np.float64)  # noqa: E731
    with np.errstate(all="ignore"):
        s, i = f(a / 127), f(127 / a)
        if bits == 3:
            m, e = np.frexp(s)
            s = np.ldexp(np.ceil(m * 8) / 8, e)
            i = f(1 / s)
        q = np.rint(f(x * i[:, None]))
    q[a < 2.0 ** -119], s[a < 2.0 ** -119] = 0, 0
    bad = ~np.isfinite(a)
    q[bad], s[bad] = 0, np.nan
    return q, s


def _act64(v, name):
    return {"none": lambda v: v, "relu": lambda v: np.maximum(v, 0), "tanh": np.tanh, "sigmoid": lambda v: 1 / (1 + np.exp(-v))}[name](v)


def _x(R, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp(torch.randn(K, generator=g)) * torch.exp(2 * torch.randn(R, 1, generator=g))
    x[:, : K // 2].clamp_(min=0)
    return x.to(dtype).cuda()


def _within(got, want, tol):
    # rounding to nearest takes a float16 of 65504 + half a step (32 / 2) or more to infinity: right where the value may be one
    inf = got.dtype == torch.float16
    got = got.detach().cpu().double().numpy()
    ok = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= tol)
    if inf:
        ok |= np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + tol >= 65520.0)
    assert ok.all(), (int((~ok).sum()), got[~ok][:5], want[~ok][:5], np.broadcast_to(tol, got.shape)[~ok][:5])


def _same(a, b):
    """Equal, a NaN (an input that float16 holds as infinity) to a NaN."""
    return a.shape == b.shape and a.dtype == b.dtype and bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("bits", [24, 3])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K", [(1, 1), (3, 2), (5, 16), (64, 168), (7, 127), (2, 129), (33, 1000), (4, 4096), (3, 9217), (2, 18432), (2, 70001)])
def test_codes_are_the_definitions(R, K, dtype, bits):
    from muzero_amd.quantized import quantize_rows
    x = _x(R, K, dtype, seed=K)
    c = quantize_rows(x, scale_bits=bits)
    q, s = _codes64(x, bits)
    assert c.codes.shape[1] % 128 == 0 and (c.codes[:, K:] == 0).all()
    np.testing.assert_array_equal(c.codes[:, :K].cpu().numpy(), q)
    np.testing.assert_array_equal(c.scales.cpu().double().numpy(), s)
    if bits == 3:
        assert set(np.frexp(s[s > 0])[0]) <= set(SHORT)
    back = c.dequantize()
    assert back.dtype == dtype and back.shape == x.shape
    np.testing.assert_array_equal(back.cpu().float().numpy(), torch.from_numpy((q * s[:, None]).astype(np.float32)).to(dtype).float().numpy())


@pytest.mark.parametrize("bits", [24, 3])
def test_hard_rows(bits):
    from muzero_amd.quantized import quantize_rows
    x = torch.randn(12, 300)
    x[0] = 0.0
    x[1] = 1e-40                                   # below float32's normal range
    x[2] *= 2.0 ** -121                            # below the smallest scale
    x[3] *= 2.0 ** -116
    x[4] = torch.finfo(torch.float32).max
    x[5, 17] = torch.inf
    x[6, 299] = torch.nan
    x[7] = 0.0
    x[7, 1] = -3.0
    x[8] = torch.arange(300) % 128 / 127.0         # every code, on the step
    x[9] = (torch.arange(300) % 254 + 0.5) / 254   # halfway between steps
    x[10] = -x[9]
    x[11, 0] = torch.finfo(torch.float32).max
    c = quantize_rows(x.cuda(), scale_bits=bits)
    q, s = _codes64(x, bits)
    np.testing.assert_array_equal(c.codes[:, :300].cpu().numpy(), q)
    np.testing.assert_array_equal(c.scales.cpu().double().numpy(), s)
    assert np.abs(q).max() <= 127 and c.dequantize()[5:7].isnan().all()


def _int8_reference(x, w, b, act, bits=24):
    (q, s), (t, v) = _codes64(x), _codes64(w)
    lin = (q @ t.T) * s[:, None] * v[None, :]
    bias = 0.0 if b is None else b.cpu().double().numpy()[None, :]
    pre = lin + bias
    # sum -> float32, scale product, product, bias: four roundings; every activation's slope is at most 1, its own
    # evaluation costs a few units of its result
    return _act64(pre, act), 4 * U * (np.abs(lin) + np.abs(pre)) + 8 * U * np.abs(_act64(pre, act)) + 1e-37


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K,N,act", [(1, 1, 1, "none"), (1, 16, 7, "relu"), (3, 168, 256, "relu"), (1, 168, 256, "tanh"), (256, 256, 7, "none"),
                                       (5, 129, 33, "sigmoid"), (16, 1000, 100, "none"), (17, 512, 130, "relu"), (64, 640, 64, "none"),
                                       (65, 127, 127, "tanh"), (128, 128, 128, "none"), (130, 300, 257, "sigmoid"), (1, 9216, 300, "relu"),
                                       (2, 18432, 65, "none"), (300, 4097, 190, "relu"), (8, 4096, 1024, "none"), (520, 260, 520, "none"),
                                       (33, 2048, 2, "none"), (1030, 64, 1, "none"), (48, 8192, 1000, "relu"), (700, 1200, 900, "none"), (3700, 100, 3601, "none"), (3601, 384, 3700, "relu"),
                                       (2000, 130, 3700, "tanh"), (2100, 700, 3300, "none"), (200, 16500, 700, "relu"), (250, 18432, 2050, "none"),
                                       (16, 1024, 40, "relu"), (16, 1025, 40, "none"), (7, 2300, 60, "tanh"), (15, 5, 3, "none"),
                                       (1, 20000, 16, "relu"), (3, 12289, 1024, "none"), (32, 13000, 5, "sigmoid"), (20, 12288, 90, "none"),
                                       (64, 300, 30000, "none"), (64, 8200, 7000, "relu"), (33, 500, 20001, "none")])
def test_int8_linear(R, K, N, act, dtype):
    from muzero_amd.quantized import int8_linear, quantize_rows
    x = _x(R, K, dtype, seed=R + K)
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(N)) / K ** 0.5
    b = torch.randn(N, generator=torch.Generator().manual_seed(1)) if N % 2 else None
    qw = quantize_rows(w.cuda())
    want, tol = _int8_reference(x, w, b, act)
    y = int8_linear(x, qw, None if b is None else b.cuda(), act)
    assert y.dtype == dtype and y.shape == (R, N)
    _within(y, want, tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype])
    coded = int8_linear(quantize_rows(x), qw, None if b is None else b.cuda(), act)
    assert _same(coded, y)                             # rows coded beforehand: the same numbers
    y32 = int8_linear(x, qw, None if b is None else b.cuda(), act, out_dtype=torch.float32)
    _within(y32, want, tol + U * np.abs(want))


@pytest.mark.parametrize("R", [1, 9, 100, 400])
def test_int8_rows_are_independent_and_nan_is_loud(R):
    from muzero_amd.quantized import int8_linear, quantize_rows
    K, N = 500, 140
    x, w = _x(R, K, torch.float32), torch.randn(N, K).cuda()
    w[3, 4] = torch.nan
    qw = quantize_rows(w)
    y = int8_linear(x, qw, activation="relu")
    assert y[:, 3].isnan().all()
    keep = [n for n in range(N) if n != 3]
    assert y[:, keep].isfinite().all()
    x2 = x.clone()
    x2[R // 2, 7] = torch.inf
    y2 = int8_linear(x2, qw, activation="relu")
    assert y2[R // 2].isnan().all()
    rest = [r for r in range(R) if r != R // 2]
    assert torch.equal(y2[rest][:, keep], y[rest][:, keep])


def test_largest_sum_stays_exact():
    from muzero_amd.quantized import int8_linear, quantize_rows
    K = 131072
    for R, N in ((1, 3), (200, 150)):
        x, w = torch.ones(R, K, device="cuda"), torch.ones(N, K, device="cuda")
        w[1] = -1.0
        y = int8_linear(x, quantize_rows(w))
        s = float(quantize_rows(x).scales[0])
        want = np.float64(127 * 127 * K) * s * s
        got = y.cpu().double().numpy()
        assert np.abs(got[:, 0] - want).max() <= 4 * U * want and np.abs(got[:, 1] + want).max() <= 4 * U * want
    with pytest.raises(ValueError):
        int8_linear(torch.ones(1, K + 1, device="cuda"), quantize_rows(torch.ones(1, K + 1, device="cuda")))


@pytest.mark.parametrize("dtype", TYPES)
def test_int8_shapes_strides_and_alignment(dtype):
    from muzero_amd.quantized import int8_linear, quantize_rows
    big = _x(40, 700, dtype)
    w = torch.randn(90, 333).cuda()
    qw, qv = quantize_rows(w), quantize_rows(torch.cat([w, w], 1)[:, :333])
    assert torch.equal(qw.codes, qv.codes)
    for view in (big[:, :333], big[:, 1:334], big[::3, 5:338], big.t()[:333].t(), big[:, : 2 * 333 : 2], big[3:4, 7:340],
                 big[:1, :333].expand(40, 333), big[:, :333].reshape(2, 5, 4, 333), big[0, :333]):
        want = int8_linear(view.contiguous().clone(), qw)
        assert torch.equal(int8_linear(view, qw), want) and want.shape == view.shape[:-1] + (90,)
        c, d = quantize_rows(view), quantize_rows(view.contiguous().clone())
        assert torch.equal(c.codes, d.codes) and torch.equal(c.scales, d.scales)
    assert int8_linear(big[:0, :333], qw).shape == (0, 90)


def _grad_reference(dz, x, bits=3):
    q, s = _codes64(x, bits)
    g = dz.detach().cpu().double().numpy()
    v = g * s[:, None]
    mag = np.abs(v).T @ np.abs(q)
    # v is rounded once and held to 22 bits (2^-39 of its column's largest at least); products are exact; a float32 sum
    # of R terms in any order is off by at most R u of the magnitudes
    tol = (2.0 ** -21 + (g.shape[0] + 8) * U) * mag + 2.0 ** -39 * np.abs(v).max(0, initial=0)[:, None] * np.abs(q).sum(0)[None, :]
    return v.T @ q, tol + 1e-37, g.sum(0), (g.shape[0] + 4) * U * np.abs(g).sum(0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K,N", [(1, 1, 1), (1, 168, 7), (2, 16, 300), (31, 129, 5), (64, 64, 64), (65, 168, 256), (256, 336, 168), (300, 100, 130),
                                   (1000, 257, 33), (257, 60, 200), (1024, 100, 65), (1025, 30, 129), (2049, 40, 50), (5000, 128, 128), (256, 1152, 640), (130, 2000, 700), (40, 3601, 3700), (200, 3700, 3601),
                                   (330, 3300, 2049), (9000, 130, 70), (9000, 1400, 900)])
def test_weight_gradient(R, K, N, dtype):
    from muzero_amd.checkpoints import save_activations, weight_grad
    x = _x(R, K, dtype, seed=R)
    g = torch.Generator().manual_seed(K)
    dz = (torch.randn(R, N, generator=g) * torch.exp(3 * torch.randn(N, generator=g)) * 1e-2)
    dz[torch.rand(R, generator=g) < 0.2] = 0.0
    dz = dz.to(dtype).cuda()
    saved = save_activations(x)
    want, tol, want_b, tol_b = _grad_reference(dz, x)
    dw, db = weight_grad(dz, saved)
    assert dw.dtype == db.dtype == dtype and dw.shape == (N, K)
    _within(dw, want, tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype])
    _within(db, want_b, tol_b + HALF[dtype] * (np.abs(want_b) + tol_b) + TINY[dtype])
    again, none = weight_grad(dz, saved, want_bias=False)
    assert none is None and _same(again, dw)


def test_weight_gradient_holds_columns_of_any_size():
    """Each output row has a range of its own; within one, values down to 2^-16 of the largest keep 22 bits."""
    from muzero_amd.checkpoints import save_activations, weight_grad
    R, K, N = 200, 96, 60
    x = _x(R, K, torch.float32)
    dz = torch.randn(R, N) * torch.logspace(-33, 30, N)[None, :]
    dz[:, 5] = 0.0
    dz[:, 6] = 1e-42
    dz[:, 7] *= torch.logspace(0, -8, R)                # a wide range inside one column
    dz = dz.cuda()
    want, tol, _, _ = _grad_reference(dz, x)
    dw, _ = weight_grad(dz, save_activations(x))
    _within(dw, want, tol + 2 * U * np.abs(want) + 1e-40)
    assert (dw[5] == 0).all()
    dz[3, 8], dz[4, 9] = torch.inf, torch.nan
    dw2, db2 = weight_grad(dz, save_activations(x))
    assert dw2[8].isnan().all() and dw2[9].isnan().all() and db2[8].isinf() and db2[9].isnan()
    keep = [n for n in range(N) if n not in (8, 9)]
    assert torch.equal(dw2[keep], dw[keep])


def test_full_scales_and_strided_gradients():
    from muzero_amd.checkpoints import save_activations, weight_grad
    from muzero_amd.quantized import quantize_rows
    R, K, N = 90, 200, 70
    for dtype in TYPES:
        x = _x(R, K, dtype)
        wide = (torch.randn(R, 3 * N) * 0.01).to(dtype).cuda()
        for dz in (wide[:, :N], wide[:, 1:N + 1], wide[:, ::3], wide[:, :N].contiguous().t().contiguous().t()):
            assert torch.equal(weight_grad(dz, save_activations(x))[0], weight_grad(dz.contiguous().clone(), save_activations(x))[0])
        want, tol, _, _ = _grad_reference(wide[:, :N], x, bits=24)
        dw, _ = weight_grad(wide[:, :N], quantize_rows(x))
        _within(dw, want, tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype])
    dw, db = weight_grad(torch.zeros(0, N, device="cuda"), save_activations(torch.zeros(0, K, device="cuda")))
    assert (dw == 0).all() and dw.shape == (N, K) and (db == 0).all()


@pytest.mark.parametrize("activation", ["none", "relu", "tanh", "sigmoid"])
@pytest.mark.parametrize("shape", [(1, 5, 3), (64, 168, 256), (33, 40, 129), (4, 300, 9)])
def test_checkpointed_layer(shape, activation):
    """Forward: the layer itself.  Backward: dz = dy act'(y) with what was kept of y, dx = dz W, dW and db from dz and
    the codes of x."""
    from muzero_amd.checkpoints import checkpointed_linear, save_activations
    R, K, N = shape
    torch.manual_seed(R)
    lin = torch.nn.Linear(K, N).cuda()
    x = torch.randn(R, K, device="cuda", requires_grad=True)
    dy = torch.randn(R, N, device="cuda")
    y = checkpointed_linear(x, lin.weight, lin.bias, activation)
    act = {"none": lambda t: t, "relu": torch.relu, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[activation]
    assert torch.equal(y, act(lin(x)))
    y.backward(dy)
    y64, g = y.detach().cpu().double().numpy(), dy.cpu().double().numpy()
    if activation == "relu":
        dz = g * (y64 > 0)
    elif activation == "tanh":
        dz = g * (1 - (np.rint(y64 * 127) / 127) ** 2)
    elif activation == "sigmoid":
        dz = g * (1 - (np.rint(254 * y64 - 127) / 127) ** 2) / 4
    else:
        dz = g
    w64 = lin.weight.detach().cpu().double().numpy()
    # a code of y next to a border may fall either way in float32 (y is then rounded to a neighbour of the same distance)
    step = 0.0 if activation in ("none", "relu") else 1e-6
    _within(x.grad, dz @ w64, (N + 8) * U * (np.abs(dz) @ np.abs(w64)) + step * np.abs(g) @ np.abs(w64) + 1e-37)
    q, s = _codes64(x, 3)
    xh = q * s[:, None]
    _within(lin.weight.grad, dz.T @ xh, (2.0 ** -20 + (R + 8) * U) * (np.abs(dz).T @ np.abs(xh)) + step * np.abs(g).T @ np.abs(xh) + 1e-37)
    _within(lin.bias.grad, dz.sum(0), (R + 8) * U * np.abs(dz).sum(0) + step * np.abs(g).sum(0) + 1e-37)
    assert torch.equal(save_activations(x).codes.cpu()[:, :K], torch.from_numpy(q).to(torch.int8))


@pytest.mark.parametrize("activation", ["relu", "tanh", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 7, 8, 65, 1000])
def test_kept_activations(N, dtype, activation):
    """What is kept of y and the gradient read from it, for every stride; NaN stays NaN."""
    from muzero_amd.checkpoints import _act_grad, _act_save
    R = 9
    y = torch.randn(R, N + 3).cuda()
    y = {"relu": torch.relu, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[activation](y).to(dtype)[:, 1:N + 1]
    dy = torch.randn(R, N + 5).to(dtype).cuda()[:, 2:N + 2]
    saved = _act_save(y, activation)
    dz = _act_grad(dy, saved, activation)
    y64, g = y.cpu().double().numpy(), dy.cpu().double().numpy()
    if activation == "relu":
        np.testing.assert_array_equal(dz.cpu().double().numpy(), g * (y64 > 0))
    else:
        # the product with 127 or 254 is one float32 rounding away from the definition: half-way cases may go either way
        t = (np.rint(y64 * 127) if activation == "tanh" else np.rint(y64 * 254 - 127)) / 127
        want = g * (1 - t * t) * (1.0 if activation == "tanh" else 0.25)
        near = np.abs(np.abs((y64 * 127 if activation == "tanh" else y64 * 254 - 127)) % 1 - 0.5) < 1e-4
        slack = np.where(near, np.abs(g) * 2 / 127, 0.0)
        _within(dz, want, slack + 8 * U * np.abs(g) + HALF[dtype] * np.abs(want) + TINY[dtype])
        y2 = y.clone()
        y2[1, 0] = torch.nan
        assert _act_grad(dy, _act_save(y2, activation), activation)[1, 0].isnan()


def test_a_row_with_an_infinity_is_loud_in_the_gradient():
    from muzero_amd.checkpoints import save_activations, weight_grad
    for R in (20, 700):
        x, dz = torch.randn(R, 50, device="cuda"), torch.randn(R, 30, device="cuda")
        x[3, 7] = torch.inf
        for t in TYPES:
            dw, db = weight_grad(dz.to(t), save_activations(x.to(t)))
            assert dw.isnan().all() and db.isfinite().all()


def test_layers_of_unusual_use():
    """No gradient wanted of some inputs, several leading dimensions, no rows at all, a strided gradient, no_grad."""
    from muzero_amd.checkpoints import checkpointed_linear
    torch.manual_seed(0)
    lin = torch.nn.Linear(40, 24).cuda()
    x = torch.randn(3, 5, 40, device="cuda")
    want = torch.relu(lin(x))
    dy = torch.randn(3, 24, 5, device="cuda").transpose(1, 2)
    full = checkpointed_linear(x.clone().requires_grad_(True), lin.weight, lin.bias, "relu")
    assert torch.equal(full, want)
    xr = x.clone().requires_grad_(True)
    ref = torch.autograd.grad(checkpointed_linear(xr, lin.weight, lin.bias, "relu"), (xr, lin.weight, lin.bias), dy)
    w, b = lin.weight.detach(), lin.bias.detach()
    got, = torch.autograd.grad(checkpointed_linear(xr, w, b, "relu"), xr, dy)
    assert torch.equal(got, ref[0]) and got.shape == x.shape
    got, = torch.autograd.grad(checkpointed_linear(x, lin.weight, b, "relu"), lin.weight, dy)
    assert torch.equal(got, ref[1])
    got, = torch.autograd.grad(checkpointed_linear(x, w, lin.bias, "relu"), lin.bias, dy)
    np.testing.assert_allclose(got.detach().cpu(), ref[2].detach().cpu(), rtol=0, atol=15 * U * float(dy.abs().max()) * 15)
    got = torch.autograd.grad(checkpointed_linear(xr, lin.weight, None, "tanh"), (xr, lin.weight), dy)
    assert all(g.isfinite().all() for g in got)
    none = torch.zeros(0, 40, device="cuda", requires_grad=True)
    got = torch.autograd.grad(checkpointed_linear(none, lin.weight, lin.bias, "relu").sum(), (none, lin.weight, lin.bias))
    assert got[0].shape == (0, 40) and all((g == 0).all() for g in got)
    with torch.no_grad():
        y = checkpointed_linear(xr, lin.weight, lin.bias, "sigmoid")
    assert not y.requires_grad and torch.equal(y, torch.sigmoid(lin(x)))
    g, = torch.autograd.grad(checkpointed_linear(xr, lin.weight, lin.bias).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_a_layer_keeps_a_quarter_of_the_bytes():
    from muzero_amd.checkpoints import checkpointed_linear
    lin = torch.nn.Linear(2048, 1024).cuda()
    x = torch.randn(4096, 2048, device="cuda", requires_grad=True)

    def kept(fn):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        src = x * 1.0                                   # an input nobody else keeps
        y = fn(src)
        del src
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated() - before - y.numel() * 4, y
    full, y0 = kept(lambda t: torch.tanh(lin(t)) + 0.0)
    small, y1 = kept(lambda t: checkpointed_linear(t, lin.weight, lin.bias, "tanh") + 0.0)
    assert torch.equal(y0, y1) and small < 0.26 * full + 65536 * 2, (small, full)


def _networks(seed=0):
    from muzero_amd.config import load_config
    from muzero_amd.neural_networks import DynamicsNetwork, PredictionNetwork, RepresentationNetwork
    cfg = load_config("config_c4_mlp.yaml")
    torch.manual_seed(seed)
    ls = cfg.networks.latent_shape
    return (RepresentationNetwork((2, 6, 7), ls, cfg.networks.representation).cuda(), DynamicsNetwork(ls, 7, cfg.networks.dynamics).cuda(),
            PredictionNetwork(ls, 7, cfg.networks.prediction).cuda())


def _batch(B, w=5, seed=0):
    from muzero_amd.learner import WindowBatch
    g = torch.Generator().manual_seed(seed)
    return WindowBatch(torch.randn(B, 3, 6, 7, generator=g), torch.randint(0, 7, (B, w + 1), generator=g),
                       torch.softmax(torch.randn(B, w + 1, 7, generator=g), -1), torch.randn(B, w + 1, generator=g),
                       torch.randn(B, w + 1, generator=g), torch.rand(B, generator=g) + 0.1).to("cuda")


class _PlainCheckpoint(torch.autograd.Function):
    """A relu or linear layer whose weight gradient reads its input back from codes, in elementary float32 operations."""

    @staticmethod
    def forward(ctx, x, weight, bias, relu):
        y = torch.nn.functional.linear(x, weight, bias)
        y = torch.relu(y) if relu else y
        q, s = _codes64(x, 3)
        ctx.save_for_backward(torch.from_numpy((q * s[:, None]).astype(np.float32)).cuda(), weight, y)
        ctx.relu = relu
        return y

    @staticmethod
    def backward(ctx, dy):
        xh, weight, y = ctx.saved_tensors
        dz = dy * (y > 0) if ctx.relu else dy
        return dz @ weight, dz.t() @ xh, dz.sum(0), None


def test_unroll_with_checkpoints(monkeypatch):
    """Same loss bit for bit, and the gradients of the same unroll with every dense layer replaced by the plain form of a
    checkpointed one: what differs then is float32 rounding.  A gradient passes at most 6 steps of 4 products of at most
    512 terms, each off by at most (512 + 8) u of its magnitudes: 24 * 520 * 2^-24 = 7.5e-4."""
    import muzero_amd.checkpoints as ck
    from muzero_amd.learner import batched_unroll_loss
    nets = _networks()
    batch = _batch(96)
    params = [p for n in nets for p in n.parameters()]
    keys = [list(n.state_dict()) for n in nets]
    loss, per_window, _ = batched_unroll_loss(*nets, batch, 5)
    loss8, per_window8, _ = batched_unroll_loss(*nets, batch, 5, checkpoints8=True)
    got = torch.autograd.grad(loss8, params)
    assert torch.equal(loss, loss8) and torch.equal(per_window, per_window8)
    assert keys == [list(n.state_dict()) for n in nets] and all("forward" not in m.__dict__ for n in nets for m in n.modules())
    calls = []
    monkeypatch.setattr(ck, "checkpointed_linear",
                        lambda x, w, b, act="none": (calls.append(act), _PlainCheckpoint.apply(x, w, b, act == "relu"))[1])
    want = torch.autograd.grad(batched_unroll_loss(*nets, batch, 5, checkpoints8=True)[0], params)
    assert len(calls) == 6 * (3 + 3) + 5 * (1 + 2)     # f six times (two heads of three layers), g five times
    for p, a, b in zip(params, want, got):
        assert float((a - b).norm()) <= 7.5e-4 * float(a.norm()), p.shape


def test_recorded_learner_step_with_checkpoints():
    from muzero_amd.learner import DataParallelLearner

    def make():
        nets = _networks(3)
        return DataParallelLearner(*nets, torch.optim.Adam([p for n in nets for p in n.parameters()], lr=1e-3, capturable=True), 5,
                                   checkpoints8=True)
    eager, recorded = make(), make()
    for step in range(4):
        b = _batch(64, seed=step)
        l0, pw0 = eager.step_local(b)
        l1, pw1 = recorded.step_local_recorded(b)
        assert abs(l0 - float(l1)) <= 1e-5 * abs(l0)
        np.testing.assert_allclose(pw0, pw1.cpu(), rtol=1e-4)
    for p, q in zip(eager.params, recorded.params):
        np.testing.assert_allclose(p.detach().cpu(), q.detach().cpu(), atol=2e-5)
    s = eager.policy_report(_batch(64), top=3)
    assert s.log_prob.shape == (64,) and s.top_actions.shape == (64, 3) and s.entropy.isfinite().all()


def test_heads_in_8_bits_and_their_scores():
    """The operators in a row, as a server uses them: a policy head in 8-bit integers and the scores of its moves.  The
    codes of x and W are off by at most half a step of 1/127 of a row's largest value each."""
    from muzero_amd.policy_scores import policy_scores
    from muzero_amd.quantized import Int8MLP, quantize_rows
    _, _, f = _networks(1)
    head = Int8MLP(f.policy_mlp)
    lat = torch.randn(200, 4, 6, 7, device="cuda")
    act = torch.randint(0, 7, (200,), device="cuda")
    with torch.no_grad():
        want = f.policy_logits(lat)
        got = head.logits(lat.reshape(200, -1))
        assert float((got - want).abs().max()) <= 0.05 * float(want.abs().max())
        assert torch.equal(head.logits(quantize_rows(lat.reshape(200, -1))), got)
        s = policy_scores(got, act, top=7)
        np.testing.assert_allclose(s.log_prob.exp().cpu(), head(lat.reshape(200, -1)).gather(1, act[:, None])[:, 0].cpu(), rtol=1e-5)
        with torch.no_grad():
            f.policy_mlp[0].weight.mul_(2.0)
        head.refresh()
        assert not torch.equal(head.logits(lat.reshape(200, -1)), got)


def test_networks_in_8_bits_are_their_layers():
    """Int8Networks against the same layers written out: rows gathered and scattered, per-node and per-row actions."""
    from muzero_amd.engine import make_networks
    from muzero_amd.quantized import int8_linear, quantize_rows
    _, g, f = _networks(2)
    nets = make_networks(g, f, int8=True)
    A, D, U = 7, 168, 5
    lat = torch.randn(40, D, device="cuda")
    rows = torch.tensor([3, 39, -1, 0, 7], dtype=torch.int32, device="cuda")
    x = torch.where((rows >= 0)[:, None], lat[rows.clamp(min=0).long()], torch.zeros((), device="cuda"))
    W, b, emb = g.fc_merge.weight.detach(), g.fc_merge.bias.detach(), g.action_embedding.weight.detach()
    base = int8_linear(x, quantize_rows(W[:, :D]))
    table = (emb.double() @ W[:, D:].double().t() + b.double()).float()

    def reward_of(nxt):
        (w0, b0, a0), (w1, b1, a1) = nets.heads[0].layers
        assert (a0, a1) == ("relu", "linear") or (a0, a1) == ("relu", "none")
        return int8_linear(int8_linear(nxt, w0, b0, "relu"), w1, b1)[:, 0]
    out, rew = torch.full((60, D), 9.0, device="cuda"), torch.empty(U, A, device="cuda")
    next_rows = (20 + torch.arange(U * A, device="cuda", dtype=torch.int32))
    next_rows[4] = -1
    nets.dynamics(lat, U * A, rows=rows, next_latent=out, next_rows=next_rows, reward=rew)
    kids = torch.relu(base[:, None] + table[None]).reshape(U * A, D)
    got = torch.where((next_rows >= 0)[:, None], out[next_rows.clamp(min=0).long()], kids)
    torch.testing.assert_close(got, kids, rtol=0, atol=1e-5)                 # the table's float32 sums of 168 terms
    assert (out[0:20] == 9.0).all() and (out[24] == 9.0).all()
    act = torch.tensor([0, 6, 2, 2, 5], dtype=torch.int32, device="cuda")
    one, col = torch.empty(U, D, device="cuda"), torch.zeros(U, 3, device="cuda")
    nets.dynamics(lat, U, rows=rows, action=act, next_latent=one, reward=col[:, 1])
    torch.testing.assert_close(one, kids.view(U, A, D)[torch.arange(U), act.long()], rtol=0, atol=1e-5)
    assert torch.equal(col[:, 1], reward_of(one)) and (col[:, 0] == 0).all()
    pol, val, arg = torch.empty(U, A, device="cuda"), torch.empty(U, device="cuda"), torch.empty(U, dtype=torch.int32, device="cuda")
    nets.prediction(lat, U, rows=rows, softmax_times=1, policy=pol, value=val, argmax=arg)
    p = torch.softmax(nets.heads[2].logits(x), 1)
    torch.testing.assert_close(pol, torch.softmax(p, 1), rtol=1e-6, atol=1e-7)
    assert torch.equal(val, nets.heads[1](x)[:, 0]) and torch.equal(arg.long(), p.argmax(1))
    before = val.clone()
    with torch.no_grad():
        f.value_mlp[0].weight.mul_(1.5)
    nets.refresh()
    nets.prediction(lat, U, rows=rows, value=val)
    assert not torch.equal(val, before)


def test_search_with_networks_in_8_bits():
    """A lock-step search on Int8Networks: its trees are the CPU oracle's on the network outputs it produced, and a whole
    self-play move runs."""
    from muzero_amd.config import load_config
    from muzero_amd.engine import BatchedMCTS, make_networks
    from muzero_amd.selfplay import SelfPlayEngine
    from oracle import tree as otree
    h, g, f = _networks(4)
    nets = make_networks(g, f, int8=True)
    G, A, S, D = 24, 7, 12, 168
    mcts = BatchedMCTS(nets, G, S, 1, discount=0.998, noise_frac=0.25)
    rng = np.random.default_rng(0)
    lat = torch.from_numpy(rng.standard_normal((G, D)).astype(np.float32)).cuda()
    eta = rng.dirichlet(np.full(A, 0.3), size=G).astype(np.float32)
    rand = rng.integers(0, A, size=(G, S + 1)).astype(np.int32)
    tp = np.ones(G, np.int8)
    trace = {}
    res = mcts.run(lat, torch.from_numpy(tp).cuda(), torch.from_numpy(eta).cuda(), torch.from_numpy(rand).cuda(), trace)
    torch.cuda.synchronize()
    pool = mcts.pool
    root_prior = torch.empty(G, A, device="cuda")
    nets.prediction(lat, G, softmax_times=1, policy=root_prior)
    prior = np.concatenate([root_prior.cpu().numpy()[:, None]] + [p.cpu().numpy()[:, None] for p in trace["prior"]], 1)
    nodes = pool.reward.cpu().numpy()
    reward = np.stack([nodes[:, 1 + e * A:1 + (e + 1) * A] for e in range(S + 1)], 1)
    rollout = np.stack([r.cpu().numpy() for r in trace["rollout"]], 1)
    ref = otree.run_batch(A, S, 1, tp, prior, reward, rand, rollout, eta, 0.25, 0.998)
    assert np.array_equal(pool.visit.cpu().numpy(), ref["visit"]) and np.array_equal(pool.value_sum.cpu().numpy(), ref["value_sum"])
    np.testing.assert_allclose(res.policy.cpu().numpy(), ref["policy"], rtol=1e-12)
    cfg = load_config("config_c4_mlp.yaml").training_data_generator
    cfg.mcts.max_iterations = 6
    eng = SelfPlayEngine(h, g, f, G=16, config=cfg, int8=True)
    obs, policy, value, action, _, _ = eng.move()
    assert policy.shape == (16, 7) and bool(policy.isfinite().all()) and bool(value.isfinite().all()) and bool((action >= 0).all())


def test_other_streams_and_replayed_graphs():
    from muzero_amd.checkpoints import save_activations, weight_grad
    from muzero_amd.quantized import int8_linear, quantize_rows
    R, K, N = 100, 400, 300
    x, dz = torch.randn(R, K, device="cuda"), torch.randn(R, N, device="cuda")
    qw = quantize_rows(torch.randn(N, K, device="cuda"))

    def step():
        saved = save_activations(x)
        return (int8_linear(x, qw, activation="tanh"), int8_linear(x[:2], qw), saved.dequantize()) + weight_grad(dz, saved)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for turn in range(3):
        x.normal_(), dz.normal_()
        want = step()
        for gr, out in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, out)), turn


def test_offsets_past_32_bits():
    from muzero_amd.checkpoints import save_activations
    R, K = 140000, 16384  # 2.3e9 values
    x = torch.zeros(R, K, dtype=torch.bfloat16, device="cuda")
    tail = _x(3, K, torch.bfloat16)
    x[-3:] = tail
    c, d = save_activations(x), save_activations(tail)
    assert torch.equal(c.codes[-3:], d.codes) and torch.equal(c.scales[-3:], d.scales) and (c.scales[:-3] == 0).all()
    assert torch.equal(c.dequantize()[-3:], d.dequantize())


def test_a_recorded_graph_follows_refreshed_weights():
    from muzero_amd.engine import make_networks
    from muzero_amd.quantized import Int8MLP
    _, g, f = _networks(6)
    head, nets = Int8MLP(f.policy_mlp), make_networks(g, f, int8=True)
    x = torch.randn(9, 168, device="cuda")
    out = torch.empty(9 * 7, 168, device="cuda")

    def step():
        nets.dynamics(x, 9 * 7, next_latent=out)
        return head(x), out.clone()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        rec = step()
    for turn in range(3):
        with torch.no_grad():
            for p in list(g.parameters()) + list(f.parameters()):
                p.normal_(0, 0.1)
        head.refresh(), nets.refresh()
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(rec, step())), turn
            fresh = Int8MLP(f.policy_mlp)(x)
        assert torch.equal(rec[0], fresh)


def test_more_rows_than_a_weight_gradient_takes_are_refused_in_front():
    from muzero_amd.checkpoints import MAX_CHECKPOINT_ROWS, checkpointed_linear
    w = torch.randn(1, 16, device="cuda", requires_grad=True)
    x = torch.randn(MAX_CHECKPOINT_ROWS + 1, 16, device="cuda")
    with pytest.raises(ValueError, match="rows"):
        checkpointed_linear(x, w)
    y = checkpointed_linear(x[1:], w)  # the largest number
    y.sum().backward()
    want = x[1:].double().sum(0)
    # codes are off by half a step of at most 1.25 / 127 of a row's largest value; the sum of 2^20 terms of one sign each
    bound = float(x[1:].abs().amax(1).double().sum()) * 1.25 / 254 + 2.0 ** -24 * 2 ** 20 * float(x.abs().max())
    assert float((w.grad[0].double() - want).abs().max()) <= bound


def test_contexts_leave_float64_layers_alone():
    from muzero_amd.checkpoints import eight_bit_checkpoints
    _, g, f = _networks(7)
    g, f = g.double(), f.double()
    lat, act = torch.randn(3, 4, 6, 7, device="cuda", dtype=torch.float64), torch.tensor([0, 3, 6], device="cuda")
    want = g(lat, act) + f(lat)
    with eight_bit_checkpoints(g, f):
        got = g(lat, act) + f(lat)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [3, 24])
@pytest.mark.parametrize("R,K,N", [(1, 5, 2), (7, 65, 33), (33, 64, 31), (255, 200, 97), (257, 130, 34), (4096, 100, 70), (4097, 100, 70),
                                   (500, 2048, 2047), (530, 2048, 2048), (90, 3000, 1500),
                                   (5000, 60, 30), (4500, 60, 60), (4500, 50, 250),
                                   (5000, 9000, 30), (4500, 2300, 120), (4500, 1100, 250), (6000, 600, 500), (2048, 70, 40), (2049, 70, 40),
                                   (40000, 33, 65), (3000, 512, 512)])
def test_weight_gradient_on_both_sides_of_its_variants(R, K, N, bits, dtype):
    """Rows on pairs of elements and off them, the last row at the end of its memory, garbage around the rest."""
    from muzero_amd.checkpoints import weight_grad
    from muzero_amd.quantized import quantize_rows
    x = _x(R, K, dtype, seed=N)
    saved = quantize_rows(x, scale_bits=bits)
    g = torch.Generator().manual_seed(R)
    dz = (torch.randn(R, N, generator=g) * 0.1).to(dtype)
    want, tol, want_b, tol_b = _grad_reference(dz, x, bits)
    first = None
    for width, at in ((N, 0), (N + 1, 0), (N + 2 + N % 2, 1), (N + 6, 6)):
        big = torch.full((R * width + at,), torch.nan, dtype=dtype, device="cuda")[: (R - 1) * width + at + N]
        view = big.as_strided((R, N), (width, 1), at)
        view.copy_(dz)
        dw, db = weight_grad(view, saved)
        _within(dw, want, tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype])
        _within(db, want_b, tol_b + HALF[dtype] * (np.abs(want_b) + tol_b) + TINY[dtype])
        first = dw if first is None else first
        assert _same(dw, first)  # x may hold fp16 infinities, whose rows make everything NaN in both


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,N", [(1, 1), (70, 8), (33, 9), (1000, 31), (513, 32), (257, 256), (130, 257), (9, 2047), (5, 2048), (3, 2049), (2, 30000), (2, 70008)])
def test_rows_in_pieces(R, N, dtype):
    """Codes, their values and kept activations for rows narrower than a wave's share up to rows of many pieces."""
    from muzero_amd.checkpoints import _act_grad, _act_save
    from muzero_amd.quantized import quantize_rows
    g = torch.Generator().manual_seed(R + N)
    x = torch.randn(R, N, generator=g).to(dtype).cuda()
    q = quantize_rows(x)
    codes, scales = _codes64(x, 24)
    assert np.array_equal(q.codes[:, :N].cpu().numpy(), codes) and (q.codes[:, N:] == 0).all()
    back = torch.from_numpy(codes.astype(np.float32)) * torch.from_numpy(scales.astype(np.float32))[:, None]
    assert torch.equal(q.dequantize().cpu(), back.to(dtype))
    dy = torch.randn(R, N, generator=g).to(dtype).cuda()
    for act, y in (("relu", torch.relu(x)), ("tanh", torch.tanh(x)), ("sigmoid", torch.sigmoid(x))):
        saved = _act_save(y, act)
        dz = _act_grad(dy, saved, act)
        if act == "relu":
            assert torch.equal(dz, torch.where(y > 0, dy, torch.zeros_like(dy)))
            continue
        # the product with 127 or 254 is one float32 rounding away: half-way cases may go either way, one step of t
        t = torch.from_numpy(saved.cpu().numpy().view(np.int8).astype(np.float64)) / 127
        y64 = y.cpu().double() if act == "tanh" else 2 * y.cpu().double() - 1
        assert float((t - y64).abs().max()) <= 0.5 / 127 + 1e-5
        want = dy.cpu().double() * (1 - t * t) * (1.0 if act == "tanh" else 0.25)
        _within(dz, want.numpy(), (16 * U * dy.cpu().double().abs() + HALF[dtype] * want.abs()).numpy() + TINY[dtype])
    inplace = dy.clone()
    from muzero_amd import _hip
    _hip.check(_hip.lib().mz_ckpt8_act_grad(inplace.data_ptr(), _hip.TYPE_F32 if dtype == torch.float32 else _hip.TYPE_BF16 if dtype == torch.bfloat16
                                            else _hip.TYPE_F16, N, saved.data_ptr(), R, N, _hip.ACT["sigmoid"], inplace.data_ptr(), N,
                                            torch.cuda.current_stream().cuda_stream), "mz_ckpt8_act_grad")
    assert torch.equal(inplace, dz)


@pytest.mark.parametrize("R,K,N", [(5, 100, 30), (40, 128, 200), (300, 130, 4200), (5000, 1000, 300)])
def test_codes_that_are_part_of_a_wider_matrix(R, K, N):
    """Rows of codes with a stride, the last one at the end of its memory: what lies between them is not theirs."""
    from muzero_amd.checkpoints import weight_grad
    from muzero_amd.quantized import QuantizedRows, int8_linear, quantize_rows
    x = _x(R, K, torch.float32)
    q = quantize_rows(x, scale_bits=3)
    width = q.codes.shape[1]
    big = torch.full((R, width + 256), 99, dtype=torch.int8, device="cuda")
    big[:, 256:] = q.codes
    part = QuantizedRows(big[:, 256:], q.scales, q.shape, q.dtype, 3)
    assert part.ld == width + 256
    assert torch.equal(part.dequantize(), q.dequantize())
    dz = torch.randn(R, N, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(weight_grad(dz, part), weight_grad(dz, q)))
    w = quantize_rows(torch.randn(N, K, device="cuda"))
    assert torch.equal(int8_linear(part, w), int8_linear(q, w))
    v = quantize_rows(torch.randn(7, K, device="cuda"))
    assert torch.equal(int8_linear(v, part), int8_linear(v, q))


def test_forward_mode_through_a_checkpointed_layer():
    """Without reverse mode the layer is torch's own operators, tangent and all; with it there is no forward-mode rule."""
    import torch.autograd.forward_ad as fwad

    from muzero_amd.checkpoints import checkpointed_linear
    lin = torch.nn.Linear(40, 24).cuda()
    x, t = torch.randn(5, 40, device="cuda"), torch.randn(5, 40, device="cuda")
    with fwad.dual_level():
        dual = fwad.make_dual(x, t)
        with pytest.raises(NotImplementedError):
            checkpointed_linear(dual, lin.weight, lin.bias, "tanh")
        with torch.no_grad():
            got = fwad.unpack_dual(checkpointed_linear(dual, lin.weight, lin.bias, "tanh")).tangent
            want = fwad.unpack_dual(torch.tanh(lin(dual))).tangent
    torch.testing.assert_close(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layers_under_autocast(dtype):
    """The forward pass of the layer under autocast; gradients of it and of a plain layer with the same weights beside it."""
    from muzero_amd.checkpoints import eight_bit_checkpoints
    _, _, f = _networks(8)
    lat = torch.randn(32, 4, 6, 7, device="cuda")
    params = list(f.policy_mlp.parameters())
    with torch.autocast("cuda", dtype):
        with eight_bit_checkpoints(f):
            policy, _ = f(lat)
        logits = f.policy_logits(lat)          # the same layers outside a context
    plain = torch.autograd.grad(logits.float().square().sum(), params)
    assert all(bool((g != 0).any()) for g in plain)
    with torch.autocast("cuda", dtype):
        want_policy, _ = f(lat)
    assert torch.equal(policy, want_policy)
    w = torch.randn(32, 7, device="cuda")
    want = torch.autograd.grad((want_policy * w).sum(), params)
    got = torch.autograd.grad((policy * w).sum(), params)
    assert all(g.dtype == torch.float32 and bool(g.isfinite().all()) and bool((g != 0).any()) for g in got)
    # the last bias: column sums of the same 16-bit dz, 32 terms in float32, rounded once to the type on each side
    assert float((want[-1] - got[-1]).abs().max()) <= 2 * HALF[dtype] * float(want[-1].abs().max()) + 64 * U * float(w.abs().sum())


def test_values_whose_sign_is_not_in_memory():
    from muzero_amd.policy_scores import policy_scores
    from muzero_amd.quantized import int8_linear, quantize_rows
    w, x, bias = quantize_rows(torch.randn(24, 40, device="cuda")), torch.randn(3, 40, device="cuda"), torch.randn(24, device="cuda")
    assert torch.equal(int8_linear(x, w, torch._neg_view(bias)), int8_linear(x, w, -bias))
    assert torch.equal(int8_linear(torch._neg_view(x), w), int8_linear(-x, w))
    z = torch.randn(1, 7, device="cuda", requires_grad=True)
    a = torch.tensor([-2], device="cuda")
    assert torch.equal(policy_scores(z, torch._neg_view(a)).log_prob, policy_scores(z, -a).log_prob)
    s = policy_scores(z, -a)
    turned = torch.complex(torch.zeros_like(s.log_prob), s.log_prob).conj() * 1j   # its real part is log_prob
    got, = torch.autograd.grad(turned.real.sum(), z)
    want, = torch.autograd.grad(policy_scores(z, -a).log_prob.sum(), z)
    assert torch.equal(got, want)


# beyond the one-launch kernel: column factors from the block itself, from up to 16 chunks of rows, from a kernel of their own
PLANES = [(90, 3000, 1500), (530, 2100, 2048), (5000, 9000, 30), (4100, 1030, 300)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K,N", PLANES)
def test_column_factors_of_any_size(R, K, N, dtype):
    """Columns of dz from the smallest to the largest a type holds, each with a power of two of its own; zeros, subnormal
    ones, a wide range inside one; an infinity or a NaN stays in its column, a NaN scale is everybody's."""
    from muzero_amd.checkpoints import save_activations, weight_grad
    from muzero_amd.quantized import QuantizedRows
    x = _x(R, K, dtype, seed=R).nan_to_num(posinf=6e4, neginf=-6e4)
    g = torch.Generator().manual_seed(N)
    span = torch.logspace(-6, 3, N) if dtype == torch.float16 else torch.logspace(-33, 30, N)
    dz = torch.randn(R, N, generator=g).clamp(-4, 4) * span[None, :]
    dz[:, 5] = 0.0
    dz[:, 6] = 1e-42 if dtype == torch.float32 else torch.finfo(dtype).tiny / 8
    dz[:, 7] *= torch.logspace(0, -8, R)
    dz = dz.to(dtype).cuda()
    want, tol, want_b, tol_b = _grad_reference(dz, x)
    saved = save_activations(x)
    dw, db = weight_grad(dz, saved)
    _within(dw, want, tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype] + 1e-40)
    _within(db, want_b, tol_b + HALF[dtype] * (np.abs(want_b) + tol_b) + TINY[dtype] + 1e-40)
    assert (dw[5] == 0).all() and (db[5] == 0).all()
    dz[3, 8], dz[R - 1, 9] = torch.inf, torch.nan
    dw2, db2 = weight_grad(dz, saved)
    assert dw2[8].isnan().all() and dw2[9].isnan().all() and db2[8].isinf() and db2[9].isnan()
    keep = [n for n in range(N) if n not in (8, 9)]
    assert torch.equal(dw2[keep], dw[keep]) and torch.equal(db2[keep], db[keep])
    scales = saved.scales.clone()
    scales[R // 2] = torch.nan
    dw3, db3 = weight_grad(dz, QuantizedRows(saved.codes, scales, saved.shape, saved.dtype, 3))
    assert dw3.isnan().all() and torch.equal(db3[keep], db[keep])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K,N", PLANES[:1] + PLANES[-1:])
def test_full_scales_and_strided_gradients_of_large_layers(R, K, N, dtype):
    from muzero_amd.checkpoints import weight_grad
    from muzero_amd.quantized import quantize_rows
    x = _x(R, K, dtype, seed=K).nan_to_num(posinf=6e4, neginf=-6e4)
    wide = (torch.randn(R, 2 * N + 1, generator=torch.Generator().manual_seed(R)) * 0.01).to(dtype).cuda()
    saved = quantize_rows(x)
    for dz in (wide[:, :N], wide[:, 1:N + 1], wide[:, : 2 * N : 2], wide[:, :N].t().contiguous().t()):
        dw, db = weight_grad(dz, saved)
        again = weight_grad(dz.contiguous().clone(), saved)
        assert torch.equal(dw, again[0]) and torch.equal(db, again[1])
    want, tol, _, _ = _grad_reference(wide[:, :N], x, bits=24)
    _within(weight_grad(wide[:, :N], saved)[0], want, tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype])


@pytest.mark.parametrize("R,K,N,act,dtype", [
    (253, 18432, 6661, "relu", torch.float32), (253, 18432, 6661, "sigmoid", torch.bfloat16),      # 256 x 256 tiles, nine parts
    (70, 131072, 8190, "none", torch.float16),                                                      # the longest sums, in parts
    (5201, 130, 5301, "tanh", torch.float32), (7301, 100, 7303, "relu", torch.bfloat16),            # results of 100 MB and more
    (7301, 100, 7304, "none", torch.float16), (64, 300, 450001, "none", torch.float32)])
def test_int8_linear_of_large_layers(R, K, N, act, dtype):
    """Against float64 products of the codes themselves, which are exact."""
    from muzero_amd.quantized import int8_linear, quantize_rows
    g = torch.Generator(device="cuda").manual_seed(R)
    x = torch.randn(R, K, generator=g, device="cuda").to(dtype)
    w = quantize_rows(torch.randn(N, K, generator=g, device="cuda") / K ** 0.5)
    b = torch.randn(N, generator=g, device="cuda")
    y = int8_linear(x, w, b, act)
    q = quantize_rows(x)
    for lo in range(0, N, 4096):
        part = slice(lo, min(N, lo + 4096))
        lin = q.codes.double() @ w.codes[part].double().t().contiguous() * q.scales.double()[:, None] * w.scales[part].double()
        pre = lin + b[part].double()
        want = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "tanh": torch.tanh, "sigmoid": torch.sigmoid}[act](pre)
        tol = 4 * U * (lin.abs() + pre.abs()) + 8 * U * want.abs() + 1e-37
        tol = tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype]
        bad = ~((y[:, part].double() - want).abs() <= tol)
        assert not bad.any(), (lo, int(bad.sum()))


def test_replayed_graphs_with_workspaces():
    """A split product and a large weight gradient: two graphs, whose workspaces are theirs, and eager calls in between."""
    from muzero_amd.checkpoints import save_activations, weight_grad
    from muzero_amd.quantized import int8_linear, quantize_rows
    x, dz = torch.randn(4100, 1030, device="cuda"), torch.randn(4100, 300, device="cuda")
    long, qw = torch.randn(100, 4096, device="cuda"), quantize_rows(torch.randn(500, 4096, device="cuda"))

    def step():
        return (int8_linear(long, qw, activation="relu"),) + weight_grad(dz, save_activations(x))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for turn in range(3):
        x.normal_(), dz.normal_(), long.normal_()
        want = step()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out in outs for a, b in zip(want, out)), turn


def test_policy_report_scores_the_recorded_moves():
    from muzero_amd.learner import DataParallelLearner
    h, g, f = _networks(9)
    learner = DataParallelLearner(h, g, f, torch.optim.SGD(f.parameters(), lr=0.1), 5)
    batch = _batch(64, seed=3)
    with torch.no_grad():
        policy = torch.cat([f(h(batch.history[i:i + 1]))[0] for i in range(64)]).double()   # one window at a time
    report = learner.policy_report(batch, top=2)
    at = torch.arange(64, device="cuda")
    # the network in float32, one window at a time or all together, differs by roundings of sums of at most 512 terms
    torch.testing.assert_close(report.log_prob.double(), policy[at, batch.actions[:, 0]].log(), rtol=0, atol=1e-3)
    torch.testing.assert_close(report.entropy.double(), -(policy * policy.log()).sum(1), rtol=0, atol=1e-3)
    torch.testing.assert_close(report.top_log_probs.double().exp(), policy.topk(2, dim=1).values, rtol=0, atol=1e-3)
    assert torch.equal(report.top_actions[:, 0], policy.argmax(1))


def test_skipped_rows_leave_row_0_to_whom_it_belongs():
    """next_rows of Int8Networks: any row may be written, row 0 too, beside rows that are skipped, or nothing at all."""
    from muzero_amd.engine import make_networks
    _, g, f = _networks(11)
    nets = make_networks(g, f, int8=True)
    B, D = 4096, 168
    lat, act = torch.randn(B, D, device="cuda"), torch.randint(0, 7, (B,), device="cuda", dtype=torch.int32)
    want = torch.empty(B, D, device="cuda")
    nets.dynamics(lat, B, action=act, next_latent=want)
    for keep in (torch.arange(B) % 3 == 0, torch.arange(B) == B - 1, torch.arange(B) < 0, torch.arange(B) >= 0):
        keep = keep.cuda()
        rows = torch.where(keep, torch.arange(B, device="cuda").flip(0) if bool(keep[-1]) else torch.arange(B, device="cuda"), -5).int()
        out = torch.full((B, D), 9.0, device="cuda")
        nets.dynamics(lat, B, action=act, next_latent=out, next_rows=rows)
        ref = torch.full((B, D), 9.0, device="cuda")
        ref[rows[keep].long()] = want[keep]
        assert torch.equal(out, ref)
    rows[0], rows[1] = B, 2 ** 31 - 1                  # behind the last row: skipped as well
    nets.dynamics(lat, B, action=act, next_latent=out, next_rows=rows)
    ref[:2] = out[:2]
    assert torch.equal(out, ref)
    wide = torch.full((B, D + 3), 9.0, device="cuda")
    nets.dynamics(lat, B, action=act, next_latent=wide[:, :D], next_rows=torch.arange(B, device="cuda"))
    assert torch.equal(wide[:, :D], want) and (wide[:, D:] == 9.0).all()
    for bad in (dict(next_latent=out, next_rows=rows[1:]), dict(next_latent=out, next_rows=rows.cpu()),
                dict(next_latent=out.half(), next_rows=rows)):
        with pytest.raises(ValueError):
            nets.dynamics(lat, B, action=act, **bad)


def test_rows_that_32_bits_do_not_hold_are_none():
    from muzero_amd.engine import make_networks
    _, g, f = _networks(12)
    nets = make_networks(g, f, int8=True)
    lat, act = torch.randn(6, 168, device="cuda"), torch.arange(6, device="cuda", dtype=torch.int32)
    want, out = torch.empty(6, 168, device="cuda"), torch.full((6, 168), 9.0, device="cuda")
    nets.dynamics(lat, 6, action=act, next_latent=want)
    rows = torch.tensor([3, (1 << 32) + 5, -(1 << 32) + 4, 6, 1, 2 ** 31], device="cuda")
    nets.dynamics(lat, 6, action=act, next_latent=out, next_rows=rows)
    assert torch.equal(out[3], want[0]) and torch.equal(out[1], want[4]) and (out[[0, 2, 4, 5]] == 9.0).all()
