"""The 4-bit Dense layer with group scales against 64-bit sums of its definition, and its quantiser
against the rounding rule in numpy."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FP4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0])


@pytest.fixture(scope="module")
def D(wb):
    import welvet.cuda_b200.decode as decode
    return decode


def make(rng, rows, cols, group, code, scale_dtype="f16"):
    import torch
    groups = -(-cols // group)
    c = rng.integers(0, 16, (rows, 2 * ((cols + 1) // 2)), dtype=np.uint8)
    codes = (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)
    s = torch.from_numpy(rng.uniform(0.002, 0.02, (rows, groups)).astype(np.float32)).to(
        torch.float16 if scale_dtype == "f16" else torch.bfloat16)
    zeros = rng.integers(0, 16, (rows, groups), dtype=np.uint8) if code == "uint4" else None
    c = c[:, :cols].astype(np.int64)
    which = np.arange(cols) // group
    if code == "fp4":
        w = FP4[c]
    elif code == "int4":
        w = np.where(c > 7, c - 16, c).astype(np.float64)
    else:
        w = c - zeros[:, which].astype(np.float64)
    return codes, s, zeros, w * s.double().numpy()[:, which]


def mount(D, codes, s, zeros, cols, group, code, **kw):
    import torch
    z = None if zeros is None else torch.from_numpy(zeros).cuda()
    return D.GroupDense.from_codes(torch.from_numpy(codes).cuda(), s.cuda(), cols, group, D.CODES[code], zeros=z, **kw)


def check(y, x, W, what=""):
    """|y - y64| <= 2^-18 * sum |W x| + 2 ulp, the tensor GEMV's bound."""
    x = x.astype(np.float64)
    y64 = x @ W.T
    bound = 2.0 ** -18 * (np.abs(x) @ np.abs(W).T) + 2 * np.spacing(np.abs(y64).astype(np.float32)).astype(np.float64)
    err = np.abs(y.astype(np.float64) - y64)
    assert np.all(err <= bound), (what, float(np.max(err - bound)))


SHAPES = [(1, 1), (1, 33), (16, 64), (17, 31), (64, 96), (100, 130), (257, 1000), (1024, 4096), (40, 16385), (4099, 515),
          (8192, 64), (300, 2048)]


@pytest.mark.parametrize("code", ["int4", "uint4", "fp4"])
@pytest.mark.parametrize("group", [32, 64, 128, 192, 4096])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_forward(D, code, group, shape):
    import torch
    rows, cols = SHAPES[shape]
    rng = np.random.default_rng(shape * 10 + group)
    codes, s, zeros, W = make(rng, rows, cols, group, code, "f16" if shape % 2 else "bf16")
    g = mount(D, codes, s, zeros, cols, group, code)
    for n in (1, 2, 3, 4, 5, 8) if shape < 6 else (1, 1 + shape % 8):
        x = rng.standard_normal((n, cols)).astype(np.float32)
        y = torch.full((n, rows), float("nan"), device="cuda")
        g.forward(torch.from_numpy(x).cuda(), y)
        check(y.cpu().numpy(), x, W, (rows, cols, n))


@pytest.mark.parametrize("n", [9, 16, 17, 40])
def test_more_rows(D, n):
    import torch
    rng = np.random.default_rng(n)
    codes, s, zeros, W = make(rng, 130, 700, 64, "uint4")
    g = mount(D, codes, s, zeros, 700, 64, "uint4")
    x = rng.standard_normal((n, 700)).astype(np.float32)
    y = torch.empty((n, 130), device="cuda")
    g.forward(torch.from_numpy(x).cuda(), y)
    check(y.cpu().numpy(), x, W)


@pytest.mark.parametrize("act", ["linear", "relu", "silu", "gelu", "tanh", "sigmoid", "leaky_relu", "relu2"])
@pytest.mark.parametrize("bias_len", [0, 7, 100])
def test_bias_and_activation(D, oracle, act, bias_len):
    """The Dense layer's epilogue: bias for rows o < bias_len, activation in 64 bits, both rounded."""
    import torch
    rng = np.random.default_rng(bias_len)
    codes, s, zeros, W = make(rng, 100, 256, 32, "fp4")
    bias = rng.standard_normal(bias_len) if bias_len else None
    g = mount(D, codes, s, zeros, 256, 32, "fp4", act=D.ACTS[act], bias=bias)
    x = rng.standard_normal((3, 256)).astype(np.float32)
    pre, y = torch.empty((3, 100), device="cuda"), torch.empty((3, 100), device="cuda")
    g.forward(torch.from_numpy(x).cuda(), y, pre)
    full = np.zeros(100)
    full[: bias_len] = 0 if bias is None else bias
    y64 = x.astype(np.float64) @ W.T + full
    got = pre.cpu().numpy().astype(np.float64)
    bound = 2.0 ** -18 * (np.abs(x) @ np.abs(W).T) + 4 * np.spacing(np.abs(y64).astype(np.float32))
    assert np.all(np.abs(got - y64) <= bound)
    f = {"linear": lambda v: v, "relu": lambda v: np.maximum(v, 0), "silu": lambda v: v / (1 + np.exp(-v)),
         "gelu": lambda v: 0.5 * v * (1 + np.tanh(0.7978845608028654 * (v + 0.044715 * v ** 3))), "tanh": np.tanh,
         "sigmoid": lambda v: 1 / (1 + np.exp(-v)), "leaky_relu": lambda v: np.where(v < 0, 0.01 * v, v),
         "relu2": lambda v: np.where(v < 0, 0, v * v)}[act]
    # post is the activation of the unrounded pre: the derivative carries its rounding (2 |v| + 1 bounds all)
    np.testing.assert_allclose(y.cpu().numpy(), f(got), rtol=4e-7, atol=1e-7 * (1 + 2 * np.abs(got).max()) * np.abs(got).max())


def test_strided_rows_streams_graph(D):
    import torch
    rng = np.random.default_rng(12)
    codes, s, zeros, W = make(rng, 512, 1030, 128, "int4")
    g = mount(D, codes, s, zeros, 1030, 128, "int4")
    wide = rng.standard_normal((4, 3001)).astype(np.float32)
    gw = torch.from_numpy(wide).cuda()
    for at in (0, 1, 1971):  # rows that start off 16-byte boundaries
        y = torch.empty((4, 512), device="cuda")
        g.forward(gw[:, at: at + 1030], y)
        check(y.cpu().numpy(), wide[:, at: at + 1030], W)
    x = torch.from_numpy(np.ascontiguousarray(wide[:, :1030])).cuda()
    y = torch.empty((4, 512), device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g.forward(x, y)
    side.synchronize()
    check(y.cpu().numpy(), wide[:, :1030], W)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.forward(x, y)
    new = rng.standard_normal((4, 1030)).astype(np.float32)
    x.copy_(torch.from_numpy(new))
    graph.replay()
    check(y.cpu().numpy(), new, W)


def test_chain_reads_what_the_layer_before_wrote(D):
    """Three layers back to back, many times: each reads the output of the one before it."""
    import torch
    rng = np.random.default_rng(13)
    parts = [make(rng, 768, 768, 64, c) for c in ("int4", "uint4", "fp4")]
    layers = [mount(D, *p[:3], 768, 64, c) for p, c in zip(parts, ("int4", "uint4", "fp4"))]
    x = torch.from_numpy(rng.standard_normal((2, 768)).astype(np.float32)).cuda()
    first = None
    for _ in range(50):
        bufs = [torch.empty((2, 768), device="cuda") for _ in range(3)]
        src = x
        for g, dst in zip(layers, bufs):
            g.forward(src, dst)
            src = dst
        torch.cuda.synchronize()
        got = [b.cpu().numpy() for b in bufs]
        if first is None:
            first = got
            src = x.cpu().numpy()
            for b, p in zip(got, parts):
                check(b, src, p[3])
                src = b
        for a, b in zip(first, got):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e6, 1e30])
def test_range_of_x(D, scale):
    """Tokens of very different magnitude share a call; large and small values share a token."""
    import torch
    rng = np.random.default_rng(14)
    codes, s, zeros, W = make(rng, 200, 2000, 64, "fp4")
    g = mount(D, codes, s, zeros, 2000, 64, "fp4")
    x = rng.standard_normal((3, 2000)).astype(np.float32)
    x[0] *= np.float32(scale)
    x[1, ::7] *= np.float32(1e-4)
    x[2] = 0
    y = torch.empty((3, 200), device="cuda")
    g.forward(torch.from_numpy(x).cuda(), y)
    check(y.cpu().numpy(), x, W)
    assert not y[2].any()


@pytest.mark.parametrize("code", ["int4", "uint4", "fp4"])
def test_non_finite_x_stays_in_its_token(D, code):
    import torch
    rng = np.random.default_rng(15)
    codes, s, zeros, W = make(rng, 200, 500, 64, code)
    g = mount(D, codes, s, zeros, 500, 64, code)
    x = rng.standard_normal((4, 500)).astype(np.float32)
    x[1, 77], x[2, 3] = np.nan, np.inf
    y = torch.empty((4, 200), device="cuda")
    g.forward(torch.from_numpy(x).cuda(), y)
    got = y.cpu().numpy()
    check(got[[0, 3]], x[[0, 3]], W)
    assert np.all(np.isnan(got[1])) and not np.any(np.isfinite(got[2]) & (W[:, 3] != 0))


def test_host_arrays(D, wb):
    """The C entry with host pointers gives the device mount's bits."""
    import ctypes

    import torch
    rng = np.random.default_rng(16)
    codes, s, zeros, W = make(rng, 70, 300, 32, "uint4")
    a = mount(D, codes, s, zeros, 300, 32, "uint4")
    h = ctypes.c_void_p()
    sb = s.view(torch.int16).numpy()
    wb.check(wb.lib().welvet_b200_gdense_mount(300, 70, 32, 15, 2, -1, codes.ctypes.data, sb.ctypes.data, zeros.ctypes.data, 0,
                                               None, 0, ctypes.byref(h)))
    b = D.GroupDense(h, 300, 70)
    x = torch.randn((2, 300), device="cuda")
    ya, yb = torch.empty((2, 70), device="cuda"), torch.empty((2, 70), device="cuda")
    a.forward(x, ya)
    b.forward(x, yb)
    assert torch.equal(ya, yb)


@pytest.mark.parametrize("code", ["int4", "uint4", "fp4"])
@pytest.mark.parametrize("scale_dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,cols,group", [(5, 64, 32), (33, 130, 64), (64, 1001, 128), (3, 31, 64)])
def test_quantize(D, code, scale_dtype, rows, cols, group):
    import torch
    rng = np.random.default_rng(cols)
    dt = torch.float16 if scale_dtype == "f16" else torch.bfloat16
    W = (rng.standard_normal((rows, cols)) * 0.05).astype(np.float32)
    W[0, : min(cols, group)] = 0
    codes, s, zeros = D.group_quantize(torch.from_numpy(W).cuda(), group, D.CODES[code], dt)
    c = codes.cpu().numpy()
    c = np.stack([c & 15, c >> 4], -1).reshape(rows, -1)
    assert not c[:, cols:].any()
    got = s.float().cpu().numpy()
    for g in range(-(-cols // group)):
        w = W[:, g * group: (g + 1) * group]
        q = c[:, g * group: min(cols, (g + 1) * group)].astype(np.int64)
        lo, hi = np.minimum(w.min(1), 0), np.maximum(w.max(1), 0)
        amax = np.maximum(-lo, hi)
        want = amax / np.float32(6) if code == "fp4" else amax / np.float32(7) if code == "int4" else (hi - lo) / np.float32(15)
        want = torch.from_numpy(want).to(dt).float().numpy()
        np.testing.assert_array_equal(got[:, g], want)
        step = np.where(want > 0, want, 1)[:, None].astype(np.float32)
        v = np.where(want[:, None] > 0, w / step, 0).astype(np.float32)
        if code == "int4":
            expect = np.clip(np.rint(v), -8, 7).astype(np.int64) & 15
        elif code == "uint4":
            z = np.where(want > 0, np.clip(np.rint(-lo / step[:, 0]), 0, 15), 0).astype(np.float32)
            np.testing.assert_array_equal(zeros.cpu().numpy()[:, g], z.astype(np.uint8))
            expect = np.clip(np.rint(v) + z[:, None], 0, 15).astype(np.int64)
        else:
            expect = np.argmin(np.abs(np.clip(v, -6, 6)[..., None] - FP4.astype(np.float32)), -1)  # ties: the lower code
        np.testing.assert_array_equal(q, expect)


@pytest.mark.parametrize("code", ["int4", "uint4", "fp4"])
def test_quantized_layer_is_near_the_layer(D, code):
    """W ~ N(0, 0.02), which one scale per tensor in FP4 turns into zeros: the relative error of y is the
    step's, about a tenth."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(0)
    W = torch.randn((1024, 2048), generator=g, device="cuda") * 0.02
    x = torch.randn((2, 2048), generator=g, device="cuda")
    y = torch.empty((2, 1024), device="cuda")
    D.GroupDense.quantize(W, 64, D.CODES[code]).forward(x, y)
    want = x.double() @ W.double().T
    assert float((y - want).norm() / want.norm()) < 0.15


def test_refusals(D, wb):
    import torch
    codes, s = torch.zeros((4, 32), dtype=torch.uint8, device="cuda"), torch.zeros((4, 1), dtype=torch.float16, device="cuda")
    z = torch.zeros((4, 1), dtype=torch.uint8, device="cuda")
    for kw, code in ((dict(code=D.UINT4), 1), (dict(code=D.INT4, zeros=z), 1), (dict(code=9), 2), (dict(code=D.FP4, act=9), 1)):
        with pytest.raises(wb.WelvetError) as e:
            c = kw.pop("code")
            D.GroupDense.from_codes(codes, s, 64, 64, c, **kw)
        assert e.value.code == code
    for group in (48, 16, 0, -64):
        with pytest.raises((wb.WelvetError, ValueError)):
            D.GroupDense.from_codes(codes, s, 64, group, D.FP4)
    for args in ((codes[:, :31], s), (codes.int(), s), (codes.cpu(), s), (codes, s.float()), (codes, s[:3])):
        with pytest.raises(ValueError):
            D.GroupDense.from_codes(*args, 64, 64, D.FP4)
    g = D.GroupDense.from_codes(codes, s, 64, 64, D.FP4)
    x, y = torch.zeros((2, 64), device="cuda"), torch.zeros((2, 4), device="cuda")
    for a in ((x[:, :32], y), (x.half(), y), (x, y[:1]), (x, y.t()), (x.cpu(), y)):
        with pytest.raises(ValueError):
            g.forward(*a)
    g.forward(x[:0], y[:0])  # no rows: nothing to do


@pytest.mark.parametrize("scale_dtype", ["f16", "bf16"])
@pytest.mark.parametrize("code", ["int4", "uint4", "fp4"])
def test_quantize_does_not_hide_what_is_not_finite(D, code, scale_dtype):
    """A group with an infinity or NaN gets a NaN scale, and its row's result is NaN; no other changes."""
    import torch
    rng = np.random.default_rng(61)
    W = torch.from_numpy(rng.standard_normal((20, 200)).astype(np.float32)).cuda()
    dt = torch.float16 if scale_dtype == "f16" else torch.bfloat16
    want = D.group_quantize(W, 64, D.CODES[code], dt)
    W[3, 70], W[7, 199], W[11, 0] = float("nan"), float("inf"), float("-inf")
    got = D.group_quantize(W, 64, D.CODES[code], dt)
    bad = torch.zeros((20, 4), dtype=torch.bool, device="cuda")
    bad[3, 1] = bad[7, 3] = bad[11, 0] = True
    assert torch.equal(torch.isnan(got[1]), bad)
    assert torch.equal(got[1][~bad], want[1][~bad])
    layer = D.GroupDense.from_codes(got[0], got[1], 200, 64, D.CODES[code], zeros=got[2])
    y = torch.empty((1, 20), device="cuda")
    layer.forward(torch.ones((1, 200), device="cuda"), y)
    assert torch.equal(torch.isnan(y[0]), bad.any(1))


@pytest.mark.parametrize("code", ["int4", "uint4", "fp4"])
@pytest.mark.parametrize("n", [1, 8])
@pytest.mark.parametrize("scale,size", [(1e31, 1e-12), (1e36, 1e-30), (2e38, 1e-35), (1e-35, 1e25), (1e-38, 1e37), (1e-30, 1e-3)])
def test_scales_at_the_ends_of_their_range(D, code, n, scale, size):
    """BFloat16 scales near the largest and smallest floats, with x that makes the results ordinary numbers."""
    import torch
    rng = np.random.default_rng(17)
    rows, cols, group = 100, 700, 64
    codes, _, zeros, W = make(rng, rows, cols, group, code, "bf16")
    s = torch.from_numpy((rng.uniform(0.5, 1.0, (rows, 11)) * scale).astype(np.float32)).to(torch.bfloat16)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)[:, :cols].astype(np.int64)
    which = np.arange(cols) // group
    v = FP4[c] if code == "fp4" else np.where(c > 7, c - 16, c) if code == "int4" else c - zeros[:, which].astype(np.float64)
    W = v * s.double().numpy()[:, which]
    g = mount(D, codes, s, zeros, cols, group, code)
    x = (rng.standard_normal((n, cols)) * size).astype(np.float32)
    y = torch.full((n, rows), float("nan"), device="cuda")
    g.forward(torch.from_numpy(x).cuda(), y)
    check(y.cpu().numpy(), x, W, (scale, size))


def big_layer(D, rows, cols, group, code, scale_dtype, seed):
    """(layer, W's rows of a block in 64 bits on the GPU) of random codes, made on the GPU."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    half, groups = (cols + 1) // 2, -(-cols // group)
    codes = torch.randint(0, 256, (rows, half), dtype=torch.uint8, device="cuda", generator=g)
    if cols % 2:
        codes[:, -1] &= 15
    s = (torch.rand((rows, groups), device="cuda", generator=g) * 0.018 + 0.002).to(scale_dtype)
    z = torch.randint(0, 16, (rows, groups), dtype=torch.uint8, device="cuda", generator=g) if code == "uint4" else None
    layer = D.GroupDense.from_codes(codes, s, cols, group, D.CODES[code], zeros=z)
    which = torch.arange(cols, device="cuda") // group
    values = torch.tensor(FP4 if code == "fp4" else [i - 16 * (i > 7) for i in range(16)] if code == "int4" else list(range(16)),
                          dtype=torch.float64, device="cuda")

    def block(at, n):
        c = torch.stack([codes[at: at + n] & 15, codes[at: at + n] >> 4], -1).reshape(-1, 2 * half)[:, :cols].long()
        w = values[c]
        if z is not None:
            w = w - z[at: at + n].double()[:, which]
        return w * s[at: at + n].double()[:, which]

    return layer, block


# rows, cols, x's rows, and the form of the launch that the shape is here for
FORMS = [
    (256, 4609, 8, dict(slabs=2, solo=0, whole=1)),           # slabs of 10 and 9 chunks, the last of one input
    (40, 40001, 3, dict(slabs=4, solo=0, whole=0, cut=12)),   # slabs, and blocks' runs that cut row groups
    (40, 40001, 1, dict(slabs=2, solo=0, whole=0, cut=6)),
    (40, 30000, 1, dict(slabs=1, solo=0, whole=1)),
    (2400, 32768, 1, dict(slabs=1, solo=0, whole=0, cut=146)),
    (250, 17400, 8, dict(slabs=4, solo=0, whole=1)),
    (38100, 600, 1, dict(slabs=1, solo=1, cut=1578)),         # warps' runs that cut row groups
    (38100, 600, 5, dict(slabs=1, solo=1, cut=1578)),
    (38100, 600, 8, dict(slabs=1, solo=1, cut=1578)),
    (19020, 4609, 8, dict(slabs=2, solo=1, cut=2117)),        # the same in slabs
    (4096, 14336, 8, dict(slabs=4, solo=0, whole=1)),
    (3000, 50000, 7, dict(slabs=11, solo=0)),
]


@pytest.mark.parametrize("code,group,scale", [("int4", 128, "f16"), ("uint4", 64, "bf16"), ("fp4", 32, "f16")])
@pytest.mark.parametrize("rows,cols,n,form", FORMS)
def test_forms_of_the_launch(D, rows, cols, n, form, code, group, scale):
    """Slabs of the inputs, runs of the warps and of the blocks, and row groups that runs cut: against 64
    bits, and the same bits in calls that follow one another with other numbers of rows between them
    (tickets and partial sums are the handle's)."""
    import torch
    plan = D.gdense_plan(cols, rows, group, D.CODES[code], n, torch.cuda.get_device_properties(0).multi_processor_count)
    assert {k: plan[k] for k in form} == form
    layer, block = big_layer(D, rows, cols, group, code, torch.float16 if scale == "f16" else torch.bfloat16, rows + n)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((17, cols), device="cuda", generator=g)
    out = {m: torch.full((m, rows), float("nan"), device="cuda") for m in {n, 1, 4, 17}}
    layer.forward(x[:n], out[n])
    first = out[n].clone()
    for at in range(0, rows, 4096):
        W = block(at, min(4096, rows - at))
        want = x[:n].double() @ W.T
        bound = 2.0 ** -18 * (x[:n].double().abs() @ W.abs().T) + 2.0 ** -22 * want.abs()
        assert bool(((first[:, at: at + 4096] - want).abs() <= bound).all())
    for m in (1, n, 17, n, 4, n, n):
        out[m].fill_(float("nan"))
        layer.forward(x[:m], out[m])
        if m == n:
            assert torch.equal(out[n], first)
        if m == 17 and n == 8:  # passes of eight
            assert torch.equal(out[17][:8], first)
    again = out[17].clone()
    layer.forward(x, out[17])
    assert torch.equal(again, out[17]) and bool(torch.isfinite(again).all())
