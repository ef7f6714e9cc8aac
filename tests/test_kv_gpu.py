"""The paged key-value cache (append, decode attention, eviction) against 64-bit statements of its
definitions, at the sizes, layouts and masks where such code goes wrong."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = ("f32", "f16", "bf16", "f8")
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def D(wb):
    import welvet.cuda_b200.decode as decode
    return decode


def types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}


def make_cache(rng, dtype, n, per, page, kv, dim, layout="slots", fill="randn", spare=3):
    """Pools (filled with NaN where `fill` is nan), a table whose pages lie in random order."""
    import torch
    pages = n * per + spare
    shape = (pages, page, kv, dim) if layout == "slots" else (pages, kv, page, dim)
    pools = []
    for _ in range(2):
        x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()
        if fill == "nan":
            x.fill_(float("nan"))
        x = x.to(types()[dtype])
        pools.append(x if layout == "slots" else x.transpose(1, 2))
    table = torch.from_numpy(rng.permutation(pages)[: n * per].reshape(n, per).astype(np.int32)).cuda()
    return pools[0], pools[1], table


def i32(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def rows_of(pool, table, b, n, h):
    """float64 [n, dim] of a sequence's first n slots of one key-value head."""
    page = pool.shape[1]
    j = np.arange(n)
    t = table.cpu().numpy()[b]
    x = pool.float().cpu().numpy()
    return x[t[j // page], j % page, h].astype(np.float64)


def attend64(q, kp, vp, table, lens, scale, window=0, alibi=False, positions=None, seen=None, ks=1.0, vs=1.0):
    """(out, weights per query head, bound on the error of out) in 64 bits. The bound: a score's fp32
    sum of dim products and the roundings of its scale move it by dz, a weight by the factor 2 dz
    (its own and the normaliser's), and the running sums of n weights add their roundings."""
    n, H, dim = q.shape
    kv = kp.shape[2]
    q = q.double().cpu().numpy()
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    ws = [np.zeros((H, max(0, int(x)))) for x in lens]
    for b in range(n):
        L = int(lens[b])
        for h in range(H):
            g = h // (H // kv)
            k, v = rows_of(kp, table, b, L, g) * ks, rows_of(vp, table, b, L, g) * vs
            pos = np.arange(L) if positions is None else positions[b, g, :L]
            last = L - 1 if positions is None else seen[b] - 1
            ok = np.ones(L, bool) if not window else pos > last - window
            if not ok.any():
                continue
            k, v, pos = k[ok], v[ok], pos[ok]
            z = (k @ q[b, h]) * scale
            if alibi:
                z = z - 2.0 ** (-8.0 * (h + 1) / H) * (last - pos)
            w = np.exp(z - z.max())
            w /= w.sum()
            out[b, h] = w @ v
            ws[b][h, ok] = w
            dz = np.max((dim + 8) * EPS * scale * (np.abs(k) @ np.abs(q[b, h])) + 4 * EPS * (np.abs(z) * 1.5 + np.abs(z.max())))
            bound[b, h] = (2 * dz + (16 + len(z) / 8) * EPS) * (w @ np.abs(v)) + EPS * np.abs(out[b, h])
    return out, ws, bound


CASES = [
    # heads, kv, dim, page, lens
    (1, 1, 64, 16, [1]),
    (4, 4, 128, 16, [0, 1, 15, 16, 17]),
    (8, 2, 128, 16, [200, 0, 333, 64]),
    (6, 2, 64, 32, [5, 700, 31, 32, 33]),
    (5, 1, 80, 24, [95, 257, 1]),
    (12, 4, 96, 7, [50, 7, 8, 129]),
    (16, 1, 256, 64, [1025, 3]),
    (24, 1, 128, 16, [300, 40]),
    (2, 2, 40, 16, [77]),
    (3, 3, 33, 5, [61, 5, 4]),
    (2, 1, 8, 1, [9, 130]),
    (2, 1, 4, 16, [33]),
    (32, 8, 128, 16, [2049, 511, 4100]),
]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attend(D, dtype, case):
    import torch
    H, kv, dim, page, lens = CASES[case]
    rng = np.random.default_rng(100 * case + DT.index(dtype))
    n, per = len(lens), max(1, -(-max(lens) // page)) + 1
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim, layout="slots" if case % 2 else "heads")
    ks, vs = (0.5, 2.0) if dtype == "f8" else (1.0, 1.0)
    q = torch.from_numpy((rng.standard_normal((n, H, dim)) * 1.5).astype(np.float32)).cuda()
    out = torch.full((n, H, dim), float("nan"), device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H, k_scale=ks, v_scale=vs)
    c.attend(q, out)
    c.check_error()
    want, _, bound = attend64(q, kp, vp, table, lens, 1.0 / math.sqrt(dim), ks=ks, vs=vs)
    err = np.abs(out.cpu().numpy() - want)
    assert np.all(err <= bound), float(np.max(err - bound))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("window,alibi", [(1, False), (16, False), (100, True), (10 ** 6, True)])
def test_attend_window_alibi(D, dtype, window, alibi):
    """Keys outside the window hold NaN and infinity, so does every slot past the length."""
    import torch
    rng = np.random.default_rng(window + DT.index(dtype))
    H, kv, dim, page, lens = 6, 2, 64, 16, [1, 40, 16, 177, 0, 1000]
    n, per = len(lens), 70
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim)
    t = table.cpu().numpy()
    bad = float("nan") if dtype == "f8" else None
    for b, L in enumerate(lens):
        for j in list(range(0, max(0, L - window))) + list(range(L, per * page)):
            value = bad if bad is not None else (float("nan"), float("inf"), -float("inf"))[j % 3]
            if j < 200 or j >= L:
                kp.view(torch.uint8 if dtype == "f8" else kp.dtype)[int(t[b, j // page]), j % page] = 0x7f if dtype == "f8" else value
                vp.view(torch.uint8 if dtype == "f8" else vp.dtype)[int(t[b, j // page]), j % page] = 0x7f if dtype == "f8" else value
    q = torch.from_numpy(rng.standard_normal((n, H, dim)).astype(np.float32)).cuda()
    out = torch.empty((n, H, dim), device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H)
    c.attend(q, out, scale=0.3, window=window, alibi=alibi)
    c.check_error()
    scale = float(np.float32(0.3))
    want, _, bound = attend64(q, kp, vp, table, lens, scale, window, alibi)
    err = np.abs(out.cpu().numpy() - want)
    assert np.all(err <= bound), float(np.max(err - bound))


@pytest.mark.parametrize("dtype", DT)
def test_attend_accumulates_weights(D, dtype):
    import torch
    rng = np.random.default_rng(7 + DT.index(dtype))
    H, kv, dim, page, lens = 12, 4, 64, 16, [1, 40, 0, 177, 1500]
    n, per = len(lens), 100
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim)
    q = torch.from_numpy(rng.standard_normal((n, H, dim)).astype(np.float32)).cuda()
    out = torch.empty((n, H, dim), device="cuda")
    w0 = torch.rand((n, kv, per * page), device="cuda")
    w = torch.full_like(w0, -7.0)
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H, weights=w)
    c.attend(q, out, accumulate=True, weights_in=w0)
    want, ws, bound = attend64(q, kp, vp, table, lens, 1.0 / math.sqrt(dim))
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)
    got, old = w.cpu().numpy(), w0.cpu().numpy()
    for b, L in enumerate(lens):
        assert np.all(got[b, :, L:] == -7.0)
        sums = ws[b].reshape(kv, H // kv, L).sum(1)
        # a weight is off by its share of the bound above: at most dz ~ 2^-13 here, far above fp32's
        np.testing.assert_allclose(got[b, :, :L] - old[b, :, :L], sums, rtol=2e-4, atol=4 * EPS)
    # in place, and the sum over slots is the number of heads of a group
    w.copy_(w0)
    c.attend(q, out, accumulate=True)
    np.testing.assert_array_equal(w.cpu().numpy()[3, :, :177], got[3, :, :177])
    total = (w - w0).double().sum(-1).cpu().numpy()
    np.testing.assert_allclose(total[[0, 1, 3, 4]], H // kv, rtol=1e-4)


def test_attend_window_goes_by_positions(D):
    """Once slots were evicted a slot's index is not its position."""
    import torch
    rng = np.random.default_rng(3)
    H, kv, dim, page, n, per = 4, 2, 64, 16, 3, 6
    lens = [90, 33, 64]
    seen = [400, 33, 5000]
    kp, vp, table = make_cache(rng, "bf16", n, per, page, kv, dim)
    positions = np.zeros((n, kv, per * page), np.int32)
    for b in range(n):
        for h in range(kv):
            positions[b, h, : lens[b]] = rng.permutation(seen[b])[: lens[b]]
    q = torch.from_numpy(rng.standard_normal((n, H, dim)).astype(np.float32)).cuda()
    out = torch.empty((n, H, dim), device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H, seen=i32(seen), positions=i32(positions))
    for window, alibi in ((200, False), (50, True), (0, True), (1, False)):
        c.attend(q, out, window=window, alibi=alibi)
        want, _, bound = attend64(q, kp, vp, table, lens, 0.125, window, alibi, positions, seen)
        assert np.all(np.abs(out.cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("dtype", DT)
def test_attend_large_and_equal_scores(D, dtype):
    """Scores in the hundreds (a weight of one), and keys that are all the same (weights 1 / n)."""
    import torch
    rng = np.random.default_rng(11)
    H, kv, dim, page, lens = 4, 1, 64, 16, [500, 129]
    kp, vp, table = make_cache(rng, dtype, 2, 40, page, kv, dim)
    q = torch.from_numpy((rng.standard_normal((2, H, dim)) * 100).astype(np.float32)).cuda()
    out = torch.empty((2, H, dim), device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H)
    c.attend(q, out)
    want, _, bound = attend64(q, kp, vp, table, lens, 0.125)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)
    kp.zero_() if dtype != "f8" else kp.view(torch.uint8).zero_()
    c.attend(q, out)
    want, _, bound = attend64(q, kp, vp, table, lens, 0.125)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)


def test_attend_strided_rows_other_stream_and_graph(D):
    """q and out as parts of wider rows, a call on a side stream, and a captured call replayed after the
    cache has grown."""
    import torch
    rng = np.random.default_rng(5)
    H, kv, dim, page, n, per = 8, 2, 128, 16, 3, 20
    kp, vp, table = make_cache(rng, "bf16", n, per, page, kv, dim)
    lens = i32([10, 200, 33])
    wide = torch.from_numpy(rng.standard_normal((n, (H + 2 * kv) * dim)).astype(np.float32)).cuda()
    outw = torch.zeros((n, 2 * H * dim), device="cuda")
    c = D.PagedKV(kp, vp, table, lens, num_heads=H)
    q = wide[:, : H * dim]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.attend(q, outw[:, H * dim:])
    side.synchronize()
    for new in ([10, 200, 33], [11, 320, 0]):
        if new[0] == 11:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                c.attend(q, outw[:, H * dim:])
            lens.copy_(i32(new))
            g.replay()
            torch.cuda.synchronize()
        want, _, bound = attend64(q.reshape(n, H, dim), kp, vp, table, new, dim ** -0.5)
        got = outw[:, H * dim:].reshape(n, H, dim).cpu().numpy()
        assert np.all(np.abs(got - want) <= bound)
        assert not outw[:, : H * dim].any()


def test_attend_same_bits_each_time(D):
    import torch
    rng = np.random.default_rng(6)
    lens = list(rng.integers(1, 3000, 9))
    kp, vp, table = make_cache(rng, "bf16", 9, 200, 16, 2, 128)
    q = torch.from_numpy(rng.standard_normal((9, 16, 128)).astype(np.float32)).cuda()
    w = torch.zeros((9, 2, 3200), device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=16, weights=w)
    got = []
    for _ in range(5):
        out = torch.empty((9, 16, 128), device="cuda")
        w.zero_()
        c.attend(q, out, accumulate=True)
        got.append((out.cpu().numpy(), w.cpu().numpy().copy()))
    for o, x in got[1:]:
        np.testing.assert_array_equal(o, got[0][0])
        np.testing.assert_array_equal(x, got[0][1])


def test_attend_long_offsets(D):
    """A pool whose offsets pass 2^31 elements: the last pages are the ones in use."""
    import torch
    page, kv, dim = 64, 8, 128
    pages = (2 ** 31 + 2 ** 24) // (page * kv * dim)
    kp = torch.empty((pages, page, kv, dim), dtype=torch.float8_e4m3fn, device="cuda")
    vp = torch.empty_like(kp)
    rng = np.random.default_rng(8)
    used = [pages - 1, pages - 3, pages - 2, 0]
    for p in used:
        for t in (kp, vp):
            t[p] = torch.from_numpy(rng.standard_normal((page, kv, dim)).astype(np.float32)).cuda().to(torch.float8_e4m3fn)
    table = i32([used])
    q = torch.from_numpy(rng.standard_normal((1, 16, dim)).astype(np.float32)).cuda()
    out = torch.empty((1, 16, dim), device="cuda")
    D.PagedKV(kp, vp, table, i32([250]), num_heads=16).attend(q, out)
    small = [t[torch.tensor(used, device="cuda")] if False else torch.stack([t[p] for p in used]) for t in (kp, vp)]
    want, _, bound = attend64(q, small[0], small[1], i32([[0, 1, 2, 3]]), [250], dim ** -0.5)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)


# ---------------------------------------------------------------- append


def stored64(x, dtype, scale):
    """x / scale in 64 bits, and half a step of the type there."""
    y = x / scale
    if dtype == "f8":
        y = np.clip(y, -448, 448)
        return y, np.maximum(np.abs(y) * 2.0 ** -4, 2.0 ** -10)
    if dtype == "f16":
        return y, np.maximum(np.abs(y) * 2.0 ** -11, 2.0 ** -25)
    return y, np.abs(y) * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23)


def rotate64(x, pos, theta):
    d = x.shape[-1]
    half = d // 2
    y = x.copy()
    if theta > 0:
        a = pos[:, None] * theta ** (-2.0 * np.arange(half) / d)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        y[..., :half] = x[..., :half] * c - x[..., half: 2 * half] * s
        y[..., half: 2 * half] = x[..., :half] * s + x[..., half: 2 * half] * c
    return y


def rotation_bound(x, theta):
    """The angle is held to 1.6 * 2^-24 (32-bit half turns), sine and cosine to an ulp, and two products
    and a sum round: 6 * 2^-24 of the pair."""
    half = x.shape[-1] // 2
    m = np.abs(x)
    b = np.zeros_like(m)
    if theta > 0:
        b[..., : half] = b[..., half: 2 * half] = 6 * EPS * (m[..., :half] + m[..., half: 2 * half])
    return b


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kv,H,dim,page,theta,new,start", [
    (2, 4, 128, 16, 10000.0, [3, 0, 17, 1], [0, 5, 31, 100]),
    (1, 1, 64, 1, 500000.0, [9], [0]),
    (3, 3, 33, 7, 10000.0, [2, 20], [6, 0]),
    (4, 8, 80, 24, 0.0, [1, 1, 1], [23, 24, 25]),
    (2, 2, 2, 16, 10000.0, [40], [3]),
    (8, 32, 256, 64, 10000.0, [5, 0, 0], [1, 2, 3]),
])
def test_append(D, dtype, kv, H, dim, page, theta, new, start):
    import torch
    rng = np.random.default_rng(dim + len(new))
    n = len(new)
    total, per = sum(new), max(1, -(-max(a + b for a, b in zip(new, start)) // page))
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim, layout="heads" if dim == 80 else "slots")
    before = [t.float().cpu().numpy().copy() for t in (kp, vp)]
    cu = np.concatenate([[0], np.cumsum(new)])
    seen = [s + 1000000 * i for i, s in enumerate(start)]
    k, v = (rng.standard_normal((total, kv, dim)).astype(np.float32) * 3 for _ in range(2))
    q = rng.standard_normal((total, H, dim)).astype(np.float32)
    if dtype == "f8":
        v[0, 0, 0] = 1e6
    gk, gv, gq = (torch.from_numpy(t).cuda() for t in (k, v, q))
    positions = i32(np.full((n, kv, per * page), -5))
    weights = torch.full((n, kv, per * page), 2.0, device="cuda")
    lens, gseen = i32([0] * n), i32([0] * n)
    ks, vs = (0.25, 0.125) if dtype == "f8" else (1.0, 1.0)
    c = D.PagedKV(kp, vp, table, lens, num_heads=H, seen=gseen, weights=weights, positions=positions, k_scale=ks, v_scale=vs)
    q_out = torch.empty_like(gq)
    c.append(gk, gv, q=gq, q_out=q_out, cu_tokens=i32(cu), theta=theta, start=i32(start), start_seen=i32(seen))
    c.check_error()
    assert lens.tolist() == [a + b for a, b in zip(start, new)] and gseen.tolist() == [a + b for a, b in zip(seen, new)]
    pos = np.concatenate([np.arange(s, s + m) for s, m in zip(seen, new)]).astype(np.float64)
    wk, wq = rotate64(k.astype(np.float64), pos, theta), rotate64(q.astype(np.float64), pos, theta)
    assert np.all(np.abs(q_out.cpu().numpy() - wq) <= rotation_bound(q, theta) + EPS * np.abs(wq))
    t = table.cpu().numpy()
    for pool, want, scale, bound, old in ((kp, wk, ks, rotation_bound(k, theta), before[0]),
                                          (vp, v.astype(np.float64), vs, 0.0, before[1])):
        got = pool.float().cpu().numpy()
        exp, tol = old.copy(), np.zeros_like(old)
        st, half = stored64(want, dtype, scale)
        for b in range(n):
            for i in range(new[b]):
                j = start[b] + i
                exp[t[b, j // page], j % page] = st[cu[b] + i]
                tol[t[b, j // page], j % page] = (half + bound / scale * (1 + 2.0 ** -4))[cu[b] + i]
        assert np.all(np.abs(got - exp) <= tol)
    p, w = positions.cpu().numpy(), weights.cpu().numpy()
    for b in range(n):
        here = slice(start[b], start[b] + new[b])
        assert np.all(p[b, :, here] == np.arange(seen[b], seen[b] + new[b])) and np.all(w[b, :, here] == 0)
        p[b, :, here], w[b, :, here] = -5, 2.0
    assert np.all(p == -5) and np.all(w == 2.0)


def test_append_in_place_from_fused_rows(D):
    """One token a sequence from rows that hold q, k and v side by side, q rotated in place, lengths
    advanced by the call; two calls follow one another."""
    import torch
    rng = np.random.default_rng(2)
    n, H, kv, dim, page, per = 5, 4, 2, 64, 16, 4
    kp, vp, table = make_cache(rng, "f32", n, per, page, kv, dim)
    lens = i32([0, 15, 16, 40, 62])
    c = D.PagedKV(kp, vp, table, lens, num_heads=H)
    start = np.array([0, 15, 16, 40, 62])
    for step in range(2):
        rows = rng.standard_normal((n, (H + 2 * kv) * dim)).astype(np.float32)
        g = torch.from_numpy(rows).cuda()
        q, k, v = g[:, : H * dim], g[:, H * dim: (H + kv) * dim], g[:, (H + kv) * dim:]
        c.append(k, v, q=q, q_out=q, theta=10000.0)
        assert lens.tolist() == list(start + step + 1)
        want = rotate64(rows[:, : H * dim].reshape(n, H, dim).astype(np.float64), (start + step).astype(np.float64), 10000.0)
        np.testing.assert_allclose(q.reshape(n, H, dim).cpu().numpy(), want, atol=3e-6)
        for b in range(n):
            j = int(start[b]) + step
            page_id = int(table[b, j // page])
            assert torch.equal(vp[page_id, j % page], v[b].reshape(kv, dim))
    c.check_error()


def test_append_past_the_end_and_bad_pages_are_reported(D, wb):
    import torch
    rng = np.random.default_rng(9)
    n, kv, dim, page, per = 3, 2, 64, 16, 2
    kp, vp, table = make_cache(rng, "bf16", n, per, page, kv, dim, fill="nan")
    k = torch.ones((n, kv, dim), device="cuda")
    lens = i32([32, 31, -4])
    c = D.PagedKV(kp, vp, table, lens, num_heads=2)
    c.append(k, k)
    with pytest.raises(wb.WelvetError) as e:
        c.check_error()
    assert e.value.code == 1 and "slots" in str(e.value)
    c.check_error()  # cleared
    assert lens.tolist()[:2] == [32, 32]
    written = torch.isfinite(kp.float()).all(-1).sum().item()
    assert written == kv  # one row of the sequence that had room
    for bad in (-1, 10 ** 6, 2 ** 31 - 1):
        broken = table.clone()
        broken[1, 0] = bad
        lens = i32([3, 3, 3])
        c = D.PagedKV(kp, vp, broken, lens, num_heads=2)
        c.append(k, k)
        with pytest.raises(wb.WelvetError) as e:
            c.check_error()
        assert "page" in str(e.value)
        q, out = torch.ones((n, 2, dim), device="cuda"), torch.empty((n, 2, dim), device="cuda")
        kp.zero_(), vp.fill_(1.0)
        c.attend(q, out)
        with pytest.raises(wb.WelvetError):
            c.check_error()
        assert torch.all(out[0] == 1.0) and torch.all(out[1] == 0.0)  # its slots are as if masked
    # entries past the length are never looked at
    broken = table.clone()
    broken[:, 1] = -1
    c = D.PagedKV(kp, vp, broken, i32([16, 15, 1]), num_heads=2)
    c.attend(q, out)
    c.check_error()


# ---------------------------------------------------------------- eviction


def evict_reference(kp, vp, table, lens, seen, weights, positions, keep, budget, sinks, recent):
    k, v, w, p = kp.copy(), vp.copy(), weights.copy(), positions.copy()
    page, out = kp.shape[1], list(lens)
    for b, n in enumerate(lens):
        if n <= budget:
            continue
        out[b] = keep
        for h in range(w.shape[1]):
            rank = sorted(range(n), key=lambda j: (not (positions[b, h, j] < sinks or positions[b, h, j] >= seen[b] - recent),
                                                   math.inf if math.isnan(weights[b, h, j]) else -float(weights[b, h, j]), j))
            stays = set(rank[:keep])
            fill = [j for j in range(keep) if j not in stays]
            take = [j for j in range(keep, n) if j in stays]
            assert len(fill) == len(take)
            for to, frm in zip(fill, take):
                a, c = (table[b, to // page], to % page, h), (table[b, frm // page], frm % page, h)
                k[a], v[a] = kp[c], vp[c]
                w[b, h, to], p[b, h, to] = weights[b, h, frm], positions[b, h, frm]
    return k, v, w, p, out


@pytest.mark.parametrize("dtype,kv,dim,page,lens,keep,budget,sinks,recent,kind", [
    ("bf16", 2, 64, 16, [100, 33, 64, 65, 0], 32, 32, 4, 8, "random"),
    ("f32", 1, 8, 4, [7, 3, 2], 1, 1, 0, 0, "random"),
    ("f8", 3, 32, 16, [500, 499], 250, 499, 2, 100, "random"),
    ("f16", 2, 33, 5, [41, 80], 40, 40, 0, 3, "ties"),
    ("bf16", 1, 128, 16, [3000, 2048, 1025], 1024, 1024, 4, 200, "zeros"),
    ("f32", 2, 20, 16, [50, 90], 30, 40, 1, 1, "special"),
    ("f8", 2, 64, 64, [9000, 5000], 4999, 5000, 16, 512, "random"),
    ("bf16", 2, 64, 16, [70], 60, 60, 20, 40, "random"),
    ("bf16", 2, 64, 16, [70], 69, 69, 0, 0, "negative"),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(D, dtype, kv, dim, page, lens, keep, budget, sinks, recent, kind, in_place):
    import torch
    rng = np.random.default_rng(keep + dim)
    n, per = len(lens), -(-max(lens) // page) + 1
    S = per * page
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim, layout="heads" if dim == 64 else "slots")
    w = rng.lognormal(-4, 3, (n, kv, S)).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 3, (n, kv, S)).astype(np.float32)
    elif kind == "zeros":
        w[rng.random(w.shape) < 0.8] = 0.0
        w[rng.random(w.shape) < 0.2] = -0.0
    elif kind == "special":
        w[rng.random(w.shape) < 0.3] = np.nan
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
    elif kind == "negative":
        w = -w
    seen = np.array([2 * x + 3 for x in lens], np.int32)
    pos = np.zeros((n, kv, S), np.int32)
    for b in range(n):
        for h in range(kv):
            pos[b, h, : lens[b]] = rng.permutation(max(1, seen[b]))[: lens[b]]
    bits = {"f32": torch.int32, "f16": torch.int16, "bf16": torch.int16, "f8": torch.uint8}[dtype]
    view = lambda t: (t.transpose(1, 2).view(bits).transpose(1, 2) if dim == 64 else t.view(bits))  # noqa: E731
    k0, v0 = view(kp).cpu().numpy().copy(), view(vp).cpu().numpy().copy()
    gl, gw, gp = i32(lens), torch.from_numpy(w).cuda(), i32(pos)
    if in_place:
        lens_o, w_o, p_o = gl, gw, gp
        args = {}
    else:
        lens_o, w_o, p_o = i32([0] * n), torch.full_like(gw, -1.0), torch.full_like(gp, -1)
        args = dict(lens_in=gl, weights_in=gw, positions_in=gp)
    c = D.PagedKV(kp, vp, table, lens_o, num_heads=kv, seen=i32(seen), weights=w_o, positions=p_o)
    c.evict(keep, budget=budget, sinks=sinks, recent=recent, **args)
    c.check_error()
    k, v, ww, pp, out = evict_reference(k0, v0, table.cpu().numpy(), lens, seen, w, pos, keep, budget, sinks, recent)
    assert lens_o.tolist() == out
    np.testing.assert_array_equal(view(kp).cpu().numpy(), k)
    np.testing.assert_array_equal(view(vp).cpu().numpy(), v)
    gotw, gotp = w_o.cpu().numpy().view(np.int32), p_o.cpu().numpy()
    for b in range(n):
        np.testing.assert_array_equal(gotw[b, :, : out[b]], ww.view(np.int32)[b, :, : out[b]])
        np.testing.assert_array_equal(gotp[b, :, : out[b]], pp[b, :, : out[b]])
        if not in_place:
            assert np.all(w_o.cpu().numpy()[b, :, out[b]:] == -1.0) and np.all(gotp[b, :, out[b]:] == -1)


def test_cache_refusals(D, wb):
    """What the host can see is refused before any launch (status 1 or 2, or a ValueError)."""
    import torch
    rng = np.random.default_rng(1)
    kp, vp, table = make_cache(rng, "bf16", 2, 4, 16, 2, 64)
    lens = i32([3, 3])
    for bad in (dict(num_heads=3), dict(num_heads=0), dict(num_heads=4, k_scale=0.0), dict(num_heads=4, v_scale=float("nan")),
                dict(num_heads=4, positions=i32(np.zeros((2, 2, 64))))):
        with pytest.raises(wb.WelvetError) as e:
            D.PagedKV(kp, vp, table, lens, **bad)
        assert e.value.code == 1
    with pytest.raises(wb.WelvetError) as e:
        big = torch.zeros((2, 4, 1, 264), device="cuda")
        D.PagedKV(big, big.clone(), table, lens, num_heads=1)
    assert e.value.code == 2
    for args in ((kp, vp.float(), table, lens), (kp.to(torch.float64), vp.to(torch.float64), table, lens),
                 (kp, vp, table.long(), lens), (kp, vp, table, lens.long()), (kp, vp, table, i32([1])),
                 (kp.cpu(), vp.cpu(), table, lens), (kp[..., ::2], vp[..., ::2], table, lens)):
        with pytest.raises(ValueError):
            D.PagedKV(*args, num_heads=4)
    c = D.PagedKV(kp, vp, table, lens, num_heads=4)
    q, out, k = torch.zeros((2, 4, 64), device="cuda"), torch.zeros((2, 4, 64), device="cuda"), torch.zeros((2, 2, 64), device="cuda")
    for f in (lambda: c.attend(q, out, accumulate=True), lambda: c.attend(q, out, window=-1),
              lambda: c.attend(q, out, scale=float("inf")), lambda: c.evict(3), lambda: c.append(k[:1], k[:1]),
              lambda: c.append(k, k, theta=float("nan")), lambda: c.append(k, k, start_seen=lens)):
        with pytest.raises(wb.WelvetError) as e:
            f()
        assert e.value.code == 1
    for f in (lambda: c.attend(q[:1], out), lambda: c.attend(q.double(), out), lambda: c.attend(q[:, :, :32], out),
              lambda: c.append(k, k[:1]), lambda: c.append(k, k, q=q), lambda: c.attend(q.cpu(), out),
              lambda: c.append(k, k, cu_tokens=i32([0, 2]))):
        with pytest.raises(ValueError):
            f()
    w = torch.zeros((2, 2, 64), device="cuda")
    c = D.PagedKV(kp, vp, table, lens, num_heads=4, seen=i32([3, 3]), weights=w, positions=i32(np.zeros((2, 2, 64))))
    for a in (dict(keep=0), dict(keep=4, budget=3), dict(keep=4, sinks=3, recent=2), dict(keep=4, sinks=-1)):
        with pytest.raises(wb.WelvetError) as e:
            c.evict(**a)
        assert e.value.code == 1
    c.check_error()


def test_append_nothing(D):
    """No new token at all: lengths are carried over, nothing is written."""
    import torch
    rng = np.random.default_rng(4)
    kp, vp, table = make_cache(rng, "bf16", 2, 4, 16, 2, 64)
    old = kp.clone()
    lens = i32([0, 0])
    c = D.PagedKV(kp, vp, table, lens, num_heads=4)
    k = torch.zeros((0, 2, 64), device="cuda")
    c.append(k, k, cu_tokens=i32([0, 0, 0]), start=i32([5, 9]))
    assert lens.tolist() == [5, 9] and torch.equal(kp, old)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [16, 48, 56, 112, 120, 192, 248])
def test_attend_dims_between_the_tiles(D, dtype, dim):
    """Head widths that fill a row of shared memory only in part."""
    import torch
    rng = np.random.default_rng(dim)
    H, kv, page, lens = 4, 2, 16, [70, 16, 129]
    kp, vp, table = make_cache(rng, dtype, 3, 9, page, kv, dim)
    q = torch.from_numpy(rng.standard_normal((3, H, dim)).astype(np.float32)).cuda()
    out = torch.empty((3, H, dim), device="cuda")
    D.PagedKV(kp, vp, table, i32(lens), num_heads=H).attend(q, out)
    want, _, bound = attend64(q, kp, vp, table, lens, 1.0 / math.sqrt(dim))
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("dim", [64, 33])
def test_attend_accumulates_within_the_window(D, dim):
    import torch
    rng = np.random.default_rng(21)
    H, kv, page, lens, window = 4, 2, 16, [1000, 30], 100
    kp, vp, table = make_cache(rng, "bf16", 2, 64, page, kv, dim)
    q = torch.from_numpy(rng.standard_normal((2, H, dim)).astype(np.float32)).cuda()
    out = torch.empty((2, H, dim), device="cuda")
    w = torch.full((2, kv, 1024), 0.5, device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H, weights=w)
    c.attend(q, out)  # leaves scores of all slots behind
    c.attend(q, out, accumulate=True, window=window)
    _, ws, _ = attend64(q, kp, vp, table, lens, 1.0 / math.sqrt(dim), window)
    got = w.cpu().numpy()
    for b, L in enumerate(lens):
        np.testing.assert_allclose(got[b, :, :L] - 0.5, ws[b].reshape(kv, 2, L).sum(1), rtol=2e-4, atol=4 * EPS)
        assert np.all(got[b, :, L:] == 0.5) and np.all(got[b, :, : max(0, L - window)] == 0.5)


def test_attend_many_sequences(D):
    """More sequences than a block has threads, most of them empty or a token long."""
    import torch
    rng = np.random.default_rng(22)
    n, H, kv, dim, page = 700, 2, 1, 64, 16
    lens = [int(x) for x in rng.choice([0, 1, 2, 17, 64, 65, 300], n)]
    kp, vp, table = make_cache(rng, "f16", n, 19, page, kv, dim)
    q = torch.from_numpy(rng.standard_normal((n, H, dim)).astype(np.float32)).cuda()
    out = torch.full((n, H, dim), float("nan"), device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H)
    for _ in range(3):
        c.attend(q, out)
    pages = [t.float().cpu() for t in (kp, vp)]
    want, _, bound = attend64(q, pages[0], pages[1], table, lens, 0.125)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("kv,lens,keep,page", [(1, [70000], 20000, 64), (2, [30001, 5, 250000], 29999, 16), (40, [3000, 2500, 10, 2049], 2048, 32)])
def test_evict_long_and_many(D, kv, lens, keep, page):
    """Heads spread over a cluster of blocks, keys beyond what shared memory holds, and more heads than SMs,
    against one stable sort."""
    import torch
    dim, n = 16, len(lens)
    per = -(-max(lens) // page)
    S = per * page
    g = torch.Generator(device="cuda").manual_seed(kv)
    kp = torch.randint(0, 256, (n * per, page, kv, dim), generator=g, device="cuda", dtype=torch.uint8)
    vp = torch.randint(0, 256, kp.shape, generator=g, device="cuda", dtype=torch.uint8)
    table = torch.randperm(n * per, generator=g, device="cuda").reshape(n, per).to(torch.int32)
    w = (torch.rand((n, kv, S), generator=g, device="cuda") * 50).floor() * 0.25  # many ties
    pos = torch.arange(S, device="cuda", dtype=torch.int32).expand(n, kv, S).contiguous()
    lens_t = i32(lens)
    k0, v0, w0 = kp.clone(), vp.clone(), w.clone()
    c = D.PagedKV(kp.view(torch.float8_e4m3fn), vp.view(torch.float8_e4m3fn), table, lens_t, num_heads=kv, seen=i32(lens), weights=w, positions=pos)
    c.evict(keep, sinks=3, recent=keep // 5)
    c.check_error()
    assert lens_t.tolist() == [min(x, keep) for x in lens]
    for b, L in enumerate(lens):
        t = table[b].long()
        old_k, old_v = k0[t].reshape(S, kv, dim), v0[t].reshape(S, kv, dim)
        new_k, new_v = kp[t].reshape(S, kv, dim), vp[t].reshape(S, kv, dim)
        m = min(L, keep)
        for h in range(kv):
            src = torch.arange(m, device="cuda")
            if L > keep:
                j = torch.arange(L, device="cuda")
                key = torch.where((j < 3) | (j >= L - keep // 5), torch.inf, w0[b, h, :L])
                stays = torch.zeros(L, dtype=torch.bool, device="cuda")
                stays[torch.sort(key, descending=True, stable=True).indices[:keep]] = True
                src[~stays[:keep]] = keep + torch.nonzero(stays[keep:]).flatten()
            assert torch.equal(pos[b, h, :m].long(), src)
            assert torch.equal(w[b, h, :m], w0[b, h, src])
            assert torch.equal(new_k[:m, h], old_k[src, h]) and torch.equal(new_v[:m, h], old_v[src, h])


def test_evict_again_and_again(D):
    """Two hundred calls with one new token between them: the tickets and lengths stay in step."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    n, kv, dim, page, per, keep = 3, 2, 64, 16, 6, 64
    kp = torch.randn((n * per, page, kv, dim), generator=g, device="cuda")
    vp, table = kp.clone(), torch.arange(n * per, device="cuda", dtype=torch.int32).reshape(n, per)
    lens, seen = i32([60, 0, 30]), i32([60, 0, 30])
    w, pos = torch.rand((n, kv, per * page), generator=g, device="cuda"), torch.zeros((n, kv, per * page), dtype=torch.int32, device="cuda")
    pos[:] = torch.arange(per * page, device="cuda", dtype=torch.int32)
    c = D.PagedKV(kp, vp, table, lens, num_heads=4, seen=seen, weights=w, positions=pos)
    q, out = torch.randn((n, 4, dim), generator=g, device="cuda"), torch.empty((n, 4, dim), device="cuda")
    for step in range(200):
        k = torch.randn((n, kv, dim), generator=g, device="cuda")
        c.append(k, k)
        c.attend(q, out, accumulate=True)
        c.evict(keep, budget=keep + 7, sinks=2, recent=16)
    c.check_error()
    assert seen.tolist() == [260, 200, 230]
    assert all(keep <= x <= keep + 7 for x in lens.tolist())
    for b in range(n):
        for h in range(kv):
            p = pos[b, h, : lens.tolist()[b]].tolist()
            assert len(set(p)) == len(p) and {0, 1} <= set(p)
            assert set(range(seen.tolist()[b] - 16, seen.tolist()[b])) <= set(p)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("page", [16, 48, 20, 64])
def test_attend_pages_and_groups(D, dtype, dim, page):
    """Every constant width, pages that hold whole 16-slot tiles and pages that end inside one, head groups
    that fill a tile of eight in part, exactly and more than once."""
    import torch
    rng = np.random.default_rng(dim + page)
    lens = [131, 64, 33, 400]
    for H, kv in ((3, 1), (16, 2), (20, 2)):
        per = -(-400 // page)
        kp, vp, table = make_cache(rng, dtype, 4, per, page, kv, dim, layout="heads" if page == 48 else "slots")
        q = torch.from_numpy(rng.standard_normal((4, H, dim)).astype(np.float32)).cuda()
        out = torch.full((4, H, dim), float("nan"), device="cuda")
        c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H)
        c.attend(q, out)
        c.check_error()
        want, _, bound = attend64(q, kp, vp, table, lens, 1.0 / math.sqrt(dim))
        assert np.all(np.abs(out.cpu().numpy() - want) <= bound), (H, kv)


def test_attend_pools_of_different_layout(D):
    """Keys by slot, values by head: the pools' strides differ."""
    import torch
    rng = np.random.default_rng(31)
    kp, _, table = make_cache(rng, "bf16", 2, 8, 32, 4, 128)
    vp = torch.from_numpy(rng.standard_normal((kp.shape[0], 4, 32, 128)).astype(np.float32)).cuda().to(torch.bfloat16).transpose(1, 2)
    q = torch.from_numpy(rng.standard_normal((2, 8, 128)).astype(np.float32)).cuda()
    out = torch.empty((2, 8, 128), device="cuda")
    D.PagedKV(kp, vp, table, i32([250, 77]), num_heads=8).attend(q, out)
    want, _, bound = attend64(q, kp, vp, table, [250, 77], 128 ** -0.5)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("dim", [33, 66, 64, 130])
@pytest.mark.parametrize("shift", [0, 1])
def test_append_rotates_q_in_place(D, dim, shift):
    """q_out = q, on rows that 16-byte accesses can serve and on rows that they cannot."""
    import torch
    rng = np.random.default_rng(dim)
    n, H, kv, page = 7, 24, 2, 16
    kp, vp, table = make_cache(rng, "f16", n, 2, page, kv, dim)
    rows = rng.standard_normal((n, H * dim + shift)).astype(np.float32)
    g = torch.from_numpy(rows).cuda()[:, shift:]
    k = torch.zeros((n, kv, dim), device="cuda")
    pos = np.arange(n) * 1001 + 5
    c = D.PagedKV(kp, vp, table, i32([3] * n), num_heads=H, seen=i32(pos))
    c.append(k, k, q=g, q_out=g, theta=10000.0)
    x = rows[:, shift:].reshape(n, H, dim).astype(np.float64)
    want = rotate64(x, pos.astype(np.float64), 10000.0)
    got = g.cpu().numpy().reshape(n, H, dim)
    assert np.all(np.abs(got - want) <= rotation_bound(x, 10000.0) + EPS * np.abs(want))


def test_create_without_memory_leaves_no_trace(D, wb):
    """Workspaces that no GPU holds: the create fails, and the next cache's launches are not blamed for it."""
    import ctypes

    import torch
    big = D._KvDesc(dtype=3, num_heads=60000, num_kv_heads=60000, head_dim=64, page_size=1024, num_pages=10, num_seqs=60000,
                    pages_per_seq=1024, k_pages=4096, v_pages=4096, k_strides=(ctypes.c_int64 * 3)(2 ** 32, 2 ** 22, 64),
                    v_strides=(ctypes.c_int64 * 3)(2 ** 32, 2 ** 22, 64), k_scale=1.0, v_scale=1.0, page_table=4096,
                    table_stride=1024, lens=4096, weights=4096)
    h = ctypes.c_void_p()
    st = wb.lib().welvet_b200_kv_create(ctypes.byref(big), ctypes.byref(h))
    assert st.code == 4 and not h
    rng = np.random.default_rng(41)
    kp, vp, table = make_cache(rng, "bf16", 1, 2, 16, 1, 33)  # the form with plain launches
    q = torch.from_numpy(rng.standard_normal((1, 2, 33)).astype(np.float32)).cuda()
    out = torch.empty((1, 2, 33), device="cuda")
    D.PagedKV(kp, vp, table, i32([20]), num_heads=2).attend(q, out)
    want, _, bound = attend64(q, kp, vp, table, [20], 33 ** -0.5)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,kv,per", [(1, 1, 2), (1, 4, 30), (3, 2, 8), (2, 8, 33)])
def test_attend_small_caches(D, dtype, n, kv, per):
    """Caches small enough for clusters: lengths that leave some of their blocks without a tile, windows that
    start inside one, weights summed."""
    import torch
    rng = np.random.default_rng(n * 100 + per)
    H, dim, page = kv * 3, 128, 16
    S = per * page
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim)
    q = torch.from_numpy(rng.standard_normal((n, H, dim)).astype(np.float32)).cuda()
    out = torch.empty((n, H, dim), device="cuda")
    w = torch.zeros((n, kv, S), device="cuda")
    lens = i32([0] * n)
    c = D.PagedKV(kp, vp, table, lens, num_heads=H, weights=w)
    for base, window in ((S, 0), (1, 0), (S - 1, 0), (S // 2 + 1, 37), (0, 0), (17, 5)):
        now = [max(0, base - 5 * i) for i in range(n)]
        lens.copy_(i32(now))
        w.zero_()
        c.attend(q, out, window=window, accumulate=True)
        want, ws, bound = attend64(q, kp, vp, table, now, dim ** -0.5, window)
        assert np.all(np.abs(out.cpu().numpy() - want) <= bound)
        got = w.cpu().numpy()
        for b, L in enumerate(now):
            np.testing.assert_allclose(got[b, :, :L], ws[b].reshape(kv, 3, L).sum(1), rtol=2e-4, atol=4 * EPS)
            assert not got[b, :, L:].any()
    c.check_error()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n,kv,group,longest", [(10, 8, 1, 900), (2, 2, 3, 6000), (1, 1, 9, 20000)])
def test_attend_joins_few_and_many_parts(D, dtype, dim, n, kv, group, longest):
    """Units cut into a few parts and into many, narrow and wide, with the attention weights: dz (see
    attend64) is below 264 * 2^-24 * 20 here, and a weight moves by twice that."""
    import torch
    rng = np.random.default_rng(31 + dim + n)
    page, H = 16, kv * group
    per = longest // page + 2
    lens = [max(0, longest - 97 * b * b) for b in range(n)]
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim)
    q = torch.from_numpy(rng.standard_normal((n, H, dim)).astype(np.float32)).cuda()
    out = torch.full((n, H, dim), float("nan"), device="cuda")
    w = torch.zeros((n, kv, per * page), device="cuda")
    c = D.PagedKV(kp, vp, table, i32(lens), num_heads=H, weights=w)
    c.attend(q, out, accumulate=True)
    want, ws, bound = attend64(q, kp, vp, table, lens, dim ** -0.5)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)
    got = w.cpu().numpy()
    for b, L in enumerate(lens):
        np.testing.assert_allclose(got[b, :, :L], ws[b].reshape(kv, group, L).sum(1), rtol=1e-3, atol=4 * EPS)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kv,H,dim,theta,seen", [(4, 8, 128, 10000.0, 0), (2, 2, 64, 500000.0, 1000000), (1, 3, 50, 10000.0, 77)])
def test_append_rounds_as_the_formula_does(D, dtype, kv, H, dim, theta, seen):
    """Keys, values and queries are bit for bit what the formula gives in fp32, one rounding an operation,
    with the angle's cosine and sine rounded once from 64 bits; stored after an exact scale."""
    import torch
    n, page = 1500, 16
    half, per = dim // 2, -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(dim)
    q, k, v = (torch.randn((n, h, dim), generator=g, device="cuda") * 2 for h in (H, kv, kv))
    kp, vp = (torch.zeros((per, page, kv, dim), dtype=types()[dtype], device="cuda") for _ in range(2))
    scale = 1 / 64 if dtype == "f8" else 1.0
    out = torch.empty_like(q)
    c = D.PagedKV(kp, vp, torch.arange(per, dtype=torch.int32, device="cuda")[None], i32([0]), num_heads=H, seen=i32([0]), k_scale=scale, v_scale=scale)
    c.append(k, v, q=q, q_out=out, cu_tokens=i32([0, n]), theta=theta, start=i32([0]), start_seen=i32([seen]))
    c.check_error()
    # half turns are a multiple of two plus what is left: the same angle
    turns = torch.tensor([math.pow(theta, -2.0 * i / dim) / math.pi for i in range(half)], dtype=torch.float64, device="cuda")
    u = (seen + torch.arange(n, dtype=torch.float64, device="cuda"))[:, None] * turns
    angle = math.pi * (u - 2.0 * torch.round(0.5 * u))
    cs, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotate(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cs - b * sn, a * sn + b * cs], -1)

    assert torch.equal(out, rotate(q))
    for pool, want in ((kp, rotate(k)), (vp, v)):
        want = want / scale
        want = (want.clamp(-448, 448) if dtype == "f8" else want).to(types()[dtype])
        assert torch.equal(pool.reshape(per * page, kv, dim)[:n].float(), want.float())


@pytest.mark.parametrize("cu,counts", [([0, 2, 7], [2, 3]), ([0, 9, 9], [5, 0]), ([3, 2, 5], [0, 3]), ([-2, 1, 5], [0, 4]),
                                       ([0, 5, 2 ** 31 - 1], [5, 0]), ([-2 ** 31, 0, 5], [0, 5])])
def test_append_rows_that_cu_tokens_do_not_fit(D, wb, cu, counts):
    """Offsets past the rows, below zero or decreasing: lengths advance by the rows that there are, never
    back, and the error word says so."""
    import torch
    rng = np.random.default_rng(19)
    kv, dim, page, per, rows = 2, 64, 16, 2, 5
    kp, vp, table = make_cache(rng, "f32", 2, per, page, kv, dim, fill="nan")
    k = torch.from_numpy(rng.standard_normal((rows, kv, dim)).astype(np.float32)).cuda()
    lens, seen = i32([4, 6]), i32([10, 20])
    c = D.PagedKV(kp, vp, table, lens, num_heads=2, seen=seen)
    c.append(k, k, cu_tokens=i32(cu))
    with pytest.raises(wb.WelvetError) as e:
        c.check_error()
    assert e.value.code == 1 and "cu_tokens" in str(e.value)
    assert lens.tolist() == [4 + counts[0], 6 + counts[1]] and seen.tolist() == [10 + counts[0], 20 + counts[1]]
    for b, (first, n) in enumerate(zip((4, 6), counts)):
        for i in range(n):
            j = first + i
            assert torch.equal(kp[int(table[b, j // page]), j % page], k[cu[b] + i])
    assert int(torch.isfinite(kp[..., 0]).sum()) == sum(counts) * kv
    c.append(k, k, cu_tokens=i32([0, 2, 5]))
    c.check_error()
    # offsets that begin or end within the rows are no error: rows before and after them are nobody's
    c.append(k, k, cu_tokens=i32([1, 2, 4]))
    c.check_error()
    assert lens.tolist() == [4 + counts[0] + 3, 6 + counts[1] + 5]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [128, 24, 33])
@pytest.mark.parametrize("ks,vs", [(0.013, 3.7), (1.0 / 448, 1.0), (2.0 ** -126, 2.0 ** 127), (1e-30, 1e30)])
def test_append_divides_by_the_scale(D, dtype, dim, ks, vs):
    """Stored values are x / scale rounded to fp32 and then to the page's type, for scales that are no
    powers of two as well."""
    import torch
    n, kv, page = 300, 3, 16
    per = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(dim)
    k, v = (torch.randn((n, kv, dim), generator=g, device="cuda") * s for s in (ks * 40, min(vs, 1e30) * 40))
    kp, vp = (torch.zeros((per, page, kv, dim), dtype=types()[dtype], device="cuda") for _ in range(2))
    c = D.PagedKV(kp, vp, torch.arange(per, dtype=torch.int32, device="cuda")[None], i32([0]), num_heads=kv, k_scale=ks, v_scale=vs)
    c.append(k, v, cu_tokens=i32([0, n]))
    c.check_error()
    for pool, x, scale in ((kp, k, ks), (vp, v, vs)):
        want = (x / torch.tensor(scale, dtype=torch.float32, device="cuda")).float()
        want = (want.clamp(-448, 448) if dtype == "f8" else want).to(types()[dtype])
        assert torch.equal(pool.reshape(per * page, kv, dim)[:n].float(), want.float())


@pytest.mark.parametrize("dtype,H,kv,dim,lens", [
    ("f32", 4, 1, 96, [1500, 40]), ("f32", 16, 4, 256, [900]), ("f32", 4, 2, 64, [333, 4000]), ("bf16", 8, 8, 192, [1200, 333]),
    ("bf16", 32, 8, 128, [700, 701, 64]), ("bf16", 3, 1, 256, [5000]), ("f16", 10, 2, 128, [2222]), ("f16", 8, 1, 256, [100, 3100]),
    ("f8", 4, 4, 96, [640, 64]), ("f8", 16, 2, 256, [1800])])
def test_attend_is_as_exact_as_fp32(D, dtype, H, kv, dim, lens):
    """Against 64 bits, the result is no further off than the formula in fp32 with one running sum a score:
    sums are held in 32 bits, and what parts of 22 bits and more lose is less than a chain of `dim`
    rounded additions does."""
    import torch
    rng = np.random.default_rng(7 * dim + H)
    n, page = len(lens), 16
    per = -(-max(lens) // page)
    kp, vp, table = make_cache(rng, dtype, n, per, page, kv, dim)
    q = torch.from_numpy((rng.standard_normal((n, H, dim)) * 1.5).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    D.PagedKV(kp, vp, table, i32(lens), num_heads=H).attend(q, out)
    got = plain = 0.0
    for b, L in enumerate(lens):
        used = table[b].long()
        k, v = (p.float()[used].reshape(-1, kv, dim)[:L].repeat_interleave(H // kv, 1) for p in (kp, vp))
        zs = [torch.einsum("hd,shd->hs", q[b].double(), k.double()), torch.zeros((H, L), device="cuda")]
        for d in range(dim):
            zs[1] += q[b, :, d: d + 1] * k[:, :, d].T
        want, fp32 = (torch.einsum("hs,shd->hd", torch.softmax(z / math.sqrt(dim), -1), v.to(z.dtype)).double() for z in zs)
        got += float((out[b].double() - want).square().sum())
        plain += float((fp32 - want).square().sum())
    assert got <= plain, (got ** 0.5, plain ** 0.5)


@pytest.mark.parametrize("dim,long", [(64, False), (64, True), (33, False), (33, True)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_skips_rows_of_bad_pages(D, wb, dim, long, in_place):
    """A row that cannot move leaves its slot as it was, its weight and position too; the others move, and
    the error word says so."""
    import torch
    rng = np.random.default_rng(dim)
    kv, page, n, keep = 2, 16, 5000 if long else 160, 2000 if long else 80
    per = -(-n // page)
    kp, vp, table = make_cache(rng, "f32", 1, per, page, kv, dim)
    broken = table.clone()
    broken[0, 0], broken[0, per - 1] = -1, 1 << 20  # of slots to fill, and of slots to take
    w = rng.random((1, kv, per * page)).astype(np.float32)
    pos = np.broadcast_to(np.arange(per * page, dtype=np.int32) * 3, w.shape).copy()
    k0, v0 = kp.clone(), vp.clone()
    w_in, p_in = torch.from_numpy(w).cuda(), i32(pos)
    w_out, p_out = (w_in.clone(), p_in.clone()) if in_place else (torch.full_like(w_in, -1), torch.full_like(p_in, -1))
    lens = i32([n])
    c = D.PagedKV(kp, vp, broken, lens, num_heads=kv, seen=i32([3 * n]), weights=w_out, positions=p_out)
    c.evict(keep, **({} if in_place else dict(weights_in=w_in, positions_in=p_in)))
    with pytest.raises(wb.WelvetError) as e:
        c.check_error()
    assert e.value.code == 1 and "page" in str(e.value) and lens.tolist() == [keep]
    t, moved, skipped = table.cpu().numpy()[0], 0, 0
    got_w, got_p = w_out.cpu().numpy(), p_out.cpu().numpy()
    kb, ka = k0.cpu().numpy(), kp.cpu().numpy()
    for h in range(kv):
        order = np.lexsort((np.arange(n), -w[0, h, :n]))
        stays = np.zeros(n, bool)
        stays[order[:keep]] = True
        src = np.arange(keep)
        fill, take = np.flatnonzero(~stays[:keep]), keep + np.flatnonzero(stays[keep:])
        ok = (fill >= page) & (take < (per - 1) * page)
        src[fill[ok]] = take[ok]
        moved, skipped = moved + int(ok.sum()), skipped + int((~ok).sum())
        np.testing.assert_array_equal(got_w[0, h, :keep], w[0, h, src])
        np.testing.assert_array_equal(got_p[0, h, :keep], pos[0, h, src])
        for j in range(keep):
            np.testing.assert_array_equal(ka[t[j // page], j % page, h], kb[t[src[j] // page], src[j] % page, h])
    assert moved and skipped
