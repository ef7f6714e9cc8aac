"""An MHA cell's prompt and decode steps over a paged cache against the cell's own forward of the whole
sequence and against 64-bit sums, and the example that runs the operators together."""
import os
import sys

import numpy as np
import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def D(wb):
    import welvet.cuda_b200.decode as decode
    return decode


def cache_for(D, n, heads, kv, dim, slots, dtype, page=16, records=False):
    import torch
    per = -(-slots // page)
    k = torch.zeros((n * per + 1, page, kv, dim), dtype=dtype, device="cuda")
    table = torch.randperm(n * per, device="cuda").reshape(n, per).to(torch.int32)
    z = lambda: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    kw = {}
    if records:
        kw = dict(weights=torch.zeros((n, kv, per * page), device="cuda"),
                  positions=torch.zeros((n, kv, per * page), dtype=torch.int32, device="cuda"))
    return D.PagedKV(k, torch.zeros_like(k), table, z(), num_heads=heads, seen=z(), **kw)


@pytest.mark.parametrize("pos", [0, 2, 3, 1])
@pytest.mark.parametrize("mask,max_seq", [(1, 200), (3, 20), (2, 200), (4, 200)])
def test_cell_steps_equal_the_whole_forward(D, wb, pos, mask, max_seq):
    """A prompt and single tokens over a float32 cache give the rows that the cell's forward of the whole
    sequence gives (causal rows; mask 2's last row sees everything up to itself, as a step does).

    The cell's attention is in 64 bits, the cache's in 32 (keys, values and query to 24 bits, scores to
    about 2^-20 of |q||k| / sqrt(dim) ~ 10): 1e-4 of the largest output holds both, and the projections'
    2^-18 bound between other batch sizes."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(pos * 10 + mask)
    d_model, heads, kv, dim, total, first = 256, 4, 2, 64, 60, 13
    w = [torch.randn((r, d_model), generator=g, device="cuda") * 0.08 for r in (heads * dim, kv * dim, kv * dim)]
    w.append(torch.randn((d_model, heads * dim), generator=g, device="cuda") * 0.08)
    cell = wb.MhaCell(*w, d_model, heads, kv, dim, max_seq, mask, pos, wb.FP8E4M3)
    x = torch.randn((total, d_model), generator=g, device="cuda")
    seen = total if mask != 3 else max_seq  # the cell's ring holds max_seq positions of one forward
    cache = cache_for(D, 1, heads, kv, dim, 100, torch.float32)
    y, attn = torch.empty((first, d_model), device="cuda"), torch.empty((first, heads * dim), device="cuda")
    D.mha_prefill(cell, cache, 0, x[:first].contiguous(), y, attn)
    got_y, got_a = [y], [attn]
    for t in range(first, seen):
        y, attn = torch.empty((1, d_model), device="cuda"), torch.empty((1, heads * dim), device="cuda")
        D.mha_decode(cell, cache, x[t: t + 1], y, attn)
        got_y.append(y)
        got_a.append(attn)
    cache.check_error()
    assert cache.lens.tolist() == [seen] and cache.seen.tolist() == [seen]
    if mask == 2:  # full: each step is compared with the last row of its own prefix
        for t in (first, first + 1, seen - 1):
            ye, ae = torch.empty((t + 1, d_model), device="cuda"), torch.empty((t + 1, heads * dim), device="cuda")
            cell.execute_device(x[: t + 1].contiguous(), 1, t + 1, ye, ae)
            for a, b in ((got_a[t - first + 1], ae[-1:]), (got_y[t - first + 1], ye[-1:])):
                assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
        return
    ye, ae = torch.empty((seen, d_model), device="cuda"), torch.empty((seen, heads * dim), device="cuda")
    cell.execute_device(x[:seen].contiguous(), 1, seen, ye, ae)
    for a, b in ((torch.cat(got_a), ae), (torch.cat(got_y), ye)):
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())


def test_window_cell_forgets(D, wb):
    """mask 3: tokens max_seq_len back no longer count."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    d_model, heads, dim, window = 128, 2, 64, 8
    w = [torch.randn((128, 128), generator=g, device="cuda") * 0.1 for _ in range(4)]
    cell = wb.MhaCell(*w, d_model, heads, heads, dim, window, 3, 1, wb.FP8E4M3)  # no positions: rows decide
    x = torch.randn((30, d_model), generator=g, device="cuda")
    outs = []
    for drop in (0, 15):  # a cache that never saw the first tokens gives the same last step
        cache = cache_for(D, 1, heads, heads, dim, 64, torch.bfloat16)
        for t in range(drop, 30):
            y = torch.empty((1, d_model), device="cuda")
            D.mha_decode(cell, cache, x[t: t + 1], y)
        outs.append(y)
    assert float((outs[0] - outs[1]).abs().max()) <= 2e-6 * float(outs[0].abs().max())


def test_refusals(D, wb):
    import torch
    w = [torch.zeros((128, 128), device="cuda") for _ in range(4)]
    cell = wb.MhaCell(*w, 128, 2, 2, 64, 64, 1, 0, wb.FP8E4M3)
    cache = cache_for(D, 3, 2, 2, 64, 32, torch.bfloat16)
    other = cache_for(D, 3, 4, 2, 64, 32, torch.bfloat16)
    x, y = torch.zeros((3, 128), device="cuda"), torch.zeros((3, 128), device="cuda")
    for f in (lambda: D.mha_decode(cell, other, x, y), lambda: D.mha_decode(cell, cache, x, y, accumulate=True),
              lambda: D.mha_prefill(cell, cache, 3, x, y), lambda: D.mha_prefill(cell, cache, -1, x, y),
              lambda: D.mha_prefill(cell, cache, 0, torch.zeros((40, 128), device="cuda"), torch.zeros((40, 128), device="cuda"))):
        with pytest.raises(wb.WelvetError) as e:
            f()
        assert e.value.code == 1
    for a in ((x[:2], y), (x, y[:, :64]), (x.half(), y)):
        with pytest.raises(ValueError):
            D.mha_decode(cell, cache, *a)
    assert cache.lens.tolist() == [0, 0, 0]


def test_example(D):
    """Replays of the captured step keep the budget, are finite, and repeat bit for bit."""
    import torch
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_step
    layer, outs = decode_step.run(steps=40, budget=48, d_model=256, heads=4, kv_heads=2, inter=512, prompts=(60, 1, 20), quiet=True)
    again = decode_step.run(steps=40, budget=48, d_model=256, heads=4, kv_heads=2, inter=512, prompts=(60, 1, 20), quiet=True)[1]
    assert all(torch.isfinite(o).all() for o in outs)
    for a, b in zip(outs, again):
        assert torch.equal(a, b)
    # one step before the capture and 40 replays (the capture itself runs nothing)
    assert layer.cache.seen.tolist() == [101, 42, 61]
    assert all(x <= 56 for x in layer.cache.lens.tolist()) and layer.cache.lens.tolist()[1] == 42


def test_example_without_eviction_equals_single_steps(D, wb):
    """The captured and the plain step agree bit for bit, and follow the cell and layers called one by one."""
    import torch
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_step
    res = []
    for captured in (False, True):
        layer = decode_step.Layer(256, 4, 2, 512, (9, 3), 64, 8, seed=3)
        g = torch.Generator(device="cuda").manual_seed(9)
        for s, n in enumerate((9, 3)):
            layer.prompt(s, torch.randn((n, 256), generator=g, device="cuda"))
        x = torch.randn((2, 256), generator=g, device="cuda")
        layer.step(x, evict=False)
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                layer.step(x, evict=False)
        outs = []
        for _ in range(5):
            graph.replay() if captured else layer.step(x, evict=False)
            outs.append(layer.out.clone())
            x.copy_(layer.out)
        res.append(outs)
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.parametrize("captured", ["decode", "prefill"])
def test_a_longer_prompt_leaves_captured_steps_alone(D, wb, captured):
    """A step (or a prompt) is captured, then prompts longer than any before go through the cell; replays
    give the bits of a cell that made the same calls without a capture."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(31)
    d_model, heads, kv, dim, n = 256, 4, 2, 64, 2
    w = [torch.randn((r, d_model), generator=g, device="cuda") * 0.08 for r in (heads * dim, kv * dim, kv * dim)]
    w.append(torch.randn((d_model, heads * dim), generator=g, device="cuda") * 0.08)
    prompt, long = (torch.randn((t, d_model), generator=g, device="cuda") for t in (9, 300))
    steps = torch.randn((6, n, d_model), generator=g, device="cuda")
    results = []
    for capture in (False, True):
        cell = wb.MhaCell(*w, d_model, heads, kv, dim, 400, 1, 0, wb.FP8E4M3)
        cache, other = (cache_for(D, s, heads, kv, dim, 400, torch.bfloat16) for s in (n, 1))
        x = prompt.clone() if captured == "prefill" else steps[0].clone()
        y, attn = torch.empty_like(x), torch.empty((x.shape[0], heads * dim), device="cuda")

        def call():
            if captured == "decode":
                D.mha_decode(cell, cache, x, y, attn)
            else:
                cache.lens.zero_()
                cache.seen.zero_()
                D.mha_prefill(cell, cache, 1, x, y, attn)

        call()
        if capture:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
        outs = []
        for i in range(1, 6):
            if i in (1, 3):  # each longer than all before
                other.lens.zero_()
                other.seen.zero_()
                p = long[: 100 * i].contiguous()
                D.mha_prefill(cell, other, 0, p, torch.empty_like(p))
                torch.cuda.synchronize()
                junk = [torch.full((1 << 16,), float("nan"), device="cuda") for _ in range(64)]  # noqa: F841
            x.mul_(0.5).add_(steps[i].repeat(5, 1)[: x.shape[0]])
            graph.replay() if capture else call()
            outs += [y.clone(), attn.clone()]
        cache.check_error()
        outs += [cache.k_pages.float(), cache.lens.clone()]
        results.append(outs)
        results.append(cache.page_table)
    (plain, t0, graphed, t1) = results
    for a, b in zip(plain[:-2], graphed[:-2]):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert torch.equal(plain[-2][t0.long()], graphed[-2][t1.long()]) and torch.equal(plain[-1], graphed[-1])


@pytest.mark.parametrize("accumulate", [False, True])
def test_step_leaves_sequences_out(D, wb, accumulate):
    """Sequences that have ended are left out of a captured step: one whose former pages belong to another
    now, one whose page-table row is no longer valid, one that is full. The others get the bits of a batch
    without them, and a sequence joins again when its flag says so."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(41)
    d_model, heads, kv, dim, n, per, page = 256, 4, 2, 64, 5, 3, 16
    w = [torch.randn((r, d_model), generator=g, device="cuda") * 0.08 for r in (heads * dim, kv * dim, kv * dim)]
    w.append(torch.randn((d_model, heads * dim), generator=g, device="cuda") * 0.08)
    cell = wb.MhaCell(*w, d_model, heads, kv, dim, 64, 1, 0, wb.FP8E4M3)
    pools = [torch.randn((n * per, page, kv, dim), generator=g, device="cuda") for _ in range(2)]
    table = torch.arange(n * per, dtype=torch.int32, device="cuda").reshape(n, per).contiguous()
    table[1] = table[0]  # its pages went to sequence 0
    table[2] = -1
    lens = torch.tensor([5, 20, 7, per * page, 30], dtype=torch.int32, device="cuda")
    flags = torch.tensor([1, 0, 0, 0, 1], dtype=torch.int32, device="cuda")
    stay = [0, 4]
    xs = torch.randn((6, n, d_model), generator=g, device="cuda")

    def cache_of(rows, pools):
        kw = {}
        if accumulate:
            kw = dict(weights=torch.full((len(rows), kv, per * page), 0.5, device="cuda"))
        return D.PagedKV(*[p.clone() for p in pools], table[rows].contiguous(), lens[rows].contiguous(), num_heads=heads,
                         seen=lens[rows].contiguous() + 3, **kw)

    cache, alone = cache_of(list(range(n)), pools), cache_of(stay, pools)
    x, y, attn = xs[0].clone(), torch.full((n, d_model), float("nan"), device="cuda"), torch.full((n, heads * dim), float("nan"), device="cuda")
    step = lambda: D.mha_decode(cell, cache, x, y, attn, accumulate=accumulate, active=flags)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    flags.zero_()
    step()  # makes the work buffers; nobody takes part
    assert not y.any() and not attn.any() and torch.equal(cache.lens, lens) and torch.equal(cache.k_pages, pools[0])
    flags.copy_(torch.tensor([1, 0, 0, 0, 1]))
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(xs[i])
        graph.replay()
        ya, aa = torch.empty((2, d_model), device="cuda"), torch.empty((2, heads * dim), device="cuda")
        D.mha_decode(cell, alone, xs[i][stay].contiguous(), ya, aa, accumulate=accumulate)
        assert torch.equal(y[stay], ya) and torch.equal(attn[stay], aa)
        assert not y[1:4].any() and not attn[1:4].any()
    cache.check_error()
    assert cache.lens.tolist() == [9, 20, 7, 48, 34] and cache.seen.tolist() == [12, 23, 10, 51, 37]
    for a, b in ((cache.k_pages, alone.k_pages), (cache.v_pages, alone.v_pages)):
        assert torch.equal(a, b)
    if accumulate:
        assert torch.equal(cache.weights[stay], alone.weights) and bool((cache.weights[1:4] == 0.5).all())
    flags.fill_(0)
    flags[1] = 1  # again, with pages of its own
    table2 = cache.page_table
    table2[1] = torch.arange(per, dtype=torch.int32) + per
    x.copy_(xs[4])
    graph.replay()
    cache.check_error()
    assert cache.lens.tolist() == [9, 21, 7, 48, 34] and bool(y[1].any()) and not y[0].any() and not y[2:].any()


def test_step_flags_are_checked(D, wb):
    import torch
    w = [torch.zeros((128, 128), device="cuda") for _ in range(4)]
    cell = wb.MhaCell(*w, 128, 2, 2, 64, 64, 1, 0, wb.FP8E4M3)
    cache = cache_for(D, 3, 2, 2, 64, 32, torch.bfloat16)
    x, y = torch.zeros((3, 128), device="cuda"), torch.zeros((3, 128), device="cuda")
    for bad in (torch.ones(3, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32)):
        with pytest.raises(ValueError):
            D.mha_decode(cell, cache, x, y, active=bad)
    assert cache.lens.tolist() == [0, 0, 0]


def test_prompt_into_a_row_that_was_used(D, wb):
    """A row whose length was reset, but not its count of tokens seen, takes a prompt as a new one does: the
    keys' positions are those of the attention just computed. A row that holds slots keeps them, with an error."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(51)
    d_model, heads, kv, dim = 256, 4, 2, 64
    w = [torch.randn((r, d_model), generator=g, device="cuda") * 0.08 for r in (heads * dim, kv * dim, kv * dim)]
    w.append(torch.randn((d_model, heads * dim), generator=g, device="cuda") * 0.08)
    cell = wb.MhaCell(*w, d_model, heads, kv, dim, 64, 1, 0, wb.FP8E4M3)
    x = torch.randn((20, d_model), generator=g, device="cuda")
    outs = []
    for used in (False, True):
        cache = cache_for(D, 3, heads, kv, dim, 64, torch.float32, records=True)
        cache.page_table.copy_(torch.arange(12, dtype=torch.int32).reshape(3, 4))
        if used:
            y = torch.empty((11, d_model), device="cuda")
            D.mha_prefill(cell, cache, 1, x[:11].flip(0).contiguous(), y)
            cache.weights.fill_(3.0)
            cache.lens.zero_()
        y = torch.empty((7, d_model), device="cuda")
        D.mha_prefill(cell, cache, 1, x[:7].contiguous(), y)
        cache.check_error()
        assert cache.lens.tolist() == [0, 7, 0] and cache.seen.tolist() == [0, 7, 0]
        assert cache.positions[1, :, :7].tolist() == [list(range(7))] * kv and not cache.weights[1, :, :7].any()
        only = torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda")
        for t in range(7, 12):
            y = torch.empty((3, d_model), device="cuda")
            D.mha_decode(cell, cache, x[t].expand(3, -1).contiguous(), y, active=only)
        outs += [y, cache.k_pages[4].clone(), cache.v_pages[4].clone(), cache.lens.clone(), cache.seen.clone()]
        outs[-3][12:], outs[-4][12:] = 0, 0  # slots not in use
    for a, b in zip(outs[:5], outs[5:]):
        assert torch.equal(a, b)
    k, positions = cache.k_pages.clone(), cache.positions.clone()
    D.mha_prefill(cell, cache, 1, x[:3].contiguous(), torch.empty((3, d_model), device="cuda"))
    with pytest.raises(wb.WelvetError) as e:
        cache.check_error()
    assert e.value.code == 1 and "holds" in str(e.value)
    cache.check_error()
    assert cache.lens.tolist() == [0, 12, 0] and cache.seen.tolist() == [0, 12, 0]
    assert torch.equal(k, cache.k_pages) and torch.equal(positions, cache.positions)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f8"])
@pytest.mark.parametrize("pos,mask,max_seq,heads,kv,dim", [(0, 1, 400, 8, 2, 128), (3, 3, 70, 4, 4, 96), (2, 1, 400, 6, 3, 40), (1, 3, 33, 16, 1, 128)])
def test_steps_against_64_bits(D, wb, dtype, pos, mask, max_seq, heads, kv, dim):
    """The cell's wiring (slots, positions, slopes, scale, window, heads' groups) held to the operators' own
    bound: prompts and single tokens of a Float32 cell, whose projections of up to 2^20 weights are sums in
    64 bits rounded once. Stored rows are within half a step of the type, attention is compared over what
    is stored, with the query off by its projection's rounding (2^-24) and its rotation's (three more of
    the pair): both move a score by no more than 4 * 2^-24 * 2 |q||k| scale."""
    import torch
    from test_kv_gpu import EPS, attend64, rotate64, rotation_bound, rows_of, stored64
    rng = np.random.default_rng(pos * 100 + dim)
    d_model, n, prompts, total = 256, 2, (150, 9), 160
    w = [(rng.standard_normal((r, d_model)) * 0.06).astype(np.float32) for r in (heads * dim, kv * dim, kv * dim)]
    w.append((rng.standard_normal((d_model, heads * dim)) * 0.06).astype(np.float32))
    cell = wb.MhaCell(*w, d_model, heads, kv, dim, max(max_seq, 150) if mask == 1 else max_seq, mask, pos, wb.FLOAT32)
    if mask == 3:
        prompts = (max_seq, 9)  # the cell's own prompt holds max_seq_len positions
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}[dtype]
    cache = cache_for(D, n, heads, kv, dim, total + 32, dt)
    xs = rng.standard_normal((n, total, d_model)).astype(np.float32)
    for s, m in enumerate(prompts):
        D.mha_prefill(cell, cache, s, torch.from_numpy(xs[s, :m].copy()).cuda(), torch.empty((m, d_model), device="cuda"))
    at = list(prompts)
    theta = 10000.0 if pos in (0, 3) else 0.0
    q64, k64, v64 = ((xs.astype(np.float64) @ m.T.astype(np.float64)) for m in w[:3])
    for step in range(10):
        x = np.stack([xs[s, at[s]] for s in range(n)])
        y, attn = torch.empty((n, d_model), device="cuda"), torch.empty((n, heads * dim), device="cuda")
        D.mha_decode(cell, cache, torch.from_numpy(x).cuda(), y, attn)
        at = [a + 1 for a in at]
    cache.check_error()
    assert cache.lens.tolist() == at
    q = np.stack([rotate64(q64[s, at[s] - 1].reshape(1, heads, dim), np.array([at[s] - 1.0]), theta)[0] for s in range(n)])
    for s in range(n):
        for pool, x64, turn in ((cache.k_pages, k64, theta), (cache.v_pages, v64, 0.0)):
            x = x64[s, : at[s]].reshape(at[s], kv, dim)
            want = rotate64(x, np.arange(at[s], dtype=np.float64), turn)
            st, half = stored64(want, dtype, 1.0)
            tol = half + (rotation_bound(x, turn) + EPS * (np.abs(x) + np.abs(np.roll(x, dim // 2, -1)))) * (1 + 2.0 ** -4)
            for h in range(kv):
                assert np.all(np.abs(rows_of(pool, cache.page_table, s, at[s], h) - st[:, h]) <= tol[:, h])
    scale = 1.0 / np.sqrt(dim)
    want, _, bound = attend64(torch.from_numpy(q).cuda(), cache.k_pages, cache.v_pages, cache.page_table, at, scale,
                              max_seq if mask == 3 else 0, pos in (2, 3))
    for s in range(n):
        for h in range(heads):
            k, v = (rows_of(p, cache.page_table, s, at[s], h // (heads // kv)) for p in (cache.k_pages, cache.v_pages))
            dq = 4 * EPS * 2 * scale * np.max(np.linalg.norm(k, axis=1)) * np.linalg.norm(q[s, h])
            bound[s, h] += 2 * dq * np.max(np.abs(v))
    got = attn.reshape(n, heads, dim).cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= bound)
    out = got.reshape(n, -1) @ w[3].T.astype(np.float64)
    assert np.all(np.abs(y.cpu().numpy() - out) <= 2 * EPS * np.abs(out) + 1e-30)


def test_steps_are_the_same_launches_after_a_longer_prompt(D, wb, monkeypatch):
    """The projections' prepared form of few rows stays available to a step whatever prompts came before it,
    and a step that is captured right after a prompt needs no allocation."""
    import ctypes

    import torch
    monkeypatch.setenv("WELVET_B200_GEMV_PREP", "1")  # the form that layers of 8192 rows take
    g = torch.Generator(device="cuda").manual_seed(61)
    d_model, heads, kv, dim, n = 1024, 9, 9, 128, 3
    w = [torch.randn((r, d_model), generator=g, device="cuda") * 0.03 for r in (heads * dim, kv * dim, kv * dim)]
    w.append(torch.randn((d_model, heads * dim), generator=g, device="cuda") * 0.03)
    x, long = (torch.randn((t, d_model), generator=g, device="cuda") for t in (n, 70))
    seen = []
    for before in (False, True):
        cell = wb.MhaCell(*w, d_model, heads, kv, dim, 400, 1, 0, wb.FP8E4M3)
        cache, other = (cache_for(D, s, heads, kv, dim, 400, torch.bfloat16) for s in (n, 1))
        y = torch.empty((n, d_model), device="cuda")
        if before:
            D.mha_prefill(cell, other, 0, long, torch.empty_like(long))
        D.mha_decode(cell, cache, x, y)
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            D.mha_decode(cell, cache, x, y)
        nodes = ctypes.c_size_t()
        assert ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
        graph.instantiate()
        graph.replay()
        seen.append((nodes.value, y))
    assert seen[0][0] == seen[1][0] and torch.equal(seen[0][1], seen[1][1])
    cell = wb.MhaCell(*w, d_model, heads, kv, dim, 400, 1, 0, wb.FP8E4M3)
    cache, other = (cache_for(D, s, heads, kv, dim, 400, torch.bfloat16) for s in (n, 1))
    D.mha_prefill(cell, other, 0, long, torch.empty_like(long))
    graph, y = torch.cuda.CUDAGraph(), torch.empty((n, d_model), device="cuda")
    with torch.cuda.graph(graph):
        D.mha_decode(cell, cache, x, y)
    other.lens.zero_()
    more = torch.cat([long] * 4)
    D.mha_prefill(cell, other, 0, more, torch.empty_like(more))
    for _ in range(2):
        graph.replay()
    assert torch.equal(y, seen[0][1]) and cache.lens.tolist() == [2] * n
