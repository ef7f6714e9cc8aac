"""The operators of a decode step, each in a plain form and through welvet.cuda_b200.decode.

    append  new tokens' keys and values, rotated and cast, into a paged key-value cache
    attend  attention of one new token per sequence over that cache
    evict   the cache cut back to a budget by accumulated attention weight
    gemv    matrix-vector products with 4-bit weights and group scales

A cache is a pool of pages [pages, page slots, key-value heads, head dim] for keys and one for
values, a page table [sequences, pages of a sequence] and lengths. Head counts and widths are
the MHA cell's (16 x 128 heads) and common grouped-query ones; the layer shapes are the Dense
layers' (4096 x 4096, 4096 / 14336, 16384 -> 65536).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "f8": 1}
SCALE = {"f32": 1.0, "f16": 1.0, "bf16": 1.0, "f8": 1.0 / 64.0}  # what one stored unit stands for
BITS = {"f32": torch.int32, "f16": torch.int16, "bf16": torch.int16, "f8": torch.uint8}  # a page's values, moved as they are
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
THETA = 10000.0
MOST = 8.0e8  # bytes that a drawn cache holds, or a drawn append moves, at most


def listed():
    return [
        # one sequence of a chat at its start on the MHA cell's heads: latency
        dict(name="attend one short", op="attend", batch=1, heads=16, kv_heads=16, dim=128, page=16, dtype="bf16",
             lo=500, hi=500, window=0, alibi=False, sums=False),
        # a serving batch of conversations of very different lengths, one of them just begun
        dict(name="attend batch ragged", op="attend", batch=64, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16",
             lo=1, hi=8191, window=0, alibi=False, sums=False),
        # a few long documents over an 8-bit cache
        dict(name="attend long", op="attend", batch=6, heads=32, kv_heads=8, dim=128, page=64, dtype="f8",
             lo=30000, hi=131072, window=0, alibi=False, sums=False),
        # the budgeted cache: the step also sums the attention weights that eviction goes by
        dict(name="attend sums f16", op="attend", batch=24, heads=24, kv_heads=8, dim=64, page=32, dtype="f16",
             lo=900, hi=5003, window=0, alibi=False, sums=True),
        # sliding window and linear biases over an unquantized cache
        dict(name="attend window f32", op="attend", batch=7, heads=12, kv_heads=6, dim=80, page=24, dtype="f32",
             lo=300, hi=6001, window=2048, alibi=True, sums=False),
        # one decode step's new tokens of a serving batch
        dict(name="append step", op="append", batch=64, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16",
             start=3000, lo=1, hi=1),
        # prompts of several sequences at once into an 8-bit cache
        dict(name="append prompts", op="append", batch=6, heads=32, kv_heads=8, dim=128, page=64, dtype="f8",
             start=17, lo=100, hi=6007),
        # each sequence a few tokens over its budget: a row or two per head moves
        dict(name="evict stream", op="evict", batch=32, kv_heads=8, dim=128, page=16, dtype="bf16",
             lo=1025, hi=1056, keep=1024, sinks=4, recent=256),
        # long contexts cut to a quarter
        dict(name="evict long", op="evict", batch=3, kv_heads=8, dim=128, page=64, dtype="f8",
             lo=40000, hi=65001, keep=16384, sinks=4, recent=2048),
        # one token through a square projection
        dict(name="gemv int4 4096", op="gemv", rows=4096, cols=4096, batch=1, code="int4", group=128, act="linear", bias=False),
        # a few sequences through an odd-sized layer with zero points
        dict(name="gemv uint4 odd", op="gemv", rows=14331, cols=4090, batch=7, code="uint4", group=64, act="silu", bias=True),
        # the widest layer, one token
        dict(name="gemv fp4 wide", op="gemv", rows=65536, cols=16384, batch=1, code="fp4", group=32, act="relu", bias=True),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "evict", "gemv", "gemv"])
    if op == "gemv":
        code = rng.choice(["int4", "uint4", "fp4"])
        c = dict(op=op, rows=log_int(rng, 256, 65536), cols=log_int(rng, 256, 16384), batch=rng.randint(1, 8), code=code,
                 group=rng.choice([32, 64, 128]), act=rng.choice(["linear", "relu", "silu"]), bias=rng.random() < 0.5)
        return c
    dtype = rng.choice(["f32", "f16", "bf16", "bf16", "f8"])
    kv, dim, page = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([16, 24, 32, 64])
    batch = log_int(rng, 1, 64)
    row = 2 * kv * dim * SIZE[dtype]
    most = max(64, min(131072, int(MOST / (row * batch))))
    if op == "attend":
        hi = log_int(rng, 33, most)
        sums = rng.random() < 0.4
        return dict(op=op, batch=batch, heads=kv * rng.choice([1, 2, 3, 4, 5, 8] if kv < 16 else [1, 2, 4]), kv_heads=kv, dim=dim,
                    page=page, dtype=dtype, lo=log_int(rng, 1, hi), hi=hi,
                    window=0 if rng.random() < 0.7 else log_int(rng, 16, hi), alibi=rng.random() < 0.2, sums=sums)
    if op == "append":
        group = rng.choice([1, 2, 4])
        hi = log_int(rng, 1, max(1, min(8192, int(MOST / (batch * dim * kv * (8 + 8 * group + 2 * SIZE[dtype]))))))
        return dict(op=op, batch=batch, heads=kv * group, kv_heads=kv, dim=dim, page=page, dtype=dtype,
                    start=rng.randint(0, 5000), lo=log_int(rng, 1, hi), hi=hi)
    hi = log_int(rng, 64, min(65536, most))
    lo = rng.randint(hi // 2, hi)
    keep = rng.randint(hi // 4, max(hi // 4, lo - 1))
    return dict(op=op, batch=batch, kv_heads=kv, dim=dim, page=page, dtype=dtype, lo=lo, hi=hi, keep=keep,
                sinks=rng.randint(0, 4), recent=rng.randint(0, keep // 3))


def counts(case):
    """The sequences' lengths (of an append: their numbers of new tokens), spread over [lo, hi]."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    return [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) if n > 1 else hi for i in range(n)]


def work(case):
    if case["op"] == "gemv":
        r, c, b = case["rows"], case["cols"], case["batch"]
        groups = -(-c // case["group"])
        return {"bytes": r * ((c + 1) // 2) + r * groups * (3 if case["code"] == "uint4" else 2) + 4 * b * (r + c) + (8 * r if case["bias"] else 0),
                "flops": 2 * r * c * b}
    kv, dim, size = case["kv_heads"], case["dim"], SIZE[case["dtype"]]
    n = counts(case)
    if case["op"] == "append":
        t = sum(n)
        return {"bytes": t * dim * (4 * (2 * kv + 2 * case["heads"]) + 2 * kv * size), "flops": 6 * t * dim * (kv + case["heads"])}
    if case["op"] == "attend":
        seen = [min(x, case["window"]) if case["window"] else x for x in n]
        return {"bytes": sum(seen) * kv * dim * 2 * size + 8 * case["batch"] * case["heads"] * dim + (8 * kv * sum(n) if case["sums"] else 0),
                "flops": 4 * sum(seen) * case["heads"] * dim}
    # weights and positions of every slot; of the kept rows at or above `keep` about the share (len - keep) / len moves
    cut = [x for x in n if x > case["keep"]]
    moved = sum(kv * case["keep"] * (x - case["keep"]) / x for x in cut)
    return {"bytes": sum(8 * kv * x for x in cut) + moved * (2 * 2 * dim * size + 16), "flops": sum(kv * x for x in cut)}


# ---------------------------------------------------------------- inputs


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def cache_of(case, g, slots, zeros=False):
    """Pools, page table and the number of slots of a sequence. The table's pages lie in random order."""
    n, page = case["batch"], case["page"]
    per = -(-slots // page)
    pages = n * per + 1
    shape = (pages, page, case["kv_heads"], case["dim"])
    dt = DTYPES[case["dtype"]]

    def pool():
        x = torch.zeros(shape, device="cuda") if zeros else torch.randn(shape, generator=g, device="cuda")
        return stored(x, dt, SCALE[case["dtype"]])

    table = torch.randperm(pages, generator=g, device="cuda")[: n * per].reshape(n, per).to(torch.int32)
    return {"k_pages": pool(), "v_pages": pool(), "table": table, "slots": per * page}


def ints(values, order):
    return torch.tensor([values[i] for i in order], dtype=torch.int32, device="cuda")


def inputs(case, seed):
    """The tensors that a program holds before the call, from the seed alone."""
    g = generator(seed)
    if case["op"] == "gemv":
        r, c, b, grp = case["rows"], case["cols"], case["batch"], case["group"]
        groups, half = -(-c // grp), (c + 1) // 2
        codes = torch.empty(r, half, dtype=torch.uint8, device="cuda")
        for at in range(0, r, 8192):  # by rows: the unquantized values of the widest layer are 4 GB
            w = torch.randn(min(8192, r - at), 2 * half, generator=g, device="cuda")
            if case["code"] == "fp4":  # sign, then the magnitude's nearest step of 0 .5 1 1.5 2 3 4 6
                m = torch.bucketize(w.abs() * 2.0, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda"))
                q = (m + 8 * (w < 0)).to(torch.uint8)
            else:
                q = (torch.round(w * 2.5).clamp(-8, 7).to(torch.int16) + (8 if case["code"] == "uint4" else 0)).to(torch.uint8) & 15
            if c % 2:
                q[:, -1] = 0
            codes[at: at + w.shape[0]] = q[:, 0::2] | (q[:, 1::2] << 4)
            del w, q
        s = {"codes": codes, "x": torch.randn(b, c, generator=g, device="cuda"), "y": torch.empty(b, r, device="cuda"),
             "scales": (torch.rand(r, groups, generator=g, device="cuda") * 0.01 + 0.002).to(torch.float16), "zeros": None, "bias": None}
        if case["code"] == "uint4":
            s["zeros"] = torch.randint(5, 11, (r, groups), generator=g, device="cuda", dtype=torch.uint8)
        if case["bias"]:
            s["bias"] = torch.randn(r, generator=g, device="cuda") * 0.1
        return s
    n, h, kv, d = case["batch"], case.get("heads"), case["kv_heads"], case["dim"]
    order = np.random.RandomState(seed % 2**32).permutation(n)
    if case["op"] == "append":
        new = ints(counts(case), order)
        t = int(sum(counts(case)))
        s = cache_of(case, g, case["start"] + max(counts(case)), zeros=True)
        cu = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        cu[1:] = torch.cumsum(new, 0)
        s |= {"q": torch.randn(t, h, d, generator=g, device="cuda"), "k": torch.randn(t, kv, d, generator=g, device="cuda"),
              "v": torch.randn(t, kv, d, generator=g, device="cuda"), "q_out": torch.empty(t, h, d, device="cuda"), "cu": cu,
              # sequences start at different lengths; one that was cut back has seen more tokens than it holds
              "start": torch.randint(case["start"] // 2, case["start"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)}
        s["start_seen"] = s["start"] * 2
        s |= {"lens": torch.empty_like(s["start"]), "seen": torch.empty_like(s["start"])}
        return s
    lens = ints(counts(case), order)
    s = cache_of(case, g, max(counts(case)))
    s["lens"] = lens
    if case["op"] == "attend":
        s |= {"q": torch.randn(n, h, d, generator=g, device="cuda") * 1.5, "out": torch.empty(n, h, d, device="cuda")}
        if case["sums"]:
            s["weights_in"] = torch.rand(n, kv, s["slots"], generator=g, device="cuda")
            s["weights"] = torch.zeros_like(s["weights_in"])
        return s
    # sums of softmax weights are spread over orders of magnitude; many slots of the newest tokens have none yet
    w = torch.exp(3.0 * torch.randn(n, kv, s["slots"], generator=g, device="cuda") - 4.0)
    s["weights_in"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.02, torch.zeros_like(w), w)
    # half of the tokens seen are still there: every second position, one of each pair
    s["positions_in"] = (2 * torch.arange(s["slots"], device="cuda", dtype=torch.int32)
                         + torch.randint(0, 2, w.shape, generator=g, device="cuda", dtype=torch.int32))
    s |= {"seen": 2 * lens, "lens_in": lens, "lens": torch.empty_like(lens), "weights": torch.zeros_like(w),
          "positions": torch.zeros_like(s["positions_in"])}
    return s


def prepare(case, seed):
    s = inputs(case, seed)
    s["case"] = case
    if own:  # the mounted layer, or the handle over the pools, that a serving program makes once
        from welvet.cuda_b200 import decode

        if case["op"] == "gemv":
            s["layer"] = decode.GroupDense.from_codes(s["codes"], s["scales"], case["cols"], case["group"], decode.CODES[case["code"]],
                                                      zeros=s["zeros"], act=decode.ACTS[case["act"]],
                                                      bias=None if s["bias"] is None else s["bias"].double().cpu().numpy())
        else:
            scale = SCALE[case["dtype"]]
            s["cache"] = decode.PagedKV(s["k_pages"], s["v_pages"], s["table"], s["lens"], num_heads=case.get("heads") or case["kv_heads"],
                                        seen=s.get("seen"), weights=s.get("weights"), positions=s.get("positions"),
                                        k_scale=scale, v_scale=scale)
    return s


# ---------------------------------------------------------------- the calls


def run(state):
    case = state["case"]
    if own:
        return RUN_OWN[case["op"]](state, case)
    return RUN_PLAIN[case["op"]](state, case)


def own_append(s, case):
    s["cache"].append(s["k"], s["v"], q=s["q"], q_out=s["q_out"], cu_tokens=s["cu"], theta=THETA, start=s["start"],
                      start_seen=s["start_seen"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "q": s["q_out"], "lens": s["lens"], "seen": s["seen"]}


def own_attend(s, case):
    if case["sums"]:
        s["cache"].attend(s["q"], s["out"], window=case["window"], alibi=case["alibi"], accumulate=True, weights_in=s["weights_in"])
        return {"out": s["out"], "weights": s["weights"]}
    s["cache"].attend(s["q"], s["out"], window=case["window"], alibi=case["alibi"])
    return {"out": s["out"]}


def own_evict(s, case):
    s["cache"].evict(case["keep"], sinks=case["sinks"], recent=case["recent"], lens_in=s["lens_in"], weights_in=s["weights_in"],
                     positions_in=s["positions_in"])
    return evicted(s)


def evicted(s):
    return {k: s[k] for k in ("k_pages", "v_pages", "weights", "positions", "lens")}


def own_gemv(s, case):
    s["layer"].forward(s["x"], s["y"])
    return s["y"]


# ---------------------------------------------------------------- plain forms


def stored(x, dt, scale):
    x = x / scale
    return (x.clamp(-448.0, 448.0) if dt is torch.float8_e4m3fn else x).to(dt)


def plain_append(s, case):
    cu, page, dt = s["cu"].long(), case["page"], DTYPES[case["dtype"]]
    t = torch.arange(s["k"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[seq]
    slot, pos = s["start"].long()[seq] + i, s["start_seen"].long()[seq] + i
    half = case["dim"] // 2
    # the angle is a function of two given numbers; 32 bits would lose it at position 10^4
    angle = pos.double()[:, None] * THETA ** (-2.0 * torch.arange(half, device="cuda").double() / case["dim"])
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotate(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)

    at = s["table"].long()[seq, slot // page], slot % page
    bits, scale = BITS[case["dtype"]], SCALE[case["dtype"]]
    s["k_pages"].view(bits)[at] = stored(rotate(s["k"]), dt, scale).view(bits)
    s["v_pages"].view(bits)[at] = stored(s["v"], dt, scale).view(bits)
    s["q_out"].copy_(rotate(s["q"]))
    n = (cu[1:] - cu[:-1]).to(torch.int32)
    torch.add(s["start"], n, out=s["lens"])
    torch.add(s["start_seen"], n, out=s["seen"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "q": s["q_out"], "lens": s["lens"], "seen": s["seen"]}


def slopes(heads):
    return torch.pow(2.0, -8.0 * torch.arange(1, heads + 1, device="cuda").float() / heads)


def plain_attend(s, case):
    n, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    scale = SCALE[case["dtype"]]
    table, bits, dt = s["table"].long(), BITS[case["dtype"]], DTYPES[case["dtype"]]
    k = s["k_pages"].view(bits)[table].view(dt).reshape(n, -1, kv, d).float()  # [n, slots, kv, d]
    z = torch.einsum("bkgd,bskd->bkgs", s["q"].reshape(n, kv, h // kv, d), k) * (scale / math.sqrt(d))
    del k
    j, last = torch.arange(s["slots"], device="cuda"), s["lens"].long()[:, None] - 1
    if case["alibi"]:
        z -= slopes(h).reshape(1, kv, h // kv, 1) * (last - j).float()[:, None, None]
    seen = j <= last
    if case["window"]:
        seen = seen & (j > last - case["window"])
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    w = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-3.0e38))
    w = w / w.sum(-1, keepdim=True).clamp(min=1.0e-38)
    v = s["v_pages"].view(bits)[table].view(dt).reshape(n, -1, kv, d).float() * seen[:, :, None, None]
    s["out"].copy_((torch.einsum("bkgs,bskd->bkgd", w, v) * scale).reshape(n, h, d))
    if case["sums"]:
        s["weights"].copy_(torch.where((j <= last)[:, None], s["weights_in"] + w.sum(2), s["weights"]))
        return {"out": s["out"], "weights": s["weights"]}
    return {"out": s["out"]}


def plain_evict(s, case):
    keep, page = case["keep"], case["page"]
    n, kv = s["weights_in"].shape[:2]
    j = torch.arange(s["slots"], device="cuda")
    lens = s["lens_in"].long()[:, None, None]
    live = (j < lens).expand_as(s["weights_in"])
    cut = lens > keep
    pos = s["positions_in"]
    safe = (pos < case["sinks"]) | (pos >= s["seen"][:, None, None] - case["recent"])
    key = torch.where(safe, math.inf, s["weights_in"]).masked_fill(~live, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))
    stays = live & ((rank < keep) | ~cut)
    b, hd, dst = torch.nonzero(cut & (j < keep) & ~stays, as_tuple=True)
    src = torch.nonzero(cut & (j >= keep) & stays, as_tuple=True)[2]
    stay_low = live & (~cut | (j < keep))
    weights = s["weights_in"].clone()
    weights[b, hd, dst] = s["weights_in"][b, hd, src]
    positions = pos.clone()
    positions[b, hd, dst] = pos[b, hd, src]
    s["weights"].copy_(torch.where(stay_low, weights, s["weights"]))
    s["positions"].copy_(torch.where(stay_low, positions, s["positions"]))
    table = s["table"].long()
    to, frm = (table[b, dst // page], dst % page, hd), (table[b, src // page], src % page, hd)
    bits = BITS[case["dtype"]]
    k, v = s["k_pages"].view(bits), s["v_pages"].view(bits)
    k[to] = k[frm]
    v[to] = v[frm]
    torch.clamp(s["lens_in"], max=keep, out=s["lens"])
    return evicted(s)


def nibbles(codes, cols):
    return torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)[:, :cols]


def spread(per_group, group, cols):
    return per_group.repeat_interleave(group, dim=1)[:, :cols]


def plain_gemv(s, case):
    cols, group = case["cols"], case["group"]
    c = nibbles(s["codes"], cols)
    if case["code"] == "fp4":
        w = torch.tensor(FP4, device="cuda")[c.int()]
    elif case["code"] == "int4":
        w = ((c ^ 8).float() - 8.0)
    else:
        w = c.float() - spread(s["zeros"].float(), group, cols)
    w *= spread(s["scales"].float(), group, cols)
    y = s["x"] @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["act"] == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    s["y"].copy_(y)
    return s["y"]


RUN_PLAIN = {"append": plain_append, "attend": plain_attend, "evict": plain_evict, "gemv": plain_gemv}
RUN_OWN = {"append": own_append, "attend": own_attend, "evict": own_evict, "gemv": own_gemv}


# ---------------------------------------------------------------- in 64 bits, from the definitions


def exact(case, seed):
    return EXACT[case["op"]](case, inputs(case, seed))


def exact_append(case, s):
    d, page, scale = case["dim"], case["page"], SCALE[case["dtype"]]
    half = d // 2
    kp, vp, q = s["k_pages"].float().double(), s["v_pages"].float().double(), torch.zeros_like(s["q"], dtype=torch.float64)
    cu, start, seen = (s[k].tolist() for k in ("cu", "start", "start_seen"))
    lens, total = [], []
    freq = torch.tensor([THETA ** (-(2.0 * i) / d) for i in range(half)], dtype=torch.float64, device="cuda")
    most = 448.0 if case["dtype"] == "f8" else math.inf
    for b in range(case["batch"]):
        rows = range(cu[b], cu[b + 1])
        n = len(rows)
        turn = torch.polar(torch.ones(1, 1, 1, dtype=torch.float64, device="cuda"),
                           (torch.arange(seen[b], seen[b] + n, device="cuda").double()[:, None] * freq)[:, None])
        k, v, x = (s[m][cu[b]: cu[b + 1]].double() for m in ("k", "v", "q"))
        k, x = (torch.complex(m[..., :half].contiguous(), m[..., half:].contiguous()) * turn for m in (k, x))
        slot = torch.arange(start[b], start[b] + n, device="cuda")
        pages = s["table"][b].long()[torch.div(slot, page, rounding_mode="floor")]
        kp[pages, slot % page] = (torch.cat([k.real, k.imag], -1) / scale).clamp(-most, most)
        vp[pages, slot % page] = (v / scale).clamp(-most, most)
        q[cu[b]: cu[b + 1]] = torch.cat([x.real, x.imag], -1)
        lens.append(start[b] + n)
        total.append(seen[b] + n)
    return {"k_pages": kp, "v_pages": vp, "q": q, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "seen": torch.tensor(total, dtype=torch.int32, device="cuda")}


def exact_attend(case, s):
    h, kv, d, page, scale = case["heads"], case["kv_heads"], case["dim"], case["page"], SCALE[case["dtype"]]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    sums = s["weights"].double() if case["sums"] else None
    keys, values = s["k_pages"].float(), s["v_pages"].float()
    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        used = s["table"][b, : -(-n // page)].long()
        if sums is not None:
            sums[b, :, :n] = s["weights_in"][b, :, :n].double()
        for g in range(kv):
            k = keys[used, :, g].reshape(-1, d)[first:n].double() * scale
            v = values[used, :, g].reshape(-1, d)[first:n].double() * scale
            heads = slice(g * (h // kv), (g + 1) * (h // kv))
            z = s["q"][b, heads].double() @ k.T / math.sqrt(d)
            if case["alibi"]:
                for i in range(h // kv):
                    m = 2.0 ** (-8.0 * (g * (h // kv) + i + 1) / h)
                    z[i] += m * (torch.arange(first, n, device="cuda").double() - (n - 1))
            w = torch.softmax(z, -1)
            out[b, heads] = w @ v
            if sums is not None:
                sums[b, g, first:n] += w.sum(0)
    return {"out": out, "weights": sums} if case["sums"] else {"out": out}


def exact_evict(case, s):
    keep, page = case["keep"], case["page"]
    kp, vp, table = s["k_pages"].float().double(), s["v_pages"].float().double(), s["table"].cpu().numpy()
    win, pin = s["weights_in"].cpu().numpy(), s["positions_in"].cpu().numpy()
    w, p = s["weights"].cpu().numpy().astype(np.float64), s["positions"].cpu().numpy()
    lens, seen = s["lens_in"].cpu().numpy(), s["seen"].cpu().numpy()
    moves = [[], [], [], [], []]
    for b in range(case["batch"]):
        n = int(lens[b])
        for g in range(case["kv_heads"]):
            m = min(n, keep)
            w[b, g, :m], p[b, g, :m] = win[b, g, :m], pin[b, g, :m]
            if n <= keep:
                continue
            safe = (pin[b, g, :n] < case["sinks"]) | (pin[b, g, :n] >= seen[b] - case["recent"])
            order = np.lexsort((np.arange(n), -win[b, g, :n].astype(np.float64), ~safe))
            stays = np.zeros(n, bool)
            stays[order[:keep]] = True
            dst, src = np.flatnonzero(~stays[:keep]), keep + np.flatnonzero(stays[keep:])
            w[b, g, dst], p[b, g, dst] = win[b, g, src], pin[b, g, src]
            for to, x in zip(moves, (table[b, dst // page], dst % page, table[b, src // page], src % page, np.full(len(dst), g))):
                to.append(x)
        lens[b] = min(n, keep)
    if moves[0]:
        a, i, c, j, g = (torch.from_numpy(np.concatenate(x).astype(np.int64)).cuda() for x in moves)
        kp[a, i, g], vp[a, i, g] = kp[c, j, g], vp[c, j, g]
    return {"k_pages": kp, "v_pages": vp, "weights": w, "positions": p, "lens": lens}


def exact_gemv(case, s):
    cols, group, rows = case["cols"], case["group"], case["rows"]
    x = s["x"].double()
    y = torch.empty(case["batch"], rows, dtype=torch.float64, device="cuda")
    which = torch.arange(cols, device="cuda") // group
    values = torch.tensor(FP4 if case["code"] == "fp4" else [i - 16 * (i > 7) for i in range(16)] if case["code"] == "int4" else list(range(16)),
                          dtype=torch.float64, device="cuda")
    for at in range(0, rows, 4096):
        c = s["codes"][at: at + 4096].long()
        both = torch.empty(c.shape[0], 2 * c.shape[1], dtype=torch.int64, device="cuda")
        both[:, 0::2], both[:, 1::2] = c % 16, c // 16
        w = values[both[:, :cols]]
        if s["zeros"] is not None:
            w = w - s["zeros"][at: at + 4096].double()[:, which]
        y[:, at: at + 4096] = x @ (w * s["scales"][at: at + 4096].double()[:, which]).T
    if s["bias"] is not None:
        y = y + s["bias"].double()
    return torch.relu(y) if case["act"] == "relu" else y * torch.sigmoid(y) if case["act"] == "silu" else y


EXACT = {"append": exact_append, "attend": exact_attend, "evict": exact_evict, "gemv": exact_gemv}
