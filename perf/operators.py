"""Two operators measured on the sizes they meet: feature rows held in 8 or 4 bits (written, read back), and draws of
indices from scores under temperature, top-k, top-p and min-p.

`own = False` computes them in elementary torch operations; `own = True` through point_slam_amd.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_QMAX = {"int8": 127.0, "int4": 7.0, "e4m3": 448.0}
_BITS = {"int8": 8, "int4": 4, "e4m3": 8}


def _store(name, n, heads, dim, group, fmt, dtype, rows, capacity):
    return {"name": name, "op": "store", "n": n, "heads": heads, "dim": dim, "group": group, "fmt": fmt, "dtype": dtype,
            "rows": rows, "capacity": capacity}


def _read(name, n, heads, dim, group, fmt, dtype, capacity):
    return {"name": name, "op": "read", "n": n, "heads": heads, "dim": dim, "group": group, "fmt": fmt, "dtype": dtype,
            "rows": "any", "capacity": capacity}


def _pick(name, rows, cols, draws, dtype, kind, temperature, top_k, top_p, min_p, per_row):
    return {"name": name, "op": "draw", "rows": rows, "cols": cols, "draws": draws, "dtype": dtype, "kind": kind,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "per_row": per_row}


def listed():
    return [
        # the three points of ONE new surface location: geometry and colour row of each, appended behind the map
        _store("store_location", 3, 2, 32, 32, "int8", "f32", "tail", 4096),
        # the new points of one mapped frame (18 000 locations x 3), the block a rank sends in an exchange
        _store("store_frame", 54000, 2, 32, 32, "int8", "f32", "tail", 1000000),
        # the whole map at the default capacity, as a checkpoint takes it
        _store("store_map", 2500000, 2, 32, 32, "e4m3", "f32", "tail", 2500000),
        # a cache of eight heads of 128, 4 bits with a scale to 32 values, rows scattered over the cache
        _store("store_heads_int4", 16384, 8, 128, 32, "int4", "bf16", "some", 65536),
        # ragged: odd row count, three heads of 80, fp16, padding rows (-1) among the destinations
        _store("store_ragged", 4099, 3, 80, 16, "int8", "f16", "padded", 20011),
        # eight neighbours of the five samples of 5 000 rays, gathered from a map of a million points
        _read("read_neighbours", 200000, 2, 32, 32, "int8", "f32", 1000000),
        # a long context read back for a product in bf16
        _read("read_context", 65536, 8, 128, 128, "e4m3", "bf16", 131072),
        # one row, one draw: the latency of a single decision
        _pick("draw_one", 1, 2048, 1, "f32", "token", 0.8, 50, 0.9, 0.0, False),
        # a batch of token rows with parameters of their own
        _pick("draw_batch", 64, 131072, 1, "bf16", "token", 0.9, 200, 0.95, 0.02, True),
        # odd sizes, fp16, a few draws from each row, only the relative floor
        _pick("draw_ragged", 7, 50021, 3, "f16", "token", 1.3, 0, 1.0, 0.05, False),
        # a tracked frame of 640 x 480: 200 iterations of 5 000 pixels by colour gradient, all at once
        _pick("draw_track", 1, 307200, 1000000, "f32", "image", 1.0, 75000, 1.0, 0.0, False),
        # a mapping window of twelve 1200 x 680 frames: 300 iterations of 416 pixels of each frame
        _pick("draw_window", 12, 816000, 124800, "f32", "image", 0.7, 0, 0.9, 0.0, False),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "store", "read", "draw", "draw", "draw"])
    if op in ("store", "read"):
        fmt = rng.choice(["int8", "e4m3", "int4"])
        dtype = rng.choice(["f32", "bf16", "f16"])
        group = rng.choice([8, 16, 32, 64, 80, 128])
        dim = group * rng.randint(1, max(1, 256 // group))
        heads = rng.choice([1, 2, 3, 4, 8])
        n = _logint(rng, 1, max(1, 100_000_000 // (heads * dim)))
        capacity = n + _logint(rng, 1, 200000)
        if op == "read":
            return _read("", n, heads, dim, group, fmt, dtype, capacity)
        return _store("", n, heads, dim, group, fmt, dtype, rng.choice(["tail", "some", "padded"]), capacity)
    if rng.random() < 0.5:
        rows = _logint(rng, 1, 128)
        cols = _logint(rng, 2, min(262144, 9_000_000 // rows))
        draws = rng.choice([1, 1, 1, 2, 5, 16])
        kind, dtype = "token", rng.choice(["f32", "bf16", "f16"])
    else:
        rows = rng.randint(1, 12)
        cols = _logint(rng, 10000, 816000)
        draws = _logint(rng, 100, 1_400_000 // rows)
        kind, dtype = "image", "f32"
    top_k = rng.choice([0, _logint(rng, 1, cols)])
    top_p = rng.choice([1.0, round(rng.uniform(0.3, 0.999), 3)])
    min_p = rng.choice([0.0, round(math.exp(rng.uniform(math.log(1e-4), math.log(0.5))), 5)])
    return _pick("", rows, cols, draws, dtype, kind, round(rng.uniform(0.3, 2.0), 2), top_k, top_p, min_p, rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _row_inputs(case, seed):
    """Values of the rows and where they go.  Feature rows start as N(0, 0.1^2) and spread as they are trained: every row
    has a magnitude of its own."""
    g = _generator(seed)
    n, h, d, cap = case["n"], case["heads"], case["dim"], case["capacity"]
    mag = torch.empty(n, h, 1, device="cuda").normal_(0, 0.7, generator=g).exp_().mul_(0.1)
    values = torch.empty(n, h, d, device="cuda").normal_(generator=g).mul_(mag).to(_DT[case["dtype"]])
    rows = None
    if case["rows"] in ("some", "padded"):
        rows = torch.randperm(cap, device="cuda", generator=g)[:n]
        if case["rows"] == "padded":
            rows = torch.where(torch.rand(n, device="cuda", generator=g) < 0.1, torch.full_like(rows, -1), rows)
    return values, rows


def _score_inputs(case, seed):
    g = _generator(seed)
    r, v, n = case["rows"], case["cols"], case["draws"]
    mask = None
    if case["kind"] == "image":
        # log of a colour-gradient magnitude: heavy-tailed, a sixth of the image flat (gradient zero exactly), holes in the depth
        grad = torch.empty(r, v, device="cuda").normal_(generator=g).abs_().mul_(0.05)
        grad *= torch.empty(r, v, device="cuda").normal_(0, 0.8, generator=g).exp_()
        grad[torch.rand(r, v, device="cuda", generator=g) < 0.16] = 0.0
        scores = (grad + 1e-3).log_()
        mask = torch.rand(r, v, device="cuda", generator=g) >= 0.08
    else:
        scores = torch.empty(r, v, device="cuda").normal_(0, 2.0, generator=g)
        peaks = torch.randint(v, (r, min(8, v)), device="cuda", generator=g)
        scores.scatter_(1, peaks, 6.0 + 3.0 * torch.rand(r, min(8, v), device="cuda", generator=g))
    scores = scores.to(_DT[case["dtype"]])
    u = torch.rand(r, n, device="cuda", generator=g)
    par = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    if case["per_row"]:
        j = torch.rand(4, r, device="cuda", generator=g)
        par["temperature"] = case["temperature"] * (0.7 + 0.6 * j[0])
        par["top_k"] = (case["top_k"] * (0.5 + 0.5 * j[1])).to(torch.int32)
        par["top_p"] = 1.0 - (1.0 - case["top_p"]) * (0.5 + j[2])
        par["min_p"] = case["min_p"] * (0.5 + j[3])
    return scores, mask, u, par


def prepare(case, seed):
    if case["op"] == "draw":
        scores, mask, u, par = _score_inputs(case, seed)
        return {"case": case, "scores": scores, "mask": mask, "u": u, "par": par}
    values, rows = _row_inputs(case, seed)
    first = case["capacity"] - case["n"] if rows is None else 0
    st = {"case": case, "values": values, "rows": rows, "first": first}
    if own:
        from point_slam_amd.row_store import QuantizedRows
        st["store"] = QuantizedRows(case["capacity"], case["heads"], case["dim"], case["fmt"], case["group"], device="cuda")
    else:
        st["store"] = _plain_store(case)
    if case["op"] == "read":
        # the whole cache is in place before the call; the call asks for rows of it, any of them, some twice
        filled = dict(case, n=case["capacity"], rows="tail")
        held, _ = _row_inputs(filled, seed)
        if own:
            st["store"].write(held, first=0)
        else:
            _plain_write(st["store"], case, held, None, 0)
        st["values"] = None
        st["rows"] = torch.randint(case["capacity"], (case["n"],), device="cuda", generator=_generator(seed + 1))
    return st


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_store(case):
    c, h, d = case["capacity"], case["heads"], case["dim"]
    codes = torch.zeros(c, h, d * _BITS[case["fmt"]] // 8, device="cuda",
                        dtype=torch.float8_e4m3fn if case["fmt"] == "e4m3" else torch.int8 if case["fmt"] == "int8" else torch.uint8)
    return {"codes": codes, "scales": torch.zeros(c, h, d // case["group"], device="cuda")}


def _plain_write(store, case, values, rows, first):
    n, h, d, g, qmax = values.shape[0], case["heads"], case["dim"], case["group"], _QMAX[case["fmt"]]
    x = values.float().reshape(n, h, d // g, g)
    amax = x.abs().amax(-1)
    # a division, not a product with the rounded reciprocal that a scalar divisor becomes
    scale = amax / torch.full_like(amax, qmax)
    scale = torch.where(torch.isfinite(amax), scale, torch.full_like(scale, float("nan")))
    # the quotient in 64 bits: x / scale in 32 lands on the middle between two codes where the true one lies beside it
    q = x.double() / scale.double()[..., None]
    q = torch.where((scale > 0)[..., None], q, torch.zeros_like(q)).clamp_(-qmax, qmax).reshape(n, h, d)
    if case["fmt"] == "int8":
        codes = q.round_().to(torch.int8)
    elif case["fmt"] == "e4m3":
        grid = torch.exp2(q.abs().log2_().floor_().clamp_(min=-6.0) - 3.0)
        codes = (torch.round(q / grid) * grid).to(torch.float8_e4m3fn)
    else:
        i = q.round_().to(torch.int32) & 15
        codes = (i[..., 0::2] | (i[..., 1::2] << 4)).to(torch.uint8)
    if rows is None:
        store["codes"][first:first + n] = codes
        store["scales"][first:first + n] = scale
        return
    keep = rows >= 0
    # torch's indexed assignment does not take fp8: the bytes go as bytes
    store["codes"].view(torch.uint8)[rows[keep]] = codes.view(torch.uint8)[keep]
    store["scales"][rows[keep]] = scale[keep]


def _plain_read(store, case, rows, first, n):
    h, d, g = case["heads"], case["dim"], case["group"]
    if rows is None:
        codes, scale = store["codes"][first:first + n], store["scales"][first:first + n]
        miss = None
    else:
        at = rows.clamp(min=0)
        codes, scale = store["codes"].view(torch.uint8)[at].view(store["codes"].dtype), store["scales"][at]
        miss = rows < 0
    if case["fmt"] == "int4":
        lo, hi = (codes & 15).to(torch.int32), (codes >> 4).to(torch.int32)
        q = torch.stack([lo, hi], -1).reshape(n, h, d)
        q = torch.where(q > 7, q - 16, q).float()
    else:
        q = codes.float()
    out = (q.reshape(n, h, d // g, g) * scale[..., None]).reshape(n, h, d)
    if miss is not None:
        out = torch.where(miss[:, None, None], torch.zeros_like(out), out)
    return out.to(_DT[case["dtype"]])


def _column(x, like):
    if torch.is_tensor(x):
        return x.to(torch.float64)[:, None]
    return torch.full((like.shape[0], 1), float(x), dtype=torch.float64, device=like.device)


def _plain_draw(scores, mask, u, par):
    """In 64 bits: a draw is decided by where u falls among cumulative sums of up to a million weights."""
    s = scores.double()
    s = torch.where(torch.isnan(s), torch.full_like(s, -math.inf), s)
    if mask is not None:
        s = torch.where(mask, s, torch.full_like(s, -math.inf))
    v = s.shape[1]
    order_s, order = torch.sort(s, dim=1, descending=True, stable=True)
    t, k, p, m = (_column(par[x], s) for x in ("temperature", "top_k", "top_p", "min_p"))
    w = torch.exp((order_s - order_s[:, :1]) / t)
    w = torch.where(order_s > -math.inf, w, torch.zeros_like(w))
    place = torch.arange(v, device=s.device, dtype=torch.float64)[None]
    keep = (place < k) | (k <= 0)
    keep[:, 0] = True
    wk = w * keep
    cum = wk.cumsum(1)
    keep &= (cum - wk < p * cum[:, -1:]) | (p >= 1)
    keep &= w >= m.clamp(max=1.0)
    keep &= order_s > -math.inf
    weight = torch.zeros_like(s).scatter_(1, order, w * keep)
    cum = weight.cumsum(1)
    total = cum[:, -1:]
    last = torch.where(weight > 0, place, -torch.ones_like(place)).amax(1, keepdim=True)
    idx = torch.searchsorted(cum, u.double() * total, right=True)
    idx = torch.minimum(idx, last.long())
    prob = torch.gather(weight, 1, idx.clamp(min=0)) / total
    prob = torch.where(idx < 0, torch.zeros_like(prob), prob)
    return idx.to(torch.int32), prob.float()


def run(state):
    case = state["case"]
    if case["op"] == "draw":
        if own:
            from point_slam_amd import frame_ops
            idx, prob = frame_ops.draw_indices(state["scores"], state["u"], mask=state["mask"], with_prob=True, **state["par"])
        else:
            idx, prob = _plain_draw(state["scores"], state["mask"], state["u"], state["par"])
        return {"idx": idx, "prob": prob}
    store, rows, first, n = state["store"], state["rows"], state["first"], case["n"]
    dtype = _DT[case["dtype"]]
    if case["op"] == "store":
        if own:
            store.write(state["values"], rows=rows, first=first, distinct=True)
        else:
            _plain_write(store, case, state["values"], rows, first)
    if own:
        out = store.read(rows=rows, first=first, count=n, dtype=dtype) if rows is None else store.read(rows=rows, dtype=dtype)
    else:
        out = _plain_read(store, case, rows, first, n)
    return {"values": out}


def work(case):
    if case["op"] == "draw":
        r, v, n = case["rows"], case["cols"], case["draws"]
        entry = _SIZE[case["dtype"]] + (1 if case["kind"] == "image" else 0)
        return {"bytes": r * v * entry + r * n * 12, "flops": r * v * 4 + r * n * 2}
    n, h, d = case["n"], case["heads"], case["dim"]
    held = h * (d * _BITS[case["fmt"]] // 8 + 4 * (d // case["group"]))
    index = 0 if case["rows"] == "tail" else 8
    one_way = n * (h * d * _SIZE[case["dtype"]] + held + index)
    if case["op"] == "read":
        return {"bytes": one_way, "flops": n * h * d}
    return {"bytes": 2 * one_way, "flops": 5 * n * h * d}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _nearest_e4m3(q):
    """Round to the nearest value of three mantissa bits and exponents -6 .. 8, ties to the even mantissa."""
    _, e = torch.frexp(q)
    step = torch.ldexp(torch.ones_like(q), (e - 1).clamp(min=-6) - 3)
    return torch.round(q / step) * step


def _exact_rows(case, values):
    """What the held rows stand for.  The scale is part of the definition: the group's largest magnitude over the largest
    code, held in 32 bits."""
    n = values.shape[0]
    x = values.double().view(n, case["heads"], -1, case["group"])
    top = _QMAX[case["fmt"]]
    s = (x.abs().amax(-1, keepdim=True) / top).float().double()
    q = x / torch.where(s > 0, s, torch.ones_like(s))
    q = _nearest_e4m3(q) if case["fmt"] == "e4m3" else torch.round(q)
    return (q.clamp(-top, top) * s).reshape(n, case["heads"], case["dim"])


def _exact_draw(scores, mask, u, t, k, p, m):
    """One row, on the host."""
    import numpy as np
    s = scores.double().cpu().numpy()
    ok = ~np.isnan(s) & (s > -np.inf)
    if mask is not None:
        ok &= mask.cpu().numpy()
    cand = np.flatnonzero(ok)
    n = u.shape[0]
    if cand.size == 0:
        return np.full(n, -1, np.int64), np.zeros(n)
    cand = cand[np.argsort(-s[cand], kind="stable")]
    top = s[cand[0]]
    if k > 0:
        cand = cand[:int(k)]
    w = np.exp((s[cand] - top) / t)
    if p < 1:
        cand = cand[:max(1, int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1)]
        w = w[:cand.size]
    cand = np.sort(cand[w >= min(m, 1.0)])
    w = np.exp((s[cand] - top) / t)
    cum = np.cumsum(w)
    at = np.minimum(np.searchsorted(cum, u.double().cpu().numpy() * cum[-1], side="right"), cand.size - 1)
    return cand[at], w[at] / cum[-1]


def exact(case, seed):
    if case["op"] == "draw":
        import numpy as np
        scores, mask, u, par = _score_inputs(case, seed)
        rows = []
        for r in range(case["rows"]):
            one = {key: float(x[r]) if torch.is_tensor(x) else float(x) for key, x in par.items()}
            rows.append(_exact_draw(scores[r], None if mask is None else mask[r], u[r],
                                    np.float64(one["temperature"]), one["top_k"], one["top_p"], one["min_p"]))
        return {"idx": torch.from_numpy(np.stack([a for a, _ in rows])).to(torch.int32),
                "prob": torch.from_numpy(np.stack([b for _, b in rows]))}
    if case["op"] == "read":
        held, _ = _row_inputs(dict(case, n=case["capacity"], rows="tail"), seed)
        rows = torch.randint(case["capacity"], (case["n"],), device="cuda", generator=_generator(seed + 1))
        return {"values": _exact_rows(case, held[rows])}
    values, rows = _row_inputs(case, seed)
    out = _exact_rows(case, values)
    if rows is not None:
        out = torch.where((rows < 0)[:, None, None], torch.zeros_like(out), out)
    return {"values": out}
