"""Measured cases of the quantised-catalog and sampling operators.

mx_quantize / mx_dequantize   rows packed to microscaled 4-bit floating point (MXFP4) and back
score_mx                      full-catalog scores of users against an MXFP4 item table
sample_rows                   draws from score rows: temperature, top-k, top-p, min-p, given randoms

``own`` false: the plain form in elementary torch operations; ``own`` true: the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # e2m1 magnitudes by code
_BLOCK = 32


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the embedding table of a small graph (2,728 rows) of an unaligned width: launch latency
        {"name": "quant_small", "op": "quant", "rows": 2728, "d": 100, "dtype": "bf16"},
        # the propagated table of the Gowalla graph, users and items
        {"name": "quant_gowalla", "op": "quant", "rows": 70839, "d": 64, "dtype": "f32"},
        # the million-item catalog
        {"name": "quant_catalog", "op": "quant", "rows": 1000000, "d": 256, "dtype": "f32"},
        # one user's request against the million-item catalog: the table's bytes
        {"name": "score_user", "op": "score", "B": 1, "items": 1000000, "d": 256, "q": "f32", "gather": False,
         "sigmoid": False, "out": "f32"},
        # a test batch of getUsersRating at the Gowalla shape, users picked out of their table
        {"name": "score_gowalla", "op": "score", "B": 2048, "items": 40981, "d": 64, "q": "mx", "gather": True,
         "sigmoid": True, "out": "f32"},
        # wide rows whose last block is ragged, bf16 queries and scores
        {"name": "score_wide", "op": "score", "B": 333, "items": 91599, "d": 1000, "q": "bf16", "gather": False,
         "sigmoid": False, "out": "bf16"},
        # a batch against the million-item catalog: the score matrix's bytes
        {"name": "score_catalog", "op": "score", "B": 1024, "items": 1000000, "d": 256, "q": "mx", "gather": False,
         "sigmoid": False, "out": "f32"},
        # four users of a small catalog, one draw each: launch latency
        {"name": "sample_small", "op": "sample", "rows": 4, "cols": 2120, "dtype": "f32", "draws": 1,
         "T": 0.8, "k": 20, "p": 0.95, "minp": 0.0},
        # one user, the whole million-item policy, many draws
        {"name": "sample_policy", "op": "sample", "rows": 1, "cols": 1000000, "dtype": "f32", "draws": 100,
         "T": 1.0, "k": 0, "p": 1.0, "minp": 0.0},
        # a test batch at the Gowalla shape, nucleus sampling
        {"name": "sample_gowalla", "op": "sample", "rows": 2048, "cols": 40981, "dtype": "f32", "draws": 1,
         "T": 1.0, "k": 0, "p": 0.9, "minp": 0.0},
        # a batch at the Amazon-book shape in bf16 (many equal scores), a list of draws from the top 100
        {"name": "sample_list", "op": "sample", "rows": 1024, "cols": 91599, "dtype": "bf16", "draws": 20,
         "T": 0.5, "k": 100, "p": 1.0, "minp": 0.02},
        # users with settings of their own against the million-item catalog
        {"name": "sample_catalog", "op": "sample", "rows": 512, "cols": 1000000, "dtype": "f32", "draws": 4,
         "per_row": True, "T": 0.7, "k": 0, "p": 0.9, "minp": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quant", "score", "sample"))
    if op == "quant":
        d = _log(rng, 1, 1024)
        return {"op": op, "rows": _log(rng, 1, min(1000000, 256000000 // d)), "d": d,
                "dtype": rng.choice(("f32", "bf16"))}
    if op == "score":
        d = _log(rng, 8, 1024)
        items = _log(rng, 100, min(1000000, 256000000 // d))
        most = 2 * 1024 * 10**6 * 256 // (2 * items * d)
        return {"op": op, "B": _log(rng, 1, max(1, min(2048, most, 1024 * 10**6 // items))), "items": items, "d": d,
                "q": rng.choice(("f32", "bf16", "mx")), "gather": rng.random() < 0.5,
                "sigmoid": rng.random() < 0.3, "out": rng.choice(("f32", "f32", "bf16"))}
    cols = _log(rng, 2, 1000000)
    case = {"op": op, "rows": _log(rng, 1, max(1, min(4096, 256000000 // cols))), "cols": cols,
            "dtype": rng.choice(("f32", "f32", "bf16")), "draws": rng.choice((1, 1, 2, 7, 20, 100)),
            "T": rng.choice((0.5, 0.7, 1.0, 1.3)), "k": rng.choice((0, 0, 1, 20, 50, 200, 1000)),
            "p": rng.choice((1.0, 1.0, 0.5, 0.9, 0.95)), "minp": rng.choice((0.0, 0.0, 0.02, 0.1))}
    if rng.random() < 0.3:
        case["per_row"] = True
    return case


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _table(rows, d, g, scale):
    """Embedding rows: normal entries, a row's size spread over a factor of ten (popular items are long)."""
    x = torch.randn(rows, d, generator=g, device="cuda")
    return x.mul_(scale * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda")))


def _pack(x):
    """(codes, scales) of float rows, in the framework's storage: element 2j of a row in the low nibble
    of byte j, one scale byte a block of 32."""
    codes, scales = [], []
    for r in x.split(1 << 17):
        c, s = _plain_codes(r.float())
        codes.append(c[:, 0::2] | (c[:, 1::2] << 4))
        scales.append(s)
    return torch.cat(codes), torch.cat(scales)


def prepare(case, seed):
    g = _gen(seed)
    state = {"case": case}
    if case["op"] == "quant":
        state["x"] = _table(case["rows"], case["d"], g, 0.1).to(_DTYPES[case["dtype"]])
    elif case["op"] == "score":
        n_q = 2 * case["B"] + 7 if case["gather"] else case["B"]
        scale = case["d"] ** -0.25
        q = _table(n_q, case["d"], g, scale)
        state["q"] = _pack(q) if case["q"] == "mx" else q.to(_DTYPES[case["q"]])
        state["items"] = _pack(_table(case["items"], case["d"], g, scale))
        state["rows"] = (torch.randint(0, n_q, (case["B"],), generator=g, device="cuda") if case["gather"] else None)
    else:
        rows, cols = case["rows"], case["cols"]
        s = torch.randn(rows, cols, generator=g, device="cuda").mul_(1.5)
        s.add_(0.7 * torch.randn(cols, generator=g, device="cuda"))  # an item's popularity
        # a user's train items are masked; one user in a larger batch has everything masked
        hits = max(1, cols // 100)
        s.scatter_(1, torch.randint(0, cols, (rows, hits), generator=g, device="cuda"), float("-inf"))
        if rows >= 64:
            s[rows // 2] = float("-inf")
        state["S"] = s.to(_DTYPES[case["dtype"]])
        state["u"] = torch.rand(rows, case["draws"], generator=g, device="cuda")
        state["T"], state["k"], state["p"], state["minp"] = case["T"], case["k"], case["p"], case["minp"]
        if case.get("per_row"):
            def pick(*values, dtype):
                t = torch.tensor(values, dtype=dtype, device="cuda")
                return t[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]
            state["T"] = pick(0.0, 0.5, 0.7, 1.0, dtype=torch.float32)
            state["k"] = pick(0, 0, 50, 1000, dtype=torch.int32)
            state["p"] = pick(1.0, 0.9, 0.95, dtype=torch.float32)
            state["minp"] = pick(0.0, 0.0, 0.05, dtype=torch.float32)
    return state


# ------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import factors_of_serendipity_recommendation_amd as lgx
    case = state["case"]
    if case["op"] == "quant":
        return lgx.mx_dequantize(lgx.mx_quantize(state["x"]))
    if case["op"] == "score":
        q = lgx.MXTable(*state["q"], case["d"]) if case["q"] == "mx" else state["q"]
        return lgx.score_mx(q, lgx.MXTable(*state["items"], case["d"]), user_rows=state["rows"],
                            apply_sigmoid=case["sigmoid"], dtype=_DTYPES[case["out"]])
    return lgx.sample_rows(state["S"], state["u"], temperature=state["T"], top_k=state["k"], top_p=state["p"],
                           min_p=state["minp"])


def _plain_codes(x):
    """f32 rows -> (e2m1 codes u8 [rows, 32 nb], scale bytes u8 [rows, nb])."""
    rows, d = x.shape
    nb = -(-d // _BLOCK)
    b = torch.zeros(rows, nb * _BLOCK, device=x.device)
    b[:, :d] = x
    b = b.view(rows, nb, _BLOCK)
    amax = b.abs().amax(2)
    e = (torch.frexp(amax).exponent - 3).clamp(-127, 127)  # floor(log2 amax) - 2
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    y = b.abs() * torch.exp2(-e.double()).float().unsqueeze(2)  # a power of two: exact
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code |= torch.signbit(b).to(torch.uint8) << 3
    bad = ~torch.isfinite(amax)
    scale = torch.where(bad, torch.full_like(e, 128), e) + 127
    return (torch.where(bad.unsqueeze(2), torch.zeros_like(code), code).view(rows, nb * _BLOCK),
            scale.to(torch.uint8))


def _plain_values(code, scale, d):
    """codes u8 [rows, 32 nb], scale bytes [rows, nb] -> f32 [rows, d]."""
    level = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=code.device)
    s = torch.exp2(scale.double() - 127).float()
    s = torch.where(scale == 255, torch.full_like(s, float("nan")), s)
    v = level[code.int()].view(code.shape[0], -1, _BLOCK) * s.unsqueeze(2)
    return v.view(code.shape[0], -1)[:, :d]


def _plain_unpack(packed, d):
    codes, scales = packed
    return _plain_values(torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1), scales, d)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "quant":
        return _plain_values(*_plain_codes(state["x"].float()), case["d"])
    if case["op"] == "score":
        d, rows = case["d"], state["rows"]
        q = _plain_unpack(state["q"], d) if case["q"] == "mx" else _plain_values(*_plain_codes(state["q"].float()), d)
        q = q if rows is None else q[rows]
        out = q @ _plain_unpack(state["items"], d).T
        if case["sigmoid"]:
            out = torch.sigmoid(out)
        return out.to(_DTYPES[case["out"]])
    return _plain_sample(state)


def _column(v, rows, like):
    t = v.to(like) if torch.is_tensor(v) else torch.full((rows,), float(v), dtype=like, device="cuda")
    return t.view(rows, 1)


def _plain_sample(state):
    rows, cols = state["S"].shape
    setting = [_column(state[n], rows, torch.float64) for n in ("T", "k", "p", "minp")]
    step = max(1, (1 << 27) // cols)
    parts = [_plain_sample_rows(state["S"][i:i + step], state["u"][i:i + step], *(v[i:i + step] for v in setting))
             for i in range(0, rows, step)]
    return tuple(torch.cat(p) for p in zip(*parts))


def _plain_sample_rows(S, u, T, k, p, minp):
    rows, cols = S.shape
    s = S.double()
    s = torch.where(s.isnan(), torch.full_like(s, float("-inf")), s)
    m = s.amax(1, keepdim=True)
    greedy = T <= 0
    w = torch.exp((s - m) / torch.where(greedy, torch.ones_like(T), T))
    w = torch.where(s == m, torch.ones_like(w), torch.where(greedy, torch.zeros_like(w), w))
    w = torch.where(s == float("-inf"), torch.zeros_like(w), w)
    ws, order = torch.sort(s, dim=1, descending=True, stable=True)
    ws = torch.gather(w, 1, order)
    pos = torch.arange(cols, device=S.device).view(1, cols)
    first = torch.where(greedy, torch.ones_like(k), torch.where(k > 0, k, torch.full_like(k, cols)))
    ws = torch.where(pos < first, ws, torch.zeros_like(ws))
    c = torch.cumsum(ws, 1)
    inside = (c - ws < p * c[:, -1:]) | (p >= 1) | (pos == 0)
    ws = torch.where(inside & (ws >= minp), ws, torch.zeros_like(ws))
    w = torch.zeros_like(w).scatter_(1, order, ws)
    c = torch.cumsum(w, 1)
    total = c[:, -1:]
    idx = torch.searchsorted(c, u.double() * total, right=True).clamp_(max=cols - 1)
    prob = torch.gather(w, 1, idx) / total
    none = total == 0
    idx = torch.where(none, torch.full_like(idx, -1), idx)
    return idx.int(), torch.where(none, torch.zeros_like(prob), prob).float()


# ------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size = {"f32": 4, "bf16": 2}
    if case["op"] == "quant":
        n = case["rows"] * case["d"]
        return {"bytes": n * (size[case["dtype"]] + 4), "flops": 4 * n}
    if case["op"] == "score":
        nb = -(-case["d"] // _BLOCK)
        q = nb * 17 if case["q"] == "mx" else case["d"] * size[case["q"]]
        return {"bytes": case["items"] * nb * 17 + case["B"] * q + case["B"] * case["items"] * size[case["out"]],
                "flops": 2 * case["B"] * case["items"] * case["d"]}
    n = case["rows"] * case["cols"]
    return {"bytes": n * size[case["dtype"]] + case["rows"] * case["draws"] * 12, "flops": 4 * n}


# ------------------------------------------------------------------------------------ 64-bit definition
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quant":
        return _exact_values(state["x"])
    if case["op"] == "score":
        d = case["d"]
        q = _exact_unpack(state["q"], d) if case["q"] == "mx" else _exact_values(state["q"])
        if state["rows"] is not None:
            q = q.index_select(0, state["rows"])
        out = torch.empty(case["B"], case["items"], dtype=torch.float64, device="cuda")
        step = max(1, (1 << 26) // d)
        codes, scales = state["items"]
        for i in range(0, case["items"], step):
            out[:, i:i + step] = torch.mm(q, _exact_unpack((codes[i:i + step], scales[i:i + step]), d).t().contiguous())
        return out.neg_().exp_().add_(1).reciprocal_() if case["sigmoid"] else out
    if case["rows"] * case["cols"] > 100_000_000:
        return None
    return _exact_sample(state)


def _exact_values(x):
    """Nearest representable value of every element, from the distances to all fifteen."""
    out = []
    grid = torch.tensor(sorted({s * v for v in _LEVELS for s in (1.0, -1.0)}), dtype=torch.float64, device="cuda")
    even = torch.tensor([0, 2, 4, 6], device="cuda")
    mags = torch.tensor(_LEVELS, dtype=torch.float64, device="cuda")
    is_even = torch.zeros(len(grid), dtype=torch.bool, device="cuda")
    is_even |= (grid.abs().view(-1, 1) == mags[even].view(1, -1)).any(1)
    for part in x.double().split(max(1, (1 << 22) // x.shape[1])):
        done = []
        for blk in part.split(_BLOCK, 1):
            a = blk.abs().amax(1, keepdim=True)
            e = torch.floor(torch.log2(a.clamp(min=1e-300)))
            e = torch.where(torch.exp2(e) > a, e - 1, torch.where(torch.exp2(e + 1) <= a, e + 1, e))  # log2 rounds
            unit = torch.exp2((e - 2).clamp(-127, 127))
            y = (blk / unit).clamp(-6, 6)
            best, far = torch.zeros_like(y), torch.full_like(y, float("inf"))
            for v, ev in zip(grid.tolist(), is_even.tolist()):
                dist = (y - v).abs()
                take = (dist < far) | ((dist == far) & ev)
                best, far = torch.where(take, torch.full_like(y, v), best), torch.minimum(dist, far)
            done.append(best * unit)
        out.append(torch.cat(done, 1))
    return torch.cat(out)


def _exact_unpack(packed, d):
    codes, scales = packed
    mags = torch.tensor(_LEVELS, dtype=torch.float64, device="cuda")
    out = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device="cuda")
    for half in (0, 1):
        nib = (codes >> (4 * half)) & 15
        v = mags[(nib & 7).long()]
        out[:, half::2] = torch.where(nib >= 8, -v, v)
    out = out.view(codes.shape[0], -1, _BLOCK) * torch.exp2(scales.double() - 127).unsqueeze(2)
    return out.reshape(codes.shape[0], -1)[:, :d].contiguous()


def _exact_sample(state):
    """Row by row on the host, the kept set as a list of indices."""
    S, u = state["S"].double().cpu().numpy(), state["u"].double().cpu().numpy()
    rows, cols = S.shape
    T, k, p, minp = (_column(state[n], rows, torch.float64).cpu().numpy()[:, 0] for n in ("T", "k", "p", "minp"))
    idx = np.full(u.shape, -1, dtype=np.int64)
    prob = np.zeros(u.shape)
    for r in range(rows):
        live = np.flatnonzero(S[r] > -np.inf)
        if not live.size:
            continue
        s = S[r, live]
        top = s.max()
        if T[r] <= 0:
            live, s = live[s == top][:1], s[s == top][:1]
            w = np.ones(1)
        else:
            w = np.exp((s - top) / T[r])
        if k[r] > 0 or p[r] < 1:
            rank = np.lexsort((live, -s))
            if k[r] > 0:
                rank = rank[:int(k[r])]
            if p[r] < 1:
                before = np.concatenate(([0.0], np.cumsum(w[rank])))
                n = int(np.searchsorted(before[:-1], p[r] * before[-1], side="left"))
                rank = rank[:max(1, n)]
            rank.sort()
            live, w = live[rank], w[rank]
        if minp[r] > 0:
            live, w = live[w >= minp[r]], w[w >= minp[r]]
        c = np.cumsum(w)
        j = np.minimum(np.searchsorted(c, u[r] * c[-1], side="right"), len(live) - 1)
        idx[r], prob[r] = live[j], w[j] / c[-1]
    return torch.from_numpy(idx).int().cuda(), torch.from_numpy(prob).cuda()
