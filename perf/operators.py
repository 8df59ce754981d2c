"""The operators of a serving loop on a key / value cache of 4-bit levels, as measurable cases: attention over the cache
(which takes the new rows in first), eviction from it by the attention weight that its positions have received, and the
draw of the next token from rows of logits.

The cache. A row of `head_dim` values is cut into blocks of 32. A block has an f16 scale d = f16(m / -8), m its value of
largest magnitude (the positive one where two tie, |d| at most 65504), and whole levels clamp(rint(x / d), -8, 7); what it
stands for is d * level. A block with d = 0 holds zeros.

Attention. Sequence s has lens[s] positions before the call and rows[s] new ones. New row i goes to position lens[s] + i,
and its query heads attend to the positions 0 .. lens[s] + i of their key / value head, softmax(q k / sqrt(head_dim)) v.
Where `mass` is kept, the weights that a position receives in the call, over all rows and the heads that share it, are
added to mass[s][kv head][position]; a new position starts from nothing.

Eviction. Of each sequence and key / value head, the last `recent` positions stay, and of the others the heaviest, up to
`budget` in all (the lower position where two weigh the same); they keep their order. Shorter sequences stay whole.

The draw. w = exp((l - max l) / max(T, 0.01)). Ids stay that are not below the k-th largest logit (top_k > 0), not below
the largest logit down to which the mass reaches top_p of the whole (top_p < 1) and have w >= min_p; of what stays,
weights under 2^-40 are nothing. The token is the first id, in index order, at which the running mass of the others
reaches u times their whole. T <= 0 takes the first of the largest logits.
"""
import math

import torch

own = False

BLOCK = 32
LEAST = 2.0 ** -40


# ---------------------------------------------------------------------------------------- the listed cases
def listed():
    return [
        # a single stream at the start of a chat on the narrow decoder (8 query heads, 2 key / value heads of 64): a step is all latency
        {"name": "step-short", "kind": "attend", "seqs": 1, "heads": 8, "kv": 2, "dim": 64, "cached": 33, "rows": 1, "ragged": False, "mass": False},
        # a single stream of the 1B-class decoder at the end of its context
        {"name": "step-1b", "kind": "attend", "seqs": 1, "heads": 32, "kv": 8, "dim": 64, "cached": 2046, "rows": 1, "ragged": False, "mass": True},
        # a full serving batch of it, every stream somewhere else in its context
        {"name": "step-batch", "kind": "attend", "seqs": 64, "heads": 32, "kv": 8, "dim": 64, "cached": 2040, "rows": 1, "ragged": True, "mass": True},
        # long documents, heads of 128: what a cache of 4 bits is for
        {"name": "step-long", "kind": "attend", "seqs": 8, "heads": 32, "kv": 8, "dim": 128, "cached": 32767, "rows": 1, "ragged": False, "mass": False},
        # drafts of up to five tokens verified at once, twelve heads of their own
        {"name": "verify", "kind": "attend", "seqs": 16, "heads": 12, "kv": 12, "dim": 64, "cached": 900, "rows": 5, "ragged": True, "mass": False},
        # the prompt of the 1B-class decoder into an empty cache, its weights kept for an eviction
        {"name": "prompt-1b", "kind": "attend", "seqs": 1, "heads": 32, "kv": 8, "dim": 64, "cached": 0, "rows": 2048, "ragged": False, "mass": True},
        # a long prompt, heads of 128: the largest case
        {"name": "prompt-long", "kind": "attend", "seqs": 1, "heads": 32, "kv": 8, "dim": 128, "cached": 0, "rows": 6007, "ragged": False, "mass": False},
        # a step's cache that has run full, back to its budget
        {"name": "evict-step", "kind": "evict", "seqs": 1, "kv": 8, "dim": 64, "length": 1152, "budget": 1024, "recent": 256, "ragged": False},
        # the caches of long prompts, cut down before the steps begin
        {"name": "evict-prompt", "kind": "evict", "seqs": 8, "kv": 8, "dim": 128, "length": 16001, "budget": 2048, "recent": 128, "ragged": True},
        # the draw of a single stream
        {"name": "draw-one", "kind": "draw", "rows": 1, "vocab": 32000, "filters": "all"},
        # a batch of requests, each with its own parameters
        {"name": "draw-batch", "kind": "draw", "rows": 64, "vocab": 50257, "filters": "mixed"},
        # many samples of long rows, where nothing but the temperature and a wide top-p narrows them
        {"name": "draw-wide", "kind": "draw", "rows": 192, "vocab": 131072, "filters": "wide"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "rows", "evict", "draw"])
    if kind in ("step", "rows"):
        kv = rng.choice([1, 2, 4, 8])
        case = {"kind": "attend", "seqs": 1, "heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv": kv, "dim": rng.choice([32, 64, 96, 128, 256]),
                "cached": 0, "rows": 1, "ragged": rng.choice([False, True]), "mass": rng.choice([False, True])}
        if kind == "step":
            case["seqs"] = _log(rng, 1, 64)
            case["cached"] = _log(rng, 1, min(40000, 60_000_000 // (case["seqs"] * kv * case["dim"])))
        else:
            case["seqs"] = _log(rng, 1, 8)
            case["rows"] = _log(rng, 2, 4096 // case["seqs"])
            case["cached"] = rng.choice([0, _log(rng, 1, 4096)])
            while work(case)["flops"] > 2.5e11:
                case["rows"], case["cached"] = case["rows"] * 2 // 3, case["cached"] * 2 // 3
        return case
    if kind == "evict":
        seqs, kv, dim = _log(rng, 1, 16), rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 96, 128, 256])
        length = _log(rng, 16, min(20000, 120_000_000 // (seqs * kv * dim)))
        budget = _log(rng, 2, length)
        return {"kind": kind, "seqs": seqs, "kv": kv, "dim": dim, "length": length, "budget": budget, "recent": rng.randint(0, budget),
                "ragged": rng.choice([False, True])}
    return {"kind": kind, "rows": _log(rng, 1, 128), "vocab": _log(rng, 100, 150000), "filters": rng.choice(["all", "mixed", "wide"])}


# ------------------------------------------------------------------------------------- inputs of one state
def _uneven(n, top, low, gen):
    """n whole numbers from low to top, the longest among them."""
    u = torch.rand(n, generator=gen)
    u[int(torch.randint(n, (1,), generator=gen))] = 1.0
    return [int(v) for v in (low + (top - low) * u).round().long()]


def _gens(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    return g, h


def _keys_values(n, kv, dim, gen):
    """Rows of keys, whose channels differ in size as those of trained heads do, and of values: [n][kv * dim] each."""
    size = torch.exp(0.5 * torch.randn((1, kv * dim), generator=gen, device="cuda"))
    k = torch.randn((n, kv * dim), generator=gen, device="cuda").mul_(size)
    return k, torch.randn((n, kv * dim), generator=gen, device="cuda")


def _cache(s, n, gen):
    """A cache that holds n positions of every sequence, with room for no more: the framework's, or levels and scales."""
    c = s["case"]
    seqs, kv, dim = c["seqs"], c["kv"], c["dim"]
    k, v = _keys_values(seqs * n, kv, dim, gen)
    if own:
        from ferrum_cpu_b200 import kv4
        cache = kv4.Kv4Cache(seqs, kv, dim, n)
        s["none"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        cache.append_dev(k.data_ptr(), v.data_ptr(), kv * dim, s["none"].data_ptr(), rows=[n] * seqs)
        torch.cuda.synchronize()   # k and v go when this returns
        return cache
    return [t for x in (k, v) for t in _quantize(x.view(seqs, n, kv, dim).transpose(1, 2))]


def _attend_inputs(case, seed):
    """What the passes of one state read, without the cache: (lengths, rows, q, k, v, mass) and the generator after them."""
    g, h = _gens(seed)
    seqs, heads, kv, dim = case["seqs"], case["heads"], case["kv"], case["dim"]
    lens = _uneven(seqs, case["cached"], case["cached"] // 8, h) if case["ragged"] else [case["cached"]] * seqs
    # how many rows each sequence brings belongs to the case: outputs of all seeds have one shape
    rows = _uneven(seqs, case["rows"], 1, torch.Generator().manual_seed(seqs + 64 * case["rows"])) if case["ragged"] else [case["rows"]] * seqs
    # q | k | v as one product leaves them
    qkv = torch.randn((sum(rows), (heads + 2 * kv) * dim), generator=g, device="cuda")
    room = case["cached"] + case["rows"]
    mass = torch.rand((seqs, kv, room), generator=g, device="cuda").pow_(4).mul_(8.0) if case["mass"] else None
    return lens, rows, qkv, mass, room, g


def _evict_inputs(case, seed):
    g, h = _gens(seed)
    seqs, kv, n = case["seqs"], case["kv"], case["length"]
    lens = _uneven(seqs, n, n // 4, h) if case["ragged"] else [n] * seqs
    # weight decays from a few heavy positions; positions that got none at all tie
    mass = torch.rand((seqs, kv, n), generator=g, device="cuda").pow_(6).mul_(20.0)
    mass[torch.rand((seqs, kv, n), generator=g, device="cuda") < 0.1] = 0.0
    return lens, mass, g


def _draw_inputs(case, seed):
    g, h = _gens(seed)
    n, V = case["rows"], case["vocab"]
    logits = torch.randn((n, V), generator=g, device="cuda").mul_(2.5)
    # a few ids stand out, and a grammar forbids a part of the others
    logits.scatter_add_(1, torch.randint(V, (n, 8), generator=g, device="cuda"), 8.0 * torch.rand((n, 8), generator=g, device="cuda"))
    logits[torch.rand((n, V), generator=g, device="cuda") < 0.05] = -math.inf
    logits[:, V // 2] = 1.0
    u = torch.rand(n, generator=g, device="cuda")
    some = lambda values: torch.tensor(values)[torch.randint(len(values), (n,), generator=h)]  # noqa: E731
    if case["filters"] == "all":
        params = [torch.full((n,), v) for v in (0.8, 40.0, 0.95, 0.05)]
    elif case["filters"] == "wide":
        params = [some([1.0, 1.3]), torch.zeros(n), some([1.0, 0.98]), torch.zeros(n)]
    else:
        params = [some([0.0, 0.6, 0.8, 1.0, 1.2]), some([0.0, 1.0, 20.0, 50.0, 1000.0]), some([1.0, 0.9, 0.95]), some([0.0, 0.05, 0.1])]
    # a row of parameters: temperature, top_k (a whole number), top_p, min_p
    rows = torch.stack([params[0], params[1].to(torch.int32).view(torch.float32), params[2], params[3]], dim=1)
    return logits, rows.cuda(), u


def prepare(case, seed):
    s = {"case": case}
    if case["kind"] == "attend":
        lens, rows, qkv, mass, room, g = _attend_inputs(case, seed)
        s.update(lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), rows=rows, qkv=qkv, mass=mass)
        s["cache"] = _cache(s, room, g)
        n, kv, dim = case["seqs"], case["kv"], case["dim"]
        s["out"] = torch.empty((sum(rows), case["heads"] * dim), device="cuda")
        s["new"] = torch.empty((2, n, case["rows"], kv, dim), device="cuda")
        if own and rows != [1] * n:
            from ferrum_cpu_b200 import kv4
            s["plan"] = kv4.row_counts(rows)
    elif case["kind"] == "evict":
        lens, mass, g = _evict_inputs(case, seed)
        s.update(lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), mass=mass)
        s["cache"] = _cache(s, case["length"], g)
        n, kv, dim, budget = case["seqs"], case["kv"], case["dim"], case["budget"]
        s["kept"] = torch.empty((n, kv, budget), dtype=torch.int32, device="cuda")
        s["left"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["left_mass"] = torch.zeros((n, kv, budget), device="cuda")
        s["values"] = torch.empty((2, n, budget, kv, dim), device="cuda")
        if own:
            from ferrum_cpu_b200 import kv4
            s["to"] = kv4.Kv4Cache(n, kv, dim, budget)
    else:
        logits, params, u = _draw_inputs(case, seed)
        s.update(logits=logits, params=params, u=u, token=torch.empty(case["rows"], dtype=torch.int32, device="cuda"),
                 prob=torch.empty(case["rows"], device="cuda"))
        if own:
            from ferrum_cpu_b200 import engine
            s["sample"] = engine.sample_rows_dev
    return s


# ------------------------------------------------------------------------------------------ one pass
def _quantize(x):
    """x [..][dim] as (levels [..][dim] int8, scales [..][dim / 32] f16)."""
    b = x.unflatten(-1, (-1, BLOCK))
    hi, lo = b.amax(-1), b.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) / -8.0).clamp(-65504.0, 65504.0).to(torch.float16)
    f = d.float().unsqueeze(-1)
    levels = torch.where(f == 0, 0.0, torch.round(b / f).clamp(-8.0, 7.0))
    return levels.to(torch.int8).flatten(-2), d


def _values(levels, d):
    return (levels.unflatten(-1, (-1, BLOCK)).float() * d.float().unsqueeze(-1)).flatten(-2)


def _attend_plain(s):
    c = s["case"]
    seqs, heads, kv, dim, R = c["seqs"], c["heads"], c["kv"], c["dim"], c["rows"]
    group, total = heads // kv, s["qkv"].shape[0]
    q, k, v = s["qkv"].split([heads * dim, kv * dim, kv * dim], dim=1)
    kq, kd, vq, vd = s["cache"]
    lens = s["lens"].long()
    rows = torch.tensor(s["rows"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), rows, output_size=total)
    at = torch.arange(total, device="cuda") - (rows.cumsum(0) - rows)[seq]      # a row's place among its sequence's new ones
    pos = lens[seq] + at
    for levels, scales, x in ((kq, kd, k), (vq, vd, v)):
        levels[seq, :, pos], scales[seq, :, pos] = _quantize(x.reshape(total, kv, dim))
    K, V = _values(kq, kd), _values(vq, vd)                                      # [seqs][kv][room][dim]
    room = K.shape[2]
    Q = torch.zeros((seqs, R, heads, dim), device="cuda")
    Q[seq, at] = q.reshape(total, heads, dim)
    Q = Q.view(seqs, R, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv, R * group, dim)
    scores = torch.matmul(Q, K.transpose(2, 3)).mul_(1.0 / math.sqrt(dim)).view(seqs, kv, R, group, room)
    i, j = torch.arange(R, device="cuda"), torch.arange(room, device="cuda")
    seen = (j[None, None, :] <= lens[:, None, None] + i[None, :, None])[:, None, :, None, :]
    scores.masked_fill_(~seen, -math.inf)
    P = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    P /= P.sum(-1, keepdim=True)
    out = torch.matmul(P.view(seqs, kv, R * group, room), V)
    out = out.view(seqs, kv, R, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, R, heads * dim)[seq, at]
    if s["mass"] is not None:
        live = (i[None, :] < rows[:, None])[:, None, :, None, None]
        got = (P * live).sum((2, 3))
        old = (j[None, :] < lens[:, None])[:, None, :]
        new = ~old & (j[None, :] < (lens + rows)[:, None])[:, None, :]
        s["mass"] += torch.where(old, got, torch.zeros_like(got))
        s["mass"].copy_(torch.where(new, got, s["mass"]))
    where = (lens[:, None] + i[None, :]).clamp(max=room - 1)                       # [seqs][R]
    here = (torch.arange(seqs, device="cuda")[:, None], slice(None), where)
    inside = (lens[:, None] + i[None, :] < room)[:, :, None, None]
    new = torch.stack([torch.where(inside, _values(a[here], b[here]), 0.0) for a, b in ((kq, kd), (vq, vd))])
    return {"out": out, "new": new, "mass": s["mass"]}


def _attend_own(s):
    c, cache, qkv, lens = s["case"], s["cache"], s["qkv"], s["lens"].data_ptr()
    kv, dim, q = c["kv"], c["dim"], qkv.data_ptr()
    ld, k = qkv.shape[1], q + 4 * c["heads"] * dim
    cache.attend_dev(q, ld, c["heads"], lens, s["out"].data_ptr(), c["heads"] * dim, k_ptr=k, v_ptr=k + 4 * kv * dim, ldkv=ld,
                     rows=s.get("plan"), mass_ptr=None if s["mass"] is None else s["mass"].data_ptr())
    new = s["new"]
    cache.read_dev(c["rows"], new[0].data_ptr(), new[1].data_ptr(), from_ptr=lens)
    return {"out": s["out"], "new": new, "mass": s["mass"]}


def _evict_plain(s):
    c = s["case"]
    n, budget, recent = c["length"], c["budget"], c["recent"]
    lens = s["lens"].long()[:, None, None]
    j = torch.arange(n, device="cuda")[None, None, :]
    # the recent ones come before all others, and those past the end behind all
    weight = torch.where(j >= lens, -2.0, torch.where((j >= lens - recent) | (lens <= budget), math.inf, s["mass"]))
    kept = weight.sort(dim=-1, descending=True, stable=True).indices[:, :, :budget].sort(dim=-1).values
    left = s["lens"].clamp(max=budget)
    there = torch.arange(budget, device="cuda")[None, None, :] < left[:, None, None]
    s["left_mass"] = torch.where(there, s["mass"].gather(2, kept), 0.0)
    at = lambda x: x.gather(2, kept[..., None].expand(-1, -1, -1, x.shape[-1]))  # noqa: E731
    kq, kd, vq, vd = s["cache"]
    values = torch.stack([_values(at(kq), at(kd)), _values(at(vq), at(vd))]).mul_(there[None, ..., None])
    return {"kept": torch.where(there, kept, -1).int(), "left": left, "mass": s["left_mass"], "values": values.transpose(2, 3)}


def _evict_own(s):
    c = s["case"]
    s["cache"].evict_dev(s["to"], s["lens"].data_ptr(), s["left"].data_ptr(), c["budget"], c["recent"], s["mass"].data_ptr(),
                         s["left_mass"].data_ptr(), s["kept"].data_ptr())
    values = s["values"]
    s["to"].read_dev(c["budget"], values[0].data_ptr(), values[1].data_ptr())
    return {"kept": s["kept"], "left": s["left"], "mass": s["left_mass"], "values": values}


def _draw_plain(s):
    logits, params = s["logits"], s["params"]
    V = logits.shape[1]
    t, top_p, min_p = params[:, 0:1].double(), params[:, 2:3].double(), params[:, 3:4].double()
    top_k = params[:, 1:2].contiguous().view(torch.int32).long()
    best = logits.amax(1, keepdim=True)
    w = ((logits.double() - best.double()) / t.clamp(min=0.01)).exp_()
    ranked, order = logits.sort(dim=1, descending=True)
    cut_k = ranked.gather(1, torch.where((top_k > 0) & (top_k < V), top_k, V) - 1)
    short = w.gather(1, order).cumsum(1) < top_p * w.sum(1, keepdim=True)          # the prefixes that do not reach top_p
    cut_p = ranked.gather(1, torch.where(top_p < 1, short.sum(1, keepdim=True), V - 1).clamp(max=V - 1))
    w = torch.where((logits >= torch.maximum(cut_k, cut_p)) & (w >= min_p) & (w >= LEAST), w, 0.0)
    w = torch.where(t > 0, w, (torch.arange(V, device="cuda") == (logits == best).int().argmax(1, keepdim=True)).double())
    cum = w.cumsum(1)
    whole = cum[:, -1:]
    token = ((cum >= s["u"].double()[:, None] * whole) & (w > 0)).int().argmax(1, keepdim=True)
    return {"token": token.int().view(-1), "prob": (w.gather(1, token) / whole).float().view(-1)}


def _draw_own(s):
    n, V = s["logits"].shape
    s["sample"](s["logits"].data_ptr(), V, n, V, s["params"].data_ptr(), s["u"].data_ptr(), s["token"].data_ptr(), s["prob"].data_ptr())
    return {"token": s["token"], "prob": s["prob"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _attend_own, "evict": _evict_own, "draw": _draw_own}[kind](state)
    return {"attend": _attend_plain, "evict": _evict_plain, "draw": _draw_plain}[kind](state)


# ------------------------------------------------------------------- the work a pass cannot do without
def work(case):
    if case["kind"] == "draw":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 32 * case["rows"], "flops": 4.0 * n}
    seqs, kv, dim = case["seqs"], case["kv"], case["dim"]
    position = 2 * kv * (dim / 2 + dim / BLOCK * 2)       # bytes of keys and values
    if case["kind"] == "evict":
        mean = case["length"] * 0.625 if case["ragged"] else case["length"]
        left = min(mean, case["budget"])
        return {"bytes": seqs * (4.0 * kv * mean + left * (2 * position + 8 * kv) + left * 8 * kv * dim), "flops": seqs * left * 2.0 * kv * dim}
    cached = case["cached"] * (0.5625 if case["ragged"] else 1.0)
    rows = (case["rows"] + 1) / 2 if case["ragged"] else case["rows"]
    seen = rows * (cached + (rows + 1) / 2)               # pairs of a query row and a position
    moved = seqs * ((cached + rows) * position + rows * 4 * (2 * case["heads"] + 4 * kv) * dim)
    if case["mass"]:
        moved += seqs * 4 * kv * (2 * cached + rows)
    return {"bytes": float(moved), "flops": 4.0 * seqs * case["heads"] * dim * seen}


# ----------------------------------------------------------------- the same from the definitions, in 64 bits
def _stands_for(x):
    """What the cache holds of x [..][dim], in 64 bits."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    up, down = b.max(-1).values, b.min(-1).values
    d = (-torch.where(up + down >= 0, up, down).double() / 8).clamp(-65504, 65504).half().double()[..., None]
    return torch.where(d == 0, 0.0, (b.double() / d).round().clamp(-8, 7) * d).reshape(x.shape)


def exact(case, seed):
    if case["kind"] == "draw":
        logits, params, u = _draw_inputs(case, seed)
        probs = []
        for row, (t, _, top_p, min_p), top_k, r in zip(logits.double(), params.double().tolist(), params[:, 1].contiguous().view(torch.int32).tolist(), u.tolist()):
            if t <= 0:
                probs.append(1.0)
                continue
            e = torch.exp((row - row.max()) / max(t, 0.01))
            falling = row.sort(descending=True).values
            stays = (e >= min_p) & (e >= LEAST)
            if 0 < top_k < row.numel():
                stays &= row >= falling[top_k - 1]
            if top_p < 1:
                heavy = torch.exp((falling - falling[0]) / max(t, 0.01)).cumsum(0)
                reached = (heavy >= top_p * e.sum()).nonzero()
                if reached.numel():
                    stays &= row >= falling[reached[0, 0]]
            ids = stays.nonzero()[:, 0]
            mass = e[ids].cumsum(0)
            probs.append(float(e[ids[torch.searchsorted(mass, r * mass[-1:]).clamp(max=ids.numel() - 1)]] / mass[-1]))
        return {"token": None, "prob": torch.tensor(probs, dtype=torch.float64)}
    seqs, kv, dim = case["seqs"], case["kv"], case["dim"]
    if case["kind"] == "evict":
        lens, mass, g = _evict_inputs(case, seed)
        n, budget, recent = case["length"], case["budget"], case["recent"]
        k, v = (_stands_for(x.view(seqs, n, kv, dim)) for x in _keys_values(seqs * n, kv, dim, g))
        kept = torch.full((seqs, kv, budget), -1, dtype=torch.int32)
        left_mass = torch.zeros((seqs, kv, budget), dtype=torch.float64, device="cuda")
        values = torch.zeros((2, seqs, budget, kv, dim), dtype=torch.float64, device="cuda")
        for s in range(seqs):
            for h in range(kv):
                old = max(0, lens[s] - recent)
                heavy = mass[s, h, :old].cpu().numpy()
                take = old if lens[s] <= budget else budget - recent
                at = sorted(sorted(range(old), key=lambda j: (-heavy[j], j))[:take]) + list(range(old, lens[s]))
                kept[s, h, :len(at)] = torch.tensor(at, dtype=torch.int32)
                there = torch.tensor(at, device="cuda", dtype=torch.long)
                left_mass[s, h, :len(at)] = mass[s, h, there].double()
                values[0, s, :len(at), h], values[1, s, :len(at), h] = k[s, there, h], v[s, there, h]
        return {"kept": kept, "left": torch.tensor([min(x, budget) for x in lens], dtype=torch.int32), "mass": left_mass, "values": values}
    lens, rows, qkv, mass, room, g = _attend_inputs(case, seed)
    heads, group, R = case["heads"], case["heads"] // kv, case["rows"]
    K, V = (_stands_for(x.view(seqs, room, kv, dim)) for x in _keys_values(seqs * room, kv, dim, g))
    first, outs, new = 0, [], torch.zeros((2, seqs, R, kv, dim), dtype=torch.float64, device="cuda")
    mass = None if mass is None else mass.double()
    for s in range(seqs):
        x = qkv[first:first + rows[s]]
        q = x[:, :heads * dim].double().view(rows[s], kv, group, dim)
        end = lens[s] + rows[s]
        K[s, lens[s]:end] = _stands_for(x[:, heads * dim:(heads + kv) * dim].reshape(rows[s], kv, dim))
        V[s, lens[s]:end] = _stands_for(x[:, (heads + kv) * dim:].reshape(rows[s], kv, dim))
        first += rows[s]
        out = torch.empty((rows[s], kv, group, dim), dtype=torch.float64, device="cuda")
        late = torch.arange(end, device="cuda")[None, :] > lens[s] + torch.arange(rows[s], device="cuda")[:, None]
        if mass is not None:
            mass[s, :, lens[s]:end] = 0
        for h in range(kv):
            for a in range(group):
                p = torch.softmax((q[:, h, a] @ K[s, :end, h].T / math.sqrt(dim)).masked_fill(late, -math.inf), dim=1)
                out[:, h, a] = p @ V[s, :end, h]
                if mass is not None:
                    mass[s, h, :end] += p.sum(0)
        outs.append(out.view(rows[s], heads * dim))
        stop = min(lens[s] + R, room)
        new[0, s, :stop - lens[s]], new[1, s, :stop - lens[s]] = K[s, lens[s]:stop], V[s, lens[s]:stop]
    return {"out": torch.cat(outs), "new": new, "mass": mass}
