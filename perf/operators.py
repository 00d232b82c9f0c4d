"""Cases, plain forms and exact values of three serving operators.

``kind`` names the operator of a case:

* ``norm_rope``: RMS norm of every query and key head, split-half rotation, and
  the paged K / V write (``KernelOps.qk_norm_rope_kv_write``);
* ``lora``: low-rank adapters of many requests added beside a shared projection
  (``KernelOps.lora_add``);
* ``sparse``: one decode step of attention over selected pages: key bounds of
  the pages just written, page selection, attention (``KernelOps.page_bounds``,
  ``attn_select``, ``attn_decode_sparse``).

Shapes are those of the framework's presets: 32 / 8 heads and hidden 4096, 64 /
8 heads and hidden 8192, their tensor-parallel shards, head_dim 128 (and 64),
pages of 16 tokens, contexts up to 131072.  ``run`` is the plain form in 32 bits
(64 for page scores, whose order decides) unless ``own`` is set; ``exact`` is
the definition in 64 bits.
"""
import math

import torch

own = False

PAGE = 16
EPS = 1e-5
DEV = "cuda"

_ops = None


def _kernels():
    global _ops
    if _ops is None:
        from lunaflux_b200.ops import KernelOps
        _ops = KernelOps()
    return _ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    """Normal values of `dtype`, made in pieces so that a large cache needs no fp32 copy of itself."""
    out = torch.empty(*shape, device=DEV, dtype=dtype)
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, device=DEV, generator=g) * scale
    return out


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _norm_rope(tokens, hq, hkv, d=128, decode=False, pad=0, max_pos=8192):
    return {"kind": "norm_rope", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "decode": decode, "pad": pad,
            "max_pos": max_pos}


def _lora(rows, k, n, rank, pool, used, slices="one", ragged=False, plain_rows=0, f32=False):
    return {"kind": "lora", "rows": rows, "k": k, "n": n, "rank": rank, "pool": pool, "used": used,
            "slices": slices, "ragged": ragged, "plain_rows": plain_rows, "f32": f32}


def _sparse(rows, hq, hkv, ctx, budget, ragged=False, first=1, last=2):
    return {"kind": "sparse", "rows": rows, "hq": hq, "hkv": hkv, "ctx": ctx, "budget": budget, "ragged": ragged,
            "first": first, "last": last}


def listed():
    cases = [
        # one user's decode step: a single token, where only latency counts
        ("norm_rope_decode_1", _norm_rope(1, 32, 8, decode=True)),
        # a full decode bucket of 256 rows, 7 of them padding of the captured batch
        ("norm_rope_decode_256", _norm_rope(256, 32, 8, decode=True, pad=7)),
        # an odd mixed prefill chunk with the wide model's heads, far positions
        ("norm_rope_chunk_1023", _norm_rope(1023, 64, 8, max_pos=131072)),
        # the largest prefill step the benchmark's scheduler packs
        ("norm_rope_prefill_8192", _norm_rope(8192, 32, 8)),
        # one request with an adapter, QKV projection, one token
        ("lora_decode_1", _lora(1, 4096, 6144, 16, 8, 1, slices="qkv")),
        # 64 requests, each with its own adapter, beside the QKV projection
        ("lora_decode_64", _lora(64, 4096, 6144, 16, 64, 64, slices="qkv")),
        # a 256-row decode bucket beside the down projection, 32 adapters of ranks 8 to 64 and rows without one
        ("lora_decode_256", _lora(256, 14336, 4096, 64, 48, 32, ragged=True, plain_rows=37)),
        # a prefill step of seven requests with adapters of different ranks beside the QKV projection
        ("lora_prefill_8192", _lora(8192, 4096, 6144, 64, 8, 7, slices="qkv", ragged=True, plain_rows=501)),
        # one request with a long prompt, small budget
        ("sparse_1x8191", _sparse(1, 32, 8, 8191, 64)),
        # a ragged batch from a handful of tokens to 32K
        ("sparse_17_ragged", _sparse(17, 32, 8, 32768, 128, ragged=True)),
        # the wide model at its longest context
        ("sparse_4x131072", _sparse(4, 64, 8, 131072, 256, first=4, last=16)),
        # a batch of 64 requests of 32K tokens
        ("sparse_64x32768", _sparse(64, 32, 8, 32768, 128)),
    ]
    return [dict(c, name=name) for name, c in cases]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """A case of the listed ones' ranges, with fewer rows where it would cost more than the largest of its kind."""
    case = _draw(rng)
    limit = [work(c) for c in listed() if c["kind"] == case["kind"]]
    size = "tokens" if case["kind"] == "norm_rope" else "rows"
    while case[size] > 1 and any(work(case)[x] > max(w[x] for w in limit) for x in ("bytes", "flops")):
        case[size] = case[size] * 7 // 8
        for part in ("pad", "plain_rows"):
            if part in case:
                case[part] = case[part] * 7 // 8
    return case


def _draw(rng):
    kind = rng.choice(["norm_rope", "lora", "sparse"])
    if kind == "norm_rope":
        hq, hkv, d = rng.choice([(32, 8, 128), (64, 8, 128), (8, 1, 128), (16, 2, 128), (4, 1, 128), (12, 12, 128),
                                 (64, 8, 64), (40, 8, 64), (16, 2, 64)])
        tokens = _log(rng, 1, 8192)
        decode = tokens <= 512 and rng.random() < 0.6
        return _norm_rope(tokens, hq, hkv, d=d, decode=decode,
                          pad=rng.randint(0, tokens // 2) if decode else 0,
                          max_pos=rng.choice([8192, 32768, 131072]))
    if kind == "lora":
        k = rng.choice([512, 1024, 2048, 4096, 8192, 14336, 1000, 4104])
        n = rng.choice([768, 1280, 2048, 4096, 6144, 8192, 10240, 1544])
        slices = "qkv" if n % 48 == 0 and rng.random() < 0.7 else "one"
        rank = rng.choice([8, 16, 24, 32, 64, 128])
        f32 = rng.random() < 0.25
        rows = _log(rng, 1, 8192)
        pool = rng.choice([1, 3, 8, 20, 64])
        return _lora(rows, k, n, rank, pool, rng.randint(1, min(pool, rows)), slices=slices,
                     ragged=rng.random() < 0.5, plain_rows=rng.randint(0, rows // 3), f32=f32)
    hq, hkv = rng.choice([(32, 8), (64, 8), (8, 1), (16, 2), (8, 4), (16, 1), (12, 4), (5, 1)])
    ctx = _log(rng, 1, 131072)
    rows = _log(rng, 1, 256)
    first, last = rng.randint(0, 4), rng.randint(1, 8)
    return _sparse(rows, hq, hkv, ctx, first + last + _log(rng, 1, 240), ragged=rng.random() < 0.6, first=first,
                   last=last)


# ---------------------------------------------------------------------------
# what a case fixes beyond its sizes
# ---------------------------------------------------------------------------
def _slices(case):
    """Column widths of the stacked projections: Q, K and V of a 4:1:1 QKV projection, or one."""
    n = case["n"]
    return (n // 6 * 4, n // 6, n // 6) if case["slices"] == "qkv" else (n,)


def _adapter_rows(case):
    """Rows of every adapter of the pool: the `used` first ones share the rows
    that have an adapter, the earlier ones with more of them where ragged."""
    total = case["rows"] - case["plain_rows"]
    used = min(case["used"], total)
    if used == 0:
        return [0] * case["pool"]
    w = [1.0 / (i + 1) if case["ragged"] else 1.0 for i in range(used)]
    counts = [1 + int((total - used) * x / sum(w)) for x in w]
    counts[0] += total - sum(counts)
    return counts + [0] * (case["pool"] - used)


def _ranks(case):
    """Rank of every adapter: the pool's, or a half, a quarter or an eighth of it where ragged."""
    r = case["rank"]
    return [max(1, r >> (i % 4)) if case["ragged"] else r for i in range(case["pool"])]


def _lens(case):
    """KV length of every row with the new token: the context, or from one
    token to it, spread over the logarithm, where ragged."""
    ctx, rows = case["ctx"], case["rows"]
    if not case["ragged"]:
        return [max(1, ctx - 5 * i % 61) for i in range(rows)]
    return [max(1, int(round(ctx ** ((i * 0.6180339887 + 1.0) % 1.0)))) if i else ctx for i in range(rows)]


def work(case):
    kind = case["kind"]
    if kind == "norm_rope":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        live = t - case["pad"]
        nbytes = 2 * 2 * d * (t * hq + live * 2 * hkv) + min(t, case["max_pos"]) * d * 4 + 8 * t + 4 * d
        return {"bytes": nbytes, "flops": t * (hq + hkv) * d * 7}
    if kind == "lora":
        k, n, s = case["k"], case["n"], len(_slices(case))
        counts, ranks = _adapter_rows(case), _ranks(case)
        es = 4 if case["f32"] else 2
        nbytes = sum(counts) * (2 * k + 2 * es * n + 4) + 12 * case["pool"]
        flops = 0
        for c, r in zip(counts, ranks):
            if c:
                nbytes += 2 * r * (s * k + n)
                flops += 2 * c * r * (s * k + n)
        return {"bytes": nbytes, "flops": flops}
    hq, hkv, d = case["hq"], case["hkv"], 128
    nbytes = flops = 0
    for length in _lens(case):
        pages = -(-length // PAGE)
        sel = min(pages, case["budget"])
        scored = pages if pages > case["budget"] else 0
        tail = length - (pages - 1) * PAGE
        kept = (sel - 1) * PAGE + tail
        nbytes += hkv * (scored * 2 * d * 2 + kept * 2 * d * 2 + 2 * d * 2) + 2 * hq * d * 2 + 4 * pages
        nbytes += 4 * hkv * case["budget"]
        flops += hq * (scored * 4 * d + kept * 4 * d)
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    return {"norm_rope": _prepare_norm_rope, "lora": _prepare_lora, "sparse": _prepare_sparse}[case["kind"]](case, seed)


def _prepare_norm_rope(case, seed):
    g = _gen(seed)
    t, hq, hkv, d, max_pos = case["tokens"], case["hq"], case["hkv"], case["d"], case["max_pos"]
    qkv = _randn(g, t, (hq + 2 * hkv) * d)
    # a projection's channels differ in scale; trained norm weights lie around one
    qkv *= (0.2 + 3.0 * torch.rand((hq + 2 * hkv) * d, device=DEV, generator=g)).bfloat16()
    wq = (1.0 + 0.3 * torch.randn(d, device=DEV, generator=g)).bfloat16()
    wk = (1.0 + 0.3 * torch.randn(d, device=DEV, generator=g)).bfloat16()
    inv = 500000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    ang = torch.arange(max_pos, device=DEV, dtype=torch.float64)[:, None] * inv[None]
    cos_sin = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    if case["decode"]:
        # every row its own sequence at its own position, each with its own last page
        pages = t + 3
        pos = torch.randint(0, max_pos, (t,), device=DEV, generator=g)
        page = torch.randperm(pages, device=DEV, generator=g)[:t]
        slots = page * PAGE + pos % PAGE
        if case["pad"]:
            slots[t - case["pad"]:] = -1
            pos[t - case["pad"]:] = 0
    else:
        # one chunk of consecutive positions in scattered pages
        start = int(torch.randint(0, max(1, max_pos - t + 1), (1,), device=DEV, generator=g))
        pos = (start + torch.arange(t, device=DEV)) % max_pos
        first = start // PAGE
        pages = t // PAGE + 5
        perm = torch.randperm(pages, device=DEV, generator=g)
        at = start + torch.arange(t, device=DEV)
        slots = perm[at // PAGE - first] * PAGE + at % PAGE
    return {"case": case, "qkv": qkv, "wq": wq, "wk": wk, "cos_sin": cos_sin, "pos": pos.int(), "slots": slots.int(),
            "kc": _randn(g, pages, hkv, PAGE, d), "vc": _randn(g, pages, hkv, PAGE, d),
            "q_out": torch.zeros(t, hq * d, device=DEV, dtype=torch.bfloat16)}


def _prepare_lora(case, seed):
    g = _gen(seed)
    t, k, n, r, pool = case["rows"], case["k"], case["n"], case["rank"], case["pool"]
    slices = _slices(case)
    dt = torch.float32 if case["f32"] else torch.bfloat16
    counts = _adapter_rows(case)
    ids = torch.full((t,), -1, device=DEV, dtype=torch.long)
    ids[:sum(counts)] = torch.repeat_interleave(torch.arange(pool, device=DEV), torch.tensor(counts, device=DEV))
    if t > 512:
        # prefill: a request's rows lie together, requests in any order
        order = torch.randperm(pool + 1, device=DEV, generator=g)
        ids = ids[torch.argsort(order[ids + 1], stable=True)]
    else:
        ids = ids[torch.randperm(t, device=DEV, generator=g)]
    # the engine's step block: rows grouped by adapter
    by = torch.argsort(ids, stable=True)
    rows = by[t - sum(counts):].int().contiguous()
    starts = torch.tensor([0] + counts, device=DEV).cumsum(0).int()
    base = _randn(g, t, n, dtype=dt)
    return {"case": case, "slices": slices, "ids": ids, "rows": rows, "starts": starts,
            "x": _randn(g, t, k), "a": _randn(g, pool, len(slices) * r, k, scale=k ** -0.5),
            "b": _randn(g, pool, n, r, scale=0.05), "scales": 0.25 + 2.0 * torch.rand(pool, device=DEV, generator=g),
            "ranks": torch.tensor(_ranks(case), device=DEV, dtype=torch.int32), "base": base, "out": base.clone()}


def _bounds(keys):
    """[.., tokens, d] -> [.., 2, d]: smallest and largest key of a page in every dimension."""
    return torch.stack([keys.amin(-2), keys.amax(-2)], -2)


def _prepare_sparse(case, seed):
    g = _gen(seed)
    rows, hq, hkv, d = case["rows"], case["hq"], case["hkv"], 128
    lens = _lens(case)
    npages = [-(-length // PAGE) for length in lens]
    width = max(npages)
    pages = 1 + sum(npages)                # physical page 0 stays the zero page
    perm = torch.randperm(pages - 1, device=DEV, generator=g) + 1
    bt = torch.zeros(rows, width, device=DEV, dtype=torch.int32)
    at = 0
    for i, p in enumerate(npages):
        bt[i, :p] = perm[at:at + p].int()
        at += p
    # keys: an offset per head and channel, a drift shared by a page's tokens, noise
    kc = _randn(g, pages, hkv, PAGE, d, scale=0.8)
    centre = _randn(g, hkv, 1, d)
    for i in range(0, pages, 4096):
        j = min(pages, i + 4096)
        kc[i:j] += _randn(g, j - i, hkv, 1, d, scale=0.7) + centre
    vc = _randn(g, pages, hkv, PAGE, d)
    kc[0] = 0
    vc[0] = 0
    bounds = torch.empty(pages, hkv, 2, d, device=DEV, dtype=torch.bfloat16)
    for i in range(0, pages, 4096):
        j = min(pages, i + 4096)
        bounds[i:j] = _bounds(kc[i:j])
    # the newest token's page holds what its bounds were before that token
    lens_t = torch.tensor(lens, device=DEV, dtype=torch.int32)
    for tail in range(1, PAGE):
        at = [i for i in range(rows) if (lens[i] - 1) % PAGE == tail]
        if at:
            last = bt[at, [npages[i] - 1 for i in at]].long()
            bounds[last] = _bounds(kc[last, :, :tail])
    qkv = _randn(g, rows, (hq + 2 * hkv) * d)
    return {"case": case, "qkv": qkv, "tok": torch.arange(rows, device=DEV, dtype=torch.int32),
            "lens": lens_t, "start": lens_t - 1, "bt": bt, "kc": kc, "vc": vc, "bounds": bounds,
            "sel": torch.full((rows, hkv, case["budget"]), -1, device=DEV, dtype=torch.int32),
            "out": torch.zeros(rows, hq * d, device=DEV, dtype=torch.bfloat16), "host_lens": lens,
            # the serving engine's workspace: page scores
            "ws": torch.zeros(rows * hkv * 2 * width, device=DEV)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"norm_rope": _run_norm_rope, "lora": _run_lora, "sparse": _run_sparse}[state["case"]["kind"]](state)


def _run_norm_rope(s):
    c = s["case"]
    t, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
    if own:
        _kernels().qk_norm_rope_kv_write(s["qkv"], s["wq"], s["wk"], EPS, s["pos"], s["slots"], s["cos_sin"],
                                         s["q_out"], s["kc"], s["vc"], hq, hkv, PAGE)
        return {"q": s["q_out"], "k": s["kc"], "v": s["vc"]}
    x = s["qkv"].view(t, hq + 2 * hkv, d).float()
    cs = s["cos_sin"][s["pos"].long()][:, None]
    cos, sin = cs[..., 0], cs[..., 1]

    def turn(x, w):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        y1, y2 = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([y1 * cos - y2 * sin, y2 * cos + y1 * sin], -1).bfloat16()

    q = turn(x[:, :hq], s["wq"]).reshape(t, hq * d)
    k = turn(x[:, hq:hq + hkv], s["wk"])
    # padding rows (slot -1) all lie at the end of a bucket
    n = t - c["pad"]
    slot = s["slots"][:n].long()
    s["kc"][slot // PAGE, :, slot % PAGE] = k[:n]
    s["vc"][slot // PAGE, :, slot % PAGE] = s["qkv"].view(t, hq + 2 * hkv, d)[:n, hq + hkv:]
    return {"q": q, "k": s["kc"], "v": s["vc"]}


def _run_lora(s):
    c = s["case"]
    if own:
        _kernels().lora_add(s["x"], s["a"], s["b"], s["scales"], s["ranks"], s["rows"], s["starts"], s["base"],
                            s["out"], s["slices"])
        return {"out": s["out"]}
    r, counts, ranks = c["rank"], _adapter_rows(c), _ranks(c)
    out = s["out"]
    at = 0
    for a, m in enumerate(counts):
        if not m:
            continue
        rows = s["rows"][at:at + m].long()
        at += m
        x = s["x"][rows].float()
        col = 0
        for i, width in enumerate(s["slices"]):
            h = x @ s["a"][a, i * r:i * r + ranks[a]].float().t()
            delta = h @ s["b"][a, col:col + width, :ranks[a]].float().t()
            y = s["base"][rows, col:col + width].float() + s["scales"][a] * delta
            out[rows, col:col + width] = y.to(out.dtype)
            col += width
    return {"out": out}


def _run_sparse(s):
    c = s["case"]
    rows, hq, hkv, d, budget = c["rows"], c["hq"], c["hkv"], 128, c["budget"]
    first, last = c["first"], c["last"]
    if own:
        ops = _kernels()
        ops.page_bounds(s["kc"], s["bounds"], s["bt"], s["start"], s["lens"], 1)
        ops.attn_select(s["qkv"], s["tok"], s["lens"], s["bt"], s["bounds"], s["sel"], first, last, hq, hkv, s["ws"])
        ops.attn_decode_sparse(s["qkv"], s["out"], s["tok"], s["lens"], s["bt"], s["sel"], s["kc"], s["vc"], hq, hkv)
        return {"bounds": s["bounds"], "sel": s["sel"], "out": s["out"]}
    kc, vc, bounds, group = s["kc"], s["vc"], s["bounds"], hq // hkv
    for r, length in enumerate(s["host_lens"]):
        pages = -(-length // PAGE)
        bt = s["bt"][r, :pages].long()
        tail = length - (pages - 1) * PAGE
        bounds[bt[-1]] = _bounds(kc[bt[-1], :, :tail])
        q = s["qkv"][r, :hq * d].view(hkv, group, d)
        if pages <= budget:
            sel = torch.arange(pages, device=DEV).expand(hkv, pages)
        else:
            # sum_d max(q lo, q hi) = q+ hi + q- lo, in 64 bits: the order of the scores decides
            b = bounds[bt].transpose(0, 1).double()                     # [hkv, pages, 2, d]
            qd = q.double()
            score = (qd.clamp(max=0) @ b[:, :, 0].transpose(1, 2) + qd.clamp(min=0) @ b[:, :, 1].transpose(1, 2))
            score = score.amax(1)                                       # [hkv, pages]
            score[:, :first] = math.inf
            score[:, pages - last:] = math.inf
            order = torch.sort(score, dim=-1, descending=True, stable=True).indices
            sel = order[:, :budget].sort(-1).values
        s["sel"][r].fill_(-1)
        s["sel"][r, :, :sel.shape[1]] = sel.int()
        head = torch.arange(hkv, device=DEV)[:, None]
        ks = kc[bt[sel], head].reshape(hkv, -1, d).float()
        vs = vc[bt[sel], head].reshape(hkv, -1, d).float()
        where = (sel[..., None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(hkv, 1, -1)
        p = (q.float() @ ks.transpose(1, 2) / math.sqrt(d)).masked_fill(where >= length, -math.inf).softmax(-1)
        s["out"][r] = (p @ vs).reshape(hq * d).bfloat16()
    return {"bounds": bounds, "sel": s["sel"], "out": s["out"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "lora": _exact_lora, "sparse": _exact_sparse}[case["kind"]](case, s)


def _exact_norm_rope(c, s):
    t, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
    half = d // 2
    table = s["cos_sin"].double()
    heads = s["qkv"].double().view(t, -1, d)
    weight = torch.cat([s["wq"].double().expand(hq, d), s["wk"].double().expand(hkv, d)])
    inv = 1.0 / (heads[:, :hq + hkv].square().sum(-1) / d + EPS).sqrt()
    normed = heads[:, :hq + hkv] * inv[..., None] * weight
    z = torch.complex(normed[..., :half].contiguous(), normed[..., half:].contiguous())
    at = table[s["pos"].long()]
    z = z * torch.complex(at[..., 0].contiguous(), at[..., 1].contiguous())[:, None]
    turned = torch.cat([z.real, z.imag], -1)
    k, v = s["kc"].double(), s["vc"].double()
    live = (s["slots"] >= 0).nonzero()[:, 0]
    slot = s["slots"][live].long()
    k.view(-1, hkv, PAGE, d)[slot // PAGE, :, slot % PAGE] = turned[live, hq:]
    v.view(-1, hkv, PAGE, d)[slot // PAGE, :, slot % PAGE] = heads[live, hq + hkv:]
    return {"q": turned[:, :hq].reshape(t, hq * d), "k": k, "v": v}


def _exact_lora(c, s):
    out = s["out"].double()
    r = c["rank"]
    edges = [0]
    for w in s["slices"]:
        edges.append(edges[-1] + w)
    for a in range(c["pool"]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        if not rows.numel():
            continue
        rank = int(s["ranks"][a])
        low = torch.einsum("tk,jk->tj", s["x"][rows].double(), s["a"][a].double())
        for i in range(len(s["slices"])):
            lo, hi = edges[i], edges[i + 1]
            up = torch.einsum("tj,cj->tc", low[:, i * r:i * r + rank], s["b"][a, lo:hi, :rank].double())
            out[rows, lo:hi] = s["base"][rows, lo:hi].double() + float(s["scales"][a]) * up
    return {"out": out}


def _exact_sparse(c, s):
    rows, hq, hkv, d, budget = c["rows"], c["hq"], c["hkv"], 128, c["budget"]
    g = hq // hkv
    bounds = s["bounds"].double()
    sel = torch.full((rows, hkv, budget), -1, dtype=torch.int32, device=DEV)
    out = torch.zeros(rows, hq * d, dtype=torch.float64, device=DEV)
    for r in range(rows):
        length = int(s["lens"][r])
        n = (length + PAGE - 1) // PAGE
        table = s["bt"][r, :n].long()
        newest = s["kc"][table[n - 1], :, :length - (n - 1) * PAGE].double()
        bounds[table[n - 1], :, 0] = newest.min(1).values
        bounds[table[n - 1], :, 1] = newest.max(1).values
        for h in range(hkv):
            q = s["qkv"][r, h * g * d:(h + 1) * g * d].double().view(g, d)
            if n <= budget:
                chosen = torch.arange(n, device=DEV)
            else:
                b = bounds[table, h]
                best = torch.full((n,), -math.inf, dtype=torch.float64, device=DEV)
                for j in range(g):
                    best = torch.maximum(best, torch.maximum(b[:, 0] * q[j], b[:, 1] * q[j]).sum(-1))
                mid = torch.arange(c["first"], n - c["last"], device=DEV)
                take = budget - c["first"] - c["last"]
                top = mid[torch.argsort(-best[mid], stable=True)[:take]]
                chosen = torch.cat([torch.arange(c["first"], device=DEV), top.sort().values,
                                    torch.arange(n - c["last"], n, device=DEV)])
            sel[r, h, :chosen.numel()] = chosen.int()
            pos = (chosen[:, None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(-1)
            keep = pos < length
            k = s["kc"][table[chosen], h].reshape(-1, d)[keep].double()
            v = s["vc"][table[chosen], h].reshape(-1, d)[keep].double()
            w = torch.exp((logit := q @ k.T / d ** 0.5) - logit.max(-1, keepdim=True).values)
            out[r, h * g * d:(h + 1) * g * d] = ((w @ v) / w.sum(-1, keepdim=True)).reshape(-1)
    return {"bounds": bounds, "sel": sel, "out": out}
