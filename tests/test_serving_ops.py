"""Head norm + rotation + KV write, low-rank adapters and attention over
selected pages, against their definitions in 64 bits: the plain operator set on
the CPU, the kernels on the GPU.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.  Sums in
the tensor cores are off by at most 17 * 2^-23 of the sum of magnitudes per step
of 16 terms.  Where inputs are small integers, every sum is exact in fp32 and the
outputs have to be equal.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
BF, I32, F32 = torch.bfloat16, torch.int32, torch.float32


@pytest.fixture(params=["torch", pytest.param("kernels", marks=gpu)])
def ops(request):
    if request.param == "torch":
        from lunaflux_b200.ops import TorchOps
        o = TorchOps("cpu")
        o.dev = "cpu"
        return o
    from lunaflux_b200.ops import KernelOps
    o = KernelOps()
    o.dev = "cuda"
    return o


@pytest.fixture
def kernels():
    from lunaflux_b200.ops import KernelOps
    o = KernelOps()
    o.dev = "cuda"
    o.read_error(True)
    return o


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _no_error(ops):
    assert ops.read_error(True)[0] == 0


def _within(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3g} over"


# ---------------------------------------------------------------------------
# head norm + rotation + KV write
# ---------------------------------------------------------------------------
def _norm_rope_inputs(T, Hq, Hkv, D, seed, page=16, max_pos=512, pad=0, extra=0):
    g = _gen(seed)
    width = (Hq + 2 * Hkv) * D
    qkv = _randn(g, T, width + extra, scale=2.0)
    pages = T + 2
    perm = torch.randperm(pages * page, generator=g)[:T]
    slots = perm.int()
    if pad:
        slots[T - pad:] = -1
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv
    return dict(qkv=qkv, wq=_randn(g, D, scale=0.3) + 1, wk=_randn(g, D, scale=0.3) + 1,
                pos=torch.randint(0, max_pos, (T,), generator=g).int(), slots=slots,
                cs=torch.stack([ang.cos(), ang.sin()], -1).float().contiguous(),
                kc=_randn(g, pages, Hkv, page, D), vc=_randn(g, pages, Hkv, page, D), width=width)


def _norm_rope_reference(x, Hq, Hkv, D, eps, page=16):
    """Values in 64 bits and the magnitude |y1| + |y2| behind every output."""
    T = x["qkv"].shape[0]
    h = x["qkv"][:, :x["width"]].double().view(T, Hq + 2 * Hkv, D)
    w = torch.cat([x["wq"].double().expand(Hq, D), x["wk"].double().expand(Hkv, D)])
    y = h[:, :Hq + Hkv] / (h[:, :Hq + Hkv].square().mean(-1, keepdim=True) + eps).sqrt() * w
    cs = x["cs"].double()[x["pos"].long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    y1, y2 = y[..., :D // 2], y[..., D // 2:]
    o = torch.cat([y1 * c - y2 * s, y2 * c + y1 * s], -1)
    mag = (y1.abs() + y2.abs()).repeat(1, 1, 2)
    kc, vc = x["kc"].double(), x["vc"].double()
    km = torch.zeros_like(kc)
    for t, slot in enumerate(x["slots"].tolist()):
        if slot >= 0:
            kc[slot // page, :, slot % page] = o[t, Hq:]
            km[slot // page, :, slot % page] = mag[t, Hq:]
            vc[slot // page, :, slot % page] = h[t, Hq + Hkv:]
    return o[:, :Hq].reshape(T, -1), mag[:, :Hq].reshape(T, -1), kc, km, vc


def _norm_rope_check(q, kc, vc, ref):
    # fp32: the sum of squares (all positive) to 2^-20, rsqrt, two products and the
    # rotation to 2^-21 each: under 2^-18 of |y1| + |y2|; then one rounding to bf16
    rq, mq, rk, mk, rv = ref
    _within(q, rq, 2.0 ** -8 * rq.abs() + 2.0 ** -18 * mq, "q")
    _within(kc, rk, torch.where(mk > 0, 2.0 ** -8 * rk.abs() + 2.0 ** -18 * mk, torch.zeros_like(rk)), "k")
    assert torch.equal(vc.double().cpu(), rv)


@pytest.mark.parametrize("T,Hq,Hkv,D", [(1, 32, 8, 128), (3, 8, 1, 128), (37, 4, 1, 64), (5, 2, 2, 256),
                                        (130, 64, 8, 128), (17, 5, 3, 128), (9, 1, 1, 64), (300, 12, 12, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_rope(ops, T, Hq, Hkv, D, in_place):
    x = _norm_rope_inputs(T, Hq, Hkv, D, T + Hq, pad=T // 5)
    ref = _norm_rope_reference(x, Hq, Hkv, D, 1e-5)
    d = {k: v.to(ops.dev) if torch.is_tensor(v) else v for k, v in x.items()}
    keep = d["qkv"].clone()
    q = d["qkv"][:, :Hq * D] if in_place else torch.full((T, Hq * D), 7.0, dtype=BF, device=ops.dev)
    ops.qk_norm_rope_kv_write(d["qkv"], d["wq"], d["wk"], 1e-5, d["pos"], d["slots"], d["cs"], q, d["kc"], d["vc"],
                              Hq, Hkv, 16)
    _norm_rope_check(q, d["kc"], d["vc"], ref)
    assert torch.equal(d["qkv"][:, Hq * D:], keep[:, Hq * D:])     # K and V columns are only read
    if not in_place:
        assert torch.equal(d["qkv"], keep)
    _no_error(ops)


def test_norm_rope_strides_and_zero_rows(ops):
    """Row-strided qkv and output, a zero head (norm 0: eps alone), no rows."""
    T, Hq, Hkv, D = 6, 4, 2, 128
    x = _norm_rope_inputs(T, Hq, Hkv, D, 3, extra=64)
    x["qkv"][2, :D] = 0
    x["qkv"][3] = 0
    ref = _norm_rope_reference(x, Hq, Hkv, D, 1e-6)
    d = {k: v.to(ops.dev) if torch.is_tensor(v) else v for k, v in x.items()}
    out = torch.full((T, Hq * D + 8), 5.0, dtype=BF, device=ops.dev)
    ops.qk_norm_rope_kv_write(d["qkv"][:, :x["width"]], d["wq"], d["wk"], 1e-6, d["pos"], d["slots"], d["cs"],
                              out[:, :Hq * D], d["kc"], d["vc"], Hq, Hkv, 16)
    _norm_rope_check(out[:, :Hq * D], d["kc"], d["vc"], ref)
    assert bool((out[:, Hq * D:] == 5.0).all())
    before = d["kc"].clone()
    ops.qk_norm_rope_kv_write(d["qkv"][:0, :x["width"]], d["wq"], d["wk"], 1e-6, d["pos"][:0], d["slots"][:0], d["cs"],
                              out[:0, :Hq * D], d["kc"], d["vc"], Hq, Hkv, 16)
    assert torch.equal(before, d["kc"])


@gpu
@pytest.mark.parametrize("T,Hq,Hkv,D", [(400, 8, 2, 128), (1023, 64, 8, 128), (297, 5, 3, 128), (300, 4, 1, 256), (297, 3, 3, 256)])
def test_norm_rope_many_tokens(kernels, T, Hq, Hkv, D):
    """More than two tokens per SM: the narrow CTAs."""
    x = _norm_rope_inputs(T, Hq, Hkv, D, T + Hq, pad=T // 7)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in x.items()}
    q = torch.full((T, Hq * D), 7.0, dtype=BF, device="cuda")
    kernels.qk_norm_rope_kv_write(d["qkv"], d["wq"], d["wk"], 1e-5, d["pos"], d["slots"], d["cs"], q, d["kc"], d["vc"],
                                  Hq, Hkv, 16)
    _norm_rope_check(q, d["kc"], d["vc"], _norm_rope_reference(x, Hq, Hkv, D, 1e-5))
    _no_error(kernels)


@gpu
def test_norm_rope_bad_position_and_slot_are_recorded(kernels):
    T, Hq, Hkv, D = 4, 2, 1, 128
    for field, value in (("pos", 512), ("pos", -1), ("slots", (T + 2) * 16)):
        x = _norm_rope_inputs(T, Hq, Hkv, D, 5)
        x[field][2] = value
        d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in x.items()}
        q = torch.zeros(T, Hq * D, dtype=BF, device="cuda")
        kernels.qk_norm_rope_kv_write(d["qkv"], d["wq"], d["wk"], 1e-5, d["pos"], d["slots"], d["cs"], q, d["kc"],
                                      d["vc"], Hq, Hkv, 16)
        code, info = kernels.read_error(True)
        assert (code, info) == (3, 2)
        if field == "slots":                       # nothing but that row's K / V is lost
            x["slots"][2] = -1
            _norm_rope_check(q, d["kc"], d["vc"], _norm_rope_reference(x, Hq, Hkv, D, 1e-5))


# ---------------------------------------------------------------------------
# low-rank adapters
# ---------------------------------------------------------------------------
def _lora_inputs(T, K, slices, R, counts, seed, ranks=None, f32=False, integer=True, order=None):
    g = _gen(seed)
    N, S, pool = sum(slices), len(slices), len(counts)
    ranks = [R] * pool if ranks is None else ranks
    if integer:
        def make(*shape, top):
            return torch.randint(-top, top + 1, shape, generator=g).to(BF)
        # |h| <= K, |delta| <= 128 * 2 * K: whole numbers below 2^24
        x, a, b = make(T, K, top=1), make(pool, S * R, K, top=1), make(pool, N, R, top=2)
        base = torch.randint(-64, 65, (T, N), generator=g).to(F32 if f32 else BF)
        scales = 2.0 ** torch.randint(-2, 3, (pool,), generator=g).float()
    else:
        x, a, b = _randn(g, T, K), _randn(g, pool, S * R, K, scale=K ** -0.5), _randn(g, pool, N, R, scale=0.2)
        base = _randn(g, T, N, dtype=F32 if f32 else BF)
        scales = torch.rand(pool, generator=g) + 0.5
    for i, r in enumerate(ranks):              # what lies past the rank is never used
        for s in range(S):
            a[i, s * R + r:(s + 1) * R] = float("nan")
        b[i, :, r:] = float("nan")
    perm = torch.randperm(T, generator=g) if order is None else order
    rows = perm[:sum(counts)].int()
    starts = torch.tensor([0] + counts).cumsum(0).int()
    return dict(x=x, a=a, b=b, base=base, scales=scales, ranks=torch.tensor(ranks, dtype=I32), rows=rows, starts=starts)


def _lora_reference(v, slices, R):
    """out in 64 bits and scale * sum_j |B| sum_k |A| |x| behind every element."""
    out = v["base"].double()
    mag = torch.zeros_like(out)
    for ad, rank in enumerate(v["ranks"].tolist()):
        rows = v["rows"][int(v["starts"][ad]):int(v["starts"][ad + 1])].long()
        c = 0
        for s, n in enumerate(slices):
            a = v["a"][ad, s * R:s * R + rank].double()
            b = v["b"][ad, c:c + n, :rank].double()
            out[rows, c:c + n] += float(v["scales"][ad]) * ((v["x"][rows].double() @ a.T) @ b.T)
            mag[rows, c:c + n] = float(v["scales"][ad]) * ((v["x"][rows].double().abs() @ a.abs().T) @ b.abs().T)
            c += n
    return out, mag


LORA_SHAPES = [
    # T, K, slices, R, rows per adapter, ranks
    (1, 64, (64,), 8, [1], None),
    (1, 4096, (512, 128, 128), 16, [0, 1, 0], None),
    (5, 8, (8,), 8, [2, 3], [1, 7]),
    (33, 1000, (40,), 24, [17, 0, 16], [24, 24, 5]),
    (40, 72, (48, 8, 16), 8, [40], [8]),
    (70, 520, (104, 24), 24, [1, 30, 5], [13, 24, 0]),
    (64, 256, (256,), 64, [1] * 64, [1 + i for i in range(64)]),
    (200, 2048, (136,), 128, [0, 150, 49], [128, 99, 128]),
    (300, 136, (64, 64, 64, 72), 40, [100, 100, 100], [40, 33, 8]),
    (1200, 512, (256, 64, 64), 16, [700, 3, 400], None),
    (700, 1024, (1032,), 64, [64, 65, 63, 128, 1, 300], [64, 32, 16, 8, 64, 64]),
    # enough rows for the large tiles
    (900, 200, (48, 8, 16), 8, [1, 800, 0, 65], [8, 3, 8, 1]),
    (800, 1000, (136, 72), 24, [400, 400], [24, 13]),
    (1000, 520, (256, 64, 64), 64, [64, 65, 63, 0, 700, 100], [64, 32, 9, 8, 41, 0]),
    (1000, 136, (72,), 128, [990], [77]),
    (1000, 264, (128, 64), 128, [500, 500], [128, 100]),
    (800, 328, (64, 8, 72, 64), 128, [31, 33, 736], [128, 50, 121]),
    (770, 8, (8,), 40, [769], [33]),
    # 64-row tiles in clusters of four, 128-row tiles in clusters of four and of two
    (3000, 136, (72,), 64, [1500, 1, 1499], [64, 40, 7]),
    (3000, 72, (64, 64), 128, [1400, 1500], [128, 101]),
    (6000, 136, (40, 32), 64, [3000, 2000, 900], [64, 33, 16]),
    (1300, 136, (72,), 64, [50] * 20 + [0] * 5 + [60] * 5, [64, 1, 33, 0, 17, 48] * 5),
    (2600, 136, (40, 32), 64, [65] * 40, [(7 * i) % 65 for i in range(40)]),
]


@pytest.mark.parametrize("T,K,slices,R,counts,ranks", LORA_SHAPES)
@pytest.mark.parametrize("f32", [False, True])
def test_lora_integers_are_exact(ops, T, K, slices, R, counts, ranks, f32):
    v = _lora_inputs(T, K, slices, R, counts, T + K, ranks, f32)
    ref, _ = _lora_reference(v, slices, R)
    d = {k: t.to(ops.dev) for k, t in v.items()}
    out = torch.full_like(d["base"], 3.0)
    args = (d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"])
    ops.lora_add(*args, d["base"], out, slices)
    listed = torch.zeros(T, dtype=torch.bool)
    listed[v["rows"].long()] = True
    want = torch.where(listed[:, None], ref.to(out.dtype), torch.tensor(3.0, dtype=out.dtype))
    assert torch.equal(out.cpu(), want)
    inout = d["base"].clone()                       # in place: rows not listed stay
    ops.lora_add(*args, inout, inout, slices)
    assert torch.equal(inout.cpu(), ref.to(out.dtype))
    _no_error(ops)


@pytest.mark.parametrize("T,K,slices,R,counts,ranks", LORA_SHAPES)
@pytest.mark.parametrize("f32", [False, True])
def test_lora_against_64_bits(ops, T, K, slices, R, counts, ranks, f32):
    v = _lora_inputs(T, K, slices, R, counts, 7 * T + K, ranks, f32, integer=False)
    ref, mag = _lora_reference(v, slices, R)
    d = {k: t.to(ops.dev) for k, t in v.items()}
    out = d["base"].clone()
    ops.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, slices)
    # with mag = scale * sum_j |B| sum_k |A| |x|: h over chains of at most K / 16 steps of 17 * 2^-23, its two
    # bf16 parts 2^-16 (three: 2^-24), the expansion at most 8 steps per part of 17 * 2^-23, the output's rounding
    steps = K // 16 + 1 + (8 if R > 64 else 4) * 3
    rel = 17 * 2.0 ** -23 * steps + (2.0 ** -24 if f32 else 2.0 ** -16)
    _within(out, ref, (2.0 ** -23 if f32 else 2.0 ** -8) * ref.abs() + rel * mag, "out")


def test_lora_strides_and_row_order(ops):
    """x, base and out as column ranges of wider buffers, rows in reverse."""
    T, K, R, slices = 50, 256, 16, (96, 32)
    v = _lora_inputs(T, K, slices, R, [20, 0, 30], 11, order=torch.arange(T - 1, -1, -1))
    ref, _ = _lora_reference(v, slices, R)
    d = {k: t.to(ops.dev) for k, t in v.items()}
    xw = torch.full((T, K + 24), float("nan"), dtype=BF, device=ops.dev)
    xw[:, 8:8 + K] = d["x"]
    ow = torch.full((T, 128 + 16), 9.0, dtype=BF, device=ops.dev)
    ow[:, 8:136] = d["base"]
    ops.lora_add(xw[:, 8:8 + K], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], ow[:, 8:136],
                 ow[:, 8:136], slices)
    assert torch.equal(ow[:, 8:136].cpu(), ref.to(BF))
    assert bool((ow[:, :8] == 9).all()) and bool((ow[:, 136:] == 9).all())


def test_lora_rows_do_not_depend_on_each_other(ops):
    """A row's result is the same alone and in any batch."""
    T, K, R, slices = 90, 512, 16, (256,)
    v = _lora_inputs(T, K, slices, R, [45, 45], 13, integer=False)
    d = {k: t.to(ops.dev) for k, t in v.items()}
    full = d["base"].clone()
    args = (d["x"], d["a"], d["b"], d["scales"], d["ranks"])
    ops.lora_add(*args, d["rows"], d["starts"], full, full, slices)
    t = int(v["rows"][50])
    one = d["base"].clone()
    ops.lora_add(*args, d["rows"][50:51].contiguous(), torch.tensor([0, 0, 1], dtype=I32, device=ops.dev), one, one,
                 slices)
    if ops.dev == "cuda":
        assert torch.equal(one[t], full[t])
    others = torch.arange(T, device=ops.dev) != t
    assert torch.equal(one[others], d["base"][others])


def test_lora_without_rows(ops):
    v = _lora_inputs(4, 64, (64,), 8, [0, 0], 17)
    d = {k: t.to(ops.dev) for k, t in v.items()}
    out = d["base"].clone()
    ops.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, (64,))
    assert torch.equal(out, d["base"])


@pytest.mark.parametrize("T,K,R,counts", [(40, 264, 16, [17, 1, 20]), (1300, 264, 64, [700, 1, 590])])
def test_lora_row_that_is_not_finite(ops, T, K, R, counts):
    """An infinity or a NaN in x stays in its row."""
    slices = (48, 24)
    v = _lora_inputs(T, K, slices, R, counts, 23, ranks=[R, R - 3, R - 9], integer=False)
    d = {k: t.to(ops.dev) for k, t in v.items()}

    def run(x):
        out = d["base"].clone()
        ops.lora_add(x, d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, slices)
        return out

    want = run(d["x"])
    bad = [int(v["rows"][3]), int(v["rows"][counts[0]]), int(v["rows"][-1])]
    x = d["x"].clone()
    for r, value in zip(bad, (float("inf"), float("nan"), float("-inf"))):
        x[r, 5] = value
    got = run(x)
    for r in bad:
        assert not bool(torch.isfinite(got[r]).any())
    others = torch.ones(T, dtype=torch.bool, device=ops.dev)
    others[bad] = False
    assert torch.equal(got[others], want[others])


# one row, 16-row tiles, large tiles
LORA_KERNELS = [(3, 72, 8, [1, 2], [5, 8]), (3, 328, 32, [0, 1, 1], [32, 32, 25]), (40, 264, 24, [17, 1, 20], [13, 24, 24]),
                (40, 264, 64, [17, 1, 20], [64, 51, 64]), (1300, 264, 64, [700, 1, 590], [64, 64, 41])]


@pytest.mark.parametrize("T,K,R,counts,ranks", LORA_KERNELS)
@pytest.mark.parametrize("f32", [False, True])
def test_lora_infinities_as_in_64_bits(ops, T, K, R, counts, ranks, f32):
    """An infinite h times weights of one sign is an infinity, not a NaN, whatever lies past the rank."""
    slices = (48, 24)
    v = _lora_inputs(T, K, slices, R, counts, 61, ranks, f32)
    for name in ("a", "b"):
        v[name] = torch.where(v[name].isnan(), v[name], v[name].abs() + 1)
    v["x"][int(v["rows"][0]), 5] = float("inf")
    v["x"][int(v["rows"][-1]), 7] = -float("inf")
    ref, _ = _lora_reference(v, slices, R)
    assert bool(ref[int(v["rows"][0])].isinf().all()) and bool(ref[int(v["rows"][-1])].isinf().all())
    d = {k: t.to(ops.dev) for k, t in v.items()}
    out = d["base"].clone()
    ops.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, slices)
    assert torch.equal(out.cpu(), ref.to(out.dtype))
    _no_error(ops)


@pytest.mark.parametrize("T,K,R,counts,ranks", LORA_KERNELS)
@pytest.mark.parametrize("f32", [False, True])
def test_lora_h_beyond_bf16(ops, T, K, R, counts, ranks, f32):
    """h between the largest bf16 and the largest fp32 value, +-(2 - 2^-9) 2^127: outputs stay finite."""
    slices = (48, 24)
    v = _lora_inputs(T, K, slices, R, counts, 62, ranks, f32)
    v["x"][:] = 0
    v["x"][:, 3:13] = torch.where(torch.arange(T) % 2 == 0, 2.0 ** 64, -2.0 ** 64)[:, None].to(BF)
    v["a"][..., 3:13] = torch.where(v["a"][..., 3:13].isnan(), v["a"][..., 3:13], (2.0 ** (63 - torch.arange(10.0))).to(BF))
    v["b"] = torch.where(v["b"].isnan(), v["b"], torch.zeros_like(v["b"]))
    v["b"][..., 0] = 2.0 ** -110
    v["base"][:] = 0
    ref, _ = _lora_reference(v, slices, R)
    assert bool((ref[v["rows"].long()].abs() > 1e4).all())
    d = {k: t.to(ops.dev) for k, t in v.items()}
    out = d["base"].clone()
    ops.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, slices)
    # every product, the sum and the two bf16 parts of h (10 bits) are exact: only the output is rounded
    assert torch.equal(out.cpu(), ref.to(out.dtype))
    _no_error(ops)


@gpu
def test_lora_bad_indices_are_recorded(kernels):
    T, K, R, slices = 40, 64, 8, (64,)
    for what in ("row", "negative", "starts", "rank"):
        v = _lora_inputs(T, K, slices, R, [20, 20], 19)
        if what == "row":
            v["rows"][5] = T
        elif what == "negative":
            v["rows"][25] = -1
        elif what == "starts":
            v["starts"][2] = 41
        else:
            v["ranks"][1] = R + 1
        d = {k: t.cuda() for k, t in v.items()}
        out = d["base"].clone()
        kernels.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, slices)
        assert kernels.read_error(True)[0] == 3, what


@gpu
@pytest.mark.parametrize("T,K,slices,R,counts,ranks", [
    (1300, 264, (72, 64), 64, [700, 590], [64, 41]),                      # 64-row tiles
    (3000, 520, (72,), 64, [1500, 1, 1400], [64, 40, 7]),                 # clusters of four
    (6000, 136, (40, 32), 64, [3000, 2000, 900], [64, 33, 16])])          # 128-row tiles
@pytest.mark.parametrize("f32", [False, True])
def test_lora_large_tiles_with_a_recorded_error(kernels, T, K, slices, R, counts, ranks, f32):
    """A bad row, offset or rank leaves the other rows' values as they are, in the call that
    records it and in the calls after it until the host has read the error."""
    for what in ("row", "negative", "starts", "rank"):
        v = _lora_inputs(T, K, slices, R, counts, 29, ranks, f32)
        ref, _ = _lora_reference(v, slices, R)
        good = {k: t.cuda() for k, t in v.items()}
        spoilt = torch.zeros(T, dtype=torch.bool)
        last = v["rows"][int(v["starts"][-2]):].long()
        if what == "row":
            spoilt[int(v["rows"][5])] = True
            v["rows"][5] = T
        elif what == "negative":
            spoilt[int(v["rows"][counts[0] - 1])] = True
            v["rows"][counts[0] - 1] = -1
        elif what == "starts":
            spoilt[last] = True
            v["starts"][-1] = sum(counts) + 1
        else:
            spoilt[last] = True
            v["ranks"][-1] = R + 1
        d = {k: t.cuda() for k, t in v.items()}

        def run(d):
            out = d["base"].clone()
            kernels.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, slices)
            return out.cpu()

        bad, after = run(d), run(good)
        assert torch.equal(bad[~spoilt], ref.to(bad.dtype)[~spoilt]), what
        assert torch.equal(bad[spoilt], v["base"][spoilt]), what
        assert torch.equal(after, ref.to(after.dtype)), what
        assert kernels.read_error(True)[0] == 3, what


@pytest.mark.parametrize("T,K,slices,R,counts,ranks", [
    (5, 1024, (96,), 32, [1, 2, 1], [32, 31, 7]), (40, 264, (72,), 32, [17, 1, 20], [32, 25, 32]),
    (64, 520, (1032,), 32, [1] * 60, [32] * 60), (50, 136, (40, 32, 24, 8), 8, [20, 30], [8, 5]),
    (50, 136, (40, 32, 24), 8, [20, 30], [8, 5])])
@pytest.mark.parametrize("f32", [False, True])
def test_lora_more_ranks_and_slices(ops, T, K, slices, R, counts, ranks, f32):
    """Rank 32 beside one projection, 24 and 32 columns of h: variants that the shapes above pass by."""
    test_lora_integers_are_exact(ops, T, K, slices, R, counts, ranks, f32)
    test_lora_against_64_bits(ops, T, K, slices, R, counts, ranks, f32)


@pytest.mark.parametrize("T,K,R,counts,ranks", LORA_KERNELS)
def test_lora_fp32_outputs_hold_h_to_24_bits(ops, T, K, R, counts, ranks):
    """h of 23 bits, exact in fp32, and one +-1 of B per column: two bf16 parts of h would lose the lowest bits."""
    slices = (48, 24)
    v = _lora_inputs(T, K, slices, R, counts, 63, ranks, True)
    g = _gen(64)
    v["x"][:] = 0
    v["x"][:, 3] = torch.randint(64, 128, (T,), generator=g).to(BF)              # h = 2^16 x[3] + x[40] a[40]
    v["x"][:, 40] = (torch.randint(0, 128, (T,), generator=g) * 2 + 1).to(BF)
    nan = v["a"][..., 3].isnan()
    v["a"][..., 3] = torch.where(nan, v["a"][..., 3], torch.full_like(v["a"][..., 3], 2.0 ** 16))
    odd = (torch.randint(0, 64, nan.shape, generator=g) * 2 + 1).to(BF)
    v["a"][..., 40] = torch.where(nan, v["a"][..., 40], odd)
    v["b"] = torch.where(v["b"].isnan(), v["b"], torch.zeros_like(v["b"]))
    for ad, rank in enumerate(ranks):
        c = torch.arange(sum(slices))
        v["b"][ad, c, c % rank] = torch.where(c % 3 == 0, -1.0, 1.0).to(BF)
    v["base"][:] = 0
    ref, _ = _lora_reference(v, slices, R)
    assert bool((ref.float().double() == ref).all()) and bool((ref[v["rows"].long()].abs() >= 2.0 ** 19).all())
    d = {k: t.to(ops.dev) for k, t in v.items()}
    out = d["base"].clone()
    ops.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], out, out, slices)
    assert torch.equal(out.cpu().double(), ref)
    _no_error(ops)


@pytest.mark.parametrize("T,K,R,counts,ranks", LORA_KERNELS)
@pytest.mark.parametrize("f32", [False, True])
def test_lora_repeats_exactly(ops, T, K, R, counts, ranks, f32):
    """The same call gives the same bits, a row by itself the same value to the sums' accuracy."""
    slices = (48, 24)
    v = _lora_inputs(T, K, slices, R, counts, 65, ranks, f32, integer=False)
    ref, mag = _lora_reference(v, slices, R)
    d = {k: t.to(ops.dev) for k, t in v.items()}
    args = (d["x"], d["a"], d["b"], d["scales"], d["ranks"])
    want = d["base"].clone()
    ops.lora_add(*args, d["rows"], d["starts"], want, want, slices)
    for _ in range(3):
        out = d["base"].clone()
        ops.lora_add(*args, d["rows"], d["starts"], out, out, slices)
        assert torch.equal(out, want)
    ad = len(counts) - 1                             # the last listed row is the last adapter's
    t = int(v["rows"][-1])
    starts = torch.tensor([0] * (ad + 1) + [1], dtype=I32, device=ops.dev)
    one = d["base"].clone()
    ops.lora_add(*args, d["rows"][-1:].contiguous(), starts, one, one, slices)
    steps = K // 16 + 1 + 4 * 3                      # as in test_lora_against_64_bits
    rel = 17 * 2.0 ** -23 * steps + (2.0 ** -24 if f32 else 2.0 ** -16)
    for got in (one, want):
        _within(got[t], ref[t], (2.0 ** -23 if f32 else 2.0 ** -8) * ref[t].abs() + rel * mag[t], "row")


# ---------------------------------------------------------------------------
# attention over selected pages
# ---------------------------------------------------------------------------
def _paged(lens, Hq, Hkv, seed, spare=3, shuffle=True, scale=1.0):
    g = _gen(seed)
    R = len(lens)
    n = [-(-x // 16) for x in lens]
    width = max(max(n), 1) + 1
    pages = 1 + sum(n) + spare
    perm = (torch.randperm(pages - 1, generator=g) if shuffle else torch.arange(pages - 1)) + 1
    bt = torch.zeros(R, width, dtype=I32)
    at = 0
    for r in range(R):
        bt[r, :n[r]] = perm[at:at + n[r]].int()
        at += n[r]
    kc = (_randn(g, pages, Hkv, 16, 128, dtype=F32) + _randn(g, pages, Hkv, 1, 128, dtype=F32)).mul(scale).to(BF)
    vc = _randn(g, pages, Hkv, 16, 128)
    kc[0] = vc[0] = 0
    T = R + 2                                            # rows of q that no sequence uses
    tok = torch.randperm(T, generator=g)[:R].int()
    return dict(q=_randn(g, T, (Hq + 2 * Hkv) * 128), bt=bt, lens=torch.tensor(lens, dtype=I32), tok=tok, kc=kc, vc=vc,
                bounds=torch.full((pages, Hkv, 2, 128), 77.0, dtype=BF), width=width)


def _bounds_reference(v, start):
    b = v["bounds"].clone()
    for r, (s, n) in enumerate(zip(start, v["lens"].tolist())):
        for p in range(max(s, 0) // 16, -(-n // 16)):
            if s < n:
                keys = v["kc"][int(v["bt"][r, p]), :, :min(16, n - p * 16)].double()
                b[int(v["bt"][r, p])] = torch.stack([keys.min(1).values, keys.max(1).values], 1).to(BF)
    return b


def _select_reference(v, Hq, Hkv, budget, first, last):
    R, G = len(v["lens"]), Hq // Hkv
    sel = torch.full((R, Hkv, budget), -1, dtype=I32)
    for r, n in enumerate(v["lens"].tolist()):
        pages = -(-n // 16)
        for h in range(Hkv):
            if pages <= budget:
                sel[r, h, :pages] = torch.arange(pages, dtype=I32)
                continue
            b = v["bounds"][v["bt"][r, :pages].long(), h].double()
            q = v["q"][int(v["tok"][r]), h * G * 128:(h + 1) * G * 128].double().view(G, 128)
            score = torch.stack([torch.maximum(b[:, 0] * x, b[:, 1] * x).sum(-1) for x in q]).amax(0)
            score = [float(s) if math.isfinite(s) else math.inf for s in score]
            mid = sorted(range(first, pages - last), key=lambda p: (-score[p], p))[:budget - first - last]
            sel[r, h] = torch.tensor(sorted(list(range(first)) + mid + list(range(pages - last, pages))), dtype=I32)
    return sel


def _attend_reference(v, sel, Hq, Hkv):
    """Outputs in 64 bits and sum p |v| behind every element, rows in the order of tok."""
    R, G, budget = len(v["lens"]), Hq // Hkv, sel.shape[2]
    out = torch.zeros(R, Hq, 128, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for r, n in enumerate(v["lens"].tolist()):
        count = min(-(-n // 16), budget)
        for h in range(Hkv):
            if not count:
                continue
            s = sel[r, h, :count].long()
            phys = v["bt"][r].long()[s]
            pos = (s[:, None] * 16 + torch.arange(16)).reshape(-1)
            k = v["kc"][phys, h].reshape(-1, 128)[pos < n].double()
            val = v["vc"][phys, h].reshape(-1, 128)[pos < n].double()
            q = v["q"][int(v["tok"][r]), h * G * 128:(h + 1) * G * 128].double().view(G, 128)
            p = ((q @ k.T) / math.sqrt(128)).softmax(-1)
            out[r, h * G:(h + 1) * G] = p @ val
            mag[r, h * G:(h + 1) * G] = p @ val.abs()
    return out.reshape(R, -1), mag.reshape(R, -1)


def _attend_check(out, v, sel, Hq, Hkv):
    ref, mag = _attend_reference(v, sel, Hq, Hkv)
    # every weight is rounded to bf16 (2^-8) and its logit to 2^-13: the weighted mean moves by at most
    # (2^-8 + 2^-12) (sum p |v| + |out|), then the output's rounding
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12) * (mag + ref.abs())
    _within(out[v["tok"].long().to(out.device)][:, :Hq * 128], ref, tol, "attention")


SPARSE = [
    # lens, Hq, Hkv, budget, first, last
    ([1], 4, 1, 1, 0, 1),
    ([0, 5, 16, 17, 33], 8, 2, 2, 0, 1),
    ([700, 1, 0, 350, 16 * 20], 8, 2, 12, 1, 2),
    ([1000, 999, 16 * 62], 16, 1, 20, 2, 3),
    ([2000, 64], 5, 1, 9, 4, 5),          # first and last fill the budget
    ([1555], 12, 4, 70, 0, 0),
    ([3000, 17, 2999, 16, 100, 1600], 32, 8, 40, 1, 2),
    ([9000], 2, 2, 129, 1, 1),
    ([40] * 50, 4, 4, 2, 0, 1),
    # 512 to 2048 pages in few and in many rows x heads; two CTAs per row and head where not all run at once
    ([16 * 700 + 3, 16 * 1030], 8, 2, 20, 1, 2),
    ([16 * 1100 - 5] + [1 + 37 * i for i in range(39)], 8, 8, 24, 0, 1),
    # eight-warp CTAs for more rows: a large budget
    ([16 * 200 + i for i in range(25)], 4, 1, 130, 1, 1),
]


@pytest.mark.parametrize("lens,Hq,Hkv,budget,first,last", SPARSE)
def test_sparse_step(ops, lens, Hq, Hkv, budget, first, last):
    """Bounds of every page, the selection, the attention over it, then one more token."""
    v = _paged(lens, Hq, Hkv, sum(lens) + budget)
    for r, n in enumerate(lens):               # what lies behind a sequence's end is never used
        if n % 16:
            v["kc"][int(v["bt"][r, n // 16]), :, n % 16:] = float("nan")
            v["vc"][int(v["bt"][r, n // 16]), :, n % 16:] = float("nan")
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    R = len(lens)
    zeros = torch.zeros(R, dtype=I32, device=ops.dev)
    ops.page_bounds(d["kc"], d["bounds"], d["bt"], zeros, d["lens"], max(max(lens), 1))
    v["bounds"] = _bounds_reference(v, [0] * R)
    assert torch.equal(d["bounds"].cpu(), v["bounds"])
    sel = torch.full((R, Hkv, budget), 99, dtype=I32, device=ops.dev)
    ws = torch.full((max(1, ops.select_workspace(R, Hkv, v["width"])),), float("nan"), device=ops.dev)
    ops.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, first, last, Hq, Hkv, ws)
    want = _select_reference(v, Hq, Hkv, budget, first, last)
    assert torch.equal(sel.cpu(), want)
    out = torch.full((d["q"].shape[0], Hq * 128), 4.0, dtype=BF, device=ops.dev)
    ops.attn_decode_sparse(d["q"], out, d["tok"], d["lens"], d["bt"], sel, d["kc"], d["vc"], Hq, Hkv)
    _attend_check(out, v, want, Hq, Hkv)
    unused = [t for t in range(out.shape[0]) if t not in v["tok"].tolist()]
    assert bool((out[unused] == 4.0).all())
    # one more token in every row that has room on its last page
    new = [n + 1 if n % 16 else n for n in lens]
    for r, n in enumerate(lens):
        if n % 16:
            k = _randn(_gen(r), Hkv, 128, scale=3.0)
            v["kc"][int(v["bt"][r, n // 16]), :, n % 16] = k
            d["kc"][int(v["bt"][r, n // 16]), :, n % 16] = k.to(ops.dev)
    v["lens"] = torch.tensor(new, dtype=I32)
    start = torch.tensor(lens, dtype=I32)
    ops.page_bounds(d["kc"], d["bounds"], d["bt"], start.to(ops.dev), v["lens"].to(ops.dev), 1)
    assert torch.equal(d["bounds"].cpu(), _bounds_reference(v, lens))
    _no_error(ops)


def test_select_ties_take_the_lowest_page(ops):
    """Equal pages, zero pages and pages that differ by less than fp32 sums resolve."""
    Hq, Hkv, budget = 4, 2, 7
    v = _paged([16 * 600, 16 * 40], Hq, Hkv, 5)
    v["kc"][:] = 0
    v["kc"][v["bt"][1, 20:30].long()] = 1.0
    g = _gen(9)
    row0 = v["bt"][0, :600].long()
    # large terms that cancel: the difference between pages is far below fp32's resolution of the sum
    v["kc"][row0, :, :, 0] = 8192.0
    v["kc"][row0, :, :, 1] = -8192.0
    v["kc"][row0, :, :, 2] = (torch.randint(0, 5, (600, 1, 1), generator=g) * 2.0 ** -12).to(BF)
    v["q"][:, :] = 1.0
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    ops.page_bounds(d["kc"], d["bounds"], d["bt"], torch.zeros(2, dtype=I32, device=ops.dev), d["lens"], 16 * 600)
    v["bounds"] = d["bounds"].cpu()
    for first, last in ((0, 1), (2, 3), (0, 0)):
        sel = torch.zeros(2, Hkv, budget, dtype=I32, device=ops.dev)
        ws = torch.zeros(max(1, ops.select_workspace(2, Hkv, v["width"])), device=ops.dev)
        ops.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, first, last, Hq, Hkv, ws)
        assert torch.equal(sel.cpu(), _select_reference(v, Hq, Hkv, budget, first, last))


def test_select_takes_pages_that_are_not_finite(ops):
    Hq, Hkv, budget = 8, 1, 6
    v = _paged([16 * 90], Hq, Hkv, 6)
    for p, value in ((30, float("inf")), (50, float("-inf")), (70, float("nan"))):
        v["kc"][int(v["bt"][0, p]), 0, 3, 17] = value
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    ops.page_bounds(d["kc"], d["bounds"], d["bt"], torch.zeros(1, dtype=I32, device=ops.dev), d["lens"], 16 * 90)
    sel = torch.zeros(1, Hkv, budget, dtype=I32, device=ops.dev)
    ws = torch.zeros(max(1, ops.select_workspace(1, Hkv, v["width"])), device=ops.dev)
    ops.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, 0, 1, Hq, Hkv, ws)
    assert {30, 50, 70, 89} <= set(sel[0, 0].tolist())


@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (24, 2)])
@pytest.mark.parametrize("n", [60, 1300])
@pytest.mark.parametrize("q,k", [(2.0 ** 70, 2.0 ** 70), (2.0 ** 64, 2.0 ** 60), (2.0 ** 60, 2.0 ** 60)])
def test_select_scores_beyond_fp32(ops, Hq, Hkv, n, q, k):
    """Finite keys and queries whose scores, or parts of them, lie beyond fp32: they are compared like others."""
    budget = 9
    v = _paged([16 * n, 16 * 20], Hq, Hkv, 51)
    v["q"] = (v["q"].float() * q).to(BF)
    v["kc"] = (v["kc"].float() * k).to(BF)
    v["kc"][v["bt"][0, 5:40:3].long()] *= 2.0 ** -20
    v["kc"][int(v["bt"][0, 17]), 0, 2, 9] = float("nan")
    assert bool(torch.isfinite(v["q"]).all())
    d = {k_: t.to(ops.dev) if torch.is_tensor(t) else t for k_, t in v.items()}
    ops.page_bounds(d["kc"], d["bounds"], d["bt"], torch.zeros(2, dtype=I32, device=ops.dev), d["lens"], 16 * n)
    v["bounds"] = d["bounds"].cpu()
    sel = torch.zeros(2, Hkv, budget, dtype=I32, device=ops.dev)
    ws = torch.zeros(max(1, ops.select_workspace(2, Hkv, v["width"])), device=ops.dev)
    ops.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, 1, 2, Hq, Hkv, ws)
    assert torch.equal(sel.cpu(), _select_reference(v, Hq, Hkv, budget, 1, 2))


@pytest.mark.parametrize("q,k", [(2.0 ** -64, 2.0 ** -64), (2.0 ** -70, 2.0 ** -70), (2.0 ** -73, 2.0 ** -70),
                                 (2.0 ** -76, 2.0 ** -74), (2.0 ** -78, 2.0 ** -76), (2.0 ** 20, 2.0 ** -130),
                                 (2.0 ** -14, 2.0 ** -130)])
def test_select_scores_below_fp32(ops, q, k):
    """Products at and below fp32's smallest numbers: pages that their fp32 sums order wrongly."""
    Hq, Hkv, n, budget = 16, 4, 1300, 24
    v = _paged([16 * n, 16 * (n - 100) - 5], Hq, Hkv, 52)
    v["q"] = (v["q"].float() * q).to(BF)
    v["kc"] = (v["kc"].float() * k).to(BF)
    d = {k_: t.to(ops.dev) if torch.is_tensor(t) else t for k_, t in v.items()}
    ops.page_bounds(d["kc"], d["bounds"], d["bt"], torch.zeros(2, dtype=I32, device=ops.dev), d["lens"], 16 * n)
    v["bounds"] = d["bounds"].cpu()
    sel = torch.zeros(2, Hkv, budget, dtype=I32, device=ops.dev)
    ws = torch.zeros(max(1, ops.select_workspace(2, Hkv, v["width"])), device=ops.dev)
    ops.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, 1, 2, Hq, Hkv, ws)
    assert torch.equal(sel.cpu(), _select_reference(v, Hq, Hkv, budget, 1, 2))


def test_select_first_and_last_fill_the_budget(ops):
    Hq, Hkv, lens = 4, 2, [16 * 40 + 1, 16 * 3, 5]
    v = _paged(lens, Hq, Hkv, 9)
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    for first, last in ((1, 2), (3, 0), (0, 3)):
        sel = torch.zeros(3, Hkv, 3, dtype=I32, device=ops.dev)
        ws = torch.zeros(max(1, ops.select_workspace(3, Hkv, v["width"])), device=ops.dev)
        ops.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, first, last, Hq, Hkv, ws)
        assert torch.equal(sel.cpu(), _select_reference(v, Hq, Hkv, 3, first, last))
    _no_error(ops)


def test_sparse_step_without_pages(ops):
    """A block table without columns: every row is empty."""
    Hq, Hkv = 4, 2
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=ops.dev)  # noqa: E731
    kc, bounds = torch.ones(2, Hkv, 16, 128, dtype=BF, device=ops.dev), z(2, Hkv, 2, 128)
    bt, lens, tok = z(3, 0, dtype=I32), z(3, dtype=I32), torch.arange(3, dtype=I32, device=ops.dev)
    ops.page_bounds(kc, bounds, bt, lens, lens, 1)
    assert not bool(bounds.any())
    q, out, sel = torch.ones(3, Hq * 128, dtype=BF, device=ops.dev), torch.ones(3, Hq * 128, dtype=BF, device=ops.dev), z(3, Hkv, 2, dtype=I32)
    ops.attn_select(q, tok, lens, bt, bounds, sel, 0, 1, Hq, Hkv, z(1, dtype=F32))
    assert bool((sel == -1).all())
    ops.attn_decode_sparse(q, out, tok, lens, bt, sel, kc, kc, Hq, Hkv)
    assert not bool(out.any())
    _no_error(ops)


def test_sparse_with_every_page_is_dense(ops):
    """A budget of all pages: the attention of the plain decode operator."""
    Hq, Hkv = 8, 2
    lens = [300, 16, 1, 77]
    v = _paged(lens, Hq, Hkv, 8)
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    sel = torch.zeros(len(lens), Hkv, v["width"], dtype=I32, device=ops.dev)
    ops.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, 0, 1, Hq, Hkv,
                    torch.zeros(max(1, ops.select_workspace(4, Hkv, v["width"])), device=ops.dev))
    out = torch.zeros(d["q"].shape[0], Hq * 128, dtype=BF, device=ops.dev)
    dense = torch.zeros_like(out)
    ops.attn_decode_sparse(d["q"], out, d["tok"], d["lens"], d["bt"], sel, d["kc"], d["vc"], Hq, Hkv)
    ops.attn_decode(d["q"], dense, d["tok"], d["lens"], d["bt"], d["kc"], d["vc"], Hq, Hkv, 1, None, None,
                    host={"seq_lens": v["lens"].numpy(), "tok": v["tok"].numpy()})
    _attend_check(out, v, sel.cpu(), Hq, Hkv)
    _attend_check(dense, v, sel.cpu(), Hq, Hkv)


@pytest.mark.parametrize("lens,Hq,Hkv,budget", [([2, 3, 16, 17, 40], 8, 1, 3), ([33, 2, 100], 12, 1, 7),
                                                ([90, 48, 7], 16, 4, 4), ([30, 31], 32, 2, 2)])
def test_sparse_weights_are_not_rounded(ops, lens, Hq, Hkv, budget):
    """Values of both signs, whose weighted mean is far smaller than its terms: weights
    rounded to 8 bits move it by up to 2^-8, which the output's own rounding does not hide."""
    v = _paged(lens, Hq, Hkv, 31 + Hq)
    g = _gen(32)
    # one dimension carries the logits: the products are exact in fp32, |log2 weight| <= 8 * 4 / 11.3 * 1.45 < 5
    v["q"][:] = 0
    v["q"][:, :Hq * 128:128] = torch.randint(1, 9, (v["q"].shape[0], Hq), generator=g).to(BF)
    v["kc"][:] = 0
    v["kc"][..., 0] = (torch.randint(0, 129, v["kc"].shape[:3], generator=g) / 32).to(BF)
    v["vc"] = torch.where(torch.rand(v["vc"].shape, generator=g) < 0.5, -1.0, 1.0).to(BF)
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    sel = torch.full((len(lens), Hkv, budget), -1, dtype=I32)
    for r, n in enumerate(lens):
        count = min(-(-n // 16), budget)
        sel[r, :, :count] = torch.arange(-(-n // 16) - count, -(-n // 16), dtype=I32)
    out = torch.zeros(d["q"].shape[0], Hq * 128, dtype=BF, device=ops.dev)
    ops.attn_decode_sparse(d["q"], out, d["tok"], d["lens"], d["bt"], sel.to(ops.dev), d["kc"], d["vc"], Hq, Hkv)
    ref, mag = _attend_reference(v, sel, Hq, Hkv)
    # a weight: its logit 5 * 2^-23, the exponential 2^-22, two bf16 parts 2^-15; a weighted sum over at most 2 steps
    # of 16 tokens per warp in two parts, 17 * 2^-23 each (2^-16.9); the sum of weights less: under 2^-14 of
    # sum p |v| + |out| in all
    _within(out[v["tok"].long().to(out.device)], ref, 2.0 ** -8 * ref.abs() + 2.0 ** -14 * (mag + ref.abs()), "attention")


@pytest.mark.parametrize("Hq,Hkv,budget", [(8, 1, 4), (8, 1, 40), (24, 2, 4)])
def test_sparse_logits_that_are_not_finite(ops, Hq, Hkv, budget):
    """Logits of -inf weigh nothing beside finite ones; where a row has no others, or one of +inf or NaN, it is NaN."""
    lens = [1, 40, 40, 40, 600, 600, 0]
    v = _paged(lens, Hq, Hkv, 70)
    v["q"][:, :Hq * 128:128] = 1.0
    neg = -float("inf")
    for r in (0, 1, 4):                              # every key
        v["kc"][v["bt"][r, :-(-lens[r] // 16)].long(), :, :, 0] = neg
    v["kc"][v["bt"][2, :3].long(), :, ::2, 0] = neg  # every second key
    v["kc"][int(v["bt"][2, 2]), :, :, 0] = neg
    v["kc"][int(v["bt"][3, 1]), :, 3, 0] = float("inf")
    v["kc"][v["bt"][5, 1:37].long(), :, :, 0] = neg  # all but the first and the last page
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    sel = torch.full((len(lens), Hkv, budget), -1, dtype=I32)
    for r, n in enumerate(lens):
        count = min(-(-n // 16), budget)
        sel[r, :, :count] = torch.tensor(([0] + list(range(-(-n // 16) - count + 1, -(-n // 16))))[:count], dtype=I32)
    out = torch.full((d["q"].shape[0], Hq * 128), 3.0, dtype=BF, device=ops.dev)
    ops.attn_decode_sparse(d["q"], out, d["tok"], d["lens"], d["bt"], sel.to(ops.dev), d["kc"], d["vc"], Hq, Hkv)
    got = out[v["tok"].long().to(out.device)].cpu()
    for r in (0, 1, 3, 4):
        assert bool(got[r].isnan().all()), r
    assert not bool(got[6].any())
    ref, mag = _attend_reference(v, sel, Hq, Hkv)
    for r in (2, 5):
        assert bool(ref[r].isfinite().all())
        _within(got[r], ref[r], 2.0 ** -8 * ref[r].abs() + 2.0 ** -11 * (mag[r] + ref[r].abs()), r)


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (24, 2)])
def test_sparse_values_that_are_infinite(ops, Hq, Hkv):
    """An infinite value of a token that weighs anything makes its dimension infinite, not NaN."""
    lens, budget = [1, 33, 200, 16], 30
    v = _paged(lens, Hq, Hkv, 71)
    v["q"][:] = (v["q"].float() * 0.25).to(BF)
    inf = float("inf")
    for r, (p, t) in enumerate(((0, 0), (1, 3), (12, 7), (0, 15))):
        v["vc"][int(v["bt"][r, p]), :, t, 17] = inf
        v["vc"][int(v["bt"][r, p]), :, t, 90] = -inf
    d = {k: t.to(ops.dev) if torch.is_tensor(t) else t for k, t in v.items()}
    sel = torch.full((len(lens), Hkv, budget), -1, dtype=I32)
    for r, n in enumerate(lens):
        sel[r, :, :-(-n // 16)] = torch.arange(-(-n // 16), dtype=I32)
    out = torch.zeros(d["q"].shape[0], Hq * 128, dtype=BF, device=ops.dev)
    ops.attn_decode_sparse(d["q"], out, d["tok"], d["lens"], d["bt"], sel.to(ops.dev), d["kc"], d["vc"], Hq, Hkv)
    got = out[v["tok"].long().to(out.device)].cpu().view(len(lens), Hq, 128)
    assert bool((got[..., 17] == inf).all()) and bool((got[..., 90] == -inf).all())
    ref, mag = (x.view(len(lens), Hq, 128) for x in _attend_reference(v, sel, Hq, Hkv))
    finite = [i for i in range(128) if i not in (17, 90)]
    _within(got[..., finite], ref[..., finite], 2.0 ** -8 * ref[..., finite].abs() + 2.0 ** -11 * (mag + ref.abs())[..., finite], "out")


@pytest.mark.parametrize("lens", [[16 * 20000 + 3], [16 * 9000, 16 * 3]])
@gpu
def test_select_long_rows(kernels, lens):
    """Rows beyond what the selection holds in registers, and one page's key repeated: many exact ties."""
    Hq, Hkv, budget = 4, 1, 100
    for tie in (False, True):
        v = _paged(lens, Hq, Hkv, 12)
        if tie:
            v["kc"][:] = v["kc"][5, 0, 0, 0].clone()
        d = {k: t.cuda() if torch.is_tensor(t) else t for k, t in v.items()}
        R = len(lens)
        kernels.page_bounds(d["kc"], d["bounds"], d["bt"], torch.zeros(R, dtype=I32, device="cuda"), d["lens"], max(lens))
        v["bounds"] = d["bounds"].cpu()
        sel = torch.zeros(R, Hkv, budget, dtype=I32, device="cuda")
        ws = torch.zeros(kernels.select_workspace(R, Hkv, v["width"]), device="cuda")
        kernels.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, 1, 2, Hq, Hkv, ws)
        assert torch.equal(sel.cpu(), _select_reference(v, Hq, Hkv, budget, 1, 2))
    _no_error(kernels)


@pytest.mark.parametrize("lens,Hq,Hkv,budget", [
    ([16 * 5000 + 3, 16 * 2100, 16 * 8000, 700, 16 * 60], 8, 2, 60),     # 2049 to 8192 pages
    ([16 * 3000 - 7, 16 * 2500], 12, 1, 700),                            # the same, two groups of query heads
    ([16 * 640, 1, 0, 17] + [16 * 30 + 5 * i for i in range(36)], 24, 2, 24),
    ([16 * 9 + i for i in range(40)], 32, 2, 4)])                        # many rows of wide groups
@gpu
def test_sparse_step_more_rows_pages_and_heads(kernels, lens, Hq, Hkv, budget):
    """Launch variants that the cases above pass by: with random keys, then with one key for all (ties)."""
    for tie in (False, True):
        v = _paged(lens, Hq, Hkv, 43)
        if tie:
            v["kc"][:] = v["kc"][5, 0, 0, 0].clone()
        d = {k: t.cuda() if torch.is_tensor(t) else t for k, t in v.items()}
        R = len(lens)
        kernels.page_bounds(d["kc"], d["bounds"], d["bt"], torch.zeros(R, dtype=I32, device="cuda"), d["lens"], max(lens))
        v["bounds"] = d["bounds"].cpu()
        sel = torch.full((R, Hkv, budget), 99, dtype=I32, device="cuda")
        ws = torch.zeros(kernels.select_workspace(R, Hkv, v["width"]), device="cuda")
        kernels.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, 1, 2, Hq, Hkv, ws)
        want = _select_reference(v, Hq, Hkv, budget, 1, 2)
        assert torch.equal(sel.cpu(), want)
        out = torch.full((d["q"].shape[0], Hq * 128), 4.0, dtype=BF, device="cuda")
        kernels.attn_decode_sparse(d["q"], out, d["tok"], d["lens"], d["bt"], sel, d["kc"], d["vc"], Hq, Hkv)
        _attend_check(out, v, want, Hq, Hkv)
    _no_error(kernels)


@pytest.mark.parametrize("first,last", [(5, 7), (12, 0), (0, 12)])
@gpu
def test_select_long_rows_without_a_free_place(kernels, first, last):
    """More pages than the selection holds in registers, and the first and last ones fill the budget."""
    Hq, Hkv, budget, lens = 8, 2, 12, [16 * 8300 + 1, 16 * 12000, 16 * 11, 16 * 13, 16 * 9000 - 3]
    v = _paged(lens, Hq, Hkv, 40)
    d = {k: t.cuda() if torch.is_tensor(t) else t for k, t in v.items()}
    R = len(lens)
    kernels.page_bounds(d["kc"], d["bounds"], d["bt"], torch.zeros(R, dtype=I32, device="cuda"), d["lens"], max(lens))
    v["bounds"] = d["bounds"].cpu()
    ws = torch.zeros(kernels.select_workspace(R, Hkv, v["width"]), device="cuda")
    want = _select_reference(v, Hq, Hkv, budget, first, last)
    for _ in range(3):
        sel = torch.full((R, Hkv, budget), 99, dtype=I32, device="cuda")
        kernels.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, first, last, Hq, Hkv, ws)
        assert torch.equal(sel.cpu(), want)
    _no_error(kernels)


@gpu
def test_sparse_bad_indices_are_recorded(kernels):
    """Bad pages, list entries, tokens and lengths: an error code, other rows unharmed."""
    Hq, Hkv, budget = 4, 1, 4
    for what in ("page", "entry", "minus", "token", "length"):
        v = _paged([200, 200], Hq, Hkv, 14)
        good = {k: t.cuda() if torch.is_tensor(t) else t for k, t in v.items()}
        zeros = torch.zeros(2, dtype=I32, device="cuda")
        kernels.page_bounds(good["kc"], good["bounds"], good["bt"], zeros, good["lens"], 200)
        sel = torch.zeros(2, Hkv, budget, dtype=I32, device="cuda")
        ws = torch.zeros(kernels.select_workspace(2, Hkv, v["width"]), device="cuda")
        kernels.attn_select(good["q"], good["tok"], good["lens"], good["bt"], good["bounds"], sel, 0, 1, Hq, Hkv, ws)
        _no_error(kernels)
        want = sel.clone()
        d = {k: t.clone() if torch.is_tensor(t) else t for k, t in good.items()}
        if what == "page":
            d["bt"][0, 12] = d["kc"].shape[0]
        elif what == "entry":
            sel[0, 0, 1] = 13
        elif what == "minus":
            sel[0, 0, 0] = -1
        elif what == "token":
            d["tok"][0] = d["q"].shape[0]
        else:
            d["lens"][0] = v["width"] * 16 + 1
        out = torch.zeros(d["q"].shape[0], Hq * 128, dtype=BF, device="cuda")
        kernels.attn_decode_sparse(d["q"], out, d["tok"], d["lens"], d["bt"], sel, d["kc"], d["vc"], Hq, Hkv)
        assert kernels.read_error(True)[0] == 3, what
        ref, mag = _attend_reference(v, want.cpu(), Hq, Hkv)
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12) * (mag + ref.abs())
        _within(out[int(v["tok"][1])], ref[1], tol[1], what)
        if what in ("page", "token", "length"):
            again = torch.zeros_like(sel)
            kernels.attn_select(d["q"], d["tok"], d["lens"], d["bt"], d["bounds"], again, 0, 1, Hq, Hkv, ws)
            assert kernels.read_error(True)[0] == 3, what
            assert torch.equal(again[1], want[1])
        if what in ("page", "length"):
            kernels.page_bounds(d["kc"], d["bounds"], d["bt"], zeros, d["lens"], 10000)
            assert kernels.read_error(True)[0] == 3, what
    kernels.page_bounds(good["kc"], good["bounds"], good["bt"], zeros, good["lens"], 199)   # more new tokens than said
    assert kernels.read_error(True)[0] == 3


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def _refuses(call, *words):
    with pytest.raises((RuntimeError, ValueError)) as e:
        call()
    assert any(w in str(e.value) for w in words), str(e.value)


@gpu
def test_refusals(kernels):
    k = kernels
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    # head norm + rotation
    T, Hq, Hkv, D = 4, 4, 1, 128
    good = dict(qkv=z(T, 6 * D), wq=z(D), wk=z(D), eps=1e-5, pos=z(T, dtype=I32), slots=z(T, dtype=I32),
                cs=z(16, D // 2, 2, dtype=F32), q=z(T, Hq * D), kc=z(3, Hkv, 16, D), vc=z(3, Hkv, 16, D), Hq=Hq,
                Hkv=Hkv, page=16)

    def norm(**change):
        a = dict(good, **change)
        _refuses(lambda: k.qk_norm_rope_kv_write(*a.values()), "lunaflux")

    for change in (dict(qkv=z(T, 6 * D, dtype=F32)), dict(qkv=z(T, 5 * D)), dict(qkv=z(T, 6 * D + 4)[:, 4:]),
                   dict(wq=z(64)), dict(wk=z(D, dtype=F32)), dict(pos=z(T - 1, dtype=I32)), dict(slots=z(T, dtype=torch.int64)),
                   dict(cs=z(16, D, 2, dtype=F32)), dict(cs=z(16, D // 2, dtype=F32)), dict(q=z(T, Hq * D + 8)),
                   dict(q=z(T - 1, Hq * D)), dict(kc=z(3, 2, 16, D)), dict(vc=z(4, Hkv, 16, D)), dict(page=8),
                   dict(kc=z(3, Hkv, 16, 96), vc=z(3, Hkv, 16, 96)), dict(eps=-1.0), dict(qkv=torch.zeros(T, 6 * D, dtype=BF)),
                   dict(pos=torch.zeros(T, dtype=I32)), dict(q=good["qkv"][:, D:5 * D])):
        norm(**change)
    # adapters
    T, K, N, R, P = 6, 64, 48, 16, 3
    lora = dict(x=z(T, K), a=z(P, R, K), b=z(P, N, R), scales=z(P, dtype=F32), ranks=z(P, dtype=I32),
                rows=z(2, dtype=I32), starts=z(P + 1, dtype=I32), base=z(T, N), out=z(T, N), slices=(N,))

    def add(**change):
        a = dict(lora, **change)
        _refuses(lambda: k.lora_add(*a.values()), "lunaflux")

    wide = z(T, 2 * N)
    for change in (dict(x=z(T, K + 8)), dict(x=z(T, K, dtype=F32)), dict(a=z(P, 2 * R, K)), dict(b=z(P - 1, N, R)),
                   dict(a=z(P, 12, K), b=z(P, N, 12)), dict(a=z(P, 136, K), b=z(P, N, 136)), dict(scales=z(P, dtype=BF)),
                   dict(ranks=z(P - 1, dtype=I32)), dict(starts=z(P, dtype=I32)), dict(rows=z(T + 1, dtype=I32)),
                   dict(base=z(T, N, dtype=F32)), dict(out=z(T, N + 8)), dict(slices=(N - 8,)), dict(slices=(N, 8)),
                   dict(slices=(44, 4)), dict(slices=(8,) * 5, a=z(P, 5 * R, K)),
                   dict(base=wide[:, :N], out=wide[:, 8:8 + N]), dict(x=z(T, 68)[:, 4:]),
                   dict(b=z(P, R, N).transpose(1, 2)), dict(rows=torch.zeros(2, dtype=I32))):
        add(**change)
    # selected pages
    Hq, Hkv, R, W, B = 8, 2, 3, 10, 4
    sp = dict(q=z(R, Hq * 128), tok=z(R, dtype=I32), lens=z(R, dtype=I32), bt=z(R, W, dtype=I32),
              bounds=z(5, Hkv, 2, 128), sel=z(R, Hkv, B, dtype=I32), first=1, last=2, Hq=Hq, Hkv=Hkv,
              ws=z(2 * R * Hkv * W, dtype=F32))

    def select(**change):
        a = dict(sp, **change)
        _refuses(lambda: k.attn_select(*a.values()), "lunaflux")

    for change in (dict(first=3), dict(last=-1), dict(Hq=9), dict(Hkv=0), dict(Hq=64, Hkv=2), dict(ws=z(2 * R * Hkv * W - 1, dtype=F32)),
                   dict(sel=z(R, Hkv, B)), dict(sel=z(R, B, Hkv, dtype=I32)), dict(bounds=z(5, Hkv, 2, 64)),
                   dict(bt=z(R - 1, W, dtype=I32)), dict(q=z(R, 7 * 128)), dict(tok=z(R - 1, dtype=I32)),
                   dict(lens=z(R, dtype=torch.int64)), dict(bt=torch.zeros(R, W, dtype=I32))):
        select(**change)
    at = dict(q=sp["q"], out=z(R, Hq * 128), tok=sp["tok"], lens=sp["lens"], bt=sp["bt"], sel=sp["sel"],
              kc=z(5, Hkv, 16, 128), vc=z(5, Hkv, 16, 128), Hq=Hq, Hkv=Hkv)

    def attend(**change):
        a = dict(at, **change)
        _refuses(lambda: k.attn_decode_sparse(*a.values()), "lunaflux")

    for change in (dict(out=z(R, 7 * 128)), dict(out=at["q"]), dict(out=z(R - 1, Hq * 128)), dict(kc=z(5, Hkv, 8, 128)),
                   dict(vc=z(6, Hkv, 16, 128)), dict(Hq=12), dict(sel=z(R, Hkv, 0, dtype=I32)), dict(kc=z(5, 1, 16, 128)),
                   dict(out=z(R, Hq * 128, dtype=F32))):
        attend(**change)
    for change in ((z(5, Hkv, 16, 64), z(5, Hkv, 2, 64)), (z(5, Hkv, 16, 128), z(4, Hkv, 2, 128))):
        _refuses(lambda: k.page_bounds(change[0], change[1], sp["bt"], sp["tok"], sp["lens"], 1), "lunaflux")
    _refuses(lambda: k.page_bounds(at["kc"], sp["bounds"], sp["bt"], sp["tok"], sp["lens"], -1), "lunaflux")
    assert k.read_error(True)[0] == 0


def test_contracts_refuse():
    """The launch contracts name the operand that does not fit (no GPU)."""
    from lunaflux_b200.ops.launch_contract import CONTRACTS, Issue, LaunchContractError, admit, launch_checks

    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)  # noqa: E731
    T, Hq, Hkv, D = 4, 4, 1, 128
    adapt = launch_checks()

    def norm(T=T, q_cols=Hq * D, D_=D, page=16):
        return adapt["qk_norm_rope_kv_write"](z(T, 6 * D), z(D), z(D), 1e-5, z(T, dtype=I32), z(T, dtype=I32),
                                              z(16, D_ // 2, 2, dtype=F32), z(T, q_cols), z(3, Hkv, 16, D),
                                              z(3, Hkv, 16, D), Hq, Hkv, page)

    admit(*norm())
    for bad, issue in ((dict(q_cols=Hq * D + 8), Issue.RULE), (dict(D_=64), Issue.RULE), (dict(page=8), Issue.SHAPE)):
        with pytest.raises(LaunchContractError) as e:
            admit(*norm(**bad))
        assert e.value.issue is issue

    def lora(slices=(48,), R=16, SR=None, L=2, base=BF):
        P, N, K = 3, 48, 64
        return adapt["lora_add"](z(6, K), z(P, SR or R, K), z(P, N, R), z(P, dtype=F32), z(P, dtype=I32), z(L, dtype=I32),
                                 z(P + 1, dtype=I32), z(6, N, dtype=base), z(6, N, dtype=base), slices)

    admit(*lora())
    admit(*lora(slices=(32, 16), SR=32, base=F32))
    for bad in (dict(slices=(40,)), dict(R=12), dict(SR=32), dict(L=7), dict(slices=(44, 4), SR=32)):
        with pytest.raises(LaunchContractError):
            admit(*lora(**bad))

    def select(first=1, ws=240, Hq=8):
        return adapt["attn_select"](z(3, 8 * 128), z(3, dtype=I32), z(3, dtype=I32), z(3, 10, dtype=I32), z(5, 4, 2, 128),
                                    z(3, 4, 4, dtype=I32), first, 2, Hq, 4, z(ws, dtype=F32))

    admit(*select())
    for bad in (dict(first=3), dict(ws=239), dict(Hq=12), dict(Hq=7)):
        with pytest.raises(LaunchContractError):
            admit(*select(**bad))
    admit(*adapt["page_bounds"](z(5, 4, 16, 128), z(5, 4, 2, 128), z(3, 10, dtype=I32), z(3, dtype=I32), z(3, dtype=I32), 1))
    with pytest.raises(LaunchContractError):
        admit(*adapt["page_bounds"](z(5, 4, 16, 128), z(4, 4, 2, 128), z(3, 10, dtype=I32), z(3, dtype=I32), z(3, dtype=I32), 1))
    ok = (z(3, 8 * 128), z(3, 8 * 128), z(3, dtype=I32), z(3, dtype=I32), z(3, 10, dtype=I32), z(3, 4, 4, dtype=I32),
          z(5, 4, 16, 128), z(5, 4, 16, 128), 8, 4)
    admit(*adapt["attn_decode_sparse"](*ok))
    with pytest.raises(LaunchContractError):
        admit(*adapt["attn_decode_sparse"](*ok[:1], z(2, 8 * 128), *ok[2:]))
    assert {"qk_norm_rope_kv_write", "lora_add", "page_bounds", "attn_select", "attn_decode_sparse"} <= set(CONTRACTS)
