"""The adapter, head-norm and selected-page operators as a decode layer runs
them: one after another, captured and replayed, on other streams, side by side."""
import pytest
import torch

from tests.test_serving_ops import (BF, F32, I32, _attend_check, _bounds_reference, _gen, _lora_inputs, _lora_reference,
                                    _norm_rope_reference, _randn, _select_reference, _within)

pytestmark = pytest.mark.gpu

HQ, HKV, H, D = 8, 2, 512, 128
N = (HQ + 2 * HKV) * D
SLICES = (HQ * D, HKV * D, HKV * D)


def _layer(lens, seed, pad=1):
    """A decode layer's weights, adapters, cache and step inputs for rows of the given lengths (with the new
    token), the last `pad` rows of the bucket being padding (slot -1, the zero page, length 1)."""
    g = _gen(seed)
    R = len(lens) + pad
    n = [-(-x // 16) for x in lens] + [1] * pad
    width = max(n) + 2
    pages = 1 + sum(n[:len(lens)])
    perm = torch.randperm(pages - 1, generator=g) + 1
    bt = torch.zeros(R, width, dtype=I32)
    at = 0
    for r, x in enumerate(n[:len(lens)]):
        bt[r, :x] = perm[at:at + x].int()
        at += x
    full = torch.tensor(list(lens) + [1] * pad, dtype=I32)
    pos = full - 1
    slots = torch.tensor([int(bt[r, (x - 1) // 16]) * 16 + (x - 1) % 16 for r, x in enumerate(lens)] + [-1] * pad, dtype=I32)
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(max(lens) + 1, dtype=torch.float64)[:, None] * inv
    kc = _randn(g, pages, HKV, 16, D, dtype=F32).add(_randn(g, pages, HKV, 1, D, dtype=F32)).to(BF)
    vc = _randn(g, pages, HKV, 16, D)
    kc[0] = vc[0] = 0
    pool, rank = 3, 16
    ids = torch.randint(-1, pool, (R,), generator=g)
    order = torch.argsort(ids, stable=True)
    counts = [int((ids == i).sum()) for i in range(pool)]
    # the row list has the bucket's length, as a captured step needs it; what lies behind the last adapter's is not read
    rows = torch.full((R,), -7, dtype=I32)
    rows[:sum(counts)] = order[R - sum(counts):].int()
    v = dict(x=_randn(g, R, H), wqkv=_randn(g, N, H, scale=H ** -0.5), wo=_randn(g, H, HQ * D, scale=0.03),
             qa=_randn(g, pool, 3 * rank, H, scale=H ** -0.5), qb=_randn(g, pool, N, rank, scale=0.3),
             oa=_randn(g, pool, rank, HQ * D, scale=0.03), ob=_randn(g, pool, H, rank, scale=0.3),
             scales=torch.rand(pool, generator=g) + 0.5, ranks=torch.tensor([16, 5, 9], dtype=I32),
             rows=rows, starts=torch.tensor([0] + counts).cumsum(0).int(),
             wq=_randn(g, D, scale=0.2) + 1, wk=_randn(g, D, scale=0.2) + 1, pos=pos, slots=slots, lens=full,
             start=full - 1, bt=bt, tok=torch.arange(R, dtype=I32), kc=kc, vc=vc,
             cs=torch.stack([ang.cos(), ang.sin()], -1).float().contiguous(),
             bounds=torch.zeros(pages, HKV, 2, D, dtype=BF))
    v["bounds"] = _bounds_reference(dict(v, lens=full - 1), [0] * R)
    d = {k: t.cuda() for k, t in v.items()}
    d["qkv"] = torch.zeros(R, N, dtype=BF, device="cuda")
    d["attn"] = torch.zeros(R, HQ * D, dtype=BF, device="cuda")
    d["out"] = torch.zeros(R, H, dtype=BF, device="cuda")
    return d, width


def _buffers(d, width, ops, budget):
    R = d["x"].shape[0]
    return (torch.zeros(R, HKV, budget, dtype=I32, device="cuda"),
            torch.zeros(ops.select_workspace(R, HKV, width), device="cuda"))


def _run(ops, d, sel, ws, budget, tap=None):
    tap = tap or (lambda name: None)
    ops.gemm(d["x"], d["wqkv"], d["qkv"])
    tap("qkv")
    ops.lora_add(d["x"], d["qa"], d["qb"], d["scales"], d["ranks"], d["rows"], d["starts"], d["qkv"], d["qkv"], SLICES)
    tap("lora")
    ops.qk_norm_rope_kv_write(d["qkv"], d["wq"], d["wk"], 1e-5, d["pos"], d["slots"], d["cs"], d["qkv"][:, :HQ * D],
                              d["kc"], d["vc"], HQ, HKV, 16)
    tap("norm")
    ops.page_bounds(d["kc"], d["bounds"], d["bt"], d["start"], d["lens"], 1)
    ops.attn_select(d["qkv"], d["tok"], d["lens"], d["bt"], d["bounds"], sel, 1, 1, HQ, HKV, ws)
    ops.attn_decode_sparse(d["qkv"], d["attn"], d["tok"], d["lens"], d["bt"], sel, d["kc"], d["vc"], HQ, HKV)
    ops.gemm(d["attn"], d["wo"], d["out"])
    tap("o")
    ops.lora_add(d["attn"], d["oa"], d["ob"], d["scales"], d["ranks"], d["rows"], d["starts"], d["out"], d["out"])


@pytest.fixture(scope="module")
def ops():
    from lunaflux_b200.ops import KernelOps
    return KernelOps()


def _lora_tolerance(mag, K):
    # as the single operator's: chains of K / 16 steps, 8 steps of expansion for each of two parts, h in two parts
    return (17 * 2.0 ** -23 * (K // 16 + 1 + 24) + 2.0 ** -16) * mag


def test_decode_layer_step_by_step(ops):
    """Every operator against its definition on what the one before it wrote."""
    lens, budget = [700, 33, 16, 1, 450, 1000], 6
    d, width = _layer(lens, 3)
    sel, ws = _buffers(d, width, ops, budget)
    kept = {}
    before = {k: d[k].cpu().clone() for k in ("kc", "vc", "bounds")}
    _run(ops, d, sel, ws, budget, lambda name: kept.update({name: {k: d[k].cpu().clone() for k in ("qkv", "kc", "vc", "out")}}))
    assert ops.read_error(True)[0] == 0
    c = {k: t.cpu() for k, t in d.items()}
    lo = dict(x=c["x"], a=c["qa"], b=c["qb"], base=kept["qkv"]["qkv"], scales=c["scales"], ranks=c["ranks"], rows=c["rows"],
              starts=c["starts"])
    ref, mag = _lora_reference(lo, SLICES, 16)
    _within(kept["lora"]["qkv"], ref, 2.0 ** -8 * ref.abs() + _lora_tolerance(mag, H), "lora")
    nr = dict(qkv=kept["lora"]["qkv"], wq=c["wq"], wk=c["wk"], pos=c["pos"], slots=c["slots"], cs=c["cs"],
              kc=before["kc"], vc=before["vc"], width=N)
    rq, mq, rk, mk, rv = _norm_rope_reference(nr, HQ, HKV, D, 1e-5)
    _within(kept["norm"]["qkv"][:, :HQ * D], rq, 2.0 ** -8 * rq.abs() + 2.0 ** -18 * mq, "q")
    _within(kept["norm"]["kc"], rk, torch.where(mk > 0, 2.0 ** -8 * rk.abs() + 2.0 ** -18 * mk, torch.zeros_like(rk)), "k")
    assert torch.equal(kept["norm"]["vc"].double(), rv)
    sp = dict(q=c["qkv"], bt=c["bt"], lens=c["lens"], tok=c["tok"], kc=c["kc"], vc=c["vc"], bounds=before["bounds"])
    want = _bounds_reference(sp, c["start"].tolist())
    assert torch.equal(c["bounds"], want)
    sp["bounds"] = want
    chosen = _select_reference(sp, HQ, HKV, budget, 1, 1)
    assert torch.equal(sel.cpu(), chosen)
    _attend_check(c["attn"], sp, chosen, HQ, HKV)
    lo = dict(x=c["attn"], a=c["oa"], b=c["ob"], base=kept["o"]["out"], scales=c["scales"], ranks=c["ranks"], rows=c["rows"],
              starts=c["starts"])
    ref, mag = _lora_reference(lo, (H,), 16)
    _within(c["out"], ref, 2.0 ** -8 * ref.abs() + _lora_tolerance(mag, HQ * D), "o lora")


def test_captured_layer_replays_with_new_inputs(ops):
    """A captured layer, replayed on new inputs in the same buffers, gives the eager layer's bits; nothing is
    allocated while it replays, and the library's stream is not the one it runs on."""
    budget = 5
    a, width = _layer([300, 90, 500, 17], 7)
    b, _ = _layer([300, 90, 500, 17], 8)
    sel, ws = _buffers(a, width, ops, budget)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _run(ops, a, sel, ws, budget)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        _run(ops, a, sel, ws, budget)
    eager = {k: t.clone() for k, t in b.items()}
    es, ew = _buffers(eager, width, ops, budget)
    _run(ops, eager, es, ew, budget)
    for k in a:
        a[k].copy_(b[k])
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    for k in ("qkv", "kc", "vc", "bounds", "attn", "out"):
        assert torch.equal(a[k], eager[k]), k
    assert torch.equal(sel, es)
    assert ops.read_error(True)[0] == 0


def test_two_streams_at_once(ops):
    """Calls with their own workspaces on two streams at the same time: the results of the calls alone.  The
    adapters are large tiles (tensor memory) beside small ones, the attention split over clusters."""
    work = []
    for i in range(2):
        v = _lora_inputs(2000, 512, (256, 64, 64), 64, [700, 900, 300], 40 + i, [64, 23, 40], integer=False)
        t = {k: x.cuda() for k, x in v.items()}
        layer, width = _layer([4000, 900, 2500], 50 + i)
        sel, ws = _buffers(layer, width, ops, 16)
        work.append((t, layer, sel, ws, torch.zeros_like(t["base"])))

    def go(i):
        t, layer, sel, ws, out = work[i]
        for _ in range(3):
            ops.lora_add(t["x"], t["a"], t["b"], t["scales"], t["ranks"], t["rows"], t["starts"], t["base"], out, (256, 64, 64))
            _run(ops, layer, sel, ws, 16)

    def results(i):
        t, layer, sel, ws, out = work[i]
        return [out.clone(), layer["out"].clone(), layer["attn"].clone(), sel.clone()]

    alone = []
    for i in range(2):
        go(i)
        torch.cuda.synchronize()
        alone.append(results(i))
        work[i][4].zero_()
        work[i][1]["out"].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                go(i)
    torch.cuda.synchronize()
    for i in range(2):
        for x, y in zip(results(i), alone[i]):
            assert torch.equal(x, y)
    assert ops.read_error(True)[0] == 0


def test_launch_checks_admit_the_layer(monkeypatch):
    """With every launch admitted against its contract the layer runs as before."""
    monkeypatch.setenv("LUNAFLUX_CHECK_LAUNCHES", "1")
    from lunaflux_b200.ops import KernelOps
    ops = KernelOps()
    d, width = _layer([100, 40], 9)
    sel, ws = _buffers(d, width, ops, 4)
    _run(ops, d, sel, ws, 4)
    assert ops.admitted == 8 and ops.read_error(True)[0] == 0


_FIRST_CALL = """
import torch
from lunaflux_b200.ops import KernelOps
from tests.test_serving_ops import _lora_inputs, _lora_reference, BF
ops = KernelOps()
for T, K, slices, R, counts in ((3, 256, (64, 32), 16, [1, 2]), (1300, 136, (72,), 64, [600, 700]),
                                (2600, 136, (40, 32), 64, [65] * 40)):
    v = _lora_inputs(T, K, slices, R, counts, T)
    d = {k: t.cuda() for k, t in v.items()}
    out = torch.zeros_like(d["base"])
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        ops.lora_add(d["x"], d["a"], d["b"], d["scales"], d["ranks"], d["rows"], d["starts"], d["base"], out, slices)
    g.replay()
    torch.cuda.synchronize()
    rows = v["rows"].long()
    assert torch.equal(out.cpu()[rows], _lora_reference(v, slices, R)[0].to(BF)[rows])
print("captured")
"""


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path
    p = subprocess.run([sys.executable, "-c", _FIRST_CALL], cwd=Path(__file__).resolve().parent.parent, timeout=300,
                       capture_output=True, text=True)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]
