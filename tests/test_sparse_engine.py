"""The engine's decode over selected pages (``EngineOptions.sparse_pages``)."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from lunaflux_b200.config import CacheConfig, SchedulerConfig
from lunaflux_b200.engine.engine import EngineOptions, LLMEngine
from lunaflux_b200.engine.step_inputs import device_views, make_layout
from lunaflux_b200.models.spec import LlamaSpec, tiny_llama
from lunaflux_b200.models.weights import build_runtime, random_checkpoint
from lunaflux_b200.ops import TorchOps
from lunaflux_b200.oracle.reference import ReferenceModel


def _prompts(vocab, lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def _cpu_engine(ck, spec, sparse, budget=64, prefix=False, overlap=False, pages=96, first=1, last=1):
    sched = SchedulerConfig(step_token_budget=budget, max_active_requests=4, prefill_chunk_tokens=budget,
                            emergency_decode_page_reserve=1, waiting_age_threshold_steps=8)
    return LLMEngine(build_runtime(spec, lambda n: ck[n]), TorchOps(), "cpu", sched, CacheConfig(prefix_enabled=prefix),
                     EngineOptions(max_context=256, num_pages=pages, graph_sizes=(), overlap_steps=overlap,
                                   sparse_pages=sparse, sparse_first=first, sparse_last=last))


def make_layout_of(runner, plan):
    """The layout of the step block that `plan` was packed into."""
    pre = [x for x in plan.rows if not x.decode]
    dec = len(plan.rows) - len(pre)
    return make_layout(plan.num_tokens, len(pre), dec, sum(1 for x in plan.rows if x.sample), runner.W) if plan.rows else None


@pytest.fixture(scope="module")
def tiny():
    spec = tiny_llama()
    return spec, random_checkpoint(spec, 0)


def test_all_pages_selected_is_the_dense_engine(tiny):
    spec, ck = tiny
    prompts = _prompts(256, (5, 40, 90, 150))
    ref = ReferenceModel(spec, ck)
    outs = _cpu_engine(ck, spec, 16).generate(prompts, 12)
    for p, o in zip(prompts, outs):
        assert o == ref.generate_greedy(p, 12)


def test_few_pages_do_not_depend_on_how_the_steps_are_cut(tiny):
    """Chunked prefill, overlapped steps and shared prefix pages give the same
    tokens: a page's bounds follow the page, not the step that wrote it."""
    spec, ck = tiny
    prompts = _prompts(256, (150, 90, 200, 30), seed=1)
    want = _cpu_engine(ck, spec, 4, budget=256).generate(prompts, 14)
    assert _cpu_engine(ck, spec, 4, budget=24).generate(prompts, 14) == want
    assert _cpu_engine(ck, spec, 4, budget=64, overlap=True).generate(prompts, 14) == want
    eng = _cpu_engine(ck, spec, 4, budget=64, prefix=True)
    assert eng.generate(prompts, 14) == want
    rids = [eng.add_request(p, 14) for p in prompts]      # the second time from cached prefix pages
    eng.run_until_done()
    assert [eng.results[r].tokens for r in rids] == want
    assert any(eng.results[r].cached_tokens for r in rids)
    # pages freed and taken again by other sequences: the bounds are those of the new owner
    small = _cpu_engine(ck, spec, 4, budget=64, pages=16)
    for p, w in zip(prompts, want):
        assert small.generate([p], 14) == [w]


def test_bounds_match_the_cache_after_every_step(tiny):
    spec, ck = tiny
    eng = _cpu_engine(ck, spec, 3, budget=32)
    for p in _prompts(256, (70, 33, 5), seed=2):
        eng.add_request(p, 20)
    r, checked = eng.runner, 0
    while eng.has_work():
        plan = eng.scheduler.schedule
        seen = []

        def note(*a, **k):
            seen.append(plan(*a, **k))
            return seen[-1]

        eng.scheduler.schedule = note
        eng.step()
        eng.scheduler.schedule = plan
        # the packed step still lies in the runner: every page the step's rows hold
        L = seen[-1] and make_layout_of(r, seen[-1])
        if not L:
            continue
        v = device_views(r.in_dev, L)
        for bt, lens in ((v["p_bt"], v["p_seqlen"]), (v["d_bt"], v["d_seqlen"])):
            for row, n in zip(bt.tolist(), lens.tolist()):
                for page in range(-(-n // 16)):
                    keys = r.kv[:, 0, row[page], :, : min(16, n - page * 16)]
                    b = r.bounds[:, row[page]]
                    assert torch.equal(b[:, :, 0], keys.amin(2)) and torch.equal(b[:, :, 1], keys.amax(2))
                    checked += 1
    assert checked > 50


def test_options_are_checked(tiny):
    spec, ck = tiny
    with pytest.raises(ValueError):
        _cpu_engine(ck, spec, 2, first=1, last=2)

    class NoSparse(TorchOps):
        attn_select = property(lambda self: (_ for _ in ()).throw(AttributeError()))

    sched = SchedulerConfig(step_token_budget=64, max_active_requests=4, prefill_chunk_tokens=64,
                            emergency_decode_page_reserve=1)
    with pytest.raises(ValueError):
        LLMEngine(build_runtime(spec, lambda n: ck[n]), NoSparse(), "cpu", sched, CacheConfig(),
                  EngineOptions(max_context=256, num_pages=64, graph_sizes=(), sparse_pages=4))


@pytest.mark.parametrize("change,words", [(dict(head_dim=64), "head_dim 128"), (dict(heads=34, kv_heads=2), "16 query heads"),
                                          (dict(), None)])
def test_kernel_limits_are_checked_at_construction(change, words):
    """A model or a table the kernels do not take is refused before any request is admitted."""
    from lunaflux_b200.ops import KernelOps

    class Limited(TorchOps):
        sparse_unsupported = staticmethod(KernelOps.sparse_unsupported)

    spec = LlamaSpec(**{**dict(hidden=64, layers=1, heads=4, kv_heads=2, head_dim=128, ffn=128, vocab=64, rope_theta=10000.0,
                               max_position=512, dtype="bf16"), **change})
    ck = random_checkpoint(spec, 0)
    w = build_runtime(spec, lambda n: ck[n], dtype=torch.bfloat16)
    sched = SchedulerConfig(step_token_budget=64, max_active_requests=4, prefill_chunk_tokens=64,
                            emergency_decode_page_reserve=1)

    def engine(**opts):
        return LLMEngine(w, Limited(), "cpu", sched, CacheConfig(), EngineOptions(**{**dict(
            max_context=256, num_pages=64, graph_sizes=(), sparse_pages=4), **opts}))

    if words:
        with pytest.raises(ValueError, match=words):
            engine()
    else:
        engine()
        with pytest.raises(ValueError, match="65536 pages"):
            engine(sparse_pages=65537)
    engine(sparse_pages=0)


def test_kernel_limits():
    from lunaflux_b200.ops import KernelOps
    at = dict(Hq=32, Hkv=8, D=128, page=16, dtype=torch.bfloat16, rows=256, width=8192, budget=64)
    assert KernelOps.sparse_unsupported(**at) is None
    assert KernelOps.sparse_unsupported(**{**at, "Hq": 16, "Hkv": 1, "width": 65536, "rows": 65535}) is None
    for change in (dict(D=64), dict(page=32), dict(dtype=torch.float16), dict(Hq=34, Hkv=2), dict(Hq=12), dict(width=65537),
                   dict(budget=65537), dict(rows=65536)):
        assert KernelOps.sparse_unsupported(**{**at, **change})


def _rank(rank, world, port, q, sp, sparse):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from lunaflux_b200.parallel.comm import TPComm
        from lunaflux_b200.parallel.tp import TPShard
        spec = tiny_llama()
        ck = random_checkpoint(spec, 0)
        sched = SchedulerConfig(step_token_budget=64, max_active_requests=4, prefill_chunk_tokens=64,
                                emergency_decode_page_reserve=1, waiting_age_threshold_steps=8)
        eng = LLMEngine(build_runtime(spec, lambda n: ck[n], TPShard(rank, world, spec)), TorchOps(), "cpu", sched,
                        CacheConfig(), EngineOptions(max_context=256, num_pages=96, graph_sizes=(), sequence_parallel=sp,
                                                     sparse_pages=sparse, sparse_first=1, sparse_last=1), comm=TPComm())
        assert eng.runner.sp == sp and eng.runner.bounds.shape[2] == max(1, spec.kv_heads // world)
        q.put((rank, eng.generate(_prompts(256, (150, 90, 30), seed=1), 10)))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world,sp,sparse", [(2, False, 4), (2, True, 4), (4, True, 16)])
def test_tensor_and_sequence_parallel_ranks(tiny, world, sp, sparse):
    """Ranks with whole KV heads select what one rank selects; with shared ones (world 4 of 2
    KV heads) a rank selects for its own query heads, so there every page is taken."""
    spec, ck = tiny
    want = _cpu_engine(ck, spec, sparse, budget=64).generate(_prompts(256, (150, 90, 30), seed=1), 10)
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, world, port, q, sp, sparse)) for r in range(world)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=240) for _ in range(world))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for r in range(world):
        assert got[r] == want, f"rank {r}"


def _gpu_engine(spec, ck, sparse, graphs):
    from lunaflux_b200.ops import KernelOps
    w = build_runtime(spec, lambda n: ck[n], device="cuda", dtype=torch.bfloat16)
    sched = SchedulerConfig(step_token_budget=256, max_active_requests=8, prefill_chunk_tokens=256,
                            emergency_decode_page_reserve=4)
    return LLMEngine(w, KernelOps(), "cuda", sched, CacheConfig(prefix_enabled=False),
                     EngineOptions(max_context=1024, num_pages=512, graph_sizes=(1, 2, 4, 8) if graphs else (),
                                   overlap_steps=graphs, sparse_pages=sparse))


@pytest.mark.gpu
def test_gpu_engine_over_selected_pages():
    """All pages: near the oracle's argmax.  A few: captured, overlapped steps
    give the eager engine's tokens, and the device reports no error."""
    spec = LlamaSpec(hidden=1024, layers=2, heads=8, kv_heads=2, head_dim=128, ffn=2816, vocab=4096,
                     rope_theta=500000.0, max_position=2048, dtype="bf16")
    ck = {k: v.bfloat16().float() for k, v in random_checkpoint(spec, 0).items()}
    prompts = _prompts(spec.vocab, (5, 70, 300, 17, 129, 800), seed=1)
    ref = ReferenceModel(spec, ck)
    outs = _gpu_engine(spec, ck, 64, True).generate(prompts, 8)
    for p, o in zip(prompts, outs):
        logits = ref.forward(list(p) + list(o))
        for i, tok in enumerate(o):
            row = logits[len(p) - 1 + i]
            assert (row.max() - row[tok]).item() <= 0.05 * row.std().item() + 1e-4
    graph, eager = _gpu_engine(spec, ck, 8, True), _gpu_engine(spec, ck, 8, False)
    assert graph.generate(prompts, 24) == eager.generate(prompts, 24)
    for e in (graph, eager):
        assert e.runner.ops.read_error(True)[0] == 0


@pytest.mark.gpu
def test_gpu_engine_launches_admitted(monkeypatch):
    """Every launch of the engine over selected pages meets its contract; the tokens are the same."""
    spec = LlamaSpec(hidden=1024, layers=2, heads=8, kv_heads=2, head_dim=128, ffn=2816, vocab=4096,
                     rope_theta=500000.0, max_position=2048, dtype="bf16")
    ck = {k: v.bfloat16().float() for k, v in random_checkpoint(spec, 1).items()}
    prompts = _prompts(spec.vocab, (5, 70, 300, 33), seed=2)
    want = _gpu_engine(spec, ck, 6, True).generate(prompts, 16)
    monkeypatch.setenv("LUNAFLUX_CHECK_LAUNCHES", "1")
    for graphs in (True, False):
        eng = _gpu_engine(spec, ck, 6, graphs)
        assert eng.generate(prompts, 16) == want
        assert eng.runner.ops.read_error(True)[0] == 0


@pytest.mark.gpu
def test_gpu_engine_refuses_what_the_kernels_do_not_take():
    spec = LlamaSpec(hidden=512, layers=1, heads=8, kv_heads=2, head_dim=64, ffn=512, vocab=256, max_position=1024, dtype="bf16")
    ck = {k: v.bfloat16().float() for k, v in random_checkpoint(spec, 0).items()}
    with pytest.raises(ValueError, match="head_dim 128"):
        _gpu_engine(spec, ck, 6, False)
