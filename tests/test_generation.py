"""Generation with the Llama stack: the decoding step's operators together, as a plan that a
user steps through — pieces of the prompt first, then one token at a time, each step's drawn tokens
the next one's input. On the CPU the plan's operator list runs with the oracle's arithmetic; on
the GPU through the native library, eagerly and as a replayed graph."""

import threading

import numpy as np
import pytest
import torch

from cpu_plan import CpuPlanRunner
from oracle import decode_ops as DR
from oracle import inputs as I
from oracle import reference_ops as R
from oracle.check import SHARDED_LAYER_ROUNDINGS, assert_parity

from lighthouse_b200 import _native as N
from lighthouse_b200.plan import ArgSpec, Plan
from lighthouse_b200.workloads import decoder as D

VOCAB = 96


class DecodeRunner(CpuPlanRunner):
    """With the decoding operators, by their definitions."""

    def _paged_append(self, op):
        q, k, v, k_pages, v_pages, slots, positions = op.operands[:7]
        maybe = lambda x: None if x is None else self.read(x)
        new_q, new_k, new_v, bad = DR.paged_append(maybe(q), self.read(k), self.read(v), self.read(k_pages), self.read(v_pages), self.read(slots), maybe(positions), op.attrs["theta"])
        assert not bad
        for view, new in ((q, new_q), (k_pages, new_k), (v_pages, new_v)):
            if view is not None:
                self.write(view, new)

    def _paged_attention(self, op):
        o, q, k_pages, v_pages, table, lengths = op.operands[:6]
        out, _, bad = DR.paged_attention(self.read(q), self.read(k_pages), self.read(v_pages), self.read(table), self.read(lengths), op.attrs["scale"])
        assert not bad
        self.write(o, out)

    def _sample(self, op):
        tokens, logprobs, logits, uniform, temperature, top_k, top_p, min_p = op.operands[:8]
        maybe = lambda x: None if x is None else self.read(x)
        got, lp = DR.sample(self.read(logits), self.read(uniform), maybe(temperature), maybe(top_k), maybe(top_p), maybe(min_p))
        self.write(tokens, got)
        if logprobs is not None:
            self.write(logprobs, lp)


class Generation:
    """The host's side of a generation: pages handed out, slots and positions of each step."""

    def __init__(self, rng, cache, batch, chunk, prompts, steps):
        self.cache, self.batch, self.chunk = cache, batch, chunk
        self.order = list(rng.permutation(cache.pages))  # pages lie anywhere in the pool
        self.table = np.full((batch, cache.columns), -1, np.int64)
        self.length = np.zeros(batch, np.int64)
        self.text = [list(p) for p in prompts]
        self.fed = [0] * batch
        self.uniform = rng.random((steps, batch), dtype=np.float32)

    def reserve(self, b, length):
        for c in range(-(-length // self.cache.page_size)):
            if self.table[b, c] < 0:
                self.table[b, c] = self.order.pop()

    def step(self, seq):
        """ids, slots, positions, table, lengths of a step of `seq` places per sequence."""
        ids, slots, positions = (np.zeros((self.batch, seq), np.int64) for _ in range(3))
        slots[:] = -1
        for b in range(self.batch):
            new = self.text[b][self.fed[b]:self.fed[b] + seq]
            n = len(new)
            self.reserve(b, self.fed[b] + n)
            at = np.arange(self.fed[b], self.fed[b] + n)
            ids[b, seq - n:], positions[b, seq - n:] = new, at
            slots[b, seq - n:] = self.table[b, at // self.cache.page_size] * self.cache.page_size + at % self.cache.page_size
            self.fed[b] += n
            self.length[b] = self.fed[b]
        return ids.reshape(-1), slots.reshape(-1), positions.reshape(-1), np.maximum(self.table, 0), self.length.copy()


def model(cfg, seed=5, std=0.1):
    w = I.llama_weights(cfg.n_layer, cfg.dim, cfg.n_heads, cfg.n_kv_heads, cfg.ffn, seed=seed, std=std)
    g = torch.Generator().manual_seed(seed + 1)
    wte = torch.randn(VOCAB, cfg.dim, generator=g).to(torch.bfloat16)
    head = (torch.randn(VOCAB, cfg.dim, generator=g) * 0.3).to(torch.bfloat16)
    return w, wte, head


def reference_logits(cfg, w, wte, head, text):
    """The logits after the last token of `text`, by the whole forward pass over it."""
    wn = I.tree_to_np(w)
    x = I.to_np(wte)[np.asarray(text)][None]
    h = R.llama_forward(x, wn["layers"], wn["norm"], cfg.n_heads, cfg.n_kv_heads, cfg.theta, cfg.eps, "bf16", fused_swiglu=True, fused_residual=True)
    return h[0, -1] @ I.to_np(head).T


def settings(batch):
    # greedy, everything on, unfiltered, top-p alone
    pick = lambda values, dt: np.array([values[b % 4] for b in range(batch)], dt)
    return pick([0.0, 0.8, 1.0, 1.3], np.float32), pick([0, 20, 0, 0], np.int32), pick([1.0, 0.9, 1.0, 0.7], np.float32), pick([0.0, 0.02, 0.0, 0.0], np.float32)


def generate(cfg, cache, prompts, steps, rng, run):
    """Feeds the prompts in pieces of `cfg.seq`, then `steps` single tokens. `run(seq, inputs)` makes a step;
    yields (generation, results) after those that draw from a sequence's whole text."""
    gen = Generation(rng, cache, cfg.batch, cfg.seq, prompts, steps + 64)
    number = 0
    while any(gen.fed[b] < len(gen.text[b]) for b in range(cfg.batch)):
        out = run(cfg.seq, gen.step(cfg.seq), gen.uniform[number])
        number += 1
    for _ in range(steps):
        tokens = out[0]
        for b in range(cfg.batch):
            gen.text[b].append(int(tokens[b]))
        out = run(1, gen.step(1), gen.uniform[number])
        yield gen, gen.uniform[number], out
        number += 1


LLAMA = D.LlamaConfig(n_layer=2, dim=128, n_heads=8, n_kv_heads=2, ffn=256, batch=3, seq=4)
CACHE = D.PagedCache(pages=14, columns=4, page_size=3)
PROMPT_LENGTHS = (4, 1, 3)  # one piece each: padded to four places at the front


def with_seq(cfg, seq):
    return D.LlamaConfig(**{**cfg.__dict__, "seq": seq})


def cpu_generation(cfg, cache, lengths, steps, rank=0, tp=1, allreduce=None):
    w, wte, head = model(cfg)
    sw = D.shard_llama_weights(w, cfg, rank, tp)
    rng = np.random.default_rng(11)
    prompts = [rng.integers(0, VOCAB, n) for n in lengths]
    caches = [np.zeros(cache.shape(cfg, tp), np.float32) for _ in range(2 * cfg.n_layer)]
    weights = [I.to_np(t) for t in [wte] + D.flatten_llama_args(sw) + [head]]
    kept = {"caches": caches}

    def run(seq, inputs, uniform):
        plan = D.build_llama_decode_plan(with_seq(cfg, seq), cache, VOCAB, rank, tp)
        n = cfg.batch
        args = [np.zeros(n, np.int64), np.zeros(n, np.float32), np.zeros((n, VOCAB), np.float32), *inputs, uniform, *settings(n), *kept["caches"], *weights]
        out = DecodeRunner(plan, allreduce, rank, tp).run(args)
        kept["caches"] = out[13:13 + 2 * cfg.n_layer]
        return out[:3]

    return [([list(t) for t in gen.text], out) for gen, _, out in generate(cfg, cache, prompts, steps, rng, run)], (w, wte, head)


# -------------------------------------------------------------------------------------- CPU
def test_steps_through_the_cache_match_the_whole_forward():
    results, (w, wte, head) = cpu_generation(LLAMA, CACHE, PROMPT_LENGTHS, steps=4)
    for text, (tokens, logprobs, logits) in results:
        want = np.stack([reference_logits(LLAMA, w, wte, head, t) for t in text])
        assert_parity(logits, want, "bf16", n_layer=LLAMA.n_layer)
        assert tokens[0] == logits[0].argmax() and logprobs[0] == 0  # the greedy one


def test_two_ranks_draw_the_same_tokens():
    barrier, parts, outs = threading.Barrier(2, timeout=60), [None, None], [None, None]

    def worker(rank):
        def allreduce(x):
            parts[rank] = np.asarray(x, np.float64)
            barrier.wait()
            total = parts[0] + parts[1]
            barrier.wait()
            return total

        outs[rank] = cpu_generation(LLAMA, CACHE, PROMPT_LENGTHS, 3, rank, 2, allreduce)

    threads = [threading.Thread(target=worker, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    w, wte, head = outs[0][1]
    for (text, a), (_, b) in zip(outs[0][0], outs[1][0]):
        assert (a[0] == b[0]).all() and (a[2] == b[2]).all()
        want = np.stack([reference_logits(LLAMA, w, wte, head, t) for t in text])
        # sharded, each contracting product also rounds both ranks' partial sums and their total to bf16: 13
        # roundings along a layer where one rank has 9, which is what the bound grows with
        assert_parity(a[2], want, "bf16", n_layer=LLAMA.n_layer, roundings_per_layer=SHARDED_LAYER_ROUNDINGS)


def test_plan_as_the_library_gets_it():
    plan = D.build_llama_decode_plan(LLAMA, CACHE, VOCAB)
    sig, nargs, temps, ntemps, ops, nops = plan.to_native()
    assert nargs == len(plan.args) and nops == len(plan.ops)
    kinds = [ops[i].kind for i in range(nops)]
    assert kinds.count(N.OP_PAGED_APPEND) == kinds.count(N.OP_PAGED_ATTENTION) == LLAMA.n_layer and kinds[-1] == N.OP_SAMPLE
    at = kinds.index(N.OP_PAGED_APPEND)
    append, attention, sample = ops[at], ops[kinds.index(N.OP_PAGED_ATTENTION)], ops[nops - 1]
    assert append.f0 == LLAMA.theta and [append.operands[i].slot for i in range(3, 7)] == [13, 14, 4, 5]
    assert attention.f0 == pytest.approx(LLAMA.head_dim**-0.5) and [attention.operands[i].slot for i in range(2, 7)] == [13, 14, 6, 7, -1]
    assert [sample.operands[i].slot for i in range(8)] == [0, 1, 2, 8, 9, 10, 11, 12]
    assert sum(plan.ops[i].flops() for i in range(nops) if plan.ops[i].kind in ("paged_append", "sample")) == 0


def test_plan_refusals():
    with pytest.raises(ValueError, match="page"):
        D.build_llama_decode_plan(LLAMA, D.PagedCache(pages=0, columns=1), VOCAB)
    with pytest.raises(ValueError, match="vocabulary"):
        D.build_llama_decode_plan(LLAMA, CACHE, 0)
    with pytest.raises(ValueError, match="ways"):
        D.build_llama_decode_plan(LLAMA, CACHE, VOCAB, 0, 3)


def test_entry_points_without_a_context(native_lib):
    none = None
    assert native_lib.lh_b200_paged_append(none, none, none, none, none, none, none, none, 0.0) == -1
    assert native_lib.lh_b200_paged_attention(none, none, none, none, none, none, none, none, 1.0) == -1
    assert native_lib.lh_b200_paged_attention_workspace(none, none, none, none) == -1
    assert native_lib.lh_b200_sample(none, none, none, none, none, none, none, none, none) == -1


def test_binding_refuses_what_it_cannot_read(native_lib):
    call, sample, append = N.binding().call, N.address("lh_b200_sample"), N.address("lh_b200_paged_append")
    x = torch.zeros(2, 8)
    some = N.memref(256, (2, 8), (8, 1), N.LH_F32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        call(sample, None, 0, None, x, None, x, x, None, None, None, None)
    with pytest.raises(TypeError, match="not list"):
        call(sample, None, 0, None, [1], None, some, some, None, None, None, None)
    for wrong in ((sample, None, 0, None, some), (append, None, 0, 1.0, some), (append, None, 0, None) + (some,) * 7, (sample,)):
        with pytest.raises(TypeError, match="operands"):
            call(*wrong)
    with pytest.raises(TypeError):
        call(append, None, 0, "theta", *(some,) * 7)
    # read, passed on, and refused there: no context
    assert call(sample, None, 0, None, some, None, some, some, None, None, None, None) == -1
    assert call(append, None, 0, 0.5, None, *(some,) * 6) == -1


def test_oracle_of_bad_pages_and_lengths():
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 3, 2, 1, 4))
    q = rng.standard_normal((1, 1, 1, 4))
    whole, _, bad = DR.paged_attention(q, k, v, np.array([[2, 0]]), [4], 1.0)
    assert not bad
    # a page outside the pool: its keys are skipped, the others keep their weights
    got, _, bad = DR.paged_attention(q, k, v, np.array([[2, 9]]), [4], 1.0)
    want, _, _ = DR.paged_attention(q, k, v, np.array([[2, 0]]), [2], 1.0)
    assert bad and np.allclose(got, want)
    # lengths beyond the table, negative, none: clamped and reported; a row without keys is zero
    got, _, bad = DR.paged_attention(q, k, v, np.array([[2, 0]]), [99], 1.0)
    assert bad and np.array_equal(got, whole)
    for n, reported in ((-1, True), (0, False)):
        got, _, bad = DR.paged_attention(q, k, v, np.array([[2, 0]]), [n], 1.0)
        assert bad == reported and not got.any()
    _, kp, vp, bad = DR.paged_append(None, rng.standard_normal((2, 1, 4)), rng.standard_normal((2, 1, 4)), k, v, [-1, 6], None, 0.0)
    assert bad and np.array_equal(kp, k) and np.array_equal(vp, v)


def test_oracle_of_sampling_by_counting():
    """The draw as its definition says it: the first index whose running weight passes u."""
    x = np.log(np.array([1.0, 4.0, 0.0001, 2.0, 4.0]))
    total = 11.0001
    for u, want in ((0.0, 0), (0.5 / total, 0), (1.5 / total, 1), (5.5 / total, 3), (7.5 / total, 4), (1.0, 4)):
        assert DR.sample_row(x, u)[0] == want
    assert DR.sample_row(x, 0.99, top_k=2)[0] == 4 and DR.sample_row(x, 0.49, top_k=2)[0] == 1
    assert DR.sample_row(x, 0.99, top_p=4 / 11)[0] == 4  # 4 / 11 of 11.0001 is above 4: both of the equal ones
    assert DR.sample_row(x, 0.99, top_p=4 / 12)[0] == 1  # 3.66: the first of them is enough
    assert DR.sample_row(x, 0.0, min_p=0.5)[0] == 1 and DR.sample_row(x, 0.7, temperature=0.0) == (1, 0.0)
    assert DR.sample_row(np.full(3, -np.inf), 0.5) == (-1, -np.inf)
    assert DR.sample_row(np.array([np.nan, 0.0, np.inf]), 0.5)[0] == 2


# -------------------------------------------------------------------------------------- GPU
GPU_LLAMA = D.LlamaConfig(n_layer=2, dim=512, n_heads=8, n_kv_heads=2, ffn=512, batch=5, seq=24)


def gpu_sessions(ctx, cfg, cache, use_graph):
    from lighthouse_b200.workloads.session import PlanSession

    return {seq: PlanSession(D.build_llama_decode_plan(with_seq(cfg, seq), cache, VOCAB), ctx=ctx, use_graph=use_graph) for seq in (cfg.seq, 1)}


@pytest.mark.gpu
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("page_size,columns", [(16, 6), (5, 17)])
def test_generation(ctx, use_graph, page_size, columns):
    cfg, cache = GPU_LLAMA, D.PagedCache(pages=5 * columns + 2, columns=columns, page_size=page_size)
    w, wte, head = model(cfg, std=0.05)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, VOCAB, n) for n in (24, 1, 17, 9, 24)]
    sessions = gpu_sessions(ctx, cfg, cache, use_graph)
    n = cfg.batch
    weights = [t.cuda().contiguous() for t in [wte] + D.flatten_llama_args(D.shard_llama_weights(w, cfg)) + [head]]
    caches = D.llama_decode_caches(cfg, cache)
    tokens, logprobs, logits = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(n, VOCAB, device="cuda")
    table, lengths, uniform = torch.zeros(n, columns, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    sets = [torch.from_numpy(s).cuda() for s in settings(n)]
    fixed = {seq: [torch.zeros(n * seq, dtype=dt, device="cuda") for dt in (torch.int32, torch.int64, torch.int32)] for seq in (cfg.seq, 1)}
    fixed[1][0] = tokens  # what was drawn goes straight in again

    def run(seq, inputs, u):
        ids, slots, positions = fixed[seq]
        for dst, src in ((ids, inputs[0]), (slots, inputs[1]), (positions, inputs[2]), (table, inputs[3]), (lengths, inputs[4]), (uniform, u)):
            if dst is tokens:
                assert (tokens.cpu().numpy() == src).all()
            else:
                dst.copy_(torch.from_numpy(np.ascontiguousarray(src)))
        sessions[seq].run([tokens, logprobs, logits, ids, slots, positions, table, lengths, uniform, *sets, *caches, *weights], sync=True)
        return tokens.cpu().numpy().copy(), logprobs.cpu().numpy().copy(), logits.cpu().numpy().copy()

    for gen, u, (got, lp, z) in generate(cfg, cache, prompts, 6, rng, run):
        want = np.stack([reference_logits(cfg, w, wte, head, t) for t in gen.text])
        assert_parity(z, want, "bf16", n_layer=cfg.n_layer)
        drawn, drawn_lp = DR.sample(z, u, *settings(n))
        assert (got == drawn).all()
        # as for the operator alone: an f32 half step, weights that are multiples of 2^-42
        assert (np.abs(lp - drawn_lp) <= 2.0**-22 * np.maximum(1.0, np.abs(drawn_lp)) + 2.0**-42 * np.exp(np.minimum(-drawn_lp, 60.0))).all()
    for s in sessions.values():
        s.close()


def attention_plan(batch, hq, columns, page, workspace=0, side=False):
    p = Plan("cached", [ArgSpec((batch, hq, 1, 64), "bf16", "o"), ArgSpec((batch, hq, 1, 64), "bf16", "q"), ArgSpec((8, page, 1, 64), "bf16", "k"), ArgSpec((8, page, 1, 64), "bf16", "v"), ArgSpec((batch, columns), "i32", "table"), ArgSpec((batch,), "i32", "lengths")])
    if side:  # forked from the main stream and joined again
        p.event_record(0)
        p.stream(1)
        p.event_wait(0)
    p.paged_attention(*(p.arg(i) for i in range(6)), 0.125, p.temp((workspace,), "f32") if workspace else None)
    if side:
        p.event_record(1)
        p.stream(0)
        p.event_wait(1)
    return p


@pytest.mark.gpu
def test_graphs_that_share_the_contexts_scratch(own_stream_ctx):
    """Two captured plans without workspaces of their own, the later one needing more scratch than the first
    was captured with; their replays alternate."""
    from lighthouse_b200.workloads.session import PlanSession

    ctx, rng = own_stream_ctx, np.random.default_rng(2)
    made = []
    for batch, hq in ((2, 4), (3, 32)):
        tensors = [torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(torch.bfloat16).cuda() for s in ((batch, hq, 1, 64), (batch, hq, 1, 64), (8, 32, 1, 64), (8, 32, 1, 64))]
        table = torch.from_numpy(rng.integers(0, 8, (batch, 8)).astype(np.int32)).cuda()
        lengths = torch.from_numpy(rng.integers(1, 257, batch).astype(np.int32)).cuda()
        torch.cuda.synchronize()
        args = tensors + [table, lengths]
        session = PlanSession(attention_plan(batch, hq, 8, 32), ctx=ctx, use_graph=True)
        session.run(args, sync=True)
        made.append((session, args, args[0].clone()))
    for _ in range(3):
        for session, args, first in made:
            args[0].zero_()
            torch.cuda.synchronize()
            session.run(args, sync=True)
            assert torch.equal(args[0], first)
            want, spread, _ = DR.paged_attention(*(a.double().cpu().numpy() for a in args[1:4]), args[4].cpu().numpy(), args[5].cpu().numpy(), 0.125)
            # weights rounded to bf16 (2^-8 of each, so of the spread), the result again
            assert (np.abs(first.double().cpu().numpy() - want) <= 2.0**-8 * 1.05 * (spread + np.abs(want)) + 1e-6).all()
    for session, _, _ in made:
        session.close()


@pytest.mark.gpu
def test_plan_workspaces(ctx):
    from lighthouse_b200.workloads.session import PlanSession

    rng = np.random.default_rng(4)
    args = [torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(torch.bfloat16).cuda() for s in ((2, 4, 1, 64), (2, 4, 1, 64), (8, 16, 1, 64), (8, 16, 1, 64))]
    args += [torch.tensor([[1, 2, 3], [4, 0, 7]], dtype=torch.int32, device="cuda"), torch.tensor([40, 48], dtype=torch.int32, device="cuda")]
    outs = []
    need = ctx.paged_attention_workspace(args[1], args[2])
    for workspace, side in ((0, False), (-(-need // 4), False), (-(-need // 4), True)):
        with PlanSession(attention_plan(2, 4, 3, 16, workspace, side), ctx=ctx) as s:
            args[0].zero_()
            ctx.sync()
            s.run(args, sync=True)
            outs.append(args[0].clone())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and bool(outs[0].float().abs().sum() > 0)
    # the context's scratch belongs to its main stream
    with PlanSession(attention_plan(2, 4, 3, 16, 0, True), ctx=ctx) as s:
        with pytest.raises(ValueError, match="workspace"):
            s.run(args, sync=True)
    # too small a workspace is refused, and the context goes on working
    with PlanSession(attention_plan(2, 4, 3, 16, 64), ctx=ctx) as s:
        with pytest.raises(MemoryError, match="bytes"):
            s.run(args, sync=True)
    with PlanSession(attention_plan(2, 4, 3, 16), ctx=ctx) as s:
        s.run(args, sync=True)
    assert torch.equal(args[0], outs[0])
