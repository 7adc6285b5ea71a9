"""Cases of the operators of a decoding step, with their plain forms.

A sequence that is being answered keeps its keys and values in pages of a shared pool. One
step of it is: the projections' new rows are rotated to their positions and written into the
pages (``append``), the new tokens' queries attend over what the pages hold (``attention``),
and the next token is drawn from the last layer's logits (``sample``).

``run`` computes a case either with elementary torch operations (``own`` false) or with the
calls that a program using this repository makes (``own`` true).
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
THETA = 10000.0
LOG2_DRAW = {"rows": 8, "length": 17, "tokens": 14}  # draw(): the ranges' upper ends, as powers of two


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of one conversation enters the cache: the smallest call, pure latency
        dict(name="append 1 token", op="append", dtype="bf16", cache="bf16", tokens=1, q_heads=32, kv_heads=8, head_dim=128, page=16, slots=4096, far=False, skip=False),
        # a serving step of 256 sequences far into their contexts
        dict(name="append 256 tokens far", op="append", dtype="bf16", cache="bf16", tokens=256, q_heads=32, kv_heads=8, head_dim=128, page=16, slots=65536, far=True, skip=False),
        # prompts of different lengths, padded to one batch of 12289 rows; f32 activations kept as f16
        dict(name="append 12289 tokens", op="append", dtype="f32", cache="f16", tokens=12289, q_heads=32, kv_heads=8, head_dim=128, page=64, slots=65536, far=False, skip=True),
        # the first answer tokens of one short conversation
        dict(name="attention 1x129", op="attention", dtype="bf16", batch=1, tokens=1, q_heads=32, kv_heads=8, head_dim=128, page=16, length=129, layout="token", idle=False),
        # one long document: 131071 keys, an odd length, split over the whole GPU
        dict(name="attention 1x131071", op="attention", dtype="bf16", batch=1, tokens=1, q_heads=32, kv_heads=8, head_dim=128, page=16, length=131071, layout="token", idle=False),
        # ordinary serving: 64 sequences of 133 to 8192 keys
        dict(name="attention 64x8192", op="attention", dtype="bf16", batch=64, tokens=1, q_heads=32, kv_heads=8, head_dim=128, page=16, length=8192, layout="token", idle=False),
        # nanoGPT's heads (12 of 64, no sharing), a full block of 1024, some rows of the batch idle
        dict(name="attention 250x1024 f16", op="attention", dtype="f16", batch=250, tokens=1, q_heads=12, kv_heads=12, head_dim=64, page=32, length=1024, layout="head", idle=True),
        # four proposed tokens of each of 16 sequences are scored at once
        dict(name="attention 16x4 tokens", op="attention", dtype="bf16", batch=16, tokens=4, q_heads=32, kv_heads=8, head_dim=128, page=64, length=4001, layout="head", idle=False),
        # f32 throughout
        dict(name="attention 8x4096 f32", op="attention", dtype="f32", batch=8, tokens=1, q_heads=16, kv_heads=4, head_dim=128, page=16, length=4096, layout="token", idle=False),
        # one conversation's next token, nanoGPT's vocabulary, every filter on
        dict(name="sample 1x50304", op="sample", dtype="f32", rows=1, vocab=50304, filters="all"),
        # a batch whose rows ask for different things (some greedy, some unfiltered)
        dict(name="sample 64x131071 bf16", op="sample", dtype="bf16", rows=64, vocab=131071, filters="mixed"),
        # the largest batch, the most used filter alone
        dict(name="sample 256x131071", op="sample", dtype="f32", rows=256, vocab=131071, filters="top_p"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(2 ** rng.uniform(math.log2(low), math.log2(high))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "sample"])
    heads = rng.choice([(32, 8, 128), (16, 4, 128), (12, 12, 64), (32, 32, 128), (16, 1, 64), (8, 2, 80), (24, 8, 96), (14, 2, 256), (40, 2, 128)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    page = rng.choice([1, 8, 16, 16, 17, 32, 64, 128])
    if op == "append":
        tokens = _log(rng, 1, 2 ** LOG2_DRAW["tokens"])
        slots = -(-max(4096, tokens + tokens // 2) // page) * page
        return dict(op=op, dtype=dtype, cache=rng.choice(["bf16", "bf16", "f16", "f32"]), tokens=tokens, q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2],
                    page=page, slots=slots, far=rng.random() < 0.5, skip=rng.random() < 0.5)
    if op == "attention":
        batch, length = _log(rng, 1, 2 ** LOG2_DRAW["rows"]), _log(rng, 1, 2 ** LOG2_DRAW["length"])
        row = heads[1] * heads[2] * BYTES[dtype]
        length = max(1, min(length, (1 << 29) // (batch * row)))  # no more keys than the largest listed case holds
        return dict(op=op, dtype=dtype, batch=batch, tokens=rng.choice([1, 1, 1, 2, 5]), q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2], page=page,
                    length=length, layout=rng.choice(["token", "head"]), idle=rng.random() < 0.3)
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, 2 ** LOG2_DRAW["rows"]), vocab=_log(rng, 100, 131072), filters=rng.choice(["all", "mixed", "top_p", "top_k", "min_p", "none", "greedy"]))


def lengths_of(case):
    """Keys that each sequence of an attention case holds: spread over (0, length] by the golden ratio; an idle row holds none."""
    n, top = case["batch"], case["length"]
    if n == 1:
        return [top]
    got = [max(1, math.ceil(top * (((b + 1) * 0.6180339887498949) % 1.0))) for b in range(n)]
    got[0] = top
    return [0 if case["idle"] and b % 7 == 5 else v for b, v in enumerate(got)]


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.default_rng(seed)
    randn = lambda *shape, dtype: torch.randn(*shape, device="cuda", generator=g, dtype=dtype)  # noqa: E731
    s = dict(case=case)
    if case["op"] == "append":
        t, hq, hkv, d, page = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
        pages, dt = case["slots"] // page, DTYPES[case["dtype"]]
        qkv = randn(t, hq + 2 * hkv, d, dtype=dt)  # the fused projection's rows: q, k and v are column blocks of it
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["k_pages"], s["v_pages"] = (randn(pages, page, hkv, d, dtype=DTYPES[case["cache"]]) for _ in range(2))
        slots = host.permutation(pages * page)[:t]
        if case["skip"]:
            slots = np.where(np.arange(t) % 5 == 3, -1, slots)  # padding rows of the batch
        s["slots"] = torch.tensor(slots, dtype=torch.int32, device="cuda")
        s["positions"] = torch.tensor(host.integers(0, 1000000 if case["far"] else 8192, t), dtype=torch.int32, device="cuda")
    elif case["op"] == "attention":
        b, t, hq, hkv, d, page = case["batch"], case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
        dt, lengths = DTYPES[case["dtype"]], lengths_of(case)
        used = [-(-n // page) for n in lengths]
        pages = max(1, sum(used))
        shape = (pages, page, hkv, d) if case["layout"] == "token" else (pages, hkv, page, d)
        s["k_pages"], s["v_pages"] = randn(*shape, dtype=dt), randn(*shape, dtype=dt)
        if case["layout"] == "head":
            s["k_pages"], s["v_pages"] = s["k_pages"].permute(0, 2, 1, 3), s["v_pages"].permute(0, 2, 1, 3)
        order, table, at = host.permutation(pages), np.zeros((b, max(1, max(used))), dtype=np.int32), 0
        for i, n in enumerate(used):
            table[i, :n] = order[at:at + n]
            at += n
        s["page_table"] = torch.tensor(table, device="cuda")
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = randn(b, t, hq, d, dtype=dt).transpose(1, 2)  # rows as the projection leaves them, seen as (B, H, S, D)
        s["o"] = torch.empty(b, t, hq, d, dtype=dt, device="cuda").transpose(1, 2)
        s["scale"] = 1.0 / math.sqrt(d)
    else:
        n, v = case["rows"], case["vocab"]
        s["logits"] = (randn(n, v, dtype=torch.float32) * 2.5).to(DTYPES[case["dtype"]])
        s["uniform"] = torch.rand(n, device="cuda", generator=g)
        put = lambda a, dt: torch.tensor(a, dtype=dt, device="cuda")  # noqa: E731
        temperature, k, p, m = host.uniform(0.6, 1.2, n), host.integers(1, 200, n), host.uniform(0.5, 0.99, n), host.uniform(0.01, 0.2, n)
        f = case["filters"]
        if f == "mixed":  # a row may be greedy, or leave any of the filters off
            temperature = np.where(host.random(n) < 0.2, 0.0, temperature)
            k, p, m = np.where(host.random(n) < 0.5, 0, k), np.where(host.random(n) < 0.5, 1.0, p), np.where(host.random(n) < 0.5, 0.0, m)
        if f == "greedy":
            temperature = np.zeros(n)
        s["temperature"] = put(temperature, torch.float32)
        s["top_k"] = put(k, torch.int32) if f in ("all", "mixed", "top_k") else None
        s["top_p"] = put(p, torch.float32) if f in ("all", "mixed", "top_p") else None
        s["min_p"] = put(m, torch.float32) if f in ("all", "mixed", "min_p") else None
        s["tokens"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(n, dtype=torch.float32, device="cuda")
    return s


# ------------------------------------------------------------------------------------- one pass
_contexts = {}


def _context():
    """The framework's handle on the current device, made once as a program does."""
    device = torch.cuda.current_device()
    if device not in _contexts:
        from lighthouse_b200.context import CudaContext

        _contexts[device] = CudaContext(device, use_torch_stream=True)
    return _contexts[device]


def run(state):
    return {"append": _append, "attention": _attention, "sample": _sample}[state["case"]["op"]](state)


def _append(s):
    """q <- rot(q, position); pages[slot] <- rot(k, position), v. A negative slot is padding: nothing of it is kept."""
    if own:
        _context().paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], s["positions"], theta=THETA)
    else:
        d = s["q"].shape[-1]
        freq = THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        angle = s["positions"].double()[:, None, None] * freq
        cos, sin = angle.cos().float(), angle.sin().float()

        def rotate(x):
            a, b = x[..., 0::2].float(), x[..., 1::2].float()
            return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).reshape(x.shape)

        s["q"].copy_(rotate(s["q"]))
        kept = s["slots"] >= 0
        at = s["slots"][kept].long()
        page = s["k_pages"].shape[1]
        s["k_pages"][at // page, at % page] = rotate(s["k"])[kept].to(s["k_pages"].dtype)
        s["v_pages"][at // page, at % page] = s["v"][kept].to(s["v_pages"].dtype)
    return {"q": s["q"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attention(s):
    """softmax(scale q k^T) v over the keys that a sequence's pages hold; token t of n sees the first length - n + t + 1 keys; zeros where it sees none."""
    if own:
        _context().paged_attention(s["o"], s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["scale"])
        return s["o"]
    q, table, lengths = s["q"].float(), s["page_table"].long(), s["lengths"]
    b, hq, t, d = q.shape
    page, hkv = s["k_pages"].shape[1:3]
    j = torch.arange(table.shape[1] * page, device="cuda")
    k, v = (x[table[:, j // page], j % page].permute(0, 2, 1, 3).float() for x in (s["k_pages"], s["v_pages"]))
    q = q.reshape(b, hkv, (hq // hkv) * t, d)
    scores = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(b, hkv, hq // hkv, t, -1)
    seen = j < (lengths[:, None] - t + 1 + torch.arange(t, device="cuda"))[..., None]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0.0, top)).exp_()
    p = (p / p.sum(-1, keepdim=True).clamp_min(1e-30)).view(b, hkv, -1, j.numel())
    s["o"].copy_((p @ v).view(b, hq, t, d))
    return s["o"]


def _sample(s):
    """Draws one token a row: weights exp((x - max) / temperature) of the tokens that top-k, then top-p, then min-p leave; the first, in index order, whose
    running sum passes uniform times the total. A temperature of zero takes the first largest."""
    if own:
        _context().sample(s["tokens"], s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], logprobs=s["logprobs"])
        return s["tokens"], s["logprobs"]
    x = s["logits"].double()
    n, v = x.shape
    greedy = s["temperature"] <= 0
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = ((x - x[:, :1]) / torch.where(greedy, 1.0, s["temperature"]).double()[:, None]).exp_()
    rank = torch.arange(v, device="cuda")
    kept = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        kept &= rank < torch.where(s["top_k"] > 0, s["top_k"], v)[:, None]
    if s["top_p"] is not None:
        mass = torch.where(kept, w, 0.0)
        before = mass.cumsum(1) - mass
        off = (s["top_p"] >= 1)[:, None]
        kept &= off | (before < s["top_p"].double()[:, None] * mass.sum(1, keepdim=True)) | (rank == 0)
    if s["min_p"] is not None:
        kept &= (w >= s["min_p"].double()[:, None]) | (x == x[:, :1])
    kept &= ~greedy[:, None] | (rank == 0)
    mass = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))  # back in index order
    run_ = mass.cumsum(1)
    total = run_[:, -1:]
    hit = (run_ > s["uniform"].double()[:, None] * total) & (mass > 0)
    s["tokens"].copy_(hit.to(torch.uint8).argmax(1))
    s["logprobs"].copy_((mass.gather(1, s["tokens"].long()[:, None]) / total).log()[:, 0])
    return s["tokens"], s["logprobs"]


# ------------------------------------------------------------------------------------- work and 64-bit values
def work(case):
    if case["op"] == "append":
        t, row, size = case["tokens"], case["kv_heads"] * case["head_dim"], BYTES[case["dtype"]]
        kept = t - (t + 1) // 5 if case["skip"] else t  # every fifth row, from the fourth on, is padding
        moved = 2 * t * case["q_heads"] * case["head_dim"] * size + 2 * kept * row * (size + BYTES[case["cache"]]) + 8 * t
        return {"bytes": moved, "flops": 3 * (t * case["q_heads"] * case["head_dim"] + kept * row)}
    if case["op"] == "attention":
        keys, rows = sum(lengths_of(case)), case["batch"] * case["tokens"]
        size, d = BYTES[case["dtype"]], case["head_dim"]
        moved = 2 * keys * case["kv_heads"] * d * size + 2 * rows * case["q_heads"] * d * size + 4 * sum(-(-n // case["page"]) for n in lengths_of(case)) + 4 * case["batch"]
        return {"bytes": moved, "flops": 4 * keys * case["tokens"] * case["q_heads"] * d}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * BYTES[case["dtype"]] + 28 * case["rows"], "flops": 3 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        d, page = case["head_dim"], case["page"]
        pair = torch.arange(d // 2, device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), s["positions"].double()[:, None] * torch.exp(-2.0 * pair / d * math.log(THETA)))

        def rotated(x):
            z = torch.view_as_complex(x.double().reshape(x.shape[0], x.shape[1], d // 2, 2).contiguous())
            return torch.view_as_real(z * turn[:, None]).reshape(x.shape)

        k_pages, v_pages, rows = s["k_pages"].double().reshape(-1, case["kv_heads"], d), s["v_pages"].double().reshape(-1, case["kv_heads"], d), torch.nonzero(s["slots"] >= 0)[:, 0]
        at = s["slots"][rows].long()
        k_pages.index_copy_(0, at, rotated(s["k"])[rows])
        v_pages.index_copy_(0, at, s["v"].double()[rows])
        shape = (-1, page, case["kv_heads"], d)
        return {"q": rotated(s["q"]), "k_pages": k_pages.view(shape), "v_pages": v_pages.view(shape)}
    if case["op"] == "attention":
        out = torch.zeros(s["o"].shape, dtype=torch.float64, device="cuda")
        group, page = case["q_heads"] // case["kv_heads"], case["page"]
        for b, n in enumerate(lengths_of(case)):
            ids = s["page_table"][b, : -(-n // page)].long()
            k, v = (x[ids].reshape(-1, case["kv_heads"], case["head_dim"])[:n].double().transpose(0, 1).repeat_interleave(group, 0) for x in (s["k_pages"], s["v_pages"]))
            for t in range(case["tokens"]):
                m = n - case["tokens"] + t + 1
                if m > 0:
                    z = torch.bmm(k[:, :m], s["q"][b, :, t].double()[..., None])[..., 0] * s["scale"]
                    out[b, :, t] = torch.bmm(torch.softmax(z, -1)[:, None], v[:, :m])[:, 0]
        return out
    n, v = case["rows"], case["vocab"]
    tokens, logprobs = torch.zeros(n, dtype=torch.int64), torch.zeros(n, dtype=torch.float64)
    setting = lambda key, off: [off] * n if s[key] is None else s[key].cpu().tolist()  # noqa: E731
    for r, (tau, k, p, m, u) in enumerate(zip(setting("temperature", 1.0), setting("top_k", 0), setting("top_p", 1.0), setting("min_p", 0.0), s["uniform"].cpu().tolist())):
        x = s["logits"][r].double().cpu().numpy()
        if tau <= 0:
            tokens[r] = int(np.flatnonzero(x == x.max())[0])
            continue
        e = np.exp((x - x.max()) / tau)
        ids = np.lexsort((np.arange(v), -x))[: k if 0 < k < v else v]
        if p < 1:
            c = np.cumsum(e[ids])
            ids = ids[: max(1, int(np.searchsorted(c, p * c[-1], side="left")) + 1)]
        ids = np.sort(ids[(e[ids] >= m) | (x[ids] == x.max())])
        c = np.cumsum(e[ids])
        hit = ids[min(int(np.searchsorted(c, u * c[-1], side="right")), len(ids) - 1)]
        tokens[r], logprobs[r] = int(hit), math.log(e[hit] / c[-1])
    return tokens.to(torch.int32), logprobs
