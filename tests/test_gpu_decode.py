"""The operators of a decoding step on the GPU, through ``CudaContext``, against 64-bit numpy
(``oracle/decode_ops.py``). Tolerances are derived where they are used."""

import numpy as np
import pytest
import torch

from oracle import decode_ops as R

from lighthouse_b200 import _native as N

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}
TINY = {"f32": 0.0, "bf16": 0.0, "f16": 2.0**-25}  # half a step among f16's subnormals


def host(t):
    return t.detach().double().cpu().numpy()


def randn(rng, *shape, dtype="f32"):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(TYPES[dtype]).cuda()


# ------------------------------------------------------------------------------------ append
def check_append(ctx, rng, q, k, v, k_pages, v_pages, slots, positions, theta, cache):
    dt = {v_: k_ for k_, v_ in TYPES.items()}[k.dtype]
    q0 = None if q is None else host(q)
    k0, kp0, vp0 = host(k), host(k_pages), host(v_pages)
    want_q, want_k, want_v, _ = R.paged_append(q0, k0, host(v), kp0, vp0, slots.cpu().numpy(), None if positions is None else positions.cpu().numpy(), theta)
    ctx.paged_append(q, k, v, k_pages, v_pages, slots, positions, theta=theta)
    ctx.sync()

    def close(got, want, dtype, size):
        # sine and cosine are off by at most 2^-22 each (angle reduced to f32 in [-pi, pi]: 2^-23 of
        # pi at most, the functions' own 2 units), two f32 products and a sum by 3 half steps: with
        # |x|, |y| <= size that is below 2 * size * (2^-21.3 + 3 * 2^-24) < size * 2^-19.5; then one rounding
        bound = (HALF_STEP[dtype] * np.abs(want) + TINY[dtype]) * 1.0001 + (size * 2.0**-19.5 if theta else 0.0)
        assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())

    size = max(1.0, float(np.abs(k0).max()), 0.0 if q0 is None else float(np.abs(q0).max()))
    if q is not None:
        close(host(q), want_q, dt, size)
    for got, want, before in ((host(k_pages), want_k, kp0), (host(v_pages), want_v, vp0)):
        same = want == before
        assert (got[same & (got != before)].size) == 0  # rows that no slot names stay as they were
        close(got, want, cache, size)


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("tokens,hq,hkv,d,page", [(1, 32, 8, 128, 16), (7, 12, 12, 64, 1), (129, 4, 1, 80, 17), (1500, 3, 3, 10, 5), (40, 2, 2, 256, 64)])
def test_append(ctx, dtype, cache, tokens, hq, hkv, d, page):
    rng = np.random.default_rng(tokens * 7 + d)
    pages = -(-(tokens + 9) // page)
    qkv = randn(rng, tokens, hq + 2 * hkv, d, dtype=dtype)
    kp, vp = randn(rng, pages, page, hkv, d, dtype=cache), randn(rng, pages, page, hkv, d, dtype=cache)
    slots = rng.permutation(pages * page)[:tokens]
    slots = np.where(rng.random(tokens) < 0.2, -1 - slots, slots)  # any negative slot is padding
    positions = rng.integers(0, 2_000_000, tokens)
    check_append(ctx, rng, qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], kp, vp, torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor(positions, dtype=torch.int64).cuda(), 10000.0, cache)


def test_append_without_rotation_strides_and_no_query(ctx):
    rng = np.random.default_rng(5)
    # odd head size, rows at odd offsets, (pages, Hkv, page, D) pools, strided slots
    for d, dtype, cache in ((7, "bf16", "f16"), (64, "f16", "f16"), (64, "bf16", "bf16")):
        buf = randn(rng, 33, 5 * d + 3, dtype=dtype)
        k, v = (buf[:, 1 + i * 2 * d:1 + (i + 1) * 2 * d].unflatten(1, (2, d)) for i in range(2))
        kp, vp = (randn(rng, 11, 2, 4, d, dtype=cache).permute(0, 2, 1, 3) for _ in range(2))
        slots = torch.tensor(rng.permutation(44)[:33], dtype=torch.int64).cuda()
        slots = torch.stack([slots, slots * 0], dim=1)[:, 0]
        check_append(ctx, rng, None, k, v, kp, vp, slots, None, 0.0, cache)
    q = randn(rng, 33, 3, 8)
    before = q.clone()
    k = randn(rng, 33, 2, 8)
    kp, vp = randn(rng, 44, 1, 2, 8), randn(rng, 44, 1, 2, 8)
    ctx.paged_append(q, k, k, kp, vp, torch.arange(33, device="cuda"), theta=0.0)
    ctx.sync()
    assert torch.equal(q, before) and torch.equal(kp[:33, 0], k) and torch.equal(vp[:33, 0], k)
    ctx.paged_append(None, k[:0], k[:0], kp, vp, torch.arange(0, device="cuda"), theta=0.0)  # no token
    ctx.sync()


def test_append_slot_outside_the_pool(ctx):
    rng = np.random.default_rng(6)
    k, kp, vp = randn(rng, 3, 2, 8), randn(rng, 4, 4, 2, 8), randn(rng, 4, 4, 2, 8)
    want_k, want_v = kp.clone(), vp.clone()
    slots = torch.tensor([5, 16, 2**31 - 1], dtype=torch.int32).cuda()
    want_k[1, 1], want_v[1, 1] = k[0], k[0]
    ctx.paged_append(None, k, k, kp, vp, slots, theta=0.0)
    with pytest.raises(N.LighthouseCudaError, match="outside its table"):
        ctx.sync()
    ctx.sync()  # reported once; the context stays usable
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


# --------------------------------------------------------------------------------- attention
def cache_of(rng, lengths, page, hkv, d, dtype, layout="token", spare=3):
    """Pages in random order; rows that no sequence owns hold NaN, so that reading one shows."""
    used = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(used) + spare
    order = rng.permutation(pages)
    table = np.full((len(lengths), max(1, max(used))), -7, np.int32)  # columns past the last page are not read
    k, v = rng.standard_normal((2, pages, page, hkv, d)).astype(np.float32)
    owned = np.zeros((pages, page), bool)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        for j in range(n):
            owned[order[at + j], : min(page, lengths[b] - j * page)] = True
        at += n
    k[~owned], v[~owned] = np.nan, np.nan
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a if layout == "token" else a.transpose(0, 2, 1, 3))).to(TYPES[dtype]).cuda()
    k, v = put(k), put(v)
    if layout == "head":
        k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    return k, v, table


def check_attention(ctx, o, q, k, v, table, lengths, scale, workspace=None, dtype=None):
    o.fill_(float("nan"))
    ctx.paged_attention(o, q, k, v, torch.as_tensor(table, dtype=torch.int32, device="cuda") if isinstance(table, np.ndarray) else table,
                        torch.as_tensor(np.asarray(lengths), dtype=torch.int32, device="cuda") if not torch.is_tensor(lengths) else lengths, scale, workspace=workspace)
    ctx.sync()
    compare_attention(o, q, k, v, table, lengths, scale)


def compare_attention(o, q, k, v, table, lengths, scale):
    dt = {v_: k_ for k_, v_ in TYPES.items()}[q.dtype]
    ot = {v_: k_ for k_, v_ in TYPES.items()}[o.dtype]
    to_np = lambda a: a.cpu().numpy() if torch.is_tensor(a) else np.asarray(a)
    want, spread, _ = R.paged_attention(host(q), np.nan_to_num(host(k)), np.nan_to_num(host(v)), to_np(table), to_np(lengths), scale)
    # A score is a sum of D products in f32: off by (D + 2) half steps of sum |q k| scale, itself at
    # most |q|_1 max|k| scale; weights are off by twice that (numerator and sum) and exp2's 2^-22.
    # 16-bit types round P once (half a step of p |v|); f32 sums of n terms in pieces below 2^-24 * (n / 4 + 64).
    n = max(1, int(to_np(lengths).max()))
    size = np.abs(host(q)).sum(-1, keepdims=True) * float(np.nanmax(np.abs(host(k)))) * abs(scale)
    rel = 2 * ((q.shape[-1] + 2) * 2.0**-24 * size + 2.0**-22) + 2.0**-24 * (n / 4 + 64)
    bound = spread * (rel + (HALF_STEP[dt] + TINY[dt] * n if dt != "f32" else 0.0)) + HALF_STEP[ot] * np.abs(want) * 1.01 + TINY[ot] + 1e-30
    off = np.abs(host(o) - want)
    assert np.isfinite(host(o)).all()
    assert (off <= bound).all(), (float((off / bound).max()), np.unravel_index(np.argmax(off / bound), off.shape))


HEADS = [(32, 8, 128), (12, 12, 64), (4, 1, 80), (14, 2, 256), (20, 1, 128), (3, 3, 96), (5, 5, 7)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("page,layout", [(16, "token"), (1, "head"), (17, "head"), (64, "token")])
def test_attention_heads_pages_types(ctx, dtype, hq, hkv, d, page, layout):
    rng = np.random.default_rng(hq * 100 + d + page)
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 130, 257]
    k, v, table = cache_of(rng, lengths, page, hkv, d, dtype, layout)
    q = randn(rng, len(lengths), hq, 1, d, dtype=dtype)
    check_attention(ctx, torch.empty_like(q), q, k, v, table, lengths, d**-0.5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [2, 4, 9])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (3, 3, 64), (2, 1, 40), (6, 1, 256)])
def test_attention_several_tokens(ctx, dtype, tokens, hq, hkv, d):
    """Token s of S sees length - S + s + 1 keys: sequences shorter than S leave rows with none."""
    rng = np.random.default_rng(tokens + d)
    lengths = [0, 1, 3, tokens, tokens + 1, 33, 64, 70, 200]
    k, v, table = cache_of(rng, lengths, 16, hkv, d, dtype)
    q = randn(rng, len(lengths), tokens, hq, d, dtype=dtype).transpose(1, 2)
    check_attention(ctx, torch.empty(len(lengths), tokens, hq, d, dtype=TYPES[dtype], device="cuda").transpose(1, 2), q, k, v, table, lengths, 0.3)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("batch,hq,hkv,d,top", [(1, 8, 2, 128, 20011), (1, 1, 1, 64, 70001), (3, 4, 1, 128, 9000), (40, 16, 2, 64, 1500), (600, 2, 1, 64, 90)])
def test_attention_long_and_ragged(ctx, dtype, batch, hq, hkv, d, top):
    """Units cut over many CTAs, CTAs with many units, batches wider than a block."""
    rng = np.random.default_rng(top)
    lengths = [top] + [int(n) for n in rng.integers(0, top, batch - 1)]
    k, v, table = cache_of(rng, lengths, 16, hkv, d, dtype)
    q = randn(rng, batch, hq, 1, d, dtype=dtype)
    check_attention(ctx, torch.empty_like(q), q, k, v, table, lengths, d**-0.5)


def test_attention_strides_and_alignment(ctx):
    rng = np.random.default_rng(11)
    lengths = [40, 7, 100]
    for dtype, d, lead in (("bf16", 64, 1), ("bf16", 64, 4), ("f16", 68, 2), ("f32", 64, 1), ("f32", 66, 2), ("bf16", 36, 8)):
        k0, v0, table = cache_of(rng, lengths, 8, 2, d, dtype)
        k, v = (torch.zeros(*t.shape[:3], d + 2 * lead, dtype=t.dtype, device="cuda")[..., lead:lead + d].copy_(t) for t in (k0, v0))  # rows at offsets that no vector load allows
        q = torch.zeros(3, 4, 1, d + 1, dtype=TYPES[dtype], device="cuda")[..., 1:].copy_(randn(rng, 3, 4, 1, d, dtype=dtype))
        o = torch.zeros(3, 4, 1, d + 3, dtype=TYPES[dtype], device="cuda")[..., 2:2 + d]
        wide = torch.full((3, 2 * table.shape[1] + 1), -1, dtype=torch.int32, device="cuda")
        wide[:, 1::2] = torch.from_numpy(table).cuda()
        lens = torch.tensor([[n, -9] for n in lengths], dtype=torch.int32, device="cuda")[:, 0]
        check_attention(ctx, o, q, k, v, wide[:, 1::2], lens, 0.2)


def test_attention_shared_prefix_other_output_type_and_repeats(ctx):
    rng = np.random.default_rng(12)
    k, v, table = cache_of(rng, [300, 280], 16, 2, 128, "bf16")
    table[1, :10] = table[0, :10]  # both sequences read the same first pages
    q = randn(rng, 2, 8, 1, 128, dtype="bf16")
    o = torch.empty(2, 8, 1, 128, device="cuda")
    check_attention(ctx, o, q, k, v, table, [300, 280], 0.09)
    first = o.clone()
    for _ in range(3):
        ctx.paged_attention(o, q, k, v, torch.from_numpy(table).cuda(), torch.tensor([300, 280], dtype=torch.int32).cuda(), 0.09)
    ctx.sync()
    assert torch.equal(o, first)  # the order of every sum is fixed


def test_attention_large_scores_and_equal_keys(ctx):
    """Scores of +-1000 (one key takes all the weight) and keys that are all alike (equal weights)."""
    rng = np.random.default_rng(13)
    for dtype in ("bf16", "f32"):
        k, v, table = cache_of(rng, [500, 64], 16, 1, 64, dtype)
        q = randn(rng, 2, 4, 1, 64, dtype=dtype)
        check_attention(ctx, torch.empty_like(q), q, k, v, table, [500, 64], 0.0)
        k2 = torch.where(torch.isnan(k), k, torch.round(k.float() * 4).to(k.dtype))  # whole numbers: products and sums are exact
        q2 = torch.round(q.float() * 8).to(q.dtype)
        check_attention(ctx, torch.empty_like(q), q2, k2, v, table, [500, 64], 4.0)


def test_attention_nan_stays_with_the_rows_that_see_it(ctx):
    rng = np.random.default_rng(14)
    for dtype in ("bf16", "f16", "f32"):
        k, v, table = cache_of(rng, [60, 61], 16, 1, 64, dtype)
        q = randn(rng, 2, 3, 3, 64, dtype=dtype)
        q[1, 1, 2] = float("nan")
        k[table[0, 59 // 16], 59 % 16] = float("inf")
        v[table[0, 59 // 16], 59 % 16] = float("nan")  # the newest key: only the last token sees it
        o = torch.empty_like(q)
        ctx.paged_attention(o, q, k, v, torch.from_numpy(table).cuda(), torch.tensor([60, 61], dtype=torch.int32).cuda(), 0.125)
        ctx.sync()
        assert torch.isnan(o[0, :, 2]).all() and torch.isfinite(o[0, :, :2]).all()
        assert torch.isnan(o[1, 1, 2]).all() and torch.isfinite(o[1, 0]).all() and torch.isfinite(o[1, 2]).all() and torch.isfinite(o[1, 1, :2]).all()
        k[table[0, 59 // 16], 59 % 16] = 0.0
        v[table[0, 59 // 16], 59 % 16] = 0.0
        compare_attention(o[:1, :, :2], q[:1, :, :2], k, v, table[:1], [59], 0.125)


def test_attention_indices_outside_their_tables(ctx):
    rng = np.random.default_rng(15)
    for dtype in ("bf16", "f32"):
        lengths = [100, 90, 33]
        k, v, table = cache_of(rng, lengths, 16, 2, 64, dtype)
        table[0, 1], table[1, 0], table[2, 2] = k.shape[0], -1, 2**31 - 1
        q = randn(rng, 3, 4, 1, 64, dtype=dtype)
        o = torch.empty_like(q)
        with pytest.raises(N.LighthouseCudaError, match="outside its table"):
            check_attention(ctx, o, q, k, v, table, lengths, 0.125)
        ctx.sync()
        compare_attention(o, q, k, v, table, lengths, 0.125)  # the other pages' keys are attended to
        k, v, table = cache_of(rng, [32, 20, 32], 16, 2, 64, dtype)
        for lens in ([33, 20, 2**31 - 1], [-5, 20, -(2**31)]):
            with pytest.raises(N.LighthouseCudaError, match="outside its table"):
                check_attention(ctx, o, q, k, v, table, lens, 0.125)
            compare_attention(o, q, k, v, table, lens, 0.125)


def test_attention_offsets_past_32_bits(ctx):
    """A pool of 2.2 G elements: pages whose offsets do not fit 32 bits, and page numbers scaled by a large stride."""
    rng = np.random.default_rng(16)
    pages, page, hkv, d = 8400, 256, 8, 128
    pool = torch.empty(pages, page, hkv, d, dtype=torch.bfloat16, device="cuda")
    assert pool.numel() > 2**31
    table = np.array([[8399, 3, 8390], [8397, 8398, 5]], np.int32)
    for pg in table.ravel():
        pool[int(pg)] = randn(rng, page, hkv, d, dtype="bf16")
    q = randn(rng, 2, 16, 1, d, dtype="bf16")
    o = torch.empty_like(q)
    lengths = [700, 513]
    ctx.paged_attention(o, q, pool, pool, torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), 0.09)
    ids = np.unique(table)
    small = pool[torch.from_numpy(ids).cuda().long()]
    ctx.sync()
    compare_attention(o, q, small, small, np.searchsorted(ids, table).astype(np.int32), lengths, 0.09)
    k = randn(rng, 2, hkv, d, dtype="bf16")
    ctx.paged_append(None, k, k, pool, pool, torch.tensor([8399 * 256 + 255, 7 * 256], dtype=torch.int32).cuda(), theta=0.0)
    ctx.sync()
    assert torch.equal(pool[8399, 255], k[0]) and torch.equal(pool[7, 0], k[1])


def test_attention_refusals(ctx):
    q = torch.zeros(2, 4, 1, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(3, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(o=q.clone(), q=q, k_pages=k, v_pages=k, page_table=table, lengths=lens, scale=1.0)
    for change in (dict(o=q[:1]), dict(q=q[..., :32]), dict(k_pages=k.float()), dict(v_pages=k[:2]), dict(page_table=table[:1]), dict(lengths=lens.long()), dict(page_table=table.long()),
                   dict(q=torch.zeros(2, 3, 1, 64, device="cuda", dtype=torch.bfloat16), o=torch.zeros(2, 3, 1, 64, device="cuda", dtype=torch.bfloat16)),
                   dict(q=q.transpose(1, 3), o=q.transpose(1, 3)), dict(o=q[:, :1].expand(2, 4, 1, 64)), dict(k_pages=k[:, :0], v_pages=k[:, :0]), dict(lengths=lens.cpu()),
                   dict(q=q[0], o=q[0]), dict(workspace=torch.empty(1 << 25, dtype=torch.uint8, device="cuda")[1:]),
                   dict(q=torch.zeros(2, 4, 1, 300, device="cuda"), o=torch.zeros(2, 4, 1, 300, device="cuda"), k_pages=torch.zeros(3, 16, 2, 300, device="cuda"), v_pages=torch.zeros(3, 16, 2, 300, device="cuda"))):
        with pytest.raises(ValueError):
            ctx.paged_attention(**{**good, **change})
    with pytest.raises(MemoryError, match="workspace"):
        ctx.paged_attention(**good, workspace=torch.empty(1024, dtype=torch.uint8, device="cuda"))
    ctx.paged_attention(**good)  # both sequences empty: zeros
    ctx.paged_attention(q[:0], q[:0], k, k, table[:0], lens[:0], 1.0)
    ctx.sync()
    assert not good["o"].any()


def test_append_refusals(ctx):
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    pages, at = torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32, device="cuda")
    good = dict(q=k.clone(), k=k, v=k, k_pages=pages, v_pages=pages.clone(), slots=at, positions=at)
    for change in (dict(q=k[:2]), dict(q=k.float()), dict(v=k[..., :32]), dict(k_pages=pages[..., :32]), dict(v_pages=pages.float()), dict(slots=at[:2]), dict(slots=at.float()),
                   dict(positions=None), dict(theta=-1.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(q=k[:, :1].expand(3, 2, 64)), dict(k_pages=pages[:1].expand(4, 16, 2, 64)),
                   dict(slots=at.cpu()), dict(k=k[0]), dict(v_pages=pages[:3])):
        with pytest.raises(ValueError):
            ctx.paged_append(**{**good, **change})
    odd = torch.zeros(3, 2, 7, device="cuda")
    with pytest.raises(ValueError):
        ctx.paged_append(None, odd, odd, torch.zeros(4, 16, 2, 7, device="cuda"), torch.zeros(4, 16, 2, 7, device="cuda"), at, at)


# ---------------------------------------------------------------------------------- sampling
def check_sample(ctx, logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, tokens_dtype=torch.int32):
    n = logits.shape[0]
    put = lambda a, dt: None if a is None else torch.as_tensor(np.asarray(a)).to(dt).cuda()
    temperature, top_p, min_p, uniform = (put(a, torch.float32) for a in (temperature, top_p, min_p, uniform))
    top_k = put(top_k, torch.int32)
    tokens = torch.full((n,), -99, dtype=tokens_dtype, device="cuda")
    logprobs = torch.full((n,), float("nan"), device="cuda")
    ctx.sample(tokens, logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, logprobs=logprobs)
    ctx.sync()
    np_of = lambda t: None if t is None else t.cpu().numpy()
    want, want_lp = R.sample(host(logits), np_of(uniform), np_of(temperature), np_of(top_k), np_of(top_p), np_of(min_p))
    got = tokens.cpu().numpy()
    assert (got == want).all(), [(int(r), int(got[r]), int(want[r])) for r in np.flatnonzero(got != want)[:5]]
    # f32's half step, and weights that are whole multiples of 2^-42: below 2^-22 for tokens above 2^-21
    finite = np.isfinite(want_lp)
    lp = logprobs.double().cpu().numpy()
    assert (lp[~finite] == want_lp[~finite]).all()
    assert (np.abs(lp - want_lp)[finite] <= 2.0**-22 * np.maximum(1.0, np.abs(want_lp[finite])) + 2.0**-42 * np.exp(np.minimum(-want_lp[finite], 60.0))).all()
    return got


FILTERS = {
    "none": {}, "top_k": dict(top_k=40), "top_p": dict(top_p=0.9), "min_p": dict(min_p=0.05), "all": dict(top_k=50, top_p=0.95, min_p=0.02),
    "top_k 1": dict(top_k=1), "top_k 2": dict(top_k=2), "top_p small": dict(top_p=0.01), "top_p near 1": dict(top_p=0.9999), "min_p 1": dict(min_p=1.0), "off": dict(top_k=0, top_p=1.0, min_p=0.0),
    "top_k wide": dict(top_k=3000), "top_k and top_p": dict(top_k=500, top_p=0.6),
}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("filters", list(FILTERS))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (5, 1000), (4, 50304), (2, 131071)])
def test_sample(ctx, dtype, filters, rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    logits = (randn(rng, rows, vocab) * 2.5).to(TYPES[dtype])
    f = {k: [v] * rows for k, v in FILTERS[filters].items()}
    check_sample(ctx, logits, rng.random(rows, dtype=np.float32), temperature=rng.uniform(0.3, 2.0, rows), **f)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_ties_and_flat_rows(ctx, dtype):
    """Rows of few different values: the borders of top-k and top-p fall inside runs of equal logits."""
    rng = np.random.default_rng(3)
    for vocab in (33, 1024, 5000, 100001):
        logits = torch.from_numpy(rng.integers(0, 4, (24, vocab)).astype(np.float32)).to(TYPES[dtype]).cuda()
        logits[0] = 1.5  # all alike
        logits[1] = -0.0
        logits[1, ::2] = 0.0
        k, p = rng.integers(1, vocab, 24), rng.uniform(0.05, 0.999, 24)
        k[:4], p[:4] = vocab // 2, 0.5
        u = rng.random(24, dtype=np.float32)
        check_sample(ctx, logits, u, top_k=k)
        check_sample(ctx, logits, u, top_p=p)
        check_sample(ctx, logits, u, top_k=k, top_p=p, min_p=p / 50)


def test_sample_edges(ctx):
    rng = np.random.default_rng(4)
    inf, nan = float("inf"), float("nan")
    x = randn(rng, 16, 300)
    x[0] = -inf
    x[1] = nan
    x[2, 5:] = -inf
    x[3, 100] = inf
    x[4, 7], x[4, 200] = inf, inf
    x[5, ::3] = nan
    x[6] = -inf
    x[6, 299] = -1e30
    x[7] *= 1e30
    x[8] = torch.finfo(torch.float32).min
    x[8, 17] = 0
    x[9] = torch.finfo(torch.float32).min  # a mask's lowest value everywhere: equal weights
    u = rng.random(16, dtype=np.float32)
    u[10], u[11], u[12], u[13] = 0.0, 1.0, nan, -3.0
    u[14], u[15] = np.float32(1.0) - np.float32(2.0**-24), 7.0
    for f in ({}, dict(top_k=[20] * 16), dict(top_p=[0.8] * 16), dict(min_p=[0.3] * 16), dict(top_k=[9] * 16, top_p=[0.7] * 16, min_p=[0.1] * 16)):
        check_sample(ctx, x, u, **f)
        check_sample(ctx, x, u, temperature=[0.0] * 16, **f)
    t = np.array([1, 1, 1e-30, 1, 1, 1, 1, 1e30, 1e-3, inf, nan, -1, 0, inf, 1e-45, 3], np.float32)
    check_sample(ctx, x, u, temperature=t, tokens_dtype=torch.int64)
    check_sample(ctx, x, u, temperature=t, top_k=[-1, 0, 1, 2, 3, 299, 300, 301, 2**31 - 1, 5, 5, 5, 5, 5, 5, 5], top_p=[0.5, nan, inf, -1, 0, 2, 1, 1e-30] * 2, min_p=[nan, -1, 0, 2, inf, 1e-30, 0.5, 1] * 2)


def test_sample_strides_and_without_logprobs(ctx):
    rng = np.random.default_rng(8)
    wide = randn(rng, 6, 1001)
    logits = wide[:, 1:1000]
    check_sample(ctx, logits, rng.random(6, dtype=np.float32), top_k=[30] * 6, top_p=[0.9] * 6)
    tokens = torch.zeros(6, 3, dtype=torch.int64, device="cuda")
    u = torch.rand(6, 2, device="cuda")
    ctx.sample(tokens[:, 1], logits[::2].repeat(2, 1), u[:, 1])
    ctx.sync()
    want, _ = R.sample(host(logits[::2].repeat(2, 1)), u[:, 1].cpu().numpy())
    assert (tokens[:, 1].cpu().numpy() == want).all() and not tokens[:, ::2].any()
    ctx.sample(tokens[:0, 0], logits[:0], u[:0, 0])
    one = torch.zeros(6, dtype=torch.int32, device="cuda")
    ctx.sample(one, logits[:1].expand(6, 999), u[:, 0], temperature=torch.ones(1, device="cuda").expand(6))  # six draws of one row
    ctx.sync()
    want, _ = R.sample(host(logits[:1].expand(6, 999)), u[:, 0].cpu().numpy())
    assert (one.cpu().numpy() == want).all()


def test_sample_frequencies(ctx):
    """Evenly spread random numbers draw every token in proportion to its weight: each count is within
    one of n * p (the running sum's two borders), and one more for numbers rounded to f32."""
    w = np.array([1, 2, 3, 4, 0, 6], np.float64)
    with np.errstate(divide="ignore"):
        x = torch.from_numpy(np.log(w).astype(np.float32)).cuda().expand(1600, 6)
    u = torch.from_numpy(((np.arange(1600) + 0.5) / 1600).astype(np.float32)).cuda()
    tokens = torch.empty(1600, dtype=torch.int32, device="cuda")
    ctx.sample(tokens, x, u)
    ctx.sync()
    counts = np.bincount(tokens.cpu().numpy(), minlength=6)
    assert (np.abs(counts - 1600 * w / w.sum()) <= 2).all()


def test_sample_refusals(ctx):
    x, t, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
    for tokens, logits, uniform, more in ((t[:2], x, u, {}), (t.float(), x, u, {}), (t, x[0], u, {}), (t, x.double(), u, {}), (t, x.t(), u, {}), (t, x, u.double(), {}), (t, x, u, dict(top_k=u)),
                                          (t, x, u, dict(top_p=u[:2])), (t, x, u, dict(temperature=t)), (t[:1].expand(3), x, u, {}), (t, x[:, :0], u, {}), (t, x, u, dict(logprobs=u[:1].expand(3))),
                                          (t, torch.zeros(1, 1, device="cuda").expand(3, (1 << 20) + 1), u, {}), (t.cpu(), x, u, {})):
        with pytest.raises(ValueError):
            ctx.sample(tokens, logits, uniform, **more)


@pytest.mark.parametrize("vocab", [200000, 400000, (1 << 20) - 3, 1 << 20])
def test_sample_wide_rows(ctx, vocab):
    """Rows that do not fit the cluster's shared memory at two CTAs an SM, and rows that do not fit it at all."""
    rng = np.random.default_rng(vocab)
    logits = randn(rng, 3, vocab) * 2.5
    logits[1] = torch.round(logits[1])
    u = rng.random(3, dtype=np.float32)
    check_sample(ctx, logits, u, top_k=[70, 100000, vocab - 1], top_p=[0.9, 0.7, 0.99])
    check_sample(ctx, logits, u, top_p=[0.9, 0.7, 0.99])
    check_sample(ctx, logits, u)


# ------------------------------------------------------------------ streams, graphs, workspaces
def test_captured_calls_follow_the_lengths_and_do_not_share_workspaces(native_lib):
    """Two graphs of the same context replayed beside one another, while the sequences grow between replays."""
    from lighthouse_b200.context import CudaContext

    rng = np.random.default_rng(21)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), CudaContext(0, use_torch_stream=True) as c:
        sets = []
        for top in (3000, 2500):
            k, v, table = cache_of(rng, [top, top // 2, top], 16, 2, 64, "bf16")
            lens = torch.tensor([5, 0, 17], dtype=torch.int32).cuda()
            q = randn(rng, 3, 8, 1, 64, dtype="bf16")
            o = torch.empty_like(q)
            tab = torch.from_numpy(table).cuda()
            c.paged_attention(o, q, k, v, tab, lens, 0.125)  # warm: an eager workspace exists
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                c.paged_attention(o, q, k, v, tab, lens, 0.125)
            sets.append((g, o, q, k, v, table, lens, top))
        other = torch.cuda.Stream()
        for step in range(4):
            for g, o, q, k, v, table, lens, top in sets:
                lens.copy_(torch.tensor([top * step // 3, top * step // 6, min(top, 17 + 900 * step)], dtype=torch.int32))
                o.fill_(float("nan"))
            torch.cuda.synchronize()
            for _ in range(5):
                sets[0][0].replay()
                with torch.cuda.stream(other):
                    sets[1][0].replay()
            torch.cuda.synchronize()
            for g, o, q, k, v, table, lens, top in sets:
                compare_attention(o, q, k, v, table, lens, 0.125)


def test_calls_on_another_stream_and_with_a_workspace_of_ones_own(native_lib, own_stream_ctx):
    rng = np.random.default_rng(22)
    c = own_stream_ctx  # launches on its own stream, not torch's
    k, v, table = cache_of(rng, [700, 900], 16, 2, 128, "f16")
    q = randn(rng, 2, 4, 1, 128, dtype="f16")
    tab, lens = torch.from_numpy(table).cuda(), torch.tensor([700, 900], dtype=torch.int32).cuda()
    o = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    c.paged_attention(o, q, k, v, tab, lens, 0.1)
    c.sync()
    compare_attention(o, q, k, v, table, [700, 900], 0.1)
    n = c.paged_attention_workspace(q, k)
    ws = torch.full((n + 512,), 0xFF, dtype=torch.uint8, device="cuda")  # whatever it holds before
    o.fill_(float("nan"))
    torch.cuda.synchronize()
    c.paged_attention(o, q, k, v, tab, lens, 0.1, workspace=ws[256:256 + n])
    c.sync()
    compare_attention(o, q, k, v, table, [700, 900], 0.1)
    assert (ws[:256] == 0xFF).all() and (ws[256 + n:] == 0xFF).all()


def test_sample_and_append_in_a_graph(native_lib):
    from lighthouse_b200.context import CudaContext

    rng = np.random.default_rng(23)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), CudaContext(0, use_torch_stream=True) as c:
        x, u, t = randn(rng, 5, 40000) * 3, torch.zeros(5, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
        p = torch.full((5,), 0.9, device="cuda")
        k = randn(rng, 5, 2, 64, dtype="bf16")
        kp, vp = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
        slots = torch.zeros(5, dtype=torch.int32, device="cuda")
        c.sample(t, x, u, top_p=p)
        c.paged_append(None, k, k, kp, vp, slots - 1, theta=0.0)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            c.sample(t, x, u, top_p=p)
            c.paged_append(None, k, k, kp, vp, slots, theta=0.0)
        for step in range(3):
            un = rng.random(5, dtype=np.float32)
            sn = rng.permutation(64)[:5].astype(np.int32)
            u.copy_(torch.from_numpy(un))
            slots.copy_(torch.from_numpy(sn))
            g.replay()
            stream.synchronize()
            want, _ = R.sample(host(x), un, top_p=[np.float32(0.9)] * 5)
            assert (t.cpu().numpy() == want).all()
            assert torch.equal(kp.view(64, 2, 64)[torch.from_numpy(sn).cuda().long()], k)


def test_a_kept_workspace_is_not_memory_that_another_stream_has_yet_to_write(own_stream_ctx):
    c = own_stream_ctx
    q = torch.zeros(1, 4, 1, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.ones(2, 16, 1, 64, device="cuda", dtype=torch.bfloat16)
    tab, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1,), 16, dtype=torch.int32, device="cuda")
    o = torch.empty_like(q)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    freed = torch.empty(c.paged_attention_workspace(q, k), dtype=torch.uint8, device="cuda")
    at = freed.data_ptr()
    del freed  # torch's current stream may have it again at once, the context's may not
    c.paged_attention(o, q, k, k, tab, lens, 0.1)
    c.sync()
    assert c._workspaces_held[-1].data_ptr() != at
    assert (o == 1).all()


def test_operands_off_their_types_boundaries_and_a_closed_context(native_lib, own_stream_ctx):
    c = own_stream_ctx
    raw = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")

    def odd(code, *shape):
        strides = N.contiguous_strides(shape)
        return N.memref(raw.data_ptr() + 1, shape, strides, code)

    q = torch.zeros(1, 2, 1, 8, device="cuda")
    k = torch.zeros(1, 16, 2, 8, device="cuda")
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = dict(o=q.clone(), q=q, k_pages=k, v_pages=k, page_table=i[None], lengths=i, scale=1.0)
    for name, bad in (("o", odd(N.LH_F32, 1, 2, 1, 8)), ("q", odd(N.LH_F32, 1, 2, 1, 8)), ("k_pages", odd(N.LH_F32, 1, 16, 2, 8)), ("v_pages", odd(N.LH_F32, 1, 16, 2, 8)), ("page_table", odd(N.LH_I32, 1, 1)), ("lengths", odd(N.LH_I32, 1))):
        with pytest.raises(ValueError, match="aligned"):
            c.paged_attention(**{**good, name: bad})
    good = dict(q=None, k=q[0, :, 0][None], v=q[0, :, 0][None], k_pages=k, v_pages=k.clone(), slots=i, positions=i)
    for name, bad in (("k", odd(N.LH_F32, 1, 2, 8)), ("v_pages", odd(N.LH_F32, 1, 16, 2, 8)), ("slots", odd(N.LH_I64, 1)), ("positions", odd(N.LH_I32, 1))):
        with pytest.raises(ValueError, match="aligned"):
            c.paged_append(**{**good, name: bad})
    x, u = torch.zeros(1, 10, device="cuda"), torch.zeros(1, device="cuda")
    for bad in (dict(tokens=odd(N.LH_I32, 1)), dict(logits=odd(N.LH_F32, 1, 10)), dict(uniform=odd(N.LH_F32, 1)), dict(top_k=odd(N.LH_I32, 1)), dict(logprobs=odd(N.LH_F32, 1))):
        with pytest.raises(ValueError, match="aligned"):
            c.sample(**{**dict(tokens=i, logits=x, uniform=u), **bad})
    from lighthouse_b200.context import CudaContext

    closed = CudaContext(0)
    closed.close()
    with pytest.raises(ValueError, match="closed"):
        closed.sample(i, x, u)
    with pytest.raises(ValueError, match="closed"):
        closed.paged_append(None, q[0], q[0], k, k, i, i)
    with pytest.raises(ValueError, match="closed"):
        closed.paged_attention(q, q, k, k, i[None], i, 1.0)


def test_the_result_may_take_the_querys_place(ctx):
    """o and q one tensor: a unit's rows of q are read by the warps of that unit alone, and written after."""
    rng = np.random.default_rng(31)
    lengths = [5, 700, 0, 4000, 33]
    k, v, table = cache_of(rng, lengths, 16, 2, 64, "bf16")
    q = randn(rng, 5, 16, 2, 64, dtype="bf16")
    tab, lens = torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    apart, both = torch.empty_like(q), q.clone()
    ctx.paged_attention(apart, q, k, v, tab, lens, 0.125)
    for _ in range(3):
        both.copy_(q)
        ctx.paged_attention(both, both, k, v, tab, lens, 0.125)
        ctx.sync()
        assert torch.equal(both, apart)


@pytest.mark.parametrize("dtype,d", [("bf16", 8), ("f16", 16), ("bf16", 24), ("bf16", 136), ("f16", 200), ("bf16", 248), ("f32", 4), ("f32", 1), ("f32", 252)])
@pytest.mark.parametrize("page", [16, 48])
def test_attention_smallest_and_odd_head_sizes(ctx, dtype, d, page):
    rng = np.random.default_rng(d + page)
    lengths = [1, 47, 48, 49, 300]
    k, v, table = cache_of(rng, lengths, page, 2, d, dtype)
    q = randn(rng, 5, 6, 1, d, dtype=dtype)
    check_attention(ctx, torch.empty_like(q), q, k, v, table, lengths, d**-0.5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens,hq,hkv,d", [(200, 8, 2, 64), (3, 100, 1, 128), (1, 64, 1, 64), (70, 2, 2, 256), (1, 33, 1, 40)])
def test_attention_many_rows_to_a_kv_head(ctx, dtype, tokens, hq, hkv, d):
    """A piece of a prompt, or many heads on one: units of more rows than one pass takes."""
    rng = np.random.default_rng(tokens + hq)
    lengths = [tokens, tokens + 130, max(1, tokens - 5), 0]
    k, v, table = cache_of(rng, lengths, 16, hkv, d, dtype)
    q = randn(rng, 4, hq, tokens, d, dtype=dtype)
    check_attention(ctx, torch.empty_like(q), q, k, v, table, lengths, d**-0.5)


def test_attention_thousands_of_sequences(ctx):
    rng = np.random.default_rng(8)
    lengths = rng.integers(0, 20, 5000).tolist()
    k, v, table = cache_of(rng, lengths, 8, 1, 32, "bf16")
    q = randn(rng, 5000, 2, 1, 32, dtype="bf16")
    check_attention(ctx, torch.empty_like(q), q, k, v, table, lengths, 0.2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_over_an_empty_pool_or_table(ctx, dtype):
    """Nothing to read: lengths of zero give zeros, others are reported and give zeros."""
    q = torch.ones(2, 4, 1, 64, dtype=TYPES[dtype], device="cuda")
    some, none = torch.ones(3, 16, 2, 64, dtype=TYPES[dtype], device="cuda"), torch.ones(0, 16, 2, 64, dtype=TYPES[dtype], device="cuda")
    columns = lambda n: torch.zeros(2, n, dtype=torch.int32, device="cuda")
    for pool, table in ((some, columns(0)), (none, columns(2)), (none, columns(0))):
        for lengths, bad in (([0, 0], False), ([5, 0], True)):
            o = torch.full_like(q, 7.0)
            ctx.paged_attention(o, q, pool, pool, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0.125)
            if bad:
                with pytest.raises(N.LighthouseCudaError, match="outside its table"):
                    ctx.sync()
            else:
                ctx.sync()
            assert not o.any()
    k = torch.ones(2, 2, 64, dtype=TYPES[dtype], device="cuda")
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    ctx.paged_append(None, k, k, none, none, at - 1, at)  # all padding
    ctx.sync()
    ctx.paged_append(None, k, k, none, none, at, at)
    with pytest.raises(N.LighthouseCudaError, match="outside its table"):
        ctx.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_top_p_borders_among_many_equal_logits(ctx, dtype):
    """More candidates than the lead ranks, with and without top-k before; borders at their first and last."""
    rng = np.random.default_rng(6)
    rows, vocab = 9, 30000
    x = torch.full((rows, vocab), -3.0, dtype=TYPES[dtype], device="cuda")
    x[:, ::7] = 1.0
    x[:, 5] = 2.0
    p = np.array([1e-6, 1e-4, 0.05, 0.3, 0.7, 0.95, 0.9999, 0.99999, 1.0], np.float32)
    for temperature in (0.5, 1.0, 4.0):
        for more in ({}, dict(top_k=[20000] * rows), dict(top_k=[2000] * rows), dict(min_p=[0.1] * rows)):
            check_sample(ctx, x, rng.random(rows, dtype=np.float32), temperature=[temperature] * rows, top_p=p, **more)


def test_on_torchs_default_stream(native_lib):
    """A context made where nobody chose a stream: the legacy default one, workspace included."""
    from lighthouse_b200.context import CudaContext

    rng = np.random.default_rng(41)
    k, v, table = cache_of(rng, [100, 300], 16, 2, 64, "bf16")
    q = randn(rng, 2, 4, 1, 64, dtype="bf16")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.default_stream()), CudaContext(0, use_torch_stream=True) as c:
        o = torch.empty_like(q)
        for _ in range(2):
            check_attention(c, o, q, k, v, table, [100, 300], 0.125)
        check_sample(c, randn(rng, 3, 1000), rng.random(3, dtype=np.float32), top_p=[0.9] * 3)
        torch.cuda.synchronize()
