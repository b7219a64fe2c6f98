"""GPU: rows of the fused QKV projection into the paged KV cache
(dmoe_kv_append_device) against the definition in 64 bits (kv_ref.py).

Bars: the norm and the rotation run in binary64 and are rounded once, so a query
is off by half an f32 step (2^-24 relative, plus 1e-12 of the row's largest
value for the 64-bit arithmetic), a cached F16 value by half a step of F16
(2^-11, 2^-25 below the normal range) beyond that, an E4M3 code by half a step
of E4M3 (2^-4, 2^-10 of the block's scale below its normal range).  Exponents
are exact, and every byte that the rows do not own stays as it was."""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu

BASE, EPS = 3e6, 1e-6


def _rows(rng, batch, nh, nkv, hd, scale=1.0):
    return (rng.standard_normal((batch.n_tokens, (nh + 2 * nkv) * hd)) * scale).astype(np.float32)


def _run(ctx, batch, cache, qkv, nh, rd, qk, gains, stream=None):
    import dmoe
    dev = "cuda:0"
    kv, b = cache.device(dmoe), batch.device(dmoe)
    ap = dmoe.attn_hparams(nh, cache.nkv, cache.hd, rd, 0, BASE, EPS, qk)
    q = torch.full((batch.n_tokens, nh, cache.hd), 7.0, device=dev)
    g = [None if x is None else torch.from_numpy(x).to(dev) for x in gains]
    x = torch.from_numpy(qkv).to(dev)
    torch.cuda.synchronize()
    ctx.kv_append_device(kv, b, ap, x, q, *g, stream=stream)
    torch.cuda.synchronize()
    return q.cpu().numpy(), R.Cache.of(kv)


def _check(batch, before, after, q, qkv, nh, rd, gains):
    nkv, hd, T = before.nkv, before.hd, batch.T
    rq, rk, rv, pos = R.rows_of(batch, qkv, nh, nkv, hd, rd, BASE, EPS, *gains)
    live = pos >= 0
    with np.errstate(invalid="ignore"):
        fine = np.isfinite(rq)
        top = np.where(fine, np.abs(rq), 0).max(-1, keepdims=True, initial=0)
        off = np.abs(q - rq) - 2.0 ** -24 * np.abs(rq) - 1e-12 * top
    assert (off[live] <= 0)[fine[live]].all() and not np.isfinite(q[live][~fine[live]]).any()
    assert (q[~live] == 7.0).all()
    want = before.copy()            # every byte that the rows do not own
    for which, rows in (("k", rk), ("v", rv)):
        old, new = before.codes(which), after.codes(which)
        expect = old.clone()
        rows32 = rows.astype(np.float32)
        for s, (o, n) in enumerate(batch.seqs):
            for p in range(o, o + n):
                at = batch.place(s, p)
                if at is None:
                    continue
                pg, t = at
                row = batch.q_start[s] + p - o
                start = p // 32 * 32
                if p == max(o, start) and before.f8:        # the first row here of this block
                    m = min(start + 32, o + n) - p
                    exps = getattr(before, which + "_exp")
                    for h in range(nkv):
                        x = np.abs(rows32[row:row + m, h])
                        e = R.exponent(float(x[np.isfinite(x)].max(initial=0)))
                        e0 = int(exps[pg, h, t // 32])
                        if p > start:
                            e = max(e, e0)
                            if e > e0:
                                lo = t // 32 * 32
                                kept = old[pg, h, lo:t].float() * 2.0 ** (e0 - e)
                                expect[pg, h, lo:t] = kept.to(R.F8)
                        getattr(want, which + "_exp")[pg, h, t // 32] = e
                for h in range(nkv):
                    got, ref = new[pg, h, t], rows[row, h]
                    expect[pg, h, t] = got
                    with np.errstate(invalid="ignore", over="ignore"):
                        if before.f8:
                            unit = 2.0 ** int(getattr(want, which + "_exp")[pg, h, t // 32])
                            ok = np.isfinite(ref) & (np.abs(rows32[row, h]) <= R.TOP * unit)
                            err = np.abs(got.double().numpy() * unit - ref)
                            assert (err <= 2.0 ** -4 * np.abs(ref) * (1 + 2.0 ** -12) + 2.0 ** -10 * unit)[ok].all()
                            assert np.isnan(got.double().numpy()[~ok]).all()
                        else:
                            assert torch.equal(torch.isnan(got), torch.from_numpy(np.isnan(rows32[row, h])))
                            err = np.abs(got.double().numpy() - ref)
                            ok = np.abs(ref) < 65504
                            assert (err <= 2.0 ** -11 * np.abs(ref) * (1 + 2.0 ** -12) + 2.0 ** -25)[ok].all()
                            assert not np.isfinite(got.double().numpy()[np.abs(ref) > 65536]).any()
        a, b = expect.contiguous().view(torch.uint8), new.contiguous().view(torch.uint8)
        if before.f8:               # a NaN may carry either sign
            nan = lambda x: (x & 0x7f) == 0x7f  # noqa: E731
            assert torch.equal(nan(a), nan(b)) and torch.equal(a[~nan(a)], b[~nan(b)])
            assert torch.equal(getattr(want, which + "_exp"), getattr(after, which + "_exp"))
        else:
            assert torch.equal(a, b)


GROUPS = {
    "one": [(0, 1)], "first_block": [(0, 32)], "tail": [(31, 1)], "past": [(32, 1)], "inside": [(5, 3)],
    "across": [(30, 5)], "long": [(17, 300)],
    "ragged": [(5, 3), (0, 0), (31, 1), (32, 40), (700, 1), (64, 32), (0, 1), (63, 70), (96, 9), (33, 0), (40, 17)],
    "singles": [(i * 7, 1) for i in range(70)],
    "many": [(i * 37 % 700, i % 6) for i in range(150)], "rows": [(i % 50, 40) for i in range(70)],
}
SHAPES = [  # n_head, n_head_kv, head_dim, rotary_dim, qk_norm, page_tokens
    (32, 4, 128, 64, True, 64), (5, 1, 64, 64, True, 32), (6, 3, 64, 20, False, 96), (3, 3, 128, 128, True, 256),
    (2, 1, 128, 6, False, 32), (4, 2, 128, 0, True, 64), (4, 2, 64, 0, False, 32), (2, 2, 128, 96, True, 32)]


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("group", GROUPS)
def test_append_groups(ctx, kvtype, group):
    nh, nkv, hd, rd, qk, T = SHAPES[0]
    _one(ctx, kvtype, group, nh, nkv, hd, rd, qk, T)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("shape", SHAPES[1:], ids=str)
def test_append_shapes(ctx, kvtype, shape):
    _one(ctx, kvtype, "ragged", *shape)


def _one(ctx, kvtype, group, nh, nkv, hd, rd, qk, T, scale=1.0, extra=3):
    print(f"case: append {kvtype} {group} {nh}/{nkv} d{hd} r{rd} page {T}", flush=True)
    rng = np.random.default_rng(len(group) + hd + rd)
    batch = R.Batch(GROUPS[group], T, seed=1, extra=extra)
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=2)
    qkv = _rows(rng, batch, nh, nkv, hd, scale)
    gains = [rng.uniform(0.5, 1.5, hd).astype(np.float32) if qk else None for _ in range(2)]
    q, after = _run(ctx, batch, cache, qkv, nh, rd, qk, gains)
    _check(batch, cache, after, q, qkv, nh, rd, gains)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_append_thousands(ctx, kvtype):
    """More sequences than one look of 64 times 64 finds, half of them with a row."""
    GROUPS["thousands"] = [(i * 7 % 60, (i * 5 + i // 64) % 2) for i in range(4300)]
    try:
        _one(ctx, kvtype, "thousands", 2, 1, 64, 32, False, 32)
    finally:
        del GROUPS["thousands"]


@pytest.mark.parametrize("scale", [1e-30, 1e-14, 1e-3, 3e3, 1e16, 1e30])
def test_append_magnitudes(ctx, scale):
    """E4M3 exponents grow over kept tokens, and end at -50 and 50: what is
    smaller rounds to zero, what is larger becomes NaN."""
    _one(ctx, "e4m3", "ragged", 4, 2, 64, 32, False, 32, scale)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_append_values_that_are_not_finite(ctx, kvtype):
    """NaN, infinities and magnitudes past the type's: they stay where they are,
    the block's other values keep their scale.  Without a rotation, so that each
    is one element."""
    nh, nkv, hd, T = 4, 2, 64, 32
    print(f"case: append {kvtype}, values that are not finite", flush=True)
    batch = R.Batch(GROUPS["ragged"], T, seed=3)
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=4)
    rng = np.random.default_rng(5)
    qkv = _rows(rng, batch, nh, nkv, hd)
    for i, x in enumerate([np.nan, np.inf, -np.inf, 0.0, -0.0, 7e4, 1e-38]):
        qkv[i::9, 11 * i + 1::97] = x
    qkv[20] = 0.0                                       # a row of zeros
    q, after = _run(ctx, batch, cache, qkv, nh, 0, False, (None, None))
    _check(batch, cache, after, q, qkv, nh, 0, (None, None))


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_append_pages_that_are_none(ctx, kvtype):
    """Entries outside the cache, a table that ends early, sequences whose
    numbers contradict each other: their tokens are skipped, the queries of
    rows with a position are formed all the same."""
    import dmoe
    nh, nkv, hd, T = 4, 2, 64, 32
    print(f"case: append {kvtype}, bad pages", flush=True)
    batch = R.Batch([(20, 80), (0, 40), (64, 33), (10, 4)], T, seed=6)
    batch.pages[0, 1], batch.pages[1, 0], batch.pages[2, 2] = -1, batch.n_pages, 2 ** 31 - 1
    batch.pages = np.ascontiguousarray(batch.pages[:, :3])      # sequences 0 and 2 go on past it
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=7)
    qkv = _rows(np.random.default_rng(8), batch, nh, nkv, hd)
    q, after = _run(ctx, batch, cache, qkv, nh, 32, False, (None, None))
    _check(batch, cache, after, q, qkv, nh, 32, (None, None))
    # contradictions: fewer cached tokens than rows; rows past the buffers
    batch.kv_len[0] = 79
    batch.q_start[4] = batch.n_tokens + 1
    kv, b = cache.device(dmoe), batch.device(dmoe)
    ap = dmoe.attn_hparams(nh, nkv, hd, 32, 0, BASE, EPS)
    q2 = torch.full((batch.n_tokens, nh, hd), 7.0, device="cuda:0")
    ctx.kv_append_device(kv, b, ap, torch.from_numpy(qkv).cuda(), q2)
    torch.cuda.synchronize()
    q2 = q2.cpu().numpy()
    assert (q2[:80] == 7.0).all() and (q2[153:] == 7.0).all() and np.array_equal(q2[80:153], q[80:153])


def test_append_far_positions(ctx):
    """Angles of positions around a million, and a page longer than that."""
    nh, nkv, hd, T = 2, 1, 64, 1 << 20
    print("case: append at position 1,048,543", flush=True)
    batch = R.Batch([((1 << 20) - 33, 33), (3, 2)], T, seed=9, spare=0)
    cache = R.Cache("e4m3", batch.n_pages, nkv, hd, T, seed=10)
    qkv = _rows(np.random.default_rng(11), batch, nh, nkv, hd)
    q, after = _run(ctx, batch, cache, qkv, nh, 64, False, (None, None))
    _check(batch, cache, after, q, qkv, nh, 64, (None, None))


def test_append_again_and_back(ctx):
    """A denoising step writes its block again: the same bytes as the first time.
    A sequence cut back to a position inside a block and continued there keeps
    the tokens before it."""
    import dmoe
    nh, nkv, hd, T = 4, 2, 128, 64
    print("case: append again, append after cutting back", flush=True)
    rng = np.random.default_rng(12)
    cache = R.Cache("e4m3", 6, nkv, hd, T, poison=True)
    kv = cache.device(dmoe)
    ap = dmoe.attn_hparams(nh, nkv, hd, 64, 32, BASE, EPS)
    pages = torch.tensor([[4, 1, 3]], dtype=torch.int32, device="cuda:0")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda:0")  # noqa: E731

    def put(old, n, seed):
        x = torch.from_numpy(np.random.default_rng(seed).standard_normal((n, 8 * hd)).astype(np.float32)).cuda()
        q = torch.empty((n, nh, hd), device="cuda:0")
        ctx.kv_append_device(kv, dmoe.KvBatch(i32([0, n]), i32([old + n]), pages, n), ap, x, q)
        torch.cuda.synchronize()
        return R.Cache.of(kv)
    put(0, 96, 1)
    first = put(96, 32, 2)
    put(96, 32, 3)
    assert put(96, 32, 2).same(first)
    back = put(70, 1, 4)
    a, b = first.values("k"), back.values("k")
    # the block of tokens 64 .. 95 kept 64 .. 69 (page 1, tokens 0 .. 5)
    e = back.k_exp[1, :, 0].double().numpy()
    assert np.all(np.abs(a[1, :, :6] - b[1, :, :6]) <= 2.0 ** -4 * np.abs(a[1, :, :6]) + 2.0 ** -10 * 2.0 ** e[:, None, None])
    assert np.array_equal(a[4], b[4]) and np.array_equal(a[1, :, 32:], b[1, :, 32:])


def test_append_on_a_side_stream_and_in_a_graph(ctx):
    """On a stream of its own, and captured: each replay reads the tables, rows
    and pages that the buffers then hold."""
    import dmoe
    nh, nkv, hd, T = 8, 2, 128, 32
    print("case: append captured in a HIP graph", flush=True)
    dev = "cuda:0"
    side = torch.cuda.Stream(dev)
    lists = [[(5, 1), (64, 1), (31, 1)], [(6, 1), (65, 1), (32, 1)], [(7, 1), (0, 1), (95, 1)]]
    batches = [R.Batch(x, T, seed=20 + i, spare=0, wide=4) for i, x in enumerate(lists)]
    for b in batches:
        b.n_pages = 12
        b.pages[b.pages >= 0] = np.random.RandomState(1).permutation(12)[:(b.pages >= 0).sum()]
    cache = R.Cache("e4m3", 12, nkv, hd, T, seed=21)
    kv = cache.device(dmoe)
    held = batches[0].device(dmoe)
    ap = dmoe.attn_hparams(nh, nkv, hd, 64, 0, BASE, EPS)
    x = torch.zeros((3, 12 * hd), device=dev)
    q = torch.zeros((3, nh, hd), device=dev)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.kv_append_device(kv, held, ap, x, q, stream=side.cuda_stream)
    for i, b in enumerate(batches):
        rows = _rows(np.random.default_rng(30 + i), b, nh, nkv, hd)
        x.copy_(torch.from_numpy(rows))
        for t, v in ((held.q_start, b.q_start), (held.kv_len, b.kv_len), (held.pages, b.pages)):
            t.copy_(torch.from_numpy(v))
        before = R.Cache.of(kv)
        g.replay()
        torch.cuda.synchronize()
        got_q, got = q.cpu().numpy(), R.Cache.of(kv)
        _check(b, before, got, got_q, rows, nh, 64, (None, None))
        eq, ecache = _run(ctx, b, before, rows, nh, 64, False, (None, None), stream=side.cuda_stream)
        assert np.array_equal(got_q, eq) and got.same(ecache)


def test_append_refusals(ctx):
    import dmoe
    print("case: append refusals", flush=True)
    batch, cache = R.Batch([(0, 4)], 32), R.Cache("e4m3", 3, 2, 64, 32)
    kv, b = cache.device(dmoe), batch.device(dmoe)
    x, q = torch.zeros((4, 8 * 64), device="cuda:0"), torch.zeros((4, 4, 64), device="cuda:0")
    E = dmoe._abi
    for ap, args, code in ((dmoe.attn_hparams(4, 2, 64, 66), (x, q), E.ERR_SHAPE),
                           (dmoe.attn_hparams(4, 1, 64, 64), (x, q), E.ERR_SHAPE),
                           (dmoe.attn_hparams(4, 2, 64, 64, use_qk_norm=True), (x, q), E.ERR_INVALID_ARG),
                           (dmoe.attn_hparams(4, 2, 64, 64), (x, x), E.ERR_INVALID_ARG),
                           (dmoe.attn_hparams(4, 2, 64, 64), (x.view(-1)[1:], q), E.ERR_INVALID_ARG)):
        with pytest.raises(dmoe.DmoeError) as e:
            ctx.kv_append_device(kv, b, ap, *args)
        assert e.value.code == code and str(e.value)
    with pytest.raises(ValueError):
        dmoe.KvCache(kv.k, kv.v.transpose(3, 4), kv.k_exp, kv.v_exp)
    with pytest.raises(ValueError):
        dmoe.KvCache(kv.k, kv.v)
    with pytest.raises(ValueError):
        dmoe.KvBatch(b.q_start, b.kv_len.long(), b.pages, 4)
    torch.cuda.synchronize()
    assert R.Cache.of(kv).same(cache)
