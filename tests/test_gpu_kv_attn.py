"""GPU: attention over the paged KV cache (dmoe_kv_attn_device) against the
definition in 64 bits on the values that the cache holds (kv_ref.py; the bar is
derived in attend_tolerance)."""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu


def _run(ctx, batch, cache, q, block, stream=None, workspace=None, kv=None):
    import dmoe
    kv = cache.device(dmoe) if kv is None else kv
    b = batch.device(dmoe)
    ap = dmoe.attn_hparams(q.shape[1], cache.nkv, cache.hd, 0, block)
    qd = torch.from_numpy(q).cuda()
    out = torch.full(q.shape, 7.0, device="cuda:0")
    torch.cuda.synchronize()
    ctx.kv_attn_device(kv, b, ap, qd, out, workspace=workspace, stream=stream)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _check(batch, cache, q, block, got, tol_scale=1.0):
    ref, top_v, top_s = R.attend(batch, cache, q, block)
    tol = tol_scale * R.attend_tolerance(top_v, top_s, cache.hd, max(batch.kv_len))
    owned = np.zeros(batch.n_tokens, bool)
    owned[:batch.q_start[-1]] = True
    assert (got[~owned] == 7.0).all()
    a, b = got[owned], ref[owned]
    fine = np.isfinite(b)
    assert np.array_equal(fine, np.isfinite(a)), "finite values elsewhere than the definition's"
    err = np.abs(a - b)[fine].max(initial=0)
    print(f"  error {err:.3e}, bar {tol:.3e}", flush=True)
    assert err <= tol
    return ref


GROUPS = {
    "one": [(0, 1)], "token": [(700, 1)], "block": [(96, 32)], "odd": [(33, 1)], "chunk": [(95, 77)],
    "ragged": [(5, 3), (0, 0), (31, 1), (32, 40), (700, 1), (64, 32), (0, 1), (63, 70), (1, 2), (33, 0), (256, 32)],
    "long": [(5000, 2), (17, 1), (2999, 33)],
    "singles": [(i * 13, 1) for i in range(70)],
}
SHAPES = [  # n_head, n_head_kv, head_dim, page_tokens
    (32, 4, 128, 64), (5, 1, 64, 32), (3, 3, 128, 96), (20, 1, 64, 256), (6, 2, 64, 64), (33, 1, 128, 32), (16, 4, 128, 64)]


def _one(ctx, kvtype, group, shape, block, seed=0, poison=True, scale=1.0):
    nh, nkv, hd, T = shape
    print(f"case: attn {kvtype} {group} {nh}/{nkv} d{hd} page {T} block {block}", flush=True)
    batch = R.Batch(GROUPS[group], T, seed=seed, extra=2)
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=seed + 1)
    if poison:
        _poison(batch, cache)
    q = (np.random.default_rng(seed + 2).standard_normal((batch.n_tokens, nh, hd)) * scale).astype(np.float32)
    got = _run(ctx, batch, cache, q, block)
    _check(batch, cache, q, block, got)
    return batch, cache, q, got


def _poison(batch, cache):
    """NaN in every token that no sequence holds; whole blocks of them get the
    largest exponents too."""
    held = np.zeros((batch.n_pages, batch.T), bool)
    for s in range(len(batch.seqs)):
        for p in range(batch.kv_len[s]):
            at = batch.place(s, p)
            if at:
                held[at] = True
    k = cache.k.view(torch.uint8 if cache.f8 else torch.int16)
    v = cache.v.view(torch.uint8 if cache.f8 else torch.int16)
    bad = 0x7f if cache.f8 else 0x7e00
    for pg, t in zip(*np.nonzero(~held)):
        k[pg, :, t] = bad
        if cache.f8:
            v[pg, :, t // 32, :, t % 32 // 8, :, t % 8] = bad
        else:
            v[pg, :, t // 32, :, t % 32] = bad
    if cache.f8:
        for pg, b in zip(*np.nonzero(~held.reshape(batch.n_pages, -1, 32).any(-1))):
            cache.k_exp[pg, :, b] = 127
            cache.v_exp[pg, :, b] = 127


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("block", [1, 32, 0])
@pytest.mark.parametrize("group", GROUPS)
def test_attn_groups(ctx, kvtype, group, block):
    _one(ctx, kvtype, group, SHAPES[0], block)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("block", [1, 5, 48])
@pytest.mark.parametrize("shape", SHAPES[1:], ids=str)
def test_attn_shapes(ctx, kvtype, shape, block):
    _one(ctx, kvtype, "ragged", shape, block, seed=block)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-4, 30.0, 1e5])
def test_attn_query_magnitudes(ctx, kvtype, scale):
    """From a uniform softmax to one that a single key takes."""
    _one(ctx, kvtype, "ragged", (8, 2, 64, 32), 32, seed=40, scale=scale)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("group", ["ragged", "long"])
def test_attn_pages_that_are_none(ctx, kvtype, group):
    """Holes in the page table, a table that ends early and a sequence without
    any page: their tokens are not seen; a row that sees nothing gives zeros."""
    nh, nkv, hd, T = 8, 2, 64, 32
    print(f"case: attn {kvtype} {group}, pages that are none", flush=True)
    batch = R.Batch(GROUPS[group], T, seed=50, extra=1)
    batch.pages[0] = -1
    batch.pages[-1, 2], batch.pages[-1, 5], batch.pages[-1, 0] = batch.n_pages, -7, 2 ** 31 - 1
    batch.pages = np.ascontiguousarray(batch.pages[:, :20])
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=51)
    _poison(batch, cache)
    q = np.random.default_rng(52).standard_normal((batch.n_tokens, nh, hd)).astype(np.float32)
    for block in (0, 1):
        got = _run(ctx, batch, cache, q, block)
        _check(batch, cache, q, block, got)
        assert (got[:batch.q_start[1]] == 0).all()


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("block", [1, 8])
def test_attn_what_is_not_seen_has_no_part(ctx, kvtype, block):
    """Keys and values that are NaN (F16: infinite too) at positions that some
    rows of a tile see and others do not: the former give NaN, the latter what
    they give without them."""
    nh, nkv, hd, T = 4, 2, 64, 32
    print(f"case: attn {kvtype} block {block}, NaN in masked places", flush=True)
    batch = R.Batch([(20, 40), (0, 64)], T, seed=60)
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=61)
    q = np.random.default_rng(62).standard_normal((batch.n_tokens, nh, hd)).astype(np.float32)
    clean = _run(ctx, batch, cache, q, block)
    dirty = cache.copy()
    pk, tk = batch.place(0, 41)
    pv, tv = batch.place(1, 25)
    if dirty.f8:
        dirty.k.view(torch.uint8)[pk, 0, tk, 3] = 0x7f
        dirty.v.view(torch.uint8)[pv, :, tv // 32, 5, tv % 32 // 8, 1, tv % 8] = 0xff
    else:
        dirty.k[pk, 0, tk, 3] = float("nan")
        dirty.v[pv, :, tv // 32, 11, tv % 32] = float("inf")
    got = _run(ctx, batch, dirty, q, block)
    _check(batch, dirty, q, block, got)
    ref = R.attend(batch, dirty, q, block)[0]
    same = np.isfinite(ref)
    assert np.array_equal(got[same], clean[same]) and not same.all()


def test_attn_exponents(ctx):
    """Blocks of zeros (the least exponent) beside large and small ones, values
    up to 2^50 times a code: a block of zero values still takes its share of the
    weights."""
    nh, nkv, hd, T = 8, 2, 128, 64
    print("case: attn e4m3, exponents from -50 to 50", flush=True)
    batch = R.Batch([(300, 1), (64, 32), (0, 10)], T, seed=70)
    for lo, hi in ((-50, -40), (-6, 3), (40, 50), (-50, 50)):
        cache = R.Cache("e4m3", batch.n_pages, nkv, hd, T, seed=71)
        rng = np.random.RandomState(72)
        cache.v_exp.copy_(torch.from_numpy(rng.randint(lo, hi + 1, cache.v_exp.shape).astype(np.int8)))
        zero = torch.from_numpy(rng.rand(*cache.v_exp.shape) < 0.4)
        cache.v.view(torch.uint8)[zero] = 0
        cache.v_exp[zero] = R.E_MIN
        q = rng.standard_normal((batch.n_tokens, nh, hd)).astype(np.float32)
        _check(batch, cache, q, 0, _run(ctx, batch, cache, q, 0))


def test_attn_queries_that_are_not_finite(ctx):
    """A NaN or infinite query is its own row's trouble only."""
    nh, nkv, hd, T = 8, 2, 64, 32
    print("case: attn, NaN and infinite queries", flush=True)
    for kvtype in ("f16", "e4m3"):
        batch = R.Batch([(100, 8)], T, seed=80)
        cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=81)
        q = np.random.default_rng(82).standard_normal((8, nh, hd)).astype(np.float32)
        clean = _run(ctx, batch, cache, q, 0)
        bad = q.copy()
        bad[2, 3, 5], bad[4, 0, 0] = np.nan, np.inf
        got = _run(ctx, batch, cache, bad, 0)
        assert np.isnan(got[2, 3]).all() and not np.isfinite(got[4, 0]).any()
        got[2, 3], got[4, 0] = clean[2, 3], clean[4, 0]
        assert np.array_equal(got, clean)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_cache_past_32_bits(ctx, kvtype):
    """Pages whose offsets need more than 32 bits, written and read."""
    import dmoe
    nh, nkv, hd, T = 4, 2, 128, 256
    print(f"case: a {kvtype} cache of more than 2^32 bytes", flush=True)
    P = (1 << 32) // (nkv * T * hd) + 40
    kv = dmoe.KvCache.empty(kvtype, P, nkv, hd, T)
    small = R.Batch([(130, 40), (300, 1)], T, seed=90, spare=0)
    far = np.array([P - 1, P - 3, P // 2 + 7])
    cache = R.Cache(kvtype, small.n_pages, nkv, hd, T, seed=91)
    for i in range(small.n_pages):
        for name in ("k", "v", "k_exp", "v_exp"):
            if getattr(cache, name) is not None:
                getattr(kv, name)[int(far[i])] = getattr(cache, name)[i].cuda()
    remote = R.Batch(small.seqs, T, seed=90, spare=0)
    remote.pages = np.where(small.pages >= 0, far[small.pages], -1).astype(np.int32)
    rng = np.random.default_rng(92)
    qkv = torch.from_numpy(rng.standard_normal((41, 8 * hd)).astype(np.float32)).cuda()
    ap = dmoe.attn_hparams(nh, nkv, hd, 64, 1)
    outs = []
    for c, b in ((cache.device(dmoe), small.device(dmoe)), (kv, remote.device(dmoe))):
        q, o = torch.empty((41, nh, hd), device="cuda:0"), torch.empty((41, nh, hd), device="cuda:0")
        ctx.kv_append_device(c, b, ap, qkv, q)
        ctx.kv_attn_device(c, b, ap, q, o)
        torch.cuda.synchronize()
        outs.append((q, o, c))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    near = R.Cache.of(outs[0][2])
    for i in range(small.n_pages):
        assert torch.equal(kv.k[int(far[i])].cpu().view(torch.uint8), near.k[i].view(torch.uint8))
        assert torch.equal(kv.v[int(far[i])].cpu().view(torch.uint8), near.v[i].view(torch.uint8))
    ref, tv, ts = R.attend(small, near, outs[0][0].cpu().numpy(), 1)
    assert np.abs(outs[1][1].cpu().numpy() - ref).max() <= R.attend_tolerance(tv, ts, hd, 301)
    del kv, outs
    torch.cuda.empty_cache()


def test_attn_same_bits_again_and_with_a_workspace(ctx):
    """No atomics whose order shows: the same call gives the same bits, on the
    context's workspace, on the caller's and on another stream; the workspace is
    asked for without tables, and too small a one is refused."""
    import dmoe
    batch, cache, q, got = _one(ctx, "e4m3", "long", SHAPES[0], 32, seed=100)
    kv, b = cache.device(dmoe), batch.device(dmoe)
    ap = dmoe.attn_hparams(32, 4, 128, 0, 32)
    n = ctx.kv_attn_workspace(kv, b, ap)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda:0")
    side = torch.cuda.Stream("cuda:0")
    for kw in ({}, dict(workspace=ws), dict(stream=side.cuda_stream), dict(stream=side.cuda_stream, workspace=ws)):
        assert np.array_equal(_run(ctx, batch, cache, q, 32, **kw), got)
    for bad in (ws[:n - 1], torch.empty(n + 16, dtype=torch.uint8, device="cuda:0")[1:]):
        with pytest.raises(dmoe.DmoeError) as e:
            _run(ctx, batch, cache, q, 32, workspace=bad)
        assert e.value.code == dmoe._abi.ERR_INVALID_ARG


def test_attn_two_streams_at_once(ctx):
    """Two calls in flight on two streams, each on a workspace of its own."""
    import dmoe
    print("case: two calls at once", flush=True)
    jobs = []
    for i in range(2):
        batch = R.Batch(GROUPS["long"], 64, seed=110 + i)
        cache = R.Cache("e4m3", batch.n_pages, 4, 128, 64, seed=112 + i)
        q = np.random.default_rng(114 + i).standard_normal((batch.n_tokens, 32, 128)).astype(np.float32)
        ref = _run(ctx, batch, cache, q, 1)
        kv, b = cache.device(dmoe), batch.device(dmoe)
        ap = dmoe.attn_hparams(32, 4, 128, 0, 1)
        ws = torch.empty(ctx.kv_attn_workspace(kv, b, ap), dtype=torch.uint8, device="cuda:0")
        jobs.append((kv, b, ap, torch.from_numpy(q).cuda(), torch.zeros(q.shape, device="cuda:0"), ws,
                     torch.cuda.Stream("cuda:0"), ref))
    torch.cuda.synchronize()
    for _ in range(5):
        for kv, b, ap, q, out, ws, st, _ in jobs:
            ctx.kv_attn_device(kv, b, ap, q, out, workspace=ws, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for *_, out, ws, st, ref in jobs:
        assert np.array_equal(out.cpu().numpy(), ref)


def test_attn_in_two_graphs(ctx):
    """Two graphs of calls of different sizes, each with a workspace, replayed in
    turn with eager calls between that make the context's own workspace grow;
    the lengths change from replay to replay.  A captured call without a
    workspace is refused."""
    import dmoe
    print("case: attention captured in two HIP graphs", flush=True)
    dev = "cuda:0"
    own = dmoe.Context(0)
    side = torch.cuda.Stream(dev)
    graphs = []
    for i, n in enumerate((1, 32)):
        batch = R.Batch([(4000 - 32 * i, n), (96, n)], 64, seed=120 + i)
        cache = R.Cache("e4m3", batch.n_pages, 4, 128, 64, seed=122 + i)
        kv, b = cache.device(dmoe), batch.device(dmoe)
        ap = dmoe.attn_hparams(32, 4, 128, 0, 32)
        ws = torch.empty(own.kv_attn_workspace(kv, b, ap), dtype=torch.uint8, device=dev)
        q, out = (torch.zeros((2 * n, 32, 128), device=dev) for _ in range(2))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            with pytest.raises(dmoe.DmoeError):
                own.kv_attn_device(kv, b, ap, q, out, stream=side.cuda_stream)
            own.kv_attn_device(kv, b, ap, q, out, workspace=ws, stream=side.cuda_stream)
        graphs.append((g, batch, cache, kv, b, q, out, n, ws))
    for turn in range(3):
        for g, batch, cache, kv, b, q, out, n, ws in graphs:
            x = np.random.default_rng(130 + turn).standard_normal(q.shape).astype(np.float32)
            q.copy_(torch.from_numpy(x))
            now = R.Batch([(o // 32 * 32 - 32 * turn, n) for o, n in batch.seqs], 64)
            now.pages, now.n_pages = batch.pages, batch.n_pages
            b.kv_len.copy_(torch.from_numpy(now.kv_len))
            out.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            _check(now, cache, x, 32, got)
            assert np.array_equal(_run(own, now, cache, x, 32), got)
    own.close()


def test_attn_refusals(ctx):
    import dmoe
    print("case: attn refusals", flush=True)
    batch, cache = R.Batch([(0, 4)], 32), R.Cache("f16", 3, 2, 64, 32)
    kv, b = cache.device(dmoe), batch.device(dmoe)
    q, out = torch.zeros((4, 4, 64), device="cuda:0"), torch.full((4, 4, 64), 7.0, device="cuda:0")
    E = dmoe._abi
    good = dmoe.attn_hparams(4, 2, 64)
    for ap, args, code in ((dmoe.attn_hparams(5, 2, 64), (q, out), E.ERR_SHAPE),
                           (dmoe.attn_hparams(4, 2, 128), (q, out), E.ERR_SHAPE),
                           (good, (q, q), E.ERR_INVALID_ARG), (good, (q, out.view(-1)[2:]), E.ERR_INVALID_ARG)):
        with pytest.raises(dmoe.DmoeError) as e:
            ctx.kv_attn_device(kv, b, ap, *args)
        assert e.value.code == code and str(e.value)
    with pytest.raises(dmoe.DmoeError):
        ctx.kv_attn_workspace(kv, b, dmoe.attn_hparams(5, 2, 64))
    torch.cuda.synchronize()
    assert (out == 7.0).all()
