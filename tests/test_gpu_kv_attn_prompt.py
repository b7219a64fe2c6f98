"""GPU: attention over the paged KV cache where it has many rows (prompts, and
prompts beside small sequences), or so many tokens that a wavefront looks up its
pages several times; and tables that contradict themselves."""
import numpy as np
import pytest
import torch

import kv_ref as R
from test_gpu_kv_attn import _poison, _run

pytestmark = pytest.mark.gpu


def attend(batch, cache, q, block):
    """R.attend by matrix products (what is not finite among the values goes to
    the rows that see it one token at a time); the bound on sum |q k| by the rows' norms (never less than the sum)."""
    nh, hd = q.shape[1:]
    G = nh // cache.nkv
    K, V = (torch.from_numpy(cache.values(w)) for w in "kv")
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    top_v = top_s = 0.0
    for s, (o, n) in enumerate(batch.seqs):
        if not n:
            continue
        length, first = o + n, int(batch.q_start[s])
        held = [batch.place(s, p) for p in range(length)]
        idx = np.array([p for p in range(length) if held[p]], np.int64)
        at = np.array([held[p] for p in idx], np.int64).reshape(-1, 2)
        k, v = (x[at[:, 0], :, at[:, 1]].transpose(0, 1).contiguous() for x in (K, V))     # [nkv, L, hd]
        rows = torch.from_numpy(q[first:first + n].astype(np.float64))
        sees = torch.tensor([int((idx < min(length, ((o + i) // block + 1) * block)).sum()) if block > 0 else len(idx)
                             for i in range(n)])
        clean = torch.where(v.isfinite(), v, 0.0)
        odd = [t for t in range(len(idx)) if not v[:, t].isfinite().all()]
        for r in range(0, n, 256):
            x = rows[r:r + 256].reshape(-1, cache.nkv, G, hd).transpose(0, 1)               # [nkv, rows, G, hd]
            m = x.shape[1]
            see = (torch.arange(len(idx)) < sees[r:r + 256, None])[None, :, None]
            w = (x.reshape(cache.nkv, m * G, hd) @ k.transpose(1, 2).contiguous()).reshape(cache.nkv, m, G, -1) / np.sqrt(hd)
            w = torch.softmax(torch.where(see, w, -np.inf), -1)
            y = (w.reshape(cache.nkv, m * G, -1) @ clean).reshape(cache.nkv, m, G, hd)
            for t in odd:
                part = w[..., t, None] * (v - clean)[:, None, None, t]
                y = y + torch.where((sees[r:r + 256] > t)[None, :, None, None], part, 0.0)
            y[:, sees[r:r + 256] == 0] = 0.0
            out[first + r:first + r + m] = y.transpose(0, 1).reshape(m, nh, hd)
        if len(idx):
            top_v = max(top_v, float(v.nan_to_num(0, 0, 0).abs().max()))
            top_s = max(top_s, float((rows.nan_to_num(0, 0, 0).norm(dim=-1).max() * k.nan_to_num(0, 0, 0).norm(dim=-1).max()) / np.sqrt(hd)))
    return out.numpy(), top_v, top_s


def _check(batch, cache, q, block, got):
    ref, top_v, top_s = attend(batch, cache, q, block)
    tol = R.attend_tolerance(top_v, top_s, cache.hd, max(batch.kv_len))
    owned = int(batch.q_start[-1])
    assert (got[owned:] == 7.0).all()
    a, b = got[:owned], ref[:owned]
    fine = np.isfinite(b)
    assert np.array_equal(fine, np.isfinite(a)), "finite values elsewhere than the definition's"
    err = np.abs(a - b)[fine].max(initial=0)
    print(f"  error {err:.3e}, bar {tol:.3e}", flush=True)
    assert err <= tol
    return ref


# rows of 8 heads to a kv head: 16 of them are 128 columns
GROUPS = {
    "one": [(0, 1800)], "after": [(90, 1795)], "long": [(2500, 1830)],
    "beside": [(5, 3), (0, 0), (2100, 513), (700, 1), (31, 16), (0, 17), (63, 70), (1, 1150), (900, 33)],
    "full": [(10, 2300)],                            # more workgroups than start at once
    "padded": [(3000, 40)],                          # fewer rows than the buffers hold
    "many": [(i * 397 % 1700, i % 6) for i in range(150)],
    "crowd": [(i * 13 % 800, 1) for i in range(70)] + [(10, 1500), (0, 0), (3000, 33), (2, 200)] + [(i * 41 % 900, i % 3) for i in range(70)],
}


def _q(batch, nh, hd, seed):
    return np.random.default_rng(seed).standard_normal((batch.n_tokens, nh, hd)).astype(np.float32)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("block", [1, 32, 0])
@pytest.mark.parametrize("group", GROUPS)
def test_prompts(ctx, kvtype, group, block):
    nh, nkv, hd, T = 32, 4, 128, 64
    print(f"case: attn {kvtype} prompt {group}, block {block}", flush=True)
    batch = R.Batch(GROUPS[group], T, seed=1, extra=1800 if group == "padded" else 3)
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=2)
    _poison(batch, cache)
    q = _q(batch, nh, hd, 3)
    _check(batch, cache, q, block, _run(ctx, batch, cache, q, block))


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("shape", [(64, 8, 64, 32), (40, 1, 64, 96), (33, 3, 128, 32), (6, 6, 64, 256), (128, 1, 128, 64)], ids=str)
def test_prompts_of_other_shapes(ctx, kvtype, shape):
    nh, nkv, hd, T = shape
    print(f"case: attn {kvtype} prompt {shape}", flush=True)
    n = -(-57344 // nh)
    for seqs in ([(77, n)], [(0, n - n // 3), (5, 1), (130, n // 3)]):
        batch = R.Batch(seqs, T, seed=4, extra=1)
        cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=5)
        _poison(batch, cache)
        q = _q(batch, nh, hd, 6)
        for block in (1, 48):
            _check(batch, cache, q, block, _run(ctx, batch, cache, q, block))


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_prompts_with_pages_that_are_none(ctx, kvtype):
    """Holes, a sequence without a page, the first 64 token tiles of one without."""
    nh, nkv, hd, T = 32, 4, 64, 32
    print(f"case: attn {kvtype} prompts, pages that are none", flush=True)
    for seqs in ([(2200, 1800)], [(40, 300), (2200, 1800), (2, 9)]):
        batch = R.Batch(seqs, T, seed=7)
        long = len(seqs) // 2
        if long:
            batch.pages[0] = -1
        batch.pages[long, :66] = -3
        batch.pages[long, 70], batch.pages[long, 90], batch.pages[long, 91] = batch.n_pages, -7, 2 ** 31 - 1
        batch.pages = np.ascontiguousarray(batch.pages[:, :96])
        cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=8)
        _poison(batch, cache)
        q = _q(batch, nh, hd, 9)
        for block in (1, 0):
            got = _run(ctx, batch, cache, q, block)
            _check(batch, cache, q, block, got)
            assert not long or (got[:300] == 0).all()


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
@pytest.mark.parametrize("block", [1, 8])
def test_prompts_what_is_not_seen_has_no_part(ctx, kvtype, block):
    """NaN and infinities at positions that some rows of a tile see."""
    nh, nkv, hd, T = 32, 2, 64, 32
    print(f"case: attn {kvtype} prompt, block {block}, NaN in masked places", flush=True)
    batch = R.Batch([(20, 1792), (0, 64)], T, seed=10)
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=11)
    q = _q(batch, nh, hd, 12)
    clean = _run(ctx, batch, cache, q, block)
    dirty = cache.copy()
    for p in (505, 1001):
        (pk, tk), (pv, tv) = batch.place(0, p), batch.place(0, p - 9)
        if dirty.f8:
            dirty.k.view(torch.uint8)[pk, 0, tk, 3] = 0x7f
            dirty.v.view(torch.uint8)[pv, 1, tv // 32, 5, tv % 32 // 8, 1, tv % 8] = 0xff
        else:
            dirty.k[pk, 0, tk, 3] = float("nan")
            dirty.v[pv, 1, tv // 32, 11, tv % 32] = float("inf")
    got = _run(ctx, batch, dirty, q, block)
    ref = _check(batch, dirty, q, block, got)
    same = np.isfinite(ref)
    assert np.array_equal(got[same], clean[same]) and not same.all()


def test_prompts_again_on_another_stream_and_in_a_graph(ctx):
    """The same bits each time; replays read the tables as they are then."""
    import dmoe
    nh, nkv, hd, T = 32, 4, 128, 64
    print("case: attn prompts, streams and a graph", flush=True)
    batch = R.Batch(GROUPS["beside"], T, seed=13, extra=3)
    cache = R.Cache("e4m3", batch.n_pages, nkv, hd, T, seed=14)
    q = _q(batch, nh, hd, 15)
    ref = _run(ctx, batch, cache, q, 32)
    side = torch.cuda.Stream("cuda:0")
    assert np.array_equal(_run(ctx, batch, cache, q, 32, stream=side.cuda_stream), ref)
    kv, b = cache.device(dmoe), batch.device(dmoe)
    ap = dmoe.attn_hparams(nh, nkv, hd, 0, 32)
    ws = torch.empty(ctx.kv_attn_workspace(kv, b, ap), dtype=torch.uint8, device="cuda:0")
    qd, out = torch.from_numpy(q).cuda(), torch.zeros(q.shape, device="cuda:0")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.kv_attn_device(kv, b, ap, qd, out, workspace=ws, stream=side.cuda_stream)
    for turn in range(3):
        now = R.Batch([(max(0, o - 40 * turn), n) for o, n in batch.seqs], T)
        now.extra, now.n_tokens, now.pages, now.n_pages = 3, batch.n_tokens, batch.pages, batch.n_pages
        b.kv_len.copy_(torch.from_numpy(now.kv_len))
        out.fill_(7.0)
        ws.fill_(0xff)                               # nothing of the last replay is left to find
        g.replay()
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert np.array_equal(_run(ctx, now, cache, q, 32), got)
        if turn != 1:
            _check(now, cache, q, 32, got)
        else:
            assert not np.array_equal(got, ref)


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_pages_looked_up_several_times(ctx, kvtype):
    """45 sequences of 10,240 tokens are a chunk each of 320 token tiles, 80 to a
    wavefront; they hold the same pages in different orders (a page may belong
    to several sequences that only read it)."""
    nh, nkv, hd, T = 8, 8, 64, 64
    print(f"case: attn {kvtype}, 320 tiles a chunk", flush=True)
    batch = R.Batch([(10239 - 7 * i, 1) for i in range(45)], T, seed=16, extra=1)
    batch.n_pages = 200
    batch.pages = np.stack([np.random.RandomState(i).permutation(200)[:160] for i in range(45)]).astype(np.int32)
    cache = R.Cache(kvtype, 200, nkv, hd, T, seed=17)
    q = _q(batch, nh, hd, 18)
    _check(batch, cache, q, 1, _run(ctx, batch, cache, q, 1))


@pytest.mark.parametrize("n", [2, 1800])
def test_rows_of_an_earlier_sequence(ctx, n):
    """Tables that decrease, with more work than there are rows: the attention
    takes the rows of a sequence that starts below an earlier entry of q_start
    for the earlier one's, and an append stays within the cache (which rows it
    takes is not defined; here all that it can take hold the same)."""
    import dmoe
    nh, nkv, hd, T = 32, 4, 64, 64
    print(f"case: tables that decrease, {n} rows", flush=True)
    S = 130
    batch = R.Batch([(900, n)] + [(300, 1)], T, seed=19)
    cache = R.Cache("f16", batch.n_pages, nkv, hd, T, seed=20)
    qkv = torch.from_numpy(_q(batch, nh + 2 * nkv, hd, 21).reshape(batch.n_tokens, -1)).cuda()
    ap = dmoe.attn_hparams(nh, nkv, hd, 64, 1)
    results = []
    for more in (0, S):
        # rows 0 .. n of the first, then n times (n .. 0, 0 .. n), then the last one's row
        starts = [0, n] + [0, n] * more + [n + 1]
        lens = [900 + n] + [900 + n] * (2 * more) + [301]
        pages = np.concatenate([batch.pages[:1], np.repeat(batch.pages[:1], 2 * more, 0), batch.pages[1:]])
        b = dmoe.KvBatch(*[torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda:0") for x in (starts, lens, pages)],
                         batch.n_tokens)
        kv = cache.device(dmoe)
        q, out = (torch.full((batch.n_tokens, nh, hd), 7.0, device="cuda:0") for _ in range(2))
        ctx.kv_append_device(kv, b, ap, qkv, q)
        if not more:
            whole, queries = kv, q
        ctx.kv_attn_device(whole, b, ap, queries, out)
        torch.cuda.synchronize()
        results.append((R.Cache.of(kv), q.cpu().numpy(), out.cpu().numpy()))
    (c0, q0, o0), (c1, q1, o1) = results
    # what the second append took is as in the first, the rest as it was
    for x, y, z in ((c0.k, c1.k, cache.k), (c0.v, c1.v, cache.v)):
        assert bool(((x == y) | (y == z)).all())
    assert ((q0 == q1) | (q1 == 7.0)).all()
    ref, top_v, top_s = attend(batch, c0, q0, 1)
    tol = R.attend_tolerance(top_v, top_s, hd, 900 + n)
    assert max(np.abs(o0 - ref).max(), np.abs(o1 - ref).max()) <= tol


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_thousands_of_sequences(ctx, kvtype):
    """More sequences than one look of 64 times 64 finds, half of them with a row."""
    nh, nkv, hd, T = 2, 1, 64, 32
    print(f"case: attn {kvtype}, 4300 sequences", flush=True)
    batch = R.Batch([(i * 7 % 60, (i * 5 + i // 64) % 2) for i in range(4299)] + [(900, 3)], T, seed=22, extra=2)
    cache = R.Cache(kvtype, batch.n_pages, nkv, hd, T, seed=23)
    _poison(batch, cache)
    q = _q(batch, nh, hd, 24)
    _check(batch, cache, q, 1, _run(ctx, batch, cache, q, 1))
