"""GPU: the attention half of a layer over a paged KV cache
(dmoe_attn_forward_cached_device): the append, the attention and the projections
run together, block by block as a sampler generates."""
import numpy as np
import pytest
import torch

import kv_ref as R
from conftest import max_rel_err

pytestmark = pytest.mark.gpu

H, NH, NKV, HD, RD = 512, 8, 2, 64, 32


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda:0")


def _layer(ctx, O, wtype=0, block=32):
    from dmoe import synth
    w = synth.host_attn(wtype, 5, O.quantize_rows, H, NH, NKV, HD, RD, block_length=block)
    return w, ctx.attn_upload(w)


def _step(ctx, layer, kv, pages, h, old, stream=None):
    """One sequence's rows h [n][H] behind `old` cached tokens."""
    import dmoe
    n = h.shape[0]
    b = dmoe.KvBatch(_i32([0, n]), _i32([old + n]), pages, n)
    x = torch.from_numpy(h).cuda()
    out, moe = torch.empty_like(x), torch.empty_like(x)
    ctx.attn_forward_cached_device(layer, kv, b, x, out, moe, stream=stream)
    torch.cuda.synchronize()
    return out.cpu().numpy(), moe.cpu().numpy()


@pytest.mark.parametrize("wtype,block", [(0, 32), (0, 1), (12, 32)])
def test_cached_steps_agree_with_one_call(ctx, O, wtype, block):
    """A window of 160 tokens in one call and in calls of 32 (the block mask) or
    of 1 to 33 (the causal mask) leave the same cache and outputs.  F32
    projections do not depend on the number of rows, so the outputs differ by
    the attention's order of summation (1e-5); Q4_K ones by their route (1e-4,
    the bar of test_gpu_attn), and then by where that moves a rounding of the
    cache (2^-11 of a score of up to ~25, 1e-2)."""
    import dmoe
    from dmoe import synth
    print(f"case: cached attention half, type {wtype}, block {block}", flush=True)
    w, layer = _layer(ctx, O, wtype, block)
    h = (synth.normal(77, synth.S_X, 160 * H).reshape(160, H) * 2).astype(np.float32)
    pages = _i32([[3, 0, 2, 4]])
    caches = [dmoe.KvCache.empty("f16", 5, NKV, HD, 64) for _ in range(2)]
    for c in caches:
        c.k.fill_(float("nan"))
        c.v.fill_(float("nan"))
    whole = _step(ctx, layer, caches[0], pages, h, 0)
    cuts = [0, 32, 64, 96, 128, 160] if block == 32 else [0, 1, 2, 33, 66, 67, 99, 130, 131, 160]
    parts = [_step(ctx, layer, caches[1], pages, h[a:b], a) for a, b in zip(cuts, cuts[1:])]
    tol = 1e-5 if wtype == 0 else 1e-2
    for i in range(2):
        assert max_rel_err(np.concatenate([p[i] for p in parts]), whole[i]) <= tol
    if wtype == 0:
        assert R.Cache.of(caches[0]).same(R.Cache.of(caches[1]))
    # the uncached half, whose keys and values stay f32: a score of up to S off by
    # 2^-11 S, S <= the product of the gains (1.5) and norms (sqrt hd) / sqrt hd
    out, _ = ctx.attn_forward(layer, h)
    assert max_rel_err(whole[0], out) <= 2 * 2.0 ** -11 * (1.5 ** 2 * HD ** 0.5) + 2.0 ** -11 + tol
    layer.free()


@pytest.mark.parametrize("kvtype", ["f16", "e4m3"])
def test_cached_half_is_its_parts(ctx, O, kvtype):
    """Two sequences and padded rows: the layer's queries, keys and values are
    those of the append, and what it adds to h is the output projection of the
    attention, both by their own entry points (F32 projections: 1e-5).  Padded
    rows keep h."""
    import dmoe
    from dmoe import synth
    print(f"case: cached attention half and its parts, {kvtype}", flush=True)
    w, layer = _layer(ctx, O)
    batch = R.Batch([(64, 32), (35, 7)], 32, seed=4, extra=5)
    N = batch.n_tokens
    h = (synth.normal(78, synth.S_X, N * H).reshape(N, H) * 2).astype(np.float32)
    cache = R.Cache(kvtype, batch.n_pages, NKV, HD, 32, seed=5)
    kv, b = cache.device(dmoe), batch.device(dmoe)
    x = torch.from_numpy(h).cuda()
    out = torch.empty_like(x)
    ws = torch.empty(ctx.attn_cached_workspace(layer, kv, b), dtype=torch.uint8, device="cuda:0").fill_(0xff)
    ctx.attn_forward_cached_device(layer, kv, b, x, out, workspace=ws)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert np.array_equal(got[batch.q_start[-1]:], h[batch.q_start[-1]:])
    # its parts, the projections on the CPU in 64 bits
    f32 = lambda t, shape: np.asarray(t).view(np.float32).reshape(shape).astype(np.float64)  # noqa: E731
    hh = h.astype(np.float64)
    xn = hh / np.sqrt((hh * hh).mean(-1, keepdims=True) + w.rms_eps) * w.attn_norm
    qkv = (xn @ f32(w.qkv, (w.qkv_dim, H)).T).astype(np.float32)
    kv2 = cache.device(dmoe)
    ap = w.hparams()
    q, att = (torch.zeros((N, NH, HD), device="cuda:0") for _ in range(2))
    gains = [torch.from_numpy(np.ascontiguousarray(g)).cuda() for g in (w.q_norm, w.k_norm)]
    ctx.kv_append_device(kv2, b, ap, torch.from_numpy(qkv).cuda(), q, *gains)
    ctx.kv_attn_device(kv, b, ap, q, att)
    torch.cuda.synchronize()
    want = hh + att.cpu().double().numpy().reshape(N, -1) @ f32(w.wo, (H, NH * HD)).T
    assert max_rel_err(got, want) <= 1e-5
    a, c = R.Cache.of(kv), R.Cache.of(kv2)
    for which in ("k", "v"):        # projections rounded differently move a code by one step at most
        x, y = a.values(which), c.values(which)
        step = 2.0 ** -3 if kvtype == "e4m3" else 2.0 ** -10
        assert np.abs(x - y).max() <= step * np.abs(y).max() and (x != y).mean() < 0.01
    layer.free()


def test_cached_half_in_place_and_captured(ctx, O):
    """h_out may be h; a captured call brings its workspace, and a decoding
    loop's replays (a token more each) give what eager calls give."""
    import dmoe
    from dmoe import synth
    print("case: cached attention half captured in a HIP graph", flush=True)
    w, layer = _layer(ctx, O, 12, 1)
    dev = "cuda:0"
    side = torch.cuda.Stream(dev)
    caches = [dmoe.KvCache.empty("e4m3", 3, NKV, HD, 32) for _ in range(2)]
    pages = _i32([[2, 0]])
    prompt = (synth.normal(79, synth.S_X, 29 * H).reshape(29, H) * 2).astype(np.float32)
    for c in caches:
        _step(ctx, layer, c, pages, prompt, 0)
    length = _i32([30])
    b = dmoe.KvBatch(_i32([0, 1]), length, pages, 1)
    x = torch.zeros((1, H), device=dev)
    moe = torch.zeros((1, H), device=dev)
    ws = torch.empty(ctx.attn_cached_workspace(layer, caches[0], b), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        with pytest.raises(dmoe.DmoeError):
            ctx.attn_forward_cached_device(layer, caches[0], b, x, x, moe, stream=side.cuda_stream)
        ctx.attn_forward_cached_device(layer, caches[0], b, x, x, moe, workspace=ws, stream=side.cuda_stream)
    for i in range(5):
        t = (synth.normal(80 + i, synth.S_X, H).reshape(1, H) * 2).astype(np.float32)
        x.copy_(torch.from_numpy(t))
        length.fill_(30 + i)
        g.replay()
        torch.cuda.synchronize()
        out, m = _step(ctx, layer, caches[1], pages, t, 29 + i)
        assert np.array_equal(x.cpu().numpy(), out) and np.array_equal(moe.cpu().numpy(), m)
    layer.free()


def test_cached_half_refusals(ctx, O):
    import dmoe
    from dmoe import synth
    print("case: cached attention half, refusals", flush=True)
    w, layer = _layer(ctx, O)
    dense = ctx.dense_upload(synth.host_dense(512, 512, 0, 5, O.quantize_rows))
    kv = dmoe.KvCache.empty("f16", 2, NKV, HD, 32)
    other = dmoe.KvCache.empty("f16", 2, NKV, 128, 32)
    b = dmoe.KvBatch(_i32([0, 4]), _i32([4]), _i32([[0]]), 4)
    h, o = torch.zeros((4, H), device="cuda:0"), torch.zeros((4, H), device="cuda:0")
    E = dmoe._abi
    for args, code in (((dense, kv, b, h, o), E.ERR_INVALID_ARG), ((layer, other, b, h, o), E.ERR_SHAPE),
                       ((layer, kv, b, h, h, h), E.ERR_INVALID_ARG), ((layer, kv, b, h, o.view(-1)[1:]), E.ERR_INVALID_ARG)):
        with pytest.raises(dmoe.DmoeError) as e:
            ctx.attn_forward_cached_device(*args)
        assert e.value.code == code
    with pytest.raises(dmoe.DmoeError):
        ctx.attn_cached_workspace(layer, other, b)
    with pytest.raises(dmoe.DmoeError):
        ctx.attn_forward_cached_device(layer, kv, b, h, o, workspace=torch.empty(256, dtype=torch.uint8, device="cuda:0"))
    layer.free()
    dense.free()
