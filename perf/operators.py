"""The paged KV cache of the attention half: what is appended to it and the
attention that reads it, as a program that generates block by block runs them.

A block-diffusion sampler runs every denoising step over the block that it is
working on (32 tokens); keys and values of the blocks before it no longer
change and stay in a cache.  A program that serves several sequences gives each
of them pages of one pool; with a block length of 1 the same calls are those
of a causal decoder, one token at a time.

Kinds
  append  rows of the fused QKV projection: QK norm, partial rotary positions,
          keys and values into the pages, queries out (kv_append_device)
  attn    queries over the pages, ragged over the sequences (kv_attn_device)

The cache holds F16, or E4M3 with one power-of-two scale per block of 32 tokens
and head.  Layouts (T tokens a page, NB = T / 32 blocks of 32 tokens):
  k      [pages, kv heads, T, head_dim]
  v      [pages, kv heads, NB, head_dim, 32]              F16
         [pages, kv heads, NB, head_dim / 2, 4, 2, 8]     E4M3: two dims of 8 tokens are adjacent
  k_exp, v_exp  int8 [pages, kv heads, NB]                E4M3: value = code * 2^exp
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
ROPE_BASE = 3e6
TOP = 448.0                 # the largest E4M3 value
E_MIN, E_MAX = -50, 50      # the scales' exponents
F8 = torch.float8_e4m3fn


def listed():
    def c(name, kind, kvtype, seqs, q, kv, heads=32, kv_heads=4, hd=128, rd=64, page=64, block=32):
        return dict(name=name, kind=kind, kvtype=kvtype, seqs=seqs, q=q, kv=kv, heads=heads, kv_heads=kv_heads,
                    hd=hd, rd=rd, page=page, block=block)
    return [
        # one chat, one token: the smallest call, all latency
        c("append_token", "append", "f16", 1, 1, 700),
        # a decoder's batch of single tokens; most fall inside a block that is kept
        c("append_tokens_s61", "append", "e4m3", 61, 1, 900, block=1),
        # a denoising step of 16 sequences: each writes its whole block anew
        c("append_blocks_s16", "append", "e4m3", 16, 32, 2048),
        # a long prompt appended behind another one that ends inside a block
        c("append_prompt_n4001", "append", "e4m3", 1, 4001, 5023),
        # one chat, one token over a short cache
        c("attn_token", "attn", "f16", 1, 1, 700),
        # a decoder's batch of single tokens, ragged lengths
        c("attn_tokens_s48", "attn", "e4m3", 48, 1, 8190, block=1),
        # one token over a very long cache
        c("attn_token_long", "attn", "e4m3", 1, 1, 131072, page=256),
        # a denoising step of one sequence over a long cache
        c("attn_block", "attn", "e4m3", 1, 32, 16384),
        # a denoising step of eight sequences of a model half as wide
        c("attn_blocks_s8", "attn", "f16", 8, 32, 4096, heads=16),
        # a chunk of a prompt over what is cached of it
        c("attn_prompt_n2000", "attn", "e4m3", 1, 2000, 6001),
        # prompts and decoding sequences in one call, small heads, odd sizes
        c("attn_mixed_s12", "attn", "e4m3", 12, 200, 2001, heads=10, kv_heads=5, hd=64, rd=64, page=32, block=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above, at most as large as the largest."""
    known = [{k: v for k, v in c.items() if k != "name"} for c in listed()]
    most = max(_cost(work(c)) for c in known)
    while True:
        heads, kv_heads, hd, rd = rng.choice(((32, 4, 128, 64), (32, 4, 128, 64), (16, 4, 128, 64), (10, 5, 64, 64),
                                              (8, 8, 128, 128), (12, 3, 64, 32)))
        q = rng.choice((1, 1, 32, 32, _log(rng, 2, 31), _log(rng, 33, 4000)))
        case = dict(kind=rng.choice(("append", "attn", "attn")), kvtype=rng.choice(("e4m3", "e4m3", "f16")),
                    seqs=_log(rng, 1, 64), q=q, kv=q + _log(rng, 1, 32768), heads=heads, kv_heads=kv_heads, hd=hd,
                    rd=rd, page=rng.choice((32, 64, 64, 256)), block=rng.choice((32, 32, 1, 0)))
        tokens, rows = case["seqs"] * case["kv"], case["seqs"] * q
        # what the plain form holds at once: padded keys and values, scores
        if tokens * kv_heads * hd > 1 << 29 or rows * heads * case["kv"] > 1 << 29 or rows > 8192:
            continue
        if _cost(work(case)) <= most and case not in known:
            return case


def _cost(w):
    return max(w["bytes"], w["flops"] / 50)


def _lengths(case):
    """([tokens of this call], [cached tokens, those included]) of each
    sequence: the first has the most, the others are spread below."""
    nq, kv = [], []
    for s in range(case["seqs"]):
        f = (s * 0.6180339887498949) % 1.0
        n = case["q"] if case["q"] in (1, 32) or s == 0 else max(1, int(case["q"] * (1 - f) ** 2))
        old = case["kv"] - case["q"]
        o = old if s == 0 else int(old * (0.1 + 0.9 * (1 - f)))
        if case["q"] == 32:
            o = o // 32 * 32            # a denoising step's block begins at a block
        nq.append(n)
        kv.append(o + n)
    return nq, kv


def work(case):
    nq, kv = _lengths(case)
    nh, nkv, hd, B = case["heads"], case["kv_heads"], case["hd"], case["block"]
    eb, n = (2 if case["kvtype"] == "f16" else 1), sum(nq)
    if case["kind"] == "append":
        return {"bytes": n * hd * (4 * (nh + 2 * nkv) + 4 * nh + 2 * nkv * eb), "flops": 0}
    pairs = 0
    for a, b in zip(nq, kv):
        if B <= 0:
            pairs += a * b
        else:
            pairs += sum(min(b, (p // B + 1) * B) for p in range(b - a, b))
    return {"bytes": 2 * n * nh * hd * 4 + sum(kv) * 2 * nkv * hd * eb, "flops": 4 * hd * nh * pairs}


# ---------------------------------------------------------------------------
# Inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _v_shape(pages, nkv, T, hd, f8):
    return (pages, nkv, T // 32, hd // 2, 4, 2, 8) if f8 else (pages, nkv, T // 32, hd, 32)


def prepare(case, seed):
    g = _gen(seed)
    nq, kv = _lengths(case)
    nh, nkv, hd, T = case["heads"], case["kv_heads"], case["hd"], case["page"]
    f8 = case["kvtype"] == "e4m3"
    need = [-(-k // T) for k in kv]
    pool, wide = sum(need) + 3, max(need)
    ids = torch.randperm(pool, generator=g, device=DEV).to(torch.int32).cpu()
    pages = torch.full((len(kv), wide), -1, dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        pages[s, :m] = ids[at:at + m]
        at += m
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    starts = [0]
    for a in nq:
        starts.append(starts[-1] + a)
    n = starts[-1]
    st = dict(case=dict(case), q_start=i32(starts), kv_len=i32(kv), pages=pages.to(DEV), n=n, most_q=max(nq),
              most_kv=max(kv))

    def cache(shape):
        # what is cached: bell-shaped values, some blocks larger than others
        x = torch.empty(shape, dtype=torch.float16, device=DEV).normal_(0, 60 if f8 else 0.7, generator=g)
        return x.clamp_(-TOP, TOP).to(F8) if f8 else x
    st["k"], st["v"] = cache((pool, nkv, T, hd)), cache(_v_shape(pool, nkv, T, hd, f8))
    if f8:
        for name in ("k_exp", "v_exp"):
            st[name] = torch.randint(-8, -5, (pool, nkv, T // 32), generator=g, device=DEV, dtype=torch.int8)
    gain = lambda m: torch.empty(m, device=DEV).uniform_(0.5, 1.5, generator=g)  # noqa: E731
    if case["kind"] == "append":
        st["qkv"] = torch.empty((n, (nh + 2 * nkv) * hd), device=DEV).normal_(0, 1.3, generator=g)
        st["q_norm"], st["k_norm"] = gain(hd), gain(hd)
    else:
        st["q"] = torch.empty((n, nh, hd), device=DEV).normal_(0, 1.0, generator=g) * gain(hd) * 1.5
    st["out"] = torch.empty((n, nh, hd), device=DEV)
    return st


# ---------------------------------------------------------------------------
# The framework's operators

_context = []


def _dmoe():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "diffuse-cpp_amd"))
    import dmoe
    if not _context:
        _context.append(dmoe.Context(0))
    return dmoe, _context[0]


def _handles(st):
    dmoe, ctx = _dmoe()
    c = st["case"]
    cache = dmoe.KvCache(st["k"], st["v"], st.get("k_exp"), st.get("v_exp"))
    batch = dmoe.KvBatch(st["q_start"], st["kv_len"], st["pages"], st["n"])
    ap = dmoe.attn_hparams(n_head=c["heads"], n_head_kv=c["kv_heads"], head_dim=c["hd"], rotary_dim=c["rd"],
                           block_length=c["block"], rope_base=ROPE_BASE, rms_eps=EPS, use_qk_norm=True)
    return ctx, cache, batch, ap


def _own(st):
    if "handles" not in st:
        st["handles"] = _handles(st)
    ctx, cache, batch, ap = st["handles"]
    stream = torch.cuda.current_stream().cuda_stream
    if st["case"]["kind"] == "append":
        ctx.kv_append_device(cache, batch, ap, st["qkv"], st["out"], st["q_norm"], st["k_norm"], stream=stream)
        return _state(st, st["out"])
    ctx.kv_attn_device(cache, batch, ap, st["q"], st["out"], stream=stream)
    return st["out"]


def _state(st, q):
    """What an append returns: the queries and the whole cache."""
    names = ("k", "v", "k_exp", "v_exp") if "k_exp" in st else ("k", "v")
    return {"q": q, **{m: st[m] for m in names}}


# ---------------------------------------------------------------------------
# The plain forms

def _rows(st):
    """Sequence and position of each row."""
    t = torch.arange(st["n"], device=DEV)
    start = st["q_start"].long()
    s = torch.bucketize(t, start[1:], right=True)
    return s, st["kv_len"].long()[s] - (start[1:] - start[:-1])[s] + t - start[:-1][s]


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, within the range of the scales."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _plain_append(st):
    c = st["case"]
    nh, nkv, hd, rd, T = c["heads"], c["kv_heads"], c["hd"], c["rd"], c["page"]
    s, pos = _rows(st)
    x = st["qkv"].view(st["n"], nh + 2 * nkv, hd)
    # norm and rotation in 64 bits: the angles of far positions need them, and
    # the scales and codes must not hang on a 32-bit rounding
    qk = x[:, :nh + nkv].double()
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    gain = torch.cat([st["q_norm"].expand(nh, hd), st["k_norm"].expand(nkv, hd)]).double()
    qk = qk * gain
    half = rd // 2
    freq = ROPE_BASE ** (torch.arange(half, device=DEV, dtype=torch.float64) * (-2.0 / rd))
    angle = pos.double()[:, None] * freq
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = qk[..., :half], qk[..., half:rd]
    qk = torch.cat([a * cos - b * sin, a * sin + b * cos, qk[..., rd:]], -1).float()
    q, k, v = qk[:, :nh].contiguous(), qk[:, nh:], x[:, nh + nkv:]
    page = st["pages"][s, pos // T].long()
    h = torch.arange(nkv, device=DEV)
    o = pos % T
    if c["kvtype"] == "f16":
        st["k"][page[:, None], h, o[:, None]] = k.half()
        st["v"][page[:, None], h, (o // 32)[:, None], :, (o % 32)[:, None]] = v.half()
        return _state(st, q)
    kc, vc = st["k"].view(torch.uint8), st["v"].view(torch.uint8)
    NB = T // 32
    # the tokens that stay in the block in which a sequence's append begins
    start = st["q_start"].long()
    first = st["kv_len"].long() - (start[1:] - start[:-1])
    fp, fb = st["pages"][torch.arange(c["seqs"], device=DEV), first // T].long(), first % T // 32
    kept = torch.arange(32, device=DEV) < (first % 32)[:, None]              # [S, 32]
    slot = page * NB + o // 32
    for name, codes, new in (("k", kc, k), ("v", vc, v)):
        exps = st[name + "_exp"]
        flat = exps.transpose(1, 2).reshape(-1, nkv).int()                   # [pages NB, nkv]
        amax = torch.zeros(flat.shape, device=DEV)
        amax.scatter_reduce_(0, slot[:, None].expand(-1, nkv), new.abs().amax(-1), "amax")
        e = _exponent(amax)
        written = torch.zeros(flat.shape[0], dtype=torch.bool, device=DEV).index_fill_(0, slot, True)
        holds = torch.zeros_like(written).index_put_((fp * NB + fb,), first % 32 > 0)
        e = torch.where(holds[:, None], torch.maximum(e, flat), e)
        e = torch.where(written[:, None], e, flat)
        fe, oe = e[fp * NB + fb], flat[fp * NB + fb]                         # [S, nkv]
        grown = torch.ldexp(torch.ones((), device=DEV), oe - fe)
        code = torch.ldexp(new, -e[slot][..., None]).to(F8).view(torch.uint8)
        if name == "k":
            w = codes.view(-1, nkv, NB, 32, hd)
            old = w[fp, :, fb]                                               # [S, nkv, 32, hd]
            re = (old.view(F8).float() * grown[..., None, None]).to(F8).view(torch.uint8)
            w[fp, :, fb] = torch.where(kept[:, None, :, None], re, old)
            w[page[:, None], h, (o // 32)[:, None], (o % 32)[:, None]] = code
        else:
            w = codes                                                        # [P, nkv, NB, hd/2, 4, 2, 8]
            old = w[fp, :, fb]
            re = (old.view(F8).float() * grown[:, :, None, None, None, None]).to(F8).view(torch.uint8)
            w[fp, :, fb] = torch.where(kept.view(-1, 1, 1, 4, 1, 8), re, old)
            g, j = (o % 32 // 8)[:, None], (o % 8)[:, None]
            w[page[:, None], h, (o // 32)[:, None], :, g, :, j] = code.view(st["n"], nkv, hd // 2, 2)
        exps.copy_(e.view(-1, NB, nkv).transpose(1, 2).to(torch.int8))
    return _state(st, q)


def _values(st, name):
    """The whole cache's keys or values as f32 [pages, T, kv heads, head_dim]."""
    x = st[name].float()
    f8 = name + "_exp" in st
    if f8:
        scale = torch.ldexp(torch.ones((), device=DEV), st[name + "_exp"].int())
    T, hd = st["case"]["page"], st["case"]["hd"]
    P, nkv = x.shape[:2]
    if name == "k":
        if f8:
            x = (x.view(P, nkv, T // 32, 32, hd) * scale[..., None, None]).view(P, nkv, T, hd)
        return x.transpose(1, 2)
    if f8:
        x = x * scale.view(P, nkv, T // 32, 1, 1, 1, 1)
        return x.permute(0, 2, 4, 6, 1, 3, 5).reshape(P, T, nkv, hd)
    return x.permute(0, 2, 4, 1, 3).reshape(P, T, nkv, hd)


def _plain_attn(st):
    c = st["case"]
    nh, nkv, hd, B, S = c["heads"], c["kv_heads"], c["hd"], c["block"], c["seqs"]
    G, L, Q = nh // nkv, st["most_kv"], st["most_q"]
    s, pos = _rows(st)
    i = torch.arange(st["n"], device=DEV) - st["q_start"].long()[s]
    held = st["pages"].long().clamp_min(0)                                   # [S, pages]
    k = _values(st, "k")[held].flatten(1, 2)[:, :L]                          # [S, L, nkv, hd]
    v = _values(st, "v")[held].flatten(1, 2)[:, :L]
    q = torch.zeros((S, Q, nh, hd), device=DEV)
    q[s, i] = st["q"]
    last = torch.zeros((S, Q), dtype=torch.long, device=DEV)                 # keys that a row sees
    seen = st["kv_len"].long()[s]
    last[s, i] = torch.minimum(seen, (pos // B + 1) * B) if B > 0 else seen
    q = q.view(S, Q, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(S * nkv, G * Q, hd)
    k = k.permute(0, 2, 3, 1).reshape(S * nkv, hd, L).contiguous()
    v = v.transpose(1, 2).reshape(S * nkv, L, hd).contiguous()
    sc = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).view(S, nkv, G, Q, L)
    sc.masked_fill_((torch.arange(L, device=DEV) >= last[..., None])[:, None, None], -math.inf)
    sc = sc.sub_(sc.amax(-1, keepdim=True).clamp_min_(-3e38)).exp_()
    den = sc.sum(-1).clamp_min_(1e-30)
    o = torch.matmul(sc.view(S * nkv, G * Q, L), v).view(S, nkv, G, Q, hd) / den[..., None]
    return o.permute(0, 3, 1, 2, 4).reshape(S, Q, nh, hd)[s, i]


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["kind"] == "append" else _plain_attn(state)


# ---------------------------------------------------------------------------
# The definition in 64 bits, one sequence after the other

def _token(x, t, f8):
    """The values of token t of a block of V [.., block's shape] -> [.., hd]."""
    return x[..., t // 8, :, t % 8].flatten(-2) if f8 else x[..., t]


def exact(case, seed):
    st = prepare(case, seed)
    nq, kv = _lengths(case)
    nh, nkv, hd, rd, T, B = (case[m] for m in ("heads", "kv_heads", "hd", "rd", "page", "block"))
    f8, pages = case["kvtype"] == "e4m3", st["pages"].cpu().tolist()
    if work(case)["flops"] > 1e12 or sum(nq) > 8192:
        return None
    row = 0
    if case["kind"] == "append":
        k, v = st["k"].double(), st["v"].double()
        ke, ve = (st["k_exp"].clone(), st["v_exp"].clone()) if f8 else (None, None)
        queries = torch.empty((st["n"], nh, hd), dtype=torch.float64, device=DEV)
        pair = torch.arange(rd // 2, dtype=torch.float64, device=DEV)
        for s, (n, length) in enumerate(zip(nq, kv)):
            x = st["qkv"][row:row + n].double().view(n, -1, hd)
            p = torch.arange(length - n, length, dtype=torch.float64, device=DEV)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                               p[:, None] * torch.exp(pair * (-2.0 / rd * math.log(ROPE_BASE))))[:, None]

            def placed(y, gain):
                y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * gain.double()
                z = torch.complex(y[..., :rd // 2], y[..., rd // 2:rd]) * turn
                return torch.cat([z.real, z.imag, y[..., rd:]], -1)
            queries[row:row + n] = placed(x[:, :nh], st["q_norm"])
            keys, vals = placed(x[:, nh:nh + nkv], st["k_norm"]), x[:, nh + nkv:]
            at = length - n
            while at < length:
                end = min(length, at // 32 * 32 + 32)
                pg, b, a, z = pages[s][at // T], at % T // 32, at % 32, at % 32 + end - at
                nk, nv = (y[at - (length - n):end - (length - n)] for y in (keys, vals))
                if f8:
                    for held, exps, new, name in ((k, ke, nk, "k"), (v, ve, nv, "v")):
                        top = new.abs().amax((0, 2)).float().tolist()
                        old = exps[pg, :, b].tolist()
                        for h in range(nkv):
                            e = E_MIN
                            while e < E_MAX and top[h] > TOP * 2.0 ** e:
                                e += 1
                            e = max(e, old[h]) if a else e
                            if a:               # what is kept stands for the same values
                                part = held[pg, h, b * 32:b * 32 + a] if name == "k" else None
                                if name == "k":
                                    part *= 2.0 ** (old[h] - e)
                                else:
                                    for t in range(a):
                                        held[pg, h, b, :, t // 8, :, t % 8] *= 2.0 ** (old[h] - e)
                            exps[pg, h, b] = e
                    nk = nk / torch.exp2(ke[pg, :, b].double())[:, None]
                    nv = nv / torch.exp2(ve[pg, :, b].double())[:, None]
                k[pg, :, b * 32 + a:b * 32 + z] = nk.transpose(0, 1)
                for t in range(a, z):
                    if f8:
                        v[pg, :, b, :, t // 8, :, t % 8] = nv[t - a].view(nkv, hd // 2, 2)
                    else:
                        v[pg, :, b, :, t] = nv[t - a]
                at = end
            row += n
        return {"q": queries, "k": k, "v": v, **({"k_exp": ke, "v_exp": ve} if f8 else {})}
    out = torch.empty((st["n"], nh, hd), dtype=torch.float64, device=DEV)
    for s, (n, length) in enumerate(zip(nq, kv)):
        pg = torch.tensor(pages[s][:-(-length // T)], device=DEV)
        x, y = st["k"][pg].double(), st["v"][pg].double()
        if f8:
            x = x * torch.exp2(st["k_exp"][pg].double()).repeat_interleave(32, -1)[..., None]
            y = torch.stack([_token(y, t, True) for t in range(32)], 3)      # [pages, nkv, NB, 32, hd]
            y = y * torch.exp2(st["v_exp"][pg].double())[..., None, None]
        else:
            y = torch.stack([_token(y, t, False) for t in range(32)], 3)
        x = x.transpose(0, 1).flatten(1, 2)[:, :length]                      # [nkv, L, hd]
        y = y.transpose(0, 1).flatten(1, 3)[:, :length]
        step = max(1, (1 << 28) // (length * (nh // nkv)))
        for i in range(0, n, step):
            m = min(step, n - i)
            q = st["q"][row + i:row + i + m].double().view(m, nkv, nh // nkv, hd)
            p = torch.arange(length - n + i, length - n + i + m, device=DEV)
            sees = torch.clamp((p // B + 1) * B, max=length) if B > 0 else torch.full_like(p, length)
            hide = torch.arange(length, device=DEV) >= sees[:, None]
            for h in range(nkv):
                w = (q[:, h].reshape(-1, hd) @ x[h].T.contiguous()).view(m, nh // nkv, length) / math.sqrt(hd)
                w = torch.softmax(w.masked_fill(hide[:, None], -math.inf), -1)
                out[row + i:row + i + m].view(m, nkv, nh // nkv, hd)[:, h] = \
                    (w.flatten(0, 1) @ y[h]).view(m, nh // nkv, hd)
        row += n
    return out
