"""The paged KV cache in numpy, 64 bits: batches for the tests, the cache's
layouts read and written one token at a time, and the definitions of the append
and of the attention."""
import numpy as np
import torch

E_MIN, E_MAX, TOP = -50, 50, 448.0
F8 = torch.float8_e4m3fn


class Batch:
    """seqs: (tokens cached before the call, rows of the call) of each sequence.
    Pages are dealt out in a shuffled order; `extra` rows follow the last
    sequence's, `spare` pages belong to no one."""

    def __init__(self, seqs, T, seed=0, extra=0, spare=2, wide=0):
        self.seqs, self.T, self.extra = list(seqs), T, extra
        self.kv_len = np.array([o + n for o, n in seqs], np.int32)
        self.q_start = np.concatenate([[0], np.cumsum([n for _, n in seqs])]).astype(np.int32)
        self.n_tokens = int(self.q_start[-1]) + extra
        need = [-(-int(k) // T) for k in self.kv_len]
        self.n_pages = sum(need) + spare
        ids = np.random.RandomState(seed).permutation(self.n_pages)
        self.pages = np.full((len(seqs), max(1, wide, max(need))), -1, np.int32)
        at = 0
        for s, m in enumerate(need):
            self.pages[s, :m] = ids[at:at + m]
            at += m

    def device(self, dmoe, dev="cuda:0"):
        t = [torch.from_numpy(np.ascontiguousarray(x)).to(dev) for x in (self.q_start, self.kv_len, self.pages)]
        return dmoe.KvBatch(*t, self.n_tokens)

    def place(self, s, p):
        """(page, token within it) of token p of sequence s, None if nothing holds it."""
        i = p // self.T
        if i >= self.pages.shape[1] or not 0 <= self.pages[s, i] < self.n_pages:
            return None
        return int(self.pages[s, i]), p % self.T


class Cache:
    """The cache's tensors on the CPU: raw bytes as they lie on the GPU."""

    def __init__(self, kvtype, n_pages, nkv, hd, T, seed=0, poison=False):
        self.f8, self.nkv, self.hd, self.T = kvtype == "e4m3", nkv, hd, T
        g = torch.Generator().manual_seed(seed)
        kshape = (n_pages, nkv, T, hd)
        vshape = (n_pages, nkv, T // 32) + ((hd // 2, 4, 2, 8) if self.f8 else (hd, 32))
        if self.f8:
            make = lambda s: (torch.randn(s, generator=g) * 60).clamp(-TOP, TOP).to(F8)  # noqa: E731
            self.k_exp, self.v_exp = (torch.randint(-9, -4, (n_pages, nkv, T // 32), generator=g, dtype=torch.int8)
                                      for _ in range(2))
        else:
            make = lambda s: torch.randn(s, generator=g).half()  # noqa: E731
            self.k_exp = self.v_exp = None
        self.k, self.v = make(kshape), make(vshape)
        if poison:                      # memory that was never written: NaN codes, any exponent
            for t in (self.k, self.v):
                t.view(torch.uint8).fill_(0xff)
            if self.f8:
                self.k_exp.fill_(127)
                self.v_exp.fill_(127)

    def copy(self):
        c = object.__new__(Cache)
        c.__dict__ = {m: (x.clone() if isinstance(x, torch.Tensor) else x) for m, x in self.__dict__.items()}
        return c

    def device(self, dmoe, dev="cuda:0"):
        return dmoe.KvCache(*[x if x is None else x.to(dev) for x in (self.k, self.v, self.k_exp, self.v_exp)])

    @classmethod
    def of(cls, kv):
        c = object.__new__(cls)
        c.k, c.v, c.k_exp, c.v_exp = [x if x is None else x.cpu() for x in (kv.k, kv.v, kv.k_exp, kv.v_exp)]
        c.f8, (_, c.nkv, c.T, c.hd) = c.k_exp is not None, c.k.shape
        return c

    def codes(self, which):
        """[n_pages, nkv, T, hd]: the stored numbers, values written out as [token][dim] (a copy for v)."""
        if which == "k":
            return self.k
        x = self.v.view(torch.uint8) if self.f8 else self.v
        x = x.permute(0, 1, 2, 4, 6, 3, 5) if self.f8 else x.transpose(3, 4)
        x = x.reshape(self.k.shape)
        return x.contiguous().view(F8) if self.f8 else x

    def values(self, which):
        x = self.codes(which).double().numpy()
        if self.f8:
            e = (self.k_exp if which == "k" else self.v_exp).double().numpy()
            x = x * np.repeat(2.0 ** e, 32, axis=2)[..., None]
        return x

    def same(self, other):
        pairs = [(self.k, other.k), (self.v, other.v)] + ([(self.k_exp, other.k_exp), (self.v_exp, other.v_exp)] if self.f8 else [])
        return all(np.array_equal(a.contiguous().view(torch.uint8).numpy(), b.contiguous().view(torch.uint8).numpy())
                   for a, b in pairs)


def exponent(amax):
    e = E_MIN
    while e < E_MAX and amax > TOP * 2.0 ** e:
        e += 1
    return e


def placed(x, gain, pos, rd, base, eps):
    """RMSNorm (gain not None) and rotation of rows x [n, heads, hd] at pos [n]."""
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    half = rd // 2
    if half:
        ang = pos.astype(np.longdouble)[:, None] * np.longdouble(base) ** (np.arange(half) * np.longdouble(-2.0) / rd)
        c, s = (f(ang).astype(np.float64)[:, None] for f in (np.cos, np.sin))
        a, b = x[..., :half].copy(), x[..., half:rd].copy()
        x = x.copy()
        x[..., :half], x[..., half:rd] = a * c - b * s, a * s + b * c
    return x


def rows_of(batch, qkv, nh, nkv, hd, rd, base, eps, qn, kn):
    """q, k, v [n_tokens, heads, hd] in 64 bits, position of each row (-1: of no sequence)."""
    x = qkv.reshape(batch.n_tokens, nh + 2 * nkv, hd)
    pos = np.full(batch.n_tokens, -1)
    for s, (o, n) in enumerate(batch.seqs):
        pos[batch.q_start[s]:batch.q_start[s] + n] = np.arange(o, o + n)
    q = placed(x[:, :nh], qn, np.maximum(pos, 0), rd, base, eps)
    k = placed(x[:, nh:nh + nkv], kn, np.maximum(pos, 0), rd, base, eps)
    return q, k, x[:, nh + nkv:].astype(np.float64), pos


def attend(batch, cache, q, block, extra_seen=None):
    """The attention's definition; q [n_tokens, nh, hd] -> the same shape, rows
    of no sequence NaN; also the largest |value| and sum of |q k| / sqrt(hd)
    that a row met."""
    nh, hd = q.shape[1:]
    G = nh // cache.nkv
    out = np.full(q.shape, np.nan)
    K, V = cache.values("k"), cache.values("v")
    top_v = top_s = 0.0
    for s, (o, n) in enumerate(batch.seqs):
        length = o + n
        held = [batch.place(s, p) for p in range(length)]
        idx = np.array([p for p in range(length) if held[p] is not None], np.int64)
        at = np.array([held[p] for p in idx], np.int64).reshape(-1, 2)
        for i in range(n):
            row, p = batch.q_start[s] + i, o + i
            see = idx < min(length, (p // block + 1) * block) if block > 0 else np.ones(len(idx), bool)
            if not see.any():
                out[row] = 0.0
                continue
            k, v = (x[at[see, 0], :, at[see, 1]] for x in (K, V))            # [L, nkv, hd]
            qq = q[row].astype(np.float64).reshape(cache.nkv, G, hd)
            with np.errstate(all="ignore"):
                sc = np.einsum("hgd,lhd->hgl", qq, k) / np.sqrt(hd)
                w = np.exp(sc - sc.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[row] = np.einsum("hgl,lhd->hgd", w, v).reshape(nh, hd)
                top_v = max(top_v, np.nanmax(np.abs(v)))
                top_s = max(top_s, np.nanmax(np.einsum("hgd,lhd->hgl", np.abs(qq), np.abs(k))) / np.sqrt(hd))
    return out, top_v, top_s


def attend_tolerance(top_v, top_s, hd, longest):
    """Largest absolute error of the attention in f32: a score is a sum of 2 hd
    / 32 MFMA results in f32 (each step off by at most 2^-24 of the partial sums,
    the operands' split by 2^-22, the factors by 2 * 2^-24), exp2 of a rounded
    argument by 2^-22 and an ulp or two; a weight is then off by that much twice
    (itself and the sum), and the output's own sum over longest / 32 tiles by
    2^-24 each, with the split probabilities' 2^-22 and the division."""
    ds = (2 * hd / 32 + 4 + 3) * 2.0 ** -24 * top_s + 2.0 ** -21
    return top_v * (2 * ds + (longest / 32 + 8) * 2.0 ** -24)
