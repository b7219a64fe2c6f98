"""CPU: what the paged KV cache's entry points refuse and how its kernels read
a batch's tables (csrc/dmoe_kv_plan.h, pure functions): every index stays in its
buffer whatever the tables hold, and the item bound covers every batch."""
import itertools
import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
BAD, TYPE, SHAPE = 1, 2, 3

PROBE = r"""
#include <cstdio>
#include <cstring>
#include "%s"
using namespace dmoe;
int main() {
  char op[16];
  long long v[40];
  while (scanf(" %%15s", op) == 1) {
    int n = 0;
    if (scanf(" %%d", &n) != 1) return 1;
    for (int i = 0; i < n; i++) if (scanf(" %%lld", &v[i]) != 1) return 1;
    if (!strcmp(op, "seq")) {
      KvSeq q = kv_seq_of(v[0], v[1], v[2], v[3]);
      printf("%%d %%d %%d %%d\n", q.q0, q.n, q.len, kv_blocks(q));
    } else if (!strcmp(op, "most")) printf("%%lld\n", (long long)kv_blocks_most(v[0], v[1]));
    else if (!strcmp(op, "byrow")) printf("%%d\n", (int)kv_by_row(v[0], v[1]));
    else if (!strcmp(op, "place")) printf("%%d\n", kv_place(v[0], v[1], v[2]));
    else if (!strcmp(op, "entry")) printf("%%d\n", kv_entry_of(v[0], v[1], v[2]));
    else if (!strcmp(op, "page")) printf("%%d\n", kv_page_of(v[0], v[1]));
    else if (!strcmp(op, "sees")) printf("%%d\n", kv_visible(v[0], kv_cached(v[1], v[2], v[3]), v[4]));
    else {
      dmoe_kv_cache kv{(int)v[0], (int)v[1], (int)v[2], (int)v[3], (int)v[4], (void *)v[5], (void *)v[6], (int8_t *)v[7], (int8_t *)v[8]};
      dmoe_kv_batch b{(int)v[9], (int)v[10], (int)v[11], (const int32_t *)v[12], (const int32_t *)v[13], (const int32_t *)v[14]};
      dmoe_attn_hparams a{(int)v[15], (int)v[16], (int)v[17], (int)v[18], (int)v[19], (int)v[20], (int)v[21], (float)v[22], (float)v[23]};
      const void *x = (void *)v[24], *y = (void *)v[25], *z = (void *)v[26], *w = (void *)v[27];
      KvRefusal r;
      if (!strcmp(op, "append")) kv_check_append(r, &kv, &b, &a, x, z, w, y);
      else if (!strcmp(op, "attn")) kv_check_attn(r, &kv, &b, &a, x, y);
      else if (!strcmp(op, "layer")) kv_check_layer(r, &kv, &b, &a, x, y, z);
      else if (!strcmp(op, "ws")) kv_check_workspace(r, x, v[25], v[26]);
      else if (!strcmp(op, "sizes")) kv_check(r, &kv, &b, &a, false);
      else if (!strcmp(op, "null")) kv_check(r, v[0] ? &kv : nullptr, v[1] ? &b : nullptr, v[2] ? &a : nullptr, true);
      else return 1;
      printf("%%d %%s\n", r.code, r.why);
    }
  }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("kvplan")
    src = d / "probe.cpp"
    src.write_text(PROBE % (ROOT / "diffuse-cpp_amd" / "csrc" / "dmoe_kv_plan.h"))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-o",
                    str(d / "probe"), str(src)], check=True)

    def f(calls):
        text = "\n".join(f"{op} {len(v)} {' '.join(str(int(x)) for x in v)}" for op, v in calls)
        out = subprocess.run([str(d / "probe")], input=text, capture_output=True, text=True, check=True).stdout
        return out.splitlines()
    return f


FIELDS = ("type n_head_kv head_dim page_tokens n_pages k v k_exp v_exp n_seqs n_tokens max_pages q_start kv_len pages "
          "n_embd n_head ap_kv ap_hd rotary_dim use_qk_norm block_length rope_base rms_eps x y z w").split()
GOOD = dict(type=1, n_head_kv=4, head_dim=128, page_tokens=64, n_pages=10, k=1 << 32, v=2 << 32, k_exp=3 << 32,
            v_exp=4 << 32, n_seqs=2, n_tokens=33, max_pages=5, q_start=5 << 32, kv_len=6 << 32, pages=7 << 32,
            n_embd=4096, n_head=32, ap_kv=4, ap_hd=128, rotary_dim=64, use_qk_norm=1, block_length=32, rope_base=10000,
            rms_eps=0, x=8 << 32, y=9 << 32, z=10 << 32, w=11 << 32)


def _call(op, **kw):
    return op, [{**GOOD, **kw}[f] for f in FIELDS]


def test_good_arguments_pass(ask):
    calls = [_call(op, **kw) for op in ("append", "attn", "layer", "sizes")
             for kw in ({}, dict(type=0, k_exp=0, v_exp=0), dict(head_dim=64, ap_hd=64), dict(n_head=4), dict(n_tokens=1),
                        dict(n_tokens=(1 << 27) // 40, x=20 << 32, y=90 << 32, z=160 << 32), dict(n_seqs=(1 << 24) // 40),
                        dict(y=(2 << 32) + 10 * 4 * 64 * 128), dict(page_tokens=32), dict(block_length=0), dict(block_length=-1), dict(rotary_dim=0),
                        dict(rotary_dim=128, head_dim=128))]
    calls += [_call("append", use_qk_norm=0, z=0, w=0), _call("layer", z=0), _call("layer", y=GOOD["x"])]
    for c, r in zip(calls, ask(calls)):
        assert r.startswith("0"), (c, r)


REFUSED = [
    ("append attn layer sizes", TYPE, dict(type=2)), ("append attn layer sizes", TYPE, dict(type=-1)),
    ("append attn layer sizes", SHAPE, dict(head_dim=96, ap_hd=96)), ("append attn layer sizes", SHAPE, dict(ap_hd=64)),
    ("append attn layer sizes", SHAPE, dict(page_tokens=48)), ("append attn layer sizes", SHAPE, dict(page_tokens=0)),
    ("append attn layer sizes", SHAPE, dict(page_tokens=-64)), ("append attn layer sizes", SHAPE, dict(n_pages=0)),
    ("append attn layer sizes", SHAPE, dict(n_head_kv=0, ap_kv=0)), ("append attn layer sizes", SHAPE, dict(n_head=30)),
    ("append attn layer sizes", SHAPE, dict(ap_kv=8)), ("append attn layer sizes", SHAPE, dict(n_head=0)),
    ("append attn layer sizes", BAD, dict(n_seqs=0)), ("append attn layer sizes", BAD, dict(n_tokens=0)),
    ("append attn layer sizes", BAD, dict(n_tokens=-1)), ("append attn layer sizes", BAD, dict(max_pages=0)),
    ("append attn layer sizes", SHAPE, dict(n_tokens=1 << 30)), ("append attn layer sizes", SHAPE, dict(n_seqs=1 << 21)),
    ("append attn layer", BAD, dict(k=0)), ("append attn layer", BAD, dict(v=0)), ("append attn layer", BAD, dict(k_exp=0)),
    ("append attn layer", BAD, dict(v_exp=0)), ("append attn layer", BAD, dict(k=(1 << 32) + 8)),
    ("append attn layer", BAD, dict(v=(2 << 32) + 1)), ("append attn layer", BAD, dict(v=(1 << 32) + 16)),
    ("append attn layer", BAD, dict(v_exp=(3 << 32) + 1)),
    ("append attn layer", BAD, dict(q_start=0)), ("append attn layer", BAD, dict(kv_len=0)),
    ("append attn layer", BAD, dict(pages=0)), ("append attn layer", BAD, dict(pages=(7 << 32) + 2)),
    ("append attn layer", BAD, dict(x=0)), ("append attn layer", BAD, dict(y=0)),
    ("append attn layer", BAD, dict(x=(8 << 32) + 4)), ("append attn layer", BAD, dict(y=(9 << 32) + 8)),
    ("append attn layer", BAD, dict(y=(8 << 32) + 16)), ("attn", BAD, dict(y=8 << 32)),
    ("append", BAD, dict(z=0)), ("append", BAD, dict(w=0)), ("append", BAD, dict(z=(10 << 32) + 2)),
    ("append", BAD, dict(y=8 << 32)), ("append", BAD, dict(y=(8 << 32) + 33 * 40 * 128 * 4 - 16)),
    ("layer", BAD, dict(z=8 << 32)), ("layer", BAD, dict(z=9 << 32)), ("layer", BAD, dict(z=(10 << 32) + 4)),
    ("append attn layer sizes", SHAPE, dict(n_tokens=(1 << 27) // 40 + 1)),
    ("append attn layer sizes", SHAPE, dict(n_seqs=(1 << 24) // 40 + 1)),
    ("append attn layer sizes", SHAPE, dict(n_tokens=(1 << 31) - 1, n_head=(1 << 31) - 1, ap_kv=(1 << 31) - 1, n_head_kv=(1 << 31) - 1)),
    ("append attn layer", BAD, dict(y=(1 << 32) + 16)), ("append attn layer", BAD, dict(y=(2 << 32) + 10 * 4 * 64 * 128 - 16)),
    ("append attn layer", BAD, dict(y=3 << 32)), ("append attn layer", BAD, dict(y=(4 << 32) - 16)),
    ("append layer", BAD, dict(x=(1 << 32) - 16)), ("layer", BAD, dict(z=2 << 32)),
    ("append layer", SHAPE, dict(rotary_dim=130)), ("append layer", SHAPE, dict(rotary_dim=63)),
    ("append layer", SHAPE, dict(rotary_dim=-2)), ("append layer", BAD, dict(rope_base=0)),
    ("append layer", BAD, dict(rope_base=-1)), ("append layer", BAD, dict(rms_eps=-1)),
]


@pytest.mark.parametrize("ops,code,change", REFUSED, ids=[f"{o.split()[0]}-{c}" for o, _, c in REFUSED])
def test_refusals(ask, ops, code, change):
    calls = [_call(op, **change) for op in ops.split()]
    for c, r in zip(calls, ask(calls)):
        status, why = r.split(" ", 1)
        assert int(status) == code and why, (c, r)


def test_refusals_of_null_structs_and_workspaces(ask):
    for r in ask([("null", [0, 1, 1]), ("null", [1, 0, 1]), ("null", [1, 1, 0])]):
        assert r.startswith("1 ")
    # (workspace, its bytes, the bytes needed)
    got = ask([_call("ws", x=1 << 32, y=b, z=256) for b in (256, 255, 0)] + [_call("ws", x=(1 << 32) + 4, y=512, z=256)])
    assert [r.split(" ")[0] for r in got] == ["0", "1", "1", "1"]


def test_sequences_of_any_table_stay_in_the_buffers(ask):
    big = 2 ** 31 - 1
    most = 1 << 30
    edge = [-2 ** 31, -1, 0, 1, 31, 32, 33, 100, 101, most, most + 1, big]
    calls = [("seq", [a, b, k, n]) for a, b, k in itertools.product(edge, edge, edge) for n in (1, 100)]
    for (_, (a, b, k, n)), r in zip(calls, ask(calls)):
        q0, rows, length, blocks = map(int, r.split())
        ok = 0 <= a <= b <= n and b - a <= k <= most
        assert rows == (b - a if ok else 0)
        if rows:
            assert 0 <= q0 and q0 + rows <= n and length - rows >= 0
            assert blocks == (length - 1) // 32 - (length - rows) // 32 + 1
        else:
            assert blocks == 0


def test_the_item_bound_covers_every_batch(ask):
    rng = random.Random(7)
    for _ in range(200):
        seqs = [(rng.choice((0, 1, 31, rng.randrange(5000))), rng.choice((0, 1, 1, 2, 32, 33, rng.randrange(300))))
                for _ in range(rng.randrange(1, 40))]
        n = sum(b for _, b in seqs)
        if n == 0:
            continue
        blocks = sum((o + b - 1) // 32 - o // 32 + 1 for o, b in seqs if b)
        assert blocks <= int(ask([("most", [len(seqs), n])])[0])


def test_pages_and_masks(ask):
    big = 2 ** 31 - 1
    assert ask([("entry", [p, 64, 5]) for p in (0, 63, 64, 319, 320, big)]) == ["0", "0", "1", "4", "-1", "-1"]
    assert ask([("page", [e, 7]) for e in (0, 6, 7, -1, big, -2 ** 31)]) == ["0", "6", "-1", "-1", "-1", "-1"]
    # (position, cached tokens, page, entries, block)
    cases = [(0, 1, 32, 9, 1), (5, 40, 32, 9, 1), (5, 40, 32, 9, 32), (39, 40, 32, 9, 32), (5, 40, 32, 9, 0),
             (5, 40, 32, 1, 0), (big - 1, big, 64, 1 << 25, 32), (big - 1, big, 64, 1 << 26, 32), (9, 40, 32, 9, big)]
    want = [1, 6, 32, 40, 40, 32, 1 << 31, big, 40]
    want[6] = min(big, 64 * (1 << 25))
    assert [int(x) for x in ask([("sees", list(c)) for c in cases])] == want


def test_structs_lie_as_in_c(tmp_path):
    """The ctypes mirrors have the size and offsets of include/dmoe.h's."""
    import ctypes
    from dmoe import _abi
    pairs = (("dmoe_kv_cache", _abi.KvCacheStruct), ("dmoe_kv_batch", _abi.KvBatchStruct))
    src = tmp_path / "layout.c"
    body = "".join(f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for f, _ in c._fields_)
                   for n, c in pairs)
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{ROOT}/include/dmoe.h"\nint main(void) {{ {body} return 0; }}\n')
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    want = [x for _, c in pairs for x in [ctypes.sizeof(c)] + [getattr(c, f).offset for f, _ in c._fields_]]
    assert got == want


def test_tensors_that_the_mirror_refuses():
    """Caches and batches of tensors that are not on a GPU, of other types, shapes or strides."""
    import dmoe
    import torch
    k = torch.zeros(3, 2, 64, 64, dtype=torch.float16)
    v = torch.zeros(3, 2, 2, 64, 32, dtype=torch.float16)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    for make in (lambda: dmoe.KvCache(k, v), lambda: dmoe.KvCache(k[0], v), lambda: dmoe.KvCache(k, v[:, :, :1]),
                 lambda: dmoe.KvCache(k.float(), v), lambda: dmoe.KvCache(k, v.transpose(3, 4)),
                 lambda: dmoe.KvCache(k[:, :, :40], v), lambda: dmoe.KvBatch(i(3), i(2), i(2, 4), 9),
                 lambda: dmoe.KvBatch(i(2), i(2), i(2, 4), 9), lambda: dmoe.KvBatch(i(3), i(2), i(3, 4), 9),
                 lambda: dmoe.KvBatch(i(3), i(2).long(), i(2, 4), 9), lambda: dmoe.KvBatch(i(3), i(2), i(4, 2).T, 9)):
        with pytest.raises(ValueError):
            make()


def test_every_block_has_a_place_of_its_own(ask):
    """kv_place's list: the blocks of ragged batches, sequences without rows among
    them, lie in disjoint places within the launch's bound, in order."""
    rng = random.Random(8)
    for _ in range(100):
        seqs = [(rng.choice((0, 1, 31, rng.randrange(5000))), rng.choice((0, 0, 1, 1, 2, 32, 33, rng.randrange(300))))
                for _ in range(rng.randrange(1, 90))]
        n = sum(b for _, b in seqs)
        if n == 0:
            continue
        starts = [sum(b for _, b in seqs[:i]) for i in range(len(seqs) + 1)]
        by_row = int(ask([("byrow", [len(seqs), n])])[0])
        places = [int(x) for x in ask([("place", [starts[i], i, by_row]) for i in range(len(seqs) + 1)])]
        most = int(ask([("most", [len(seqs), n])])[0])
        for i, (o, b) in enumerate(seqs):
            blocks = (o + b - 1) // 32 - o // 32 + 1 if b else 0
            assert places[i] + blocks <= places[i + 1] <= most
