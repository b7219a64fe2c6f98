// k_kv_attn.hip — attention over a paged KV cache (the cached form of
// src/diffuse-moe-graph.cpp:158-170): out[t, h] = sum_j softmax_j(q[t, h] .
// k[j] / sqrt(hd)) v[j] over the tokens j that row t's mask (:19-55) shows it,
// one pass over the cache with the running maximum and sum of the softmax.
//
// The products run on v_mfma_f32_16x16x32_f16 with tokens as rows and
// (query, head) pairs of one kv head as columns, S^T = K Q^T and O^T = V^T P^T:
// every lane then holds scores of one column, and the probabilities it forms
// are, in place, its operand of the second product (no exchange through LDS).
// Cached F16 and E4M3 values are exact in f16; a query row is scaled by a power
// of two to a largest magnitude of 128 to 256 and split into f16 hi + lo, a
// probability (times 2^KA_SHIFT) likewise: 22 significant bits with the low part well
// inside f16's range, f32 accumulation, so two MFMAs per product give the f32
// result to within its own rounding whatever the magnitude of the queries.
//
// E4M3: key and value of token j are code * 2^ke and code * 2^ve of its block.
// 2^ke goes into the scores' factor; ve is added to the exponent of the
// probabilities (p' = 2^(s + ve - m'), at most 2^KA_SLACK), and the
// sum takes p' 2^-ve: no operand is rescaled.  With exponents within 100 of
// each other no p' that counts in the sum underflows.
#include <algorithm>
#include <type_traits>

#include "dmoe_kv.h"

#pragma clang fp contract(off)

namespace dmoe {

// Times: 32 query and 4 kv heads of 128, kernel and join, in us.
constexpr int KA_WAVES = 4;              // wavefronts of a workgroup
constexpr int KW_WAVES = 4;              // .. of k_kv_attn_wide
constexpr int KA_SHIFT = 4;              // probabilities are held times 2^KA_SHIFT
// .. and may pass that by 2^KA_SLACK (f16 reaches 2^16) before their column's
// reference is raised: a block of 32 rows on 16,384 tokens 29.2, with 0 34.8
constexpr int KA_SLACK = 8;
constexpr int KA_COLS = 32;              // columns of an item at most
// A sequence of up to KA_WHOLE token tiles has one chunk, the others chunks of
// KA_CHUNK tiles at least: one row on 512 F16 tokens takes 12.4 whole, cut 9.3 and
// 3.6 for the join; on 700 14.8 whole, 9.5 + 3.4 in chunks of four tiles, 11.3 +
// 3.8 of eight.  A CU takes in about 50 GB/s, so that more of them pay early.
constexpr int KA_WHOLE = 16;
constexpr int KA_CHUNK = 4;
// Items wanted of a call, two workgroups for each of 256 CUs.  (256 of eight
// wavefronts: 131,072 tokens of one row the same, 48 sequences of one row 61, not 48.)
constexpr int KA_ITEMS = 512;
// Columns of all kv heads from which on k_kv_attn_wide runs, a workgroup for 128
// of them: it reads a token tile once for them, where k_kv_attn does it for 32, but
// needs a workgroup on every CU, two for E4M3 whose tiles are half the bytes.
// Prompts of 1024, 1536 and 2000 rows, wide against not: F16 50 / 56, 69 / 87,
// 89 / 129, E4M3 47 / 43, 67 / 68, 86 / 99; 1024 rows beside 48 of one on 1000
// tokens 77 / 68 and 69 / 49, beside 16 blocks of 32 on 2048 104 / 106 and 99 / 80,
// 1792 beside 8 103 / 133 and 100 / 101.
constexpr int KA_WIDE_F16 = 32768, KA_WIDE_E4M3 = 57344;
// It does not cut a sequence's tokens, so beside others it takes those with up to
// KA_LONG token tiles or 1 / KA_SHARE of the tiles of all its workgroups (an item's
// share is 1 / KA_ITEMS), which no one waits for long.  31 blocks of 32 rows on
// 1024 tokens and one on 32,768: 115 (F16) and 100 (E4M3), with KA_LONG 16 390 and
// 332, without a limit 1495 and 1433; four times 512 rows on 4000 tokens 270 and
// 258, cut 401 and 283; prompts of 2000, 500 on 6000 and 300 on 1000 252 and 209,
// all of them taken (a 256th) 263 and 262.
constexpr int KA_LONG = 64, KA_SHARE = 384;

// one 16-byte piece of cache as f16: F16 8 values, E4M3 16
template <bool F8>
__device__ __forceinline__ void kv_widen(const uint4 &x, kv_h8 (&o)[F8 ? 2 : 1])
{
    if constexpr (F8) {
        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const kv_h2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u[i], 1.0f, false);
            const kv_h2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u[i], 1.0f, true);
            o[i / 2][4 * (i % 2) + 0] = lo[0];
            o[i / 2][4 * (i % 2) + 1] = lo[1];
            o[i / 2][4 * (i % 2) + 2] = hi[0];
            o[i / 2][4 * (i % 2) + 3] = hi[1];
        }
    } else {
        o[0] = __builtin_bit_cast(kv_h8, x);
    }
}

// f16(p - hi), both halves: the difference is exact in f32
__device__ __forceinline__ kv_h2 kv_rest(const kv_f2 &p, const kv_h2 &hi)
{
    kv_f2 r;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(hi), "v"(p[0]));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(hi), "v"(p[1]));
    return __builtin_convertvector(r, kv_h2);
}

// tokens 8 g .. 8 g + 7 of a block, those from `lim` on set to zero
__device__ __forceinline__ kv_h8 kv_cut(const kv_h8 &v, int g, int lim)
{
    uint4 x = __builtin_bit_cast(uint4, v);
    uint32_t *u = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
    for (int i = 0; i < 4; i++)
        u[i] &= (8 * g + 2 * i < lim ? 0xffffu : 0u) | (8 * g + 2 * i + 1 < lim ? 0xffff0000u : 0u);
    return __builtin_bit_cast(kv_h8, x);
}

// ---------------------------------------------------------------------------
// Work items.  A sequence's columns (query, head of a kv head) form tiles of 16
// (up to 16 columns in all) or 32, its cached tokens tiles of 32; an item is
// one column tile of one kv head over one chunk of token tiles.  The chunk
// length is common to all sequences, so that ragged ones spread over the chip
// like one: the total of (column tile, token tile) pairs over the items wanted,
// at least KA_CHUNK.  A sequence's chunks are then made equally long, and one of
// up to KA_WHOLE token tiles is not cut.
//
// A sequence's items lie kv heads first, then chunks, then column tiles: what
// reads the same keys is a multiple of the kv heads apart, and as workgroups go
// to the 8 XCDs in turn, it shares few L2s (with 4 or 8 kv heads an XCD meets
// two heads or one).
struct KvItem {
    KvSeq q;
    int s, kvh, tile, split;             // sequence, kv head, column tile, chunk
    int cb;                              // 16-column blocks of a tile
    int ks, chunk;                       // chunks of the sequence, token tiles of each
    int part, unit;                      // of a sequence with several chunks: among such items, and among such
                                         // (column tile, kv head)s
};

// 16-column blocks of a tile of a sequence with `cols` columns.  (Two for few
// columns too: one row on 700 tokens 11.0, not 9.5, on 131,072 33.0, not 30.3.)
__device__ __forceinline__ int kv_blocks_of_tile(int cols) { return cols <= 16 ? 1 : 2; }

__device__ __forceinline__ int kv_token_tiles(const KvAttnArgs &a, const KvSeq &q)
{
    return q.n ? (kv_cached(q.len, a.c.T, a.b.max_pages) + 31) / 32 : 0;
}

// The most token tiles of a sequence that k_kv_attn_wide takes beside others, from
// the sum of what it could take.
__device__ __forceinline__ float kv_wide_work(const KvAttnArgs &a, const KvSeq &q, int G)
{
    const int cols = q.n * G;
    return cols > a.wide ? (float)((cols + 32 * KW_WAVES - 1) / (32 * KW_WAVES)) * (float)kv_token_tiles(a, q) : 0.0f;
}

__device__ __forceinline__ float kv_longest(const KvAttnArgs &a, float work)
{
    return fmaxf((float)KA_LONG, work * (float)a.nkv * (1.0f / (float)KA_SHARE));
}

// Whether k_kv_attn_wide takes a sequence of a call in which it runs.
__device__ __forceinline__ bool kv_is_wide(const KvAttnArgs &a, const KvSeq &q, int G, float longest)
{
    return q.n * G > a.wide && (a.wide == 0 || (float)kv_token_tiles(a, q) <= longest);
}

__device__ __forceinline__ int kv_col_tiles(const KvAttnArgs &a, const KvSeq &q, int G, float longest)
{
    const int cols = q.n * G, per = 16 * kv_blocks_of_tile(cols);
    return kv_is_wide(a, q, G, longest) ? 0 : (cols + per - 1) / per;
}

// Column tiles of the sequences that are not cut and of the others, and their pairs
// of tiles (exact enough: lengths, not indexes).
struct KvWork {
    float few, many, rest, work;
};
__device__ __forceinline__ void kv_add_work(const KvAttnArgs &a, const KvSeq &q, int G, float longest, KvWork &sum)
{
    const float tiles = (float)kv_col_tiles(a, q, G, longest);
    const int length = kv_token_tiles(a, q);
    (length > KA_WHOLE ? sum.many : sum.few) += tiles;
    (length > KA_WHOLE ? sum.work : sum.rest) += tiles * (float)length;
}

// Chunks of a sequence.
__device__ __forceinline__ int kv_cuts(int length, int C)
{
    return length > KA_WHOLE ? (int)((uint32_t)(length + C - 1) / (uint32_t)C) : 1;
}

// The chunk length.  What all can start at once is shared out; a column tile's last
// chunk is half empty on average, and where that is not enough the count of chunks
// says by how much.  If that would make a chunk twice as long as an item's share of
// all the work, the items start one after the other anyhow, and the share it is.
__device__ __forceinline__ float kv_chunk(const KvAttnArgs &a, const KvWork &sum)
{
    const float all = (float)KA_ITEMS / (float)a.nkv;
    return sum.work / fmaxf(all - sum.few - 0.5f * sum.many, 0.25f * all) + 1.0f;
}
__device__ __forceinline__ float kv_chunks(const KvAttnArgs &a, const KvSeq &q, int G, float longest, float c)
{
    const int length = kv_token_tiles(a, q), C = max(KA_CHUNK, (int)c);
    return length > KA_WHOLE ? (float)(kv_col_tiles(a, q, G, longest) * kv_cuts(length, C)) : 0.0f;
}
__device__ __forceinline__ int kv_chunk(const KvAttnArgs &a, const KvWork &sum, float c, float count)
{
    const float all = (float)KA_ITEMS / (float)a.nkv, share = (sum.work + sum.rest) / all + 1.0f;
    if (count > all - sum.few) c = fmaxf(fmaxf((float)KA_CHUNK, floorf(c)), c * count / fmaxf(all - sum.few, 0.25f * all) + 1.0f);
    return max(KA_CHUNK, (int)(c > 2.0f * share ? share : c));
}

// What lies at the start of the workspace, and, of more than 64 sequences, what
// comes before each 64 of them (k_kv_list).  Else each workgroup would pass over all
// of them: 1024 rows of as many sequences of 1000 tokens take 161 us with the list,
// 357 without, 4096 of 200 353 and 3041, 256 of 200 28 and 24.
struct KvHeader {
    int32_t units;                       // of the join: written by k_kv_attn
    int32_t C;
    float longest;
    int32_t pad[5];
};
struct KvGroup {
    int32_t items, parts, units, wide, top;              // wide: items of k_kv_attn_wide
    int32_t pad[3];
};

// The last group with key(group) <= item, its first sequence in `base`.
template <class Key>
__device__ __forceinline__ KvGroup kv_group(const KvAttnArgs &a, int item, Key &&key, int &base)
{
    const int lane = threadIdx.x & 63;
    int first = 0, n = (a.b.n_seqs + 63) / 64;
    while (n > 1) {
        const int part = (n + 63) / 64, i = lane * part;
        const uint64_t before = __ballot(i < n && key(a.groups[first + min(i, n - 1)]) <= item);
        const int k = 63 - __builtin_clzll(before | 1);
        first += k * part;
        n = min(part, n - k * part);
    }
    base = 64 * first;
    return a.groups[first];
}

// Item `item` of the call, or false past the last.  One wavefront.
__device__ __forceinline__ bool kv_item(const KvAttnArgs &a, int G, int item, KvItem &it)
{
    int base = 0, top = 0, parts = 0, units = 0;
    float longest = 0.0f;
    if (a.b.n_seqs > 64) {
        const KvGroup g = kv_group(a, item, [](const KvGroup &r) { return r.items; }, base);
        top = g.top;
        item -= g.items;
        parts = g.parts;
        units = g.units;
        longest = ((const KvHeader *)a.ws)->longest;
    }
    const KvSeq q = kv_seqs(a.b, base, top);
    if (a.b.n_seqs <= 64 && a.wide > 0 && a.wide < 0x7fffffff) longest = kv_longest(a, kv_wave_last(kv_wave_scan(kv_wide_work(a, q, G))));
    int C = 0x7fffffff;
    if (a.b.n_seqs > 64) {
        C = ((const KvHeader *)a.ws)->C;
    } else if (a.split) {
        KvWork sum{};
        kv_add_work(a, q, G, longest, sum);
        sum.few = kv_wave_last(kv_wave_scan(sum.few));
        sum.many = kv_wave_last(kv_wave_scan(sum.many));
        sum.rest = kv_wave_last(kv_wave_scan(sum.rest));
        sum.work = kv_wave_last(kv_wave_scan(sum.work));
        const float c = kv_chunk(a, sum);
        C = kv_chunk(a, sum, c, kv_wave_last(kv_wave_scan(kv_chunks(a, q, G, longest, c))));
    }
    const int tiles = kv_col_tiles(a, q, G, longest), length = kv_token_tiles(a, q), ks = kv_cuts(length, C);
    const int count = tiles * ks * a.nkv, part = ks > 1 ? tiles * ks : 0, unit = ks > 1 ? tiles : 0;
    const int end = kv_wave_scan(count), parts_end = kv_wave_scan(part), units_end = kv_wave_scan(unit);
    const uint64_t past = __ballot(end > item);
    if (past) {
        const int l = __builtin_ctzll(past);
        auto at = [&](int v) { return (uint32_t)__builtin_amdgcn_readlane(v, l); };
        const uint32_t n = at(ks), i = (uint32_t)item - (at(end) - at(count));
        it.s = base + l;
        it.q = KvSeq{(int)at(q.q0), (int)at(q.n), (int)at(q.len)};
        it.cb = kv_blocks_of_tile(it.q.n * G);
        it.ks = (int)n;
        it.chunk = (int)((at(length) + n - 1) / n);
        it.kvh = (int)(i % (uint32_t)a.nkv);
        it.split = (int)(i / (uint32_t)a.nkv % n);
        it.tile = (int)(i / (uint32_t)a.nkv / n);
        it.part = (parts + (int)(at(parts_end) - at(part))) * a.nkv + (int)i;
        it.unit = (units + (int)(at(units_end) - at(unit)) + it.tile) * a.nkv + it.kvh;
        return true;
    }
    units += kv_wave_last(units_end);
    it.unit = units * a.nkv;             // how many there are
    return false;
}

// The workspace of a call whose sequences can have several chunks: how many
// units the join has, for each what it has to know, then per item of them its
// columns' sums [KA_COLS][HD] and their (m, l).  A unit of several chunks is
// longer than a chunk, whose length is at least the work over KA_ITEMS: there
// are at most KA_ITEMS units and 2 KA_ITEMS items of this kind, however many
// columns the call has.
struct KvDesc {
    int32_t ks, part, tile, kvh, q0, cols, cb, pad;      // part: the unit's first
};

template <int HD>
__device__ __forceinline__ float *kv_part(const KvAttnArgs &a, int part)
{
    return (float *)((KvDesc *)a.ws + 1 + a.units) + (size_t)part * KA_COLS * (HD + 2);
}

// ---------------------------------------------------------------------------
// What a wavefront holds of its 16 CB columns, and the steps of a token tile.
template <int HD, bool F8, int CB>
struct KvWave {
    static constexpr int NC = HD / 32;             // 32-dim chunks of a row
    static constexpr int NB = HD / 16;             // 16-dim blocks of O
    static constexpr int EB = F8 ? 1 : 2, NE = F8 ? 2 : 1;       // bytes of a value; operands that a 16-byte piece makes
    static constexpr int NK = HD * EB / 32;        // 16-byte pieces a lane has of a tile's keys, and of its values

    // lane: column r16 of each 16-column block, and of the operands' 32 inner
    // positions the 8 of group g
    int lane, r16, g;
    int vis[CB];                                   // tokens 0 .. vis - 1 are what a column sees
    int least, last;                               // the least and the most of the live columns' vis
    float cmul[CB];                                // log2(e) / sqrt(hd) over the query's power of two
    // m: the columns' reference of s + ve, raised when a score passes it by
    // KA_SLACK (-inf: nothing seen; at least -FLT_MAX else, so that a row whose
    // every score is -inf ends as 0 / 0, not as empty); l: this lane's share of
    // the sum; o: the sums of values, [block of dims], rows 4 g + i
    float m[CB], l[CB];
    kv_f4 o[CB][NB];

    // column `col` of sequence q: query q.q0 + col / G, head kvh G + col % G
    __device__ __forceinline__ void start(const KvAttnArgs &a, const KvSeq &q, int G, int col0)
    {
        lane = threadIdx.x & 63;
        r16 = lane & 15;
        g = lane >> 4;
        const int cached = kv_cached(q.len, a.c.T, a.b.max_pages);
        last = 0;
        least = cached;
#pragma unroll
        for (int cb = 0; cb < CB; cb++) {
            const int col = col0 + 16 * cb + r16;
            const bool live = col < q.n * G;
            vis[cb] = live ? kv_visible(q.len - q.n + (int)((uint32_t)col / (uint32_t)G), cached, a.block) : 0;
            last = max(last, vis[cb]);
            if (live) least = min(least, vis[cb]);
            m[cb] = -__builtin_inff();
            l[cb] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) o[cb][b] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) {
            last = max(last, __shfl_xor(last, d, 64));
            least = min(least, __shfl_xor(least, d, 64));
        }
        last = __builtin_amdgcn_readfirstlane(last);
        least = __builtin_amdgcn_readfirstlane(least);
    }

    // The queries of 16 columns from col0 on: chunk 2 p + e of a lane holds dims
    // 64 p + 16 g + 8 e .. + 7 (its 16 dims of a 64-dim half are one piece of an
    // E4M3 key row).  fetch() reads them, form() makes the operands of them:
    // put(c, hi, lo) takes chunk c; it returns cmul.
    struct Queries {
        float x[NC][8];
        bool live;
    };
    static __device__ __forceinline__ void fetch(Queries &r, const KvAttnArgs &a, const KvSeq &q, int G, int kvh, int col0)
    {
        const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
        const int col = col0 + r16;
        r.live = col < q.n * G;
        const uint32_t qi = r.live ? (uint32_t)col / (uint32_t)G : 0, hg = r.live ? (uint32_t)col % (uint32_t)G : 0;
        const float *src = a.q + ((size_t)(q.q0 + (int)qi) * a.nh + (size_t)kvh * G + hg) * HD + 16 * g;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(src + 64 * (c / 2) + 8 * (c % 2) + j);
                r.x[c][j] = v.x;
                r.x[c][j + 1] = v.y;
                r.x[c][j + 2] = v.z;
                r.x[c][j + 3] = v.w;
            }
    }
    template <class Put>
    static __device__ __forceinline__ float form(Queries &r, const KvAttnArgs &a, Put &&put)
    {
        float amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                r.x[c][j] = r.live ? r.x[c][j] : 0.0f;
                amax = fmaxf(amax, fabsf(r.x[c][j]));
            }
        amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
        amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
        int up = 0;
        if (amax > 0.0f && amax <= 3.402823466e38f) {
            int ex;
            (void)frexpf(amax, &ex);
            up = min(8 - ex, 100);
        }
        const float mul = ldexpf(1.0f, up);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            kv_h8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = r.x[c][j] * mul;
                hi[j] = (_Float16)y;
                lo[j] = (_Float16)(y - (float)hi[j]);
            }
            put(c, hi, lo);
        }
        return ldexpf(a.scale * 1.44269504088896341f, -up);
    }

    // A tile's first byte, kept in scalar registers beside the lane's 32-bit
    // offset (the empty asm statements): their sums, formed ahead of the loop,
    // would take vector registers, which are short.
    typedef const __attribute__((address_space(1))) uint8_t *Bytes;
    typedef const __attribute__((address_space(1))) kv_u4 *Piece;
    static __device__ __forceinline__ Bytes at(const void *p, size_t byte)
    {
        Bytes tile = (Bytes)(uintptr_t)p + byte;
        asm volatile("" : "+s"(tile));
        return tile;
    }

    // Where a lane's pieces of a tile lie, in bytes from the tile's keys or
    // values.  Row r of key block kb is token 8 (r / 4) + 4 kb + r % 4, so that
    // the scores of a lane are those of tokens 8 g + 4 kb + i.
    static __device__ __forceinline__ uint32_t key_at()
    {
        const uint32_t l = lane_again(), r = l & 15;
        return ((8 * (r >> 2) + (r & 3)) * HD + 16 * (l >> 4)) * EB;
    }
    static __device__ __forceinline__ uint32_t value_at()
    {
        const uint32_t l = lane_again();
        return ((l & 15) * 4 + (l >> 4)) * 16;
    }
    // The lane, formed anew: a few instructions per tile instead of a register
    // held through the loop, or, worse, a load of a spilled one.
    static __device__ __forceinline__ uint32_t lane_again()
    {
        uint32_t l;
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
        return l;
    }
    static __device__ __forceinline__ uint4 key_piece(Bytes tile, uint32_t at, int i)
    {
        // key block, then chunk (F16) or pair of chunks (E4M3)
        const int kb = i / (NK / 2), ch = i % (NK / 2) * NE;
        return __builtin_bit_cast(uint4, *(Piece)(tile + at + (4 * kb * HD + 64 * (ch / 2) + 8 * (ch % 2)) * EB));
    }
    static __device__ __forceinline__ uint4 value_piece(Bytes tile, uint32_t at, int i)
    {
        return __builtin_bit_cast(uint4, *(Piece)(tile + at + 1024 * i));
    }
    // One tile of 32 tokens from k0 on.  FULL: every column sees all of it.
    template <bool FULL>
    struct Step {
        kv_f4 sc[CB][2];
        float c[CB], mt[CB];
        int k0, ke, ve;
        kv_h8 ph[CB], pl[CB];
    };
    template <bool FULL>
    __device__ __forceinline__ bool seen(const Step<FULL> &s, int cb, int kb, int e) const
    {
        return FULL || s.k0 + 8 * g + 4 * kb + e < vis[cb];
    }

    // the scores; true if one passes its column's reference by KA_SLACK
    template <bool FULL, class Key, class Query>
    __device__ __forceinline__ bool scores(Step<FULL> &s, Key &&key, Query &&query)
    {
#pragma unroll
        for (int cb = 0; cb < CB; cb++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++) s.sc[cb][kb] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ch = 0; ch < NC; ch += NE) {
            kv_h8 kf[2][NE];
            key(ch, kf);
#pragma unroll
            for (int e = 0; e < NE; e++)
#pragma unroll
                for (int part = 0; part < 2; part++)           // the small half first
#pragma unroll
                    for (int cb = 0; cb < CB; cb++) {
                        const kv_h8 qf = query(cb, ch + e, 1 - part);
#pragma unroll
                        for (int kb = 0; kb < 2; kb++)
                            s.sc[cb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kb][e], qf, s.sc[cb][kb], 0, 0, 0);
                    }
            if (!F8 && ch == NC / 2 - 1) __builtin_amdgcn_sched_barrier(0);    // else every query operand is read ahead
        }
        bool above = false;
#pragma unroll
        for (int cb = 0; cb < CB; cb++) {
            s.c[cb] = F8 ? ldexpf(cmul[cb], s.ke) : cmul[cb];
            float smax = -__builtin_inff();
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    smax = fmaxf(smax, seen<FULL>(s, cb, kb, e) ? s.sc[cb][kb][e] : -__builtin_inff());
            s.mt[cb] = fmaxf(__builtin_fmaf(smax, s.c[cb], (float)s.ve), -3.402823466e38f);
            if (!FULL) s.mt[cb] = vis[cb] > s.k0 ? s.mt[cb] : -__builtin_inff();
            above |= s.mt[cb] > m[cb] + (float)KA_SLACK;
        }
        return __any(above);
    }

    // the maximum over the lanes of a column
    __device__ __forceinline__ float column_max(float x) const
    {
        x = fmaxf(x, __shfl_xor(x, 16, 64));
        return fmaxf(x, __shfl_xor(x, 32, 64));
    }

    // raises the references to what a tile's scores have met
    __device__ __forceinline__ void raise(const float (&top)[CB])
    {
#pragma unroll
        for (int cb = 0; cb < CB; cb++) {
            const float mn = fmaxf(m[cb], column_max(top[cb]));
            const float corr = m[cb] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m[cb] - mn);
            m[cb] = mn;
            l[cb] *= corr;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[cb][b][e] *= corr;
        }
    }

    // the probabilities, in place the operand of the second product
    template <bool FULL>
    __device__ __forceinline__ void weights(Step<FULL> &s)
    {
#pragma unroll
        for (int cb = 0; cb < CB; cb++) {
            const float k = (float)(s.ve + KA_SHIFT) - (!FULL && m[cb] == -__builtin_inff() ? 0.0f : m[cb]);
            float sum = 0.0f;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    kv_f2 p;
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        p[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s.sc[cb][kb][e + x], s.c[cb], k));
                        p[x] = seen<FULL>(s, cb, kb, e + x) ? p[x] : 0.0f;
                        sum += p[x];
                    }
                    const kv_h2 hi = __builtin_convertvector(p, kv_h2), lo = kv_rest(p, hi);
                    s.ph[cb][4 * kb + e] = hi[0];
                    s.ph[cb][4 * kb + e + 1] = hi[1];
                    s.pl[cb][4 * kb + e] = lo[0];
                    s.pl[cb][4 * kb + e + 1] = lo[1];
                }
            l[cb] = F8 ? __builtin_fmaf(sum, ldexpf(1.0f, -s.ve), l[cb]) : l[cb] + sum;
        }
    }

    // o += V^T P^T.  O rows are dims 16 b + row (F16), 32 (b / 2) + 2 row + b % 2 (E4M3).
    template <bool FULL, class Value>
    __device__ __forceinline__ void add(Step<FULL> &s, Value &&value)
    {
        constexpr std::integral_constant<bool, FULL> full{};
        if (FULL) {
#pragma unroll
            for (int p = 0; p < NK; p++) {
                kv_h8 vf[NE];
                value(full, p, vf);
#pragma unroll
                for (int part = 0; part < 2; part++)
#pragma unroll
                    for (int e = 0; e < NE; e++)
#pragma unroll
                        for (int cb = 0; cb < CB; cb++)
                            o[cb][p * NE + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[e], part ? s.ph[cb] : s.pl[cb],
                                                                                       o[cb][p * NE + e], 0, 0, 0);
            }
            return;
        }
        // What a column does not see may hold anything, and 0 times a NaN is
        // one: tokens that no column sees are set to zero, and if the others are
        // not all finite, the columns of each limit in turn add a product whose
        // values end there.
        // (Any that is not makes a product with zeros NaN.)
        const kv_h8 zero = {};
        kv_f4 probe = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < NK; p++) {
            kv_h8 vf[NE];
            value(full, p, vf);
#pragma unroll
            for (int e = 0; e < NE; e++)
                probe = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_cut(vf[e], g, last - s.k0), zero, probe, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);                 // one piece at a time: registers are short
        }
        const bool one = __all(probe[0] + probe[1] + probe[2] + probe[3] == 0.0f);
        for (int done = s.k0;;) {
            int lim = 0x7fffffff;
#pragma unroll
            for (int cb = 0; cb < CB; cb++)
                if (vis[cb] > done) lim = min(lim, vis[cb]);
#pragma unroll
            for (int d = 8; d >= 1; d >>= 1) lim = min(lim, __shfl_xor(lim, d, 64));
            lim = one ? last : __builtin_amdgcn_readfirstlane(lim);
            if (lim == 0x7fffffff) break;
#pragma unroll
            for (int p = 0; p < NK; p++) {
                kv_h8 vf[NE];
                value(full, p, vf);
#pragma unroll
                for (int e = 0; e < NE; e++) {
                    const kv_h8 y = kv_cut(vf[e], g, lim - s.k0);
#pragma unroll
                    for (int cb = 0; cb < CB; cb++) {
                        const bool mine = one || (vis[cb] > done && (vis[cb] == lim || lim >= s.k0 + 32));
                        kv_f4 t = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, s.pl[cb], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, s.ph[cb], t, 0, 0, 0);
#pragma unroll
                        for (int x = 0; x < 4; x++) o[cb][p * NE + e][x] += mine ? t[x] : 0.0f;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (one || lim >= s.k0 + 32) break;
            done = lim;
        }
    }

    // l over the lanes of a column; column r16's sums times f to dst [HD]
    __device__ __forceinline__ float total(int cb) const
    {
        const float x = l[cb] + __shfl_xor(l[cb], 16, 64);
        return x + __shfl_xor(x, 32, 64);
    }
    __device__ __forceinline__ void store(int cb, float f, float *dst) const
    {
#pragma unroll
        for (int b = 0; b < NB; b += NE)
            if constexpr (F8) {
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    *reinterpret_cast<float4 *>(dst + 16 * b + 8 * g + 2 * i) =
                        make_float4(o[cb][b][i] * f, o[cb][b + 1][i] * f, o[cb][b][i + 1] * f, o[cb][b + 1][i + 1] * f);
            } else {
                *reinterpret_cast<float4 *>(dst + 16 * b + 4 * g) =
                    make_float4(o[cb][b][0] * f, o[cb][b][1] * f, o[cb][b][2] * f, o[cb][b][3] * f);
            }
    }
};

// The token tiles of a chunk that a wavefront walks: up to 64 at a time, a lane
// looks up the page and the exponents of one, and the loop takes them from
// there.
template <int HD, bool F8>
struct KvWalk {
    int base, step, end;                           // lane n's tile is base + step n, below end
    int kes, ves;
    uint32_t blo, bhi;
    uint64_t todo;                                 // tiles still to do, by lane; `now` is the first of them (or the last)
    int now;

    __device__ __forceinline__ void look(const KvAttnArgs &a, int s, int kvh)
    {
        const int tt = base + step * (int)(threadIdx.x & 63);
        int page = -1;
        if (tt < end) page = kv_page(a.b, a.c, s, 32 * tt);
        const size_t slot = ((size_t)max(page, 0) * a.nkv + kvh) * (a.c.T / 32) + (uint32_t)tt % (uint32_t)(a.c.T / 32);
        const size_t byte = slot * 32 * HD * (F8 ? 1 : 2);
        blo = (uint32_t)byte;
        bhi = (uint32_t)(byte >> 32);
        todo = __ballot(page >= 0);
        now = todo ? __builtin_ctzll(todo) : 0;
        kes = ves = 0;
        if (F8 && page >= 0) {
            kes = a.c.k_exp[slot];
            ves = a.c.v_exp[slot];
        }
    }
    // (past the last tile `now` stays: it is loaded again, since a wait counts
    // loads and there must always be some)
    __device__ __forceinline__ void next()
    {
        todo &= todo - 1;
        if (todo) now = __builtin_ctzll(todo);
    }
    __device__ __forceinline__ size_t byte() const
    {
        return (size_t)(uint32_t)__builtin_amdgcn_readlane(bhi, now) << 32 | (uint32_t)__builtin_amdgcn_readlane(blo, now);
    }
    __device__ __forceinline__ int k0() const { return 32 * (base + step * now); }
    __device__ __forceinline__ int ke() const { return F8 ? __builtin_amdgcn_readlane(kes, now) : 0; }
    __device__ __forceinline__ int ve() const { return F8 ? __builtin_amdgcn_readlane(ves, now) : 0; }
};

// One item's columns, 16 CB of them: the workgroup's wavefronts take its token
// tiles in turn and join their results in LDS.  Few rows are bound by the bytes:
// 48 of 8190 E4M3 tokens each, 229 MB, 48.2 us and 4.8 of the join (4.75 TB/s of
// the 5.15 that a large copy reaches), one of 131,072, 134 MB, 30.3 and 5.3.  Blocks
// by the products: 32 rows on 16,384 tokens, 17.2 GFLOP with both halves, 29.2 and
// 4.6, of them 7.7 until the first scores stand (work list, page, tile: three
// loads one after the other), 15 for the tiles (14.4 at the rate of a large
// library product) and 2.7 to join the wavefronts.  A tile's keys and values go
// straight from global memory to the registers that hold them as operands; the
// next tile's keys are loaded once a tile's scores stand, its values once its
// sums do, so that loads are always in flight and no second set of registers
// is needed.
template <int HD, bool F8, int CB>
__device__ __forceinline__ void kv_attend(const KvAttnArgs &a, const KvItem &it, int G, float *s_o, float *s_m, float *s_l)
{
    typedef KvWave<HD, F8, CB> Wave;
    constexpr int NC = Wave::NC, NK = Wave::NK, NE = Wave::NE;
    constexpr int LO = HD + 4;                     // row of O in LDS: padded against bank conflicts
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const KvSeq q = it.q;
    const int kvh = it.kvh;
    const float inf = __builtin_inff();
    Wave wave;
    wave.start(a, q, G, it.tile * CB * 16);

    uint4 kr[NK], vr[NK];
    auto load_k = [&](size_t byte) {
        const typename Wave::Bytes tile = Wave::at(a.c.k, byte);
        const uint32_t at = Wave::key_at();
#pragma unroll
        for (int i = 0; i < NK; i++) kr[i] = Wave::key_piece(tile, at, i);
    };
    auto load_v = [&](size_t byte) {
        const typename Wave::Bytes tile = Wave::at(a.c.v, byte);
        const uint32_t at = Wave::value_at();
#pragma unroll
        for (int i = 0; i < NK; i++) vr[i] = Wave::value_piece(tile, at, i);
    };
    typename Wave::Queries queries;
    if (w < CB) Wave::fetch(queries, a, q, G, kvh, (it.tile * CB + w) * 16);
    KvWalk<HD, F8> walk;
    walk.base = it.split * it.chunk + w;
    walk.step = KA_WAVES;
    walk.end = min((it.split + 1) * it.chunk, (wave.last + 31) / 32);
    walk.look(a, it.s, kvh);
    if (walk.todo) {
        load_k(walk.byte());
        load_v(walk.byte());
    }
    // the queries in LDS, [16-column block][chunk][hi, lo][lane]: every
    // wavefront has the same, and registers are short
    kv_h8 *s_q = reinterpret_cast<kv_h8 *>(s_o);
    if (w < CB) {
        const float c = Wave::form(queries, a, [&](int ch, const kv_h8 &hi, const kv_h8 &lo) {
            s_q[((w * NC + ch) * 2 + 0) * 64 + lane] = hi;
            s_q[((w * NC + ch) * 2 + 1) * 64 + lane] = lo;
        });
        if (wave.g == 0) s_m[16 * w + wave.r16] = c;
    }
    __syncthreads();
#pragma unroll
    for (int cb = 0; cb < CB; cb++) wave.cmul[cb] = s_m[16 * cb + wave.r16];

    // Tiles while `more` of them.  The references are raised outside the loop
    // over tiles (the tile's scores are then formed again): a conditional change
    // of the sums inside it costs a copy of them all per tile.
    auto run = [&](auto full, auto &&more) {
        constexpr bool FULL = decltype(full)::value;
        for (;;) {
            float mt[CB];
            bool raise = false;
            while (more()) {
                typename Wave::template Step<FULL> st;
                st.k0 = walk.k0();
                st.ke = walk.ke();
                st.ve = walk.ve();
                int at = lane;
                asm volatile("" : "+v"(at));       // the queries are read again each tile, not kept in registers
                if (wave.template scores<FULL>(
                    st,
                    [&](int ch, kv_h8(&kf)[2][NE]) {
#pragma unroll
                        for (int kb = 0; kb < 2; kb++) kv_widen<F8>(kr[kb * (NK / 2) + ch / NE], kf[kb]);
                    },
                    [&](int cb, int ch, int low) { return s_q[((cb * NC + ch) * 2 + low) * 64 + at]; })) {
                    raise = true;
#pragma unroll
                    for (int cb = 0; cb < CB; cb++) mt[cb] = st.mt[cb];
                    break;
                }
                walk.next();
                const size_t next = walk.byte();
                if (FULL) load_k(next);            // (registers are short in the other path, and its tiles few)
                wave.template weights<FULL>(st);
                wave.template add<FULL>(st, [&](auto once, int p, kv_h8(&vf)[NE]) {
                    uint4 x = vr[p];
                    // (used again per limit: not to be kept widened in between)
                    if (!once && F8) asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w));
                    kv_widen<F8>(x, vf);
                });
                if (!FULL) load_k(next);
                load_v(next);
            }
            if (!raise) break;
            wave.raise(mt);
        }
    };
    for (;;) {
        run(std::true_type{}, [&] { return walk.todo && walk.k0() + 32 <= wave.least; });
        run(std::false_type{}, [&] { return walk.todo != 0; });
        walk.base += 64 * KA_WAVES;
        if (walk.base >= walk.end) break;
        walk.look(a, it.s, kvh);
        if (walk.todo) {
            load_k(walk.byte());
            load_v(walk.byte());
        }
    }

    // the wavefronts' results joined in LDS: [wavefront][column][dim]
    __syncthreads();                               // the queries' place, no longer needed
    constexpr int COLS = 16 * CB;
#pragma unroll
    for (int cb = 0; cb < CB; cb++) {
        const int c = w * COLS + 16 * cb + wave.r16;
        const float total = wave.total(cb);
        wave.store(cb, 1.0f, s_o + c * LO);
        if (wave.g == 0) {
            s_m[c] = wave.m[cb];
            s_l[c] = total;
        }
    }
    __syncthreads();
    const int cols = min(COLS, q.n * G - it.tile * COLS);
    for (int e = threadIdx.x; e < cols * (HD / 4); e += KA_WAVES * 64) {
        const int c = e / (HD / 4), d = e % (HD / 4) * 4;
        float M = s_m[c];
#pragma unroll
        for (int i = 1; i < KA_WAVES; i++) M = fmaxf(M, s_m[i * COLS + c]);
        float L = 0.0f;
        float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < KA_WAVES; i++) {
            const float mi = s_m[i * COLS + c], f = mi == -inf ? 0.0f : __builtin_amdgcn_exp2f(mi - M);
            const float4 x = *reinterpret_cast<const float4 *>(&s_o[(i * COLS + c) * LO + d]);
            L += s_l[i * COLS + c] * f;
            O.x += x.x * f;
            O.y += x.y * f;
            O.z += x.z * f;
            O.w += x.w * f;
        }
        if (it.ks == 1) {
            const int cc = it.tile * COLS + c;
            const float inv = M == -inf ? 0.0f : 1.0f / L;         // nothing seen: zeros
            *reinterpret_cast<float4 *>(a.out + ((size_t)(q.q0 + cc / G) * a.nh + (size_t)kvh * G + cc % G) * HD + d) =
                make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
        } else {
            float *part = kv_part<HD>(a, it.part);
            *reinterpret_cast<float4 *>(part + c * HD + d) = O;
            if (d == 0) *reinterpret_cast<float2 *>(part + KA_COLS * HD + 2 * c) = make_float2(M, L);
        }
    }
}

// The list of more than 64 sequences, in one workgroup, 1024 at a time.
__global__ __launch_bounds__(1024) void k_kv_list(KvAttnArgs a)
{
    __shared__ float s_f[16];
    __shared__ int s_i[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, G = a.nh / a.nkv;
    // the sum over the workgroup
    auto total = [&](float v) {
        v = kv_wave_scan(v);
        __syncthreads();
        if (lane == 63) s_f[w] = v;
        __syncthreads();
        v = 0.0f;
        for (int i = 0; i < 16; i++) v += s_f[i];
        return v;
    };
    // op over the wavefronts before this one and `v` (the last one's with it)
    auto before = [&](int mine, int &v, auto &&op) {
        __syncthreads();
        if (lane == 0) s_i[w] = mine;
        __syncthreads();
        int r = v;
        for (int i = 0; i < 16; i++) {
            if (i < w) r = op(r, s_i[i]);
            v = op(v, s_i[i]);
        }
        return r;
    };
    auto most = [](int x, int y) { return max(x, y); };
    auto sum = [](int x, int y) { return x + y; };
    // f(first sequence of the wavefront's 64, what came before them), q a lane's
    KvSeq q;
    auto each = [&](auto &&f) {
        int top = 0;
        for (int base = 0; base < a.b.n_seqs; base += 1024) {
            int own = 0;
            (void)kv_seqs(a.b, base + 64 * w, own);
            int from = before(own, top, most);
            const int met = from;
            q = kv_seqs(a.b, base + 64 * w, from);
            f(base + 64 * w, met);
        }
    };
    float longest = 0.0f;
    if (a.wide > 0 && a.wide < 0x7fffffff) {
        float work = 0.0f;
        each([&](int, int) { work += kv_wide_work(a, q, G); });
        longest = kv_longest(a, total(work));
    }
    int C = 0x7fffffff;
    if (a.split) {
        KvWork all{};
        each([&](int, int) { kv_add_work(a, q, G, longest, all); });
        all.few = total(all.few);
        all.many = total(all.many);
        all.rest = total(all.rest);
        all.work = total(all.work);
        const float c = kv_chunk(a, all);
        float count = 0.0f;
        each([&](int, int) { count += kv_chunks(a, q, G, longest, c); });
        C = kv_chunk(a, all, c, total(count));
    }
    int items = 0, parts = 0, units = 0, wide = 0;
    const int per = 32 * KW_WAVES;
    each([&](int base, int met) {
        const int tiles = kv_col_tiles(a, q, G, longest), ks = kv_cuts(kv_token_tiles(a, q), C);
        KvGroup g{};
        g.top = met;
        g.items = before(kv_wave_last(kv_wave_scan(tiles * ks * a.nkv)), items, sum);
        g.parts = before(kv_wave_last(kv_wave_scan(ks > 1 ? tiles * ks : 0)), parts, sum);
        g.units = before(kv_wave_last(kv_wave_scan(ks > 1 ? tiles : 0)), units, sum);
        g.wide = before(kv_wave_last(kv_wave_scan(kv_is_wide(a, q, G, longest) ? (q.n * G + per - 1) / per : 0)), wide, sum);
        if (lane == 0 && base < a.b.n_seqs) a.groups[base / 64] = g;
    });
    if (threadIdx.x == 0) {
        ((KvHeader *)a.ws)->C = C;
        ((KvHeader *)a.ws)->longest = longest;
    }
}

// Many columns of one sequence (prompts): a workgroup takes 32 KW_WAVES of
// them, each wavefront 32, over all the tokens they see.  A token tile is
// loaded once for all four wavefronts, a quarter by each, widened to f16 and
// left in LDS as operands (lane-contiguous: no bank conflicts); the next tile's
// loads are in flight during its products.  The queries stay in registers.
// Bound by the products: 2000 rows on 4001 cached tokens and themselves, 328 GFLOP
// with both halves, in 270 us, 1,215 TFLOP/s, where a large f16 product of the
// library reaches 1,160 to 1,310.  A tile takes a wavefront 3,270 cycles, two of
// them on a SIMD: 1,024 of its MFMAs each, of which 8 cycles apiece are lost to
// its about 140 other vector instructions (measured apart: 16 MFMAs beside 64 fma
// of another wavefront take 384 us where either alone takes 265).
template <int HD, bool F8>
__global__ __launch_bounds__(KW_WAVES * 64, 2) void k_kv_attn_wide(KvAttnArgs a)
{
    constexpr int CB = 2;
    typedef KvWave<HD, F8, CB> Wave;
    constexpr int NC = Wave::NC, NK = Wave::NK, NE = Wave::NE, NB = Wave::NB;
    constexpr int NP = NK / 2;                     // pieces of a tile that a wavefront loads (of 2 NK)
    __shared__ __align__(16) kv_h8 s_kv[2][(2 * NC + NB) * 64];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The last column tiles see the most: they start first, and of the workgroups
    // that start at once the second of a CU is the shorter the longer its first.
    const int places = min((int)gridDim.x, KA_ITEMS), block = blockIdx.x;
    const int rank = block >= KA_ITEMS / 2 && block < places ? KA_ITEMS / 2 + places - 1 - block : block;
    const int G = a.nh / a.nkv, kvh = rank % a.nkv;
    int s, tile;
    KvSeq q;
    const int per = 16 * CB * KW_WAVES;
    int item = (int)gridDim.x / a.nkv - 1 - rank / a.nkv;
    {
        int base = 0, top = 0;
        float longest = 0.0f;
        if (a.b.n_seqs > 64) {
            const KvGroup g = kv_group(a, item, [](const KvGroup &r) { return r.wide; }, base);
            top = g.top;
            item -= g.wide;
            longest = ((const KvHeader *)a.ws)->longest;
        }
        const KvSeq r = kv_seqs(a.b, base, top);
        if (a.b.n_seqs <= 64 && a.wide > 0) longest = kv_longest(a, kv_wave_last(kv_wave_scan(kv_wide_work(a, r, G))));
        const int count = kv_is_wide(a, r, G, longest) ? (r.n * G + per - 1) / per : 0, end = kv_wave_scan(count);
        const uint64_t past = __ballot(end > item);
        if (!past) return;
        const int l = __builtin_ctzll(past);
        s = base + l;
        q = KvSeq{__builtin_amdgcn_readlane(r.q0, l), __builtin_amdgcn_readlane(r.n, l), __builtin_amdgcn_readlane(r.len, l)};
        tile = item - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(count, l));
    }
    const int col0 = tile * per + w * 16 * CB;
    Wave wave;
    wave.start(a, q, G, col0);
    const int cached = kv_cached(q.len, a.c.T, a.b.max_pages);
    const int most = kv_visible(q.len - q.n + (min((tile + 1) * per, q.n * G) - 1) / G, cached, a.block);

    uint4 r[NP];
    // wavefronts 0 and 1: keys, 2 and 3: values
    auto load = [&](size_t byte) {
        const typename Wave::Bytes tile = Wave::at(w < KW_WAVES / 2 ? a.c.k : a.c.v, byte);
        const uint32_t at = w < KW_WAVES / 2 ? Wave::key_at() : Wave::value_at();
#pragma unroll
        for (int j = 0; j < NP; j++)
            r[j] = w < KW_WAVES / 2 ? Wave::key_piece(tile, at, w * NP + j) : Wave::value_piece(tile, at, w * NP + j - NK);
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int j = 0; j < NP; j++) {
            kv_h8 x[NE];
            kv_widen<F8>(r[j], x);
#pragma unroll
            for (int e = 0; e < NE; e++) s_kv[buf][((w * NP + j) * NE + e) * 64 + lane] = x[e];
        }
    };
    KvWalk<HD, F8> walk;
    walk.base = 0;
    walk.step = 1;
    walk.end = (most + 31) / 32;
    walk.look(a, s, kvh);
    if (walk.todo) load(walk.byte());
    kv_h8 qf[CB][NC][2];
#pragma unroll
    for (int cb = 0; cb < CB; cb++) {
        typename Wave::Queries queries;
        Wave::fetch(queries, a, q, G, kvh, col0 + 16 * cb);
        wave.cmul[cb] = Wave::form(queries, a, [&](int ch, const kv_h8 &hi, const kv_h8 &lo) {
            qf[cb][ch][0] = hi;
            qf[cb][ch][1] = lo;
        });
    }
    int buf = 0;
    stage(0);
    __syncthreads();
    // Every wavefront meets the same tiles and barriers: those whose columns no
    // longer see a tile only help to load the next.
    auto run = [&](auto full, auto &&more) {
        constexpr bool FULL = decltype(full)::value;
        for (;;) {
            float mt[CB];
            bool raise = false;
            while (more()) {
                typename Wave::template Step<FULL> st;
                st.k0 = walk.k0();
                st.ke = walk.ke();
                st.ve = walk.ve();
                const kv_h8 *kv = s_kv[buf];
                if (wave.template scores<FULL>(
                    st,
                    [&](int ch, kv_h8(&kf)[2][NE]) {
#pragma unroll
                        for (int kb = 0; kb < 2; kb++)
#pragma unroll
                            for (int e = 0; e < NE; e++) kf[kb][e] = kv[(kb * NC + ch + e) * 64 + lane];
                    },
                    [&](int cb, int ch, int low) { return qf[cb][ch][low]; })) {
                    raise = true;
#pragma unroll
                    for (int cb = 0; cb < CB; cb++) mt[cb] = st.mt[cb];
                    break;
                }
                walk.next();
                load(walk.byte());
                __builtin_amdgcn_sched_barrier(0);             // not later, for fewer registers
                wave.template weights<FULL>(st);
                wave.template add<FULL>(st, [&](auto once, int p, kv_h8(&vf)[NE]) {
                    int at = lane;
                    if (!once) asm volatile("" : "+v"(at));
#pragma unroll
                    for (int e = 0; e < NE; e++) vf[e] = kv[(2 * NC + p * NE + e) * 64 + at];
                });
                buf ^= 1;
                stage(buf);
                __syncthreads();
            }
            if (!raise) break;
            wave.raise(mt);
        }
    };
    for (;;) {
        run(std::true_type{}, [&] { return walk.todo && walk.k0() + 32 <= wave.least; });
        run(std::false_type{}, [&] { return walk.todo && walk.k0() < wave.last; });
        while (walk.todo) {
            walk.next();
            load(walk.byte());
            buf ^= 1;
            stage(buf);
            __syncthreads();
        }
        walk.base += 64;
        if (walk.base >= walk.end) break;
        walk.look(a, s, kvh);
        if (walk.todo) load(walk.byte());
        __syncthreads();                           // the tile before is done with
        stage(buf);
        __syncthreads();
    }
#pragma unroll
    for (int cb = 0; cb < CB; cb++) {
        const int col = col0 + 16 * cb + wave.r16;
        const float L = wave.total(cb);
        if (col >= q.n * G) continue;
        const float inv = wave.m[cb] == -__builtin_inff() ? 0.0f : 1.0f / L;       // nothing seen: zeros
        wave.store(cb, inv, a.out + ((size_t)(q.q0 + col / G) * a.nh + (size_t)kvh * G + col % G) * HD);
    }
}

template <int HD, bool F8>
__global__ __launch_bounds__(KA_WAVES * 64, 2) void k_kv_attn(KvAttnArgs a)
{
    __shared__ __align__(16) float s_o[KA_WAVES * KA_COLS * (HD + 4)];
    __shared__ float s_m[KA_WAVES * KA_COLS], s_l[KA_WAVES * KA_COLS];
    const int G = a.nh / a.nkv;
    KvItem it;
    if (!kv_item(a, G, blockIdx.x, it)) {
        // (the launch's bound on the items is never reached)
        if (a.split && threadIdx.x == 0 && blockIdx.x == gridDim.x - 1) ((KvHeader *)a.ws)->units = it.unit;
        return;
    }
    if (it.ks > 1 && it.split == 0 && threadIdx.x == 0)
        ((KvDesc *)a.ws)[1 + it.unit] = KvDesc{it.ks, it.part, it.tile, it.kvh, it.q.q0,
                                               min(16 * it.cb, it.q.n * G - it.tile * 16 * it.cb), it.cb, 0};
    if (it.cb == 1)
        kv_attend<HD, F8, 1>(a, it, G, s_o, s_m, s_l);
    else
        kv_attend<HD, F8, 2>(a, it, G, s_o, s_m, s_l);
}

// Joins the chunks of a unit: a workgroup takes COLS of its columns, its
// threads four dims of a column and every PARTS-th chunk.
template <int HD, int DIMS, int COLS, int THREADS>
__global__ __launch_bounds__(THREADS) void k_kv_join(KvAttnArgs a)
{
    constexpr int ND = DIMS / 4, PARTS = THREADS / (COLS * ND);
    __shared__ __align__(16) float4 s_o[PARTS][COLS][ND];
    __shared__ float s_m[PARTS][COLS], s_l[PARTS][COLS];
    const int units = ((const KvHeader *)a.ws)->units;
    const KvDesc d = ((const KvDesc *)a.ws)[1 + blockIdx.x];
    const int c0 = (int)blockIdx.y / (HD / DIMS) * COLS, d0 = (int)blockIdx.y % (HD / DIMS) * DIMS;
    if ((int)blockIdx.x >= units || c0 >= d.cols) return;
    const int e = threadIdx.x % ND, ci = threadIdx.x / ND % COLS, part = threadIdx.x / (ND * COLS);
    const int c = min(c0 + ci, d.cols - 1);
    const float inf = __builtin_inff();
    float m = -inf, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int j = part; j < d.ks; j += PARTS) {
        const float *p = kv_part<HD>(a, d.part + j * a.nkv);
        const float2 ml = *reinterpret_cast<const float2 *>(p + KA_COLS * HD + 2 * c);
        const float4 x = *reinterpret_cast<const float4 *>(p + c * HD + d0 + 4 * e);
        const float mn = fmaxf(m, ml.x);
        const float f = m == -inf ? 0.0f : __builtin_amdgcn_exp2f(m - mn), h = ml.x == -inf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
        m = mn;
        l = l * f + ml.y * h;
        o = make_float4(o.x * f + x.x * h, o.y * f + x.y * h, o.z * f + x.z * h, o.w * f + x.w * h);
    }
    s_o[part][ci][e] = o;
    if (e == 0) {
        s_m[part][ci] = m;
        s_l[part][ci] = l;
    }
    __syncthreads();
    if (part > 0 || c0 + ci >= d.cols) return;
#pragma unroll
    for (int i = 1; i < PARTS; i++) m = fmaxf(m, s_m[i][ci]);
    l = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < PARTS; i++) {
        const float f = s_m[i][ci] == -inf ? 0.0f : __builtin_amdgcn_exp2f(s_m[i][ci] - m);
        const float4 x = s_o[i][ci][e];
        l += s_l[i][ci] * f;
        o = make_float4(o.x + x.x * f, o.y + x.y * f, o.z + x.z * f, o.w + x.w * f);
    }
    const int G = a.nh / a.nkv, col = d.tile * 16 * d.cb + c;
    const float inv = m == -inf ? 0.0f : 1.0f / l;
    *reinterpret_cast<float4 *>(a.out + ((size_t)(d.q0 + col / G) * a.nh + (size_t)d.kvh * G + col % G) * HD + d0 + 4 * e) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// What the launches take: the items at most, and whether any sequence can have
// several chunks (from the page table's width: the lengths are on the GPU).
struct KvAttnPlan {
    int64_t items, wide_items;           // of k_kv_attn and k_kv_attn_wide at most
    int64_t units, parts;                // what the workspace holds
    int32_t wide;                        // columns above which a sequence can be k_kv_attn_wide's
    bool split;
    size_t groups, bytes;                // where the workspace holds the groups, and its size
};

static KvAttnPlan kv_attn_plan(const KvAttnArgs &a)
{
    KvAttnPlan p;
    const int64_t cols = (int64_t)a.b.n_tokens * (a.nh / a.nkv);
    const int64_t seqs = std::min(a.b.n_seqs, a.b.n_tokens);       // .. with rows
    const bool many = cols * a.nkv >= (a.c.type == DMOE_KV_E4M3 ? KA_WIDE_E4M3 : KA_WIDE_F16);
    p.wide = many ? (seqs == 1 ? 0 : 32 * KW_WAVES) : 0x7fffffff;
    p.wide_items = many ? (cols / (32 * KW_WAVES) + seqs) * a.nkv : 0;
    // a sequence of c columns has at most c / 32 + 1 column tiles, and one that
    // is not k_kv_attn_wide's has less than the columns of KA_SHARE workgroups
    const int64_t most = (KA_SHARE / a.nkv + 1) * (int64_t)(32 * KW_WAVES);
    const int64_t tiles = p.wide == 0 ? 0 : std::min(cols / KA_COLS + seqs, many ? seqs * (most / KA_COLS + 1) : cols + seqs);
    p.split = tiles > 0 && (int64_t)a.b.max_pages * (a.c.T / 32) > KA_WHOLE;
    // chunks: less than one more per unit than its share of those wanted
    p.items = tiles * a.nkv + (p.split ? KA_ITEMS + 1 : 0);
    p.units = std::min<int64_t>(tiles * a.nkv, KA_ITEMS);
    p.parts = p.split ? std::min<int64_t>(p.items, 2 * KA_ITEMS) : 0;
    p.groups = (size_t)(1 + p.units) * sizeof(KvDesc) + (size_t)p.parts * KA_COLS * (a.hd + 2) * 4;
    p.bytes = p.groups + (a.b.n_seqs > 64 ? (size_t)(a.b.n_seqs + 63) / 64 * sizeof(KvGroup) : 0);
    return p;
}

size_t kv_attn_ws_bytes(const KvAttnArgs &a)
{
    return kv_attn_plan(a).bytes;
}

hipError_t launch_kv_attn(const KvAttnArgs &args, hipStream_t s)
{
    KvAttnArgs a = args;
    if (a.nkv <= 0 || a.nh % a.nkv) return hipErrorInvalidValue;
    const KvAttnPlan p = kv_attn_plan(a);
    a.units = (int32_t)p.units;
    a.split = p.split;
    a.wide = p.wide;
    a.groups = (KvGroup *)((uint8_t *)a.ws + p.groups);
    if (a.b.n_seqs > 64) {
        hipLaunchKernelGGL(k_kv_list, dim3(1), dim3(1024), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.wide_items) {
        const dim3 g((unsigned)p.wide_items), block(KW_WAVES * 64);
        switch (a.hd * (a.c.type == DMOE_KV_E4M3 ? -1 : 1)) {
        case 64: hipLaunchKernelGGL((k_kv_attn_wide<64, false>), g, block, 0, s, a); break;
        case 128: hipLaunchKernelGGL((k_kv_attn_wide<128, false>), g, block, 0, s, a); break;
        case -64: hipLaunchKernelGGL((k_kv_attn_wide<64, true>), g, block, 0, s, a); break;
        case -128: hipLaunchKernelGGL((k_kv_attn_wide<128, true>), g, block, 0, s, a); break;
        default: return hipErrorInvalidValue;
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (!p.items) return hipSuccess;
    const dim3 grid((unsigned)p.items), block(KA_WAVES * 64);
    switch (a.hd * (a.c.type == DMOE_KV_E4M3 ? -1 : 1)) {
    case 64: hipLaunchKernelGGL((k_kv_attn<64, false>), grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL((k_kv_attn<128, false>), grid, block, 0, s, a); break;
    case -64: hipLaunchKernelGGL((k_kv_attn<64, true>), grid, block, 0, s, a); break;
    case -128: hipLaunchKernelGGL((k_kv_attn<128, true>), grid, block, 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.split) return e;
    // Few units can have many chunks each (KA_ITEMS in all): 32 of them at a time
    // then, a workgroup per column and 64 dims (4 units of 128 chunks 5.3 us, the
    // other form 11.2).  Else a workgroup per four columns: most of the launch,
    // which has places for every column a unit could have, only starts and ends
    // (32 units of 16 chunks 4.6 against 8.7, 4 units of 6 chunks 3.4 against 4.0).
    const bool deep = p.units <= 32 && (int64_t)a.b.max_pages * (a.c.T / 32) > 16 * KA_CHUNK;
    const unsigned cols = deep ? KA_COLS * (a.hd / 64) : KA_COLS / 4;
    const dim3 join((unsigned)p.units, cols), threads(deep ? 512 : 256);
    if (a.hd == 64 && deep)
        hipLaunchKernelGGL((k_kv_join<64, 64, 1, 512>), join, threads, 0, s, a);
    else if (a.hd == 64)
        hipLaunchKernelGGL((k_kv_join<64, 64, 4, 256>), join, threads, 0, s, a);
    else if (deep)
        hipLaunchKernelGGL((k_kv_join<128, 64, 1, 512>), join, threads, 0, s, a);
    else
        hipLaunchKernelGGL((k_kv_join<128, 128, 4, 256>), join, threads, 0, s, a);
    return hipGetLastError();
}

} // namespace dmoe
