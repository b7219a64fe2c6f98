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
// probabilities (p' = 2^(s + ve - m'), at most 1 by the choice of m'), and the
// sum takes p' 2^-ve: no operand is rescaled.  With exponents within 100 of
// each other no p' that counts in the sum underflows.
#include "dmoe_kv.h"

#pragma clang fp contract(off)

namespace dmoe {

constexpr int KA_WAVES = 4;              // wavefronts of a workgroup
constexpr int KA_COLS = 16;              // columns of an item
constexpr int KA_SHIFT = 4;              // probabilities are held times 2^KA_SHIFT
constexpr int KA_SLACK = 8;              // .. and may pass that by 2^KA_SLACK before their reference is raised
constexpr int KA_CHUNK = 16;             // token tiles of a chunk at least
constexpr int KA_ITEMS = 512;            // items wanted of a call

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
// Work items.  A sequence's columns form tiles of KA_COLS, its cached tokens
// tiles of 32; an item is one column tile of one kv head over one chunk of
// token tiles.  The chunk length is common to all sequences, so that ragged
// ones spread over the chip like one: the total of (column tile, token tile)
// pairs over the items wanted, at least KA_CHUNK.  A sequence's chunks are then
// made equally long.
struct KvItem {
    int s, tile;                         // sequence, column tile
    KvSeq q;
    int ks, chunk;                       // chunks of the sequence, token tiles of each
    int split, first;                    // this item's chunk; the column tile's first item
};

__device__ __forceinline__ int kv_col_tiles(const KvSeq &q, int G) { return (int)(((int64_t)q.n * G + KA_COLS - 1) / KA_COLS); }

__device__ __forceinline__ int kv_token_tiles(const KvAttnArgs &a, const KvSeq &q)
{
    return (kv_cached(q.len, a.c.T, a.b.max_pages) + 31) / 32;
}

// The common chunk length, by one wavefront.
__device__ __forceinline__ int kv_chunk(const KvAttnArgs &a, int G)
{
    const int lane = threadIdx.x & 63;
    float w = 0.0f;                      // exact enough: a length, not an index
    for (int base = 0; base < a.b.n_seqs; base += 64)
        if (base + lane < a.b.n_seqs) {
            const KvSeq q = kv_seq(a.b, base + lane);
            w += (float)kv_col_tiles(q, G) * (float)kv_token_tiles(a, q);
        }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) w += __shfl_xor(w, d, 64);
    // rounded up beyond what the sum's rounding can hide
    return max(KA_CHUNK, (int)(w / (float)a.items * 1.001f) + 1);
}

// Item `item` of the call (units: column tiles, whatever their chunks), or
// false past the last.
__device__ __forceinline__ bool kv_item(const KvAttnArgs &a, int G, int item, bool units, KvItem &it)
{
    const int lane = threadIdx.x & 63;
    const int C = a.split ? kv_chunk(a, G) : 0x7fffffff;
    int first = 0;
    for (int base = 0; base < a.b.n_seqs; base += 64) {
        KvSeq q{0, 0, 0};
        int nt = 0, ks = 0;
        if (base + lane < a.b.n_seqs) {
            q = kv_seq(a.b, base + lane);
            nt = kv_col_tiles(q, G);
            // (a sequence without tokens still has its rows to zero)
            ks = max(1, a.split ? (kv_token_tiles(a, q) + C - 1) / C : 1);
        }
        const int mine = nt * ks, count = units ? nt : mine;
        const int end = kv_wave_scan(count), items_end = units ? kv_wave_scan(mine) : end;
        const uint64_t past = __ballot(end > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            it.s = base + l;
            it.q = KvSeq{at(q.q0), at(q.n), at(q.len)};
            it.ks = at(ks);
            const int tiles = kv_token_tiles(a, it.q), i = item - (at(end) - at(count));
            it.chunk = (tiles + it.ks - 1) / it.ks;
            it.tile = units ? i : i / it.ks;
            it.split = units ? 0 : i % it.ks;
            it.first = first + at(items_end) - at(mine) + it.tile * it.ks;
            return true;
        }
        item -= __builtin_amdgcn_readlane(end, 63);
        first += __builtin_amdgcn_readlane(items_end, 63);
    }
    return false;
}

// Partial results of an item in the workspace: its columns' sums [KA_COLS][HD],
// then their (m, l).
template <int HD>
__device__ __forceinline__ float *kv_part(const KvAttnArgs &a, int item, int kvh)
{
    return (float *)a.ws + ((size_t)item * a.nkv + kvh) * KA_COLS * (HD + 2);
}

template <int HD, bool F8>
__global__ __launch_bounds__(KA_WAVES * 64, 2) void k_kv_attn(KvAttnArgs a)
{
    constexpr int NC = HD / 32;                    // 32-dim chunks of a row
    constexpr int NB = HD / 16;                    // 16-dim blocks of O
    constexpr int EB = F8 ? 1 : 2;
    constexpr int NK = HD * EB / 32;               // 16-byte pieces a lane loads of a tile's keys, and of its values
    constexpr int LO = HD + 4;                     // row of O in LDS: padded against bank conflicts
    __shared__ __align__(16) float s_o[KA_WAVES][KA_COLS * LO];
    __shared__ float s_m[KA_WAVES][KA_COLS], s_l[KA_WAVES][KA_COLS];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.nh / a.nkv, kvh = blockIdx.x % a.nkv;
    KvItem it;
    if (!kv_item(a, G, blockIdx.x / a.nkv, false, it)) return;
    const KvSeq q = it.q;
    // this lane's column: query q.q0 + qi, head kvh G + hg
    const int col = it.tile * KA_COLS + r16;
    const bool live = col < q.n * G;
    const int qi = live ? col / G : 0, hg = live ? col % G : 0;
    const size_t at = ((size_t)(q.q0 + qi) * a.nh + (size_t)kvh * G + hg) * HD;
    // tokens the column sees: 0 .. vis - 1
    const int cached = kv_cached(q.len, a.c.T, a.b.max_pages);
    const int vis = live ? kv_visible(q.len - q.n + qi, cached, a.block) : 0;
    int last = vis, least = live ? vis : cached;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) {
        last = max(last, __shfl_xor(last, d, 64));
        least = min(least, __shfl_xor(least, d, 64));
    }
    last = __builtin_amdgcn_readfirstlane(last);
    least = __builtin_amdgcn_readfirstlane(least);
    // this wavefront's token tiles: tile0 + w, every KA_WAVES-th, up to tile1
    const int tile0 = it.split * it.chunk, tile1 = min(tile0 + it.chunk, (last + 31) / 32);

    // queries: chunk 2 p + e of this lane holds dims 64 p + 16 g + 8 e .. + 7
    // (a lane's 16 dims of a 64-dim half are one piece of an E4M3 key row)
    kv_h8 qh[NC], ql[NC];
    float cmul;
    {
        float x[NC][8], amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const float *src = a.q + at + 64 * (c / 2) + 16 * g + 8 * (c % 2);
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 v = live ? *reinterpret_cast<const float4 *>(src + j) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[c][j] = v.x;
                x[c][j + 1] = v.y;
                x[c][j + 2] = v.z;
                x[c][j + 3] = v.w;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(x[c][j]));
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
        cmul = ldexpf(a.scale * 1.44269504088896341f, -up);
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = x[c][j] * mul;
                qh[c][j] = (_Float16)y;
                ql[c][j] = (_Float16)(y - (float)qh[c][j]);
            }
    }

    // m: the columns' reference of s + ve, raised when a score passes it by
    // KA_SLACK (-inf: nothing seen; at least -FLT_MAX else, so that a row whose
    // every score is -inf ends as 0 / 0, not as empty); l: this lane's share of
    // the sum
    const float inf = __builtin_inff(), low = -3.402823466e38f;
    float m = -inf, l = 0.0f;
    kv_f4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) o[b] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};

    struct Tile {
        uint4 k[NK], v[NK];
    };
    // row r of key block kb is token 8 (r / 4) + 4 kb + r % 4, so that the
    // scores of a lane are those of tokens 8 g + 4 kb + i
    const uint32_t koff = (8 * (r16 >> 2) + (r16 & 3)) * HD * EB + 16 * EB * g;
    const uint32_t voff = (r16 * 4 + g) * 16;
    auto load = [&](Tile &x, size_t byte) {
        const uint8_t *K = (const uint8_t *)a.c.k + byte, *V = (const uint8_t *)a.c.v + byte;
#pragma unroll
        for (int i = 0; i < NK; i++) {
            // key block, then chunk (F16) or pair of chunks (E4M3)
            const int kb = i / (NK / 2), ch = i % (NK / 2) * (F8 ? 2 : 1);
            x.k[i] = *reinterpret_cast<const uint4 *>(K + koff + 4 * kb * HD * EB + (64 * (ch / 2) + 8 * (ch % 2)) * EB);
        }
#pragma unroll
        for (int i = 0; i < NK; i++) x.v[i] = *reinterpret_cast<const uint4 *>(V + voff + 1024 * i);
    };
    auto compute = [&](const Tile &x, int k0, int ke, int ve) {
        const float c = F8 ? ldexpf(cmul, ke) : cmul, back = F8 ? ldexpf(1.0f, -ve) : 1.0f;
        kv_f4 sc[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            sc[kb] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ch = 0; ch < NC; ch += F8 ? 2 : 1) {
                kv_h8 kf[F8 ? 2 : 1];
                kv_widen<F8>(x.k[kb * (NK / 2) + ch / (F8 ? 2 : 1)], kf);
#pragma unroll
                for (int e = 0; e < (F8 ? 2 : 1); e++) {
                    sc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[e], ql[ch + e], sc[kb], 0, 0, 0);
                    sc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[e], qh[ch + e], sc[kb], 0, 0, 0);
                }
            }
        }
        const bool whole = k0 + 32 <= least;       // every column sees the tile
        float smax = -inf;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                smax = fmaxf(smax, whole || k0 + 8 * g + 4 * kb + i < vis ? sc[kb][i] : -inf);
        float mt = __builtin_fmaf(smax, c, (float)ve);
        mt = vis > k0 ? fmaxf(mt, low) : -inf;
        if (__any(mt > m + (float)KA_SLACK)) {
            mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
            mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
            const float mn = fmaxf(m, mt);
            const float corr = m == -inf ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[b][i] *= corr;
        }
        const float k = (float)ve + (float)KA_SHIFT - (m == -inf ? 0.0f : m);
        float sum = 0.0f;
        kv_h8 ph, pl;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][i], c, k));
                p = whole || k0 + 8 * g + 4 * kb + i < vis ? p : 0.0f;
                sum += p;
                ph[4 * kb + i] = (_Float16)p;
                pl[4 * kb + i] = (_Float16)(p - (float)ph[4 * kb + i]);
            }
        l = __builtin_fmaf(sum, back, l);
        // values: O rows are dims 16 b + row (F16), 32 (b / 2) + 2 row + b % 2 (E4M3)
        kv_h8 vf[NB];
#pragma unroll
        for (int i = 0; i < NK; i++) {
            kv_h8 y[F8 ? 2 : 1];
            kv_widen<F8>(x.v[i], y);
#pragma unroll
            for (int e = 0; e < (F8 ? 2 : 1); e++) vf[i * (F8 ? 2 : 1) + e] = y[e];
        }
        if (whole) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], pl, o[b], 0, 0, 0);
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], ph, o[b], 0, 0, 0);
            }
            return;
        }
        // some column does not see all 32 tokens: what it does not see may hold
        // anything (0 times a NaN is one), so the columns of each limit in turn
        // add a product whose values end there
        for (int done = k0;;) {
            int lim = vis > done ? vis : 0x7fffffff;
#pragma unroll
            for (int d = 8; d >= 1; d >>= 1) lim = min(lim, __shfl_xor(lim, d, 64));
            lim = __builtin_amdgcn_readfirstlane(lim);
            if (lim == 0x7fffffff) break;
            const bool mine = vis > done && (vis == lim || lim >= k0 + 32);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const kv_h8 y = kv_cut(vf[b], g, lim - k0);
                kv_f4 t = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pl, t, 0, 0, 0);
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ph, t, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) o[b][i] += mine ? t[i] : 0.0f;
            }
            if (lim >= k0 + 32) break;
            done = lim;
        }
    };

    // up to 64 of the wavefront's tiles at a time: a lane looks up one tile's
    // page and exponents, and the loop takes them from there
    for (int base = tile0 + w; base < tile1; base += 64 * KA_WAVES) {
        const int t = base + KA_WAVES * lane, k0 = 32 * t;
        int page = -1, ke = 0, ve = 0;
        if (t < tile1) page = kv_page(a.b, a.c, it.s, k0);
        const size_t slot = ((size_t)max(page, 0) * a.nkv + kvh) * (a.c.T / 32) + k0 % a.c.T / 32;
        if (F8 && page >= 0) {
            ke = a.c.k_exp[slot];
            ve = a.c.v_exp[slot];
        }
        const size_t byte = slot * 32 * HD * EB;
        const uint32_t blo = (uint32_t)byte, bhi = (uint32_t)(byte >> 32);
        auto where = [&](int i) {
            return (size_t)(uint32_t)__builtin_amdgcn_readlane(bhi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(blo, i);
        };
        uint64_t todo = __ballot(page >= 0);
        if (!todo) continue;
        // the next tile's loads are in flight during a tile's products (past
        // the last one, that tile again: a wait counts loads, so there must
        // always be some)
        Tile x, y;
        int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        load(x, where(i));
        auto step = [&](Tile &now, Tile &next) {
            const int j = todo ? __builtin_ctzll(todo) : i;
            load(next, where(j));
            compute(now, 32 * (base + KA_WAVES * i), __builtin_amdgcn_readlane(ke, i), __builtin_amdgcn_readlane(ve, i));
            const bool more = todo != 0;
            todo &= todo - 1;
            i = j;
            return more;
        };
        while (step(x, y) && step(y, x)) {
        }
    }

    // the wavefronts' results joined in LDS
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int b = 0; b < NB; b += F8 ? 2 : 1)
        if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < 4; i += 2)
                *reinterpret_cast<float4 *>(&s_o[w][r16 * LO + 16 * b + 8 * g + 2 * i]) =
                    make_float4(o[b][i], o[b + 1][i], o[b][i + 1], o[b + 1][i + 1]);
        } else {
            *reinterpret_cast<float4 *>(&s_o[w][r16 * LO + 16 * b + 4 * g]) = make_float4(o[b][0], o[b][1], o[b][2], o[b][3]);
        }
    if (g == 0) {
        s_m[w][r16] = m;
        s_l[w][r16] = l;
    }
    __syncthreads();
    const int cols = min(KA_COLS, q.n * G - it.tile * KA_COLS);
    for (int e = threadIdx.x; e < cols * (HD / 4); e += KA_WAVES * 64) {
        const int c = e / (HD / 4), d = e % (HD / 4) * 4;
        float M = s_m[0][c];
#pragma unroll
        for (int i = 1; i < KA_WAVES; i++) M = fmaxf(M, s_m[i][c]);
        float L = 0.0f;
        float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < KA_WAVES; i++) {
            const float f = s_m[i][c] == -inf ? 0.0f : __builtin_amdgcn_exp2f(s_m[i][c] - M);
            const float4 x = *reinterpret_cast<const float4 *>(&s_o[i][c * LO + d]);
            L += s_l[i][c] * f;
            O.x += x.x * f;
            O.y += x.y * f;
            O.z += x.z * f;
            O.w += x.w * f;
        }
        if (it.ks == 1) {
            const int cc = it.tile * KA_COLS + c;
            const float inv = M == -inf ? 0.0f : 1.0f / L;         // nothing seen: zeros
            *reinterpret_cast<float4 *>(a.out + ((size_t)(q.q0 + cc / G) * a.nh + (size_t)kvh * G + cc % G) * HD + d) =
                make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
        } else {
            float *part = kv_part<HD>(a, it.first + it.split, kvh);
            *reinterpret_cast<float4 *>(part + c * HD + d) = O;
            if (d == 0) *reinterpret_cast<float2 *>(part + KA_COLS * HD + 2 * c) = make_float2(M, L);
        }
    }
}

// Joins the chunks of a column: a workgroup takes one column, its wavefronts
// every KA_WAVES-th chunk.
template <int HD>
__global__ __launch_bounds__(KA_WAVES * 64) void k_kv_join(KvAttnArgs a)
{
    constexpr int ND = HD / 64;                    // dims of a lane
    __shared__ float s_o[KA_WAVES][HD], s_l[KA_WAVES];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int G = a.nh / a.nkv, kvh = blockIdx.y % a.nkv, c = blockIdx.y / a.nkv;
    KvItem it;
    if (!kv_item(a, G, blockIdx.x, true, it) || it.ks == 1) return;
    const int col = it.tile * KA_COLS + c;
    if (col >= it.q.n * G) return;
    const float inf = __builtin_inff();
    // the chunks' references: every lane those of chunks lane, lane + 64, ..
    float M = -inf;
    for (int j = lane; j < it.ks; j += 64) M = fmaxf(M, kv_part<HD>(a, it.first + j, kvh)[KA_COLS * HD + 2 * c]);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
    float o[ND] = {}, l = 0.0f;
#pragma unroll 8
    for (int j = w; j < it.ks; j += KA_WAVES) {
        const float *part = kv_part<HD>(a, it.first + j, kvh);
        const float2 ml = *reinterpret_cast<const float2 *>(part + KA_COLS * HD + 2 * c);
        const float f = ml.x == -inf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
        l += ml.y * f;
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] += part[c * HD + ND * lane + d] * f;
    }
#pragma unroll
    for (int d = 0; d < ND; d++) s_o[w][ND * lane + d] = o[d];
    if (lane == 0) s_l[w] = l;
    __syncthreads();
    if (threadIdx.x >= HD) return;
    float O = 0.0f, L = 0.0f;
#pragma unroll
    for (int i = 0; i < KA_WAVES; i++) {
        O += s_o[i][threadIdx.x];
        L += s_l[i];
    }
    a.out[((size_t)(it.q.q0 + col / G) * a.nh + (size_t)kvh * G + col % G) * HD + threadIdx.x] = M == -inf ? 0.0f : O / L;
}

// What the launches take: the items wanted per kv head and at most, and whether
// any sequence can have several chunks (from the page table's width: the
// lengths themselves are on the GPU).
struct KvAttnPlan {
    int64_t units, items;                // column tiles, items at most
    int32_t want;
    bool split;
};

static KvAttnPlan kv_attn_plan(const KvAttnArgs &a)
{
    KvAttnPlan p;
    p.units = (int64_t)a.b.n_tokens * (a.nh / a.nkv) / KA_COLS + a.b.n_seqs;
    p.want = (KA_ITEMS + a.nkv - 1) / a.nkv;
    const int64_t tiles = (int64_t)a.b.max_pages * (a.c.T / 32);
    p.split = tiles > KA_CHUNK;
    // a column tile has at most one chunk more than its share of those wanted
    p.items = p.split ? p.want + p.units : p.units;
    return p;
}

size_t kv_attn_ws_bytes(const KvAttnArgs &a)
{
    const KvAttnPlan p = kv_attn_plan(a);
    return p.split ? (size_t)p.items * a.nkv * KA_COLS * (a.hd + 2) * 4 : 256;
}

hipError_t launch_kv_attn(const KvAttnArgs &args, hipStream_t s)
{
    KvAttnArgs a = args;
    if (a.nkv <= 0 || a.nh % a.nkv) return hipErrorInvalidValue;
    const KvAttnPlan p = kv_attn_plan(a);
    a.items = p.want;
    a.split = p.split;
    const dim3 grid((unsigned)(p.items * a.nkv)), block(KA_WAVES * 64);
    switch (a.hd * (a.c.type == DMOE_KV_E4M3 ? -1 : 1)) {
    case 64: hipLaunchKernelGGL((k_kv_attn<64, false>), grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL((k_kv_attn<128, false>), grid, block, 0, s, a); break;
    case -64: hipLaunchKernelGGL((k_kv_attn<64, true>), grid, block, 0, s, a); break;
    case -128: hipLaunchKernelGGL((k_kv_attn<128, true>), grid, block, 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.split) return e;
    const dim3 join((unsigned)p.units, KA_COLS * a.nkv);
    if (a.hd == 64)
        hipLaunchKernelGGL((k_kv_join<64>), join, block, 0, s, a);
    else
        hipLaunchKernelGGL((k_kv_join<128>), join, block, 0, s, a);
    return hipGetLastError();
}

} // namespace dmoe
