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

constexpr int KA_COLS = 16;              // columns of a wavefront
constexpr int KA_SHIFT = 4;              // probabilities are held times 2^KA_SHIFT

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

template <int HD, bool F8>
__global__ __launch_bounds__(256) void k_kv_attn(KvAttnArgs a)
{
    constexpr int NC = HD / 32;                    // 32-dim chunks of a row
    constexpr int NB = HD / 16;                    // 16-dim blocks of O
    constexpr int EB = F8 ? 1 : 2;
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int G = a.nh / a.nkv, kvh = blockIdx.y;
    int s, tile;
    KvSeq q;
    if (!kv_find(a.b, blockIdx.x * 4 + (threadIdx.x >> 6),
                 [=](const KvSeq &r) { return (int)(((long)r.n * G + KA_COLS - 1) / KA_COLS); }, s, q, tile))
        return;
    // this lane's column: query q.q0 + qi, head kvh G + hg
    const int col = tile * KA_COLS + r16;
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

    // m: the largest s + ve so far (-inf: nothing seen; at least -FLT_MAX else,
    // so that a row whose every score is -inf ends as 0 / 0, not as empty)
    const float inf = __builtin_inff(), low = -3.402823466e38f;
    float m = -inf, l = 0.0f;
    kv_f4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) o[b] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < last; k0 += 32) {
        const int page = kv_page(a.b, a.c, s, k0);
        if (page < 0) continue;
        const size_t slot = ((size_t)page * a.nkv + kvh) * (a.c.T / 32) + k0 % a.c.T / 32;
        const uint8_t *K = (const uint8_t *)a.c.k + slot * 32 * HD * EB;
        const uint8_t *V = (const uint8_t *)a.c.v + slot * 32 * HD * EB;
        float c = cmul, ve = 0.0f, back = 1.0f;
        if (F8) {
            c = ldexpf(cmul, a.c.k_exp[slot]);
            ve = (float)a.c.v_exp[slot];
            back = ldexpf(1.0f, -a.c.v_exp[slot]);
        }
        // row r of key block kb is token 8 (r / 4) + 4 kb + r % 4, so that the
        // scores of a lane are those of tokens 8 g + 4 kb + i
        kv_f4 sc[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            sc[kb] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
            const uint8_t *kr = K + (8 * (r16 >> 2) + 4 * kb + (r16 & 3)) * HD * EB;
#pragma unroll
            for (int ch = 0; ch < NC; ch += F8 ? 2 : 1) {
                kv_h8 kf[F8 ? 2 : 1];
                kv_widen<F8>(*reinterpret_cast<const uint4 *>(kr + (64 * (ch / 2) + 16 * g + 8 * (ch % 2)) * EB), kf);
#pragma unroll
                for (int e = 0; e < (F8 ? 2 : 1); e++) {
                    sc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[e], ql[ch + e], sc[kb], 0, 0, 0);
                    sc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[e], qh[ch + e], sc[kb], 0, 0, 0);
                }
            }
        }
        float mt = vis > k0 ? low : -inf;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool ok = k0 + 8 * g + 4 * kb + i < vis;
                sc[kb][i] = ok ? __builtin_fmaf(sc[kb][i], c, ve) : -inf;
                mt = fmaxf(mt, sc[kb][i]);
            }
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        const float mn = fmaxf(m, mt), ref = mn == -inf ? 0.0f : mn;
        const float corr = m == -inf ? 0.0f : __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        float sum = 0.0f;
        kv_h8 ph, pl;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __builtin_amdgcn_exp2f(sc[kb][i] - ref + (float)KA_SHIFT);
                sum += p;
                ph[4 * kb + i] = (_Float16)p;
                pl[4 * kb + i] = (_Float16)(p - (float)ph[4 * kb + i]);
            }
        l = l * corr + sum * back;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[b][i] *= corr;
        // values: O rows are dims 16 b + row (F16), 32 (b / 2) + 2 row + b % 2 (E4M3)
        kv_h8 vf[NB];
#pragma unroll
        for (int b = 0; b < NB; b += F8 ? 2 : 1) {
            kv_h8 x[F8 ? 2 : 1];
            kv_widen<F8>(*reinterpret_cast<const uint4 *>(V + (size_t)((16 * (F8 ? b / 2 : b) + r16) * 4 + g) * 16), x);
#pragma unroll
            for (int e = 0; e < (F8 ? 2 : 1); e++) vf[b + e] = x[e];
        }
        if (k0 + 32 <= least) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], pl, o[b], 0, 0, 0);
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], ph, o[b], 0, 0, 0);
            }
            continue;
        }
        // some column does not see all 32 tokens: what it does not see may hold
        // anything (0 times a NaN is one), so the columns of each limit in turn
        // add a product whose values end there
        for (int done = k0;;) {
            int lim = live && vis > done ? vis : 0x7fffffff;
#pragma unroll
            for (int d = 8; d >= 1; d >>= 1) lim = min(lim, __shfl_xor(lim, d, 64));
            lim = __builtin_amdgcn_readfirstlane(lim);
            if (lim == 0x7fffffff) break;
            const bool mine = live && vis > done && (vis == lim || lim >= k0 + 32);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const kv_h8 x = kv_cut(vf[b], g, lim - k0);
                kv_f4 t = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl, t, 0, 0, 0);
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph, t, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) o[b][i] += mine ? t[i] : 0.0f;
            }
            if (lim >= k0 + 32) break;
            done = lim;
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (!live) return;
    float *dst = a.out + at;
    // nothing seen: zeros
    const float inv = m == -inf ? 0.0f : 1.0f / l;
    if constexpr (F8) {
#pragma unroll
        for (int b = 0; b < NB; b += 2)
#pragma unroll
            for (int i = 0; i < 4; i += 2)
                *reinterpret_cast<float4 *>(dst + 16 * b + 8 * g + 2 * i) =
                    make_float4(o[b][i] * inv, o[b + 1][i] * inv, o[b][i + 1] * inv, o[b + 1][i + 1] * inv);
    } else {
#pragma unroll
        for (int b = 0; b < NB; b++)
            *reinterpret_cast<float4 *>(dst + 16 * b + 4 * g) =
                make_float4(o[b][0] * inv, o[b][1] * inv, o[b][2] * inv, o[b][3] * inv);
    }
}

size_t kv_attn_ws_bytes(const KvAttnArgs &) { return 256; }

hipError_t launch_kv_attn(const KvAttnArgs &a, hipStream_t s)
{
    if (a.nkv <= 0 || a.nh % a.nkv) return hipErrorInvalidValue;
    const long tiles = (long)a.b.n_tokens * (a.nh / a.nkv) / KA_COLS + a.b.n_seqs;
    const dim3 grid((unsigned)((tiles + 3) / 4), a.nkv);
    switch (a.hd * (a.c.type == DMOE_KV_E4M3 ? -1 : 1)) {
    case 64: hipLaunchKernelGGL((k_kv_attn<64, false>), grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL((k_kv_attn<128, false>), grid, dim3(256), 0, s, a); break;
    case -64: hipLaunchKernelGGL((k_kv_attn<64, true>), grid, dim3(256), 0, s, a); break;
    case -128: hipLaunchKernelGGL((k_kv_attn<128, true>), grid, dim3(256), 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

} // namespace dmoe
