// k_kv_append.hip — rows of the fused QKV projection into a paged KV cache
// (the position-dependent half of src/diffuse-moe-graph.cpp:132-155, which the
// reference repeats for the whole window every step).
//
// Per row and head: QK RMSNorm, the NEOX rotation of the first rd dims at the
// row's position, queries to q_out (f32), keys and values to their page (F16,
// or E4M3 with a power-of-two scale per block of 32 tokens and head).
//
// The norm and the rotation run in binary64 and are rounded once to f32: the
// angle of a far position has no correct digits left in f32 (position 131,072
// times a frequency rounded to 2^-24 is off by 0.008 rad), the launch waits for
// memory, and an f64 multiply-add has an f32 one's rate here.
//
// E4M3: a block's exponent e is the least whole number with amax <= 448 2^e
// (in KV_EMIN .. KV_EMAX), so a code is the value over a power of two, rounded
// once: half a step, 2^-4 relative (2^-10 2^e below 2^-6 2^e).  A power of two
// costs a floating code no precision, keeps the attention's rescaling exact,
// and lets a block's exponent grow: rows that begin inside a block keep the
// tokens before them, whose codes are divided by 2^(e - e_old) (exact, but for
// codes that fall under 2^-6) where e exceeds theirs.
#include "dmoe_kv.h"

#pragma clang fp contract(off)

namespace dmoe {

constexpr int KA_WAVES = 4;

// f32 -> E4M3 (round to nearest even); what the type does not hold (inf, NaN,
// and values over 448, which only KV_EMAX lets through) becomes its NaN.
__device__ __forceinline__ uint32_t kv_e4m3x2(float a, float b)
{
    const float nan = __builtin_nanf("");
    a = fabsf(a) <= 448.0f ? a : nan;
    b = fabsf(b) <= 448.0f ? b : nan;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

// The least e with amax <= 448 * 2^e, in KV_EMIN .. KV_EMAX.  amax finite.
__device__ __forceinline__ int kv_exponent(float amax)
{
    if (!(amax > 0.0f)) return KV_EMIN;
    int x;
    const float m = frexpf(amax, &x);              // amax = m 2^x, 448 = 0.875 * 2^9
    const int e = m <= 0.875f ? x - 9 : x - 8;
    return min(max(e, KV_EMIN), KV_EMAX);
}

// One workgroup: one block's rows (up to 32) of KA_WAVES heads.  A wavefront
// takes up to eight rows of a head, so 1, 2 or 4 of them share a head by the
// block's rows and the heads take 1, 2 or 4 passes; the cosines and sines of
// the rows are formed once for all of them.  A lane holds two dims of a row
// (hd 64: a wavefront two rows at a time).
template <int HD, bool F8>
__global__ __launch_bounds__(KA_WAVES * 64) void k_kv_append(KvAppendArgs a)
{
    constexpr int TPW = 128 / HD;                  // rows per wavefront step
    constexpr int STEPS = 8 / TPW;
    constexpr int EB = F8 ? 1 : 2;
    constexpr int LROW = HD * EB + 16;             // bytes of a row in the tile
    __shared__ __align__(16) uint8_t s_tile[32 * LROW];
    __shared__ float s_amax[KA_WAVES];
    extern __shared__ __align__(16) double2 s_rot[];                 // [rows][rd / 2]
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int half = a.rd / 2, heads = a.nh + 2 * a.nkv;

    if (blockIdx.x >= (unsigned)a.blocks) {
        // a layer's padded rows, past the last sequence's: their attention is zero
        const int64_t first = (int64_t)min(max(a.b.q_start[a.b.n_seqs], 0), a.b.n_tokens) * a.nh * HD;
        const int64_t n = (int64_t)a.b.n_tokens * a.nh * HD - first;
        const int64_t step = (int64_t)(gridDim.x - a.blocks) * gridDim.y * KA_WAVES * 64 * 4;
        const int64_t i0 = ((int64_t)(blockIdx.x - a.blocks) * gridDim.y + blockIdx.y) * KA_WAVES * 64 + threadIdx.x;
        for (int64_t i = 4 * i0; i < n; i += step)
            *reinterpret_cast<float4 *>(a.rest + first + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        return;
    }
    int s, blk;
    KvSeq q;
    if (!kv_find(a.b, blockIdx.x, [](const KvSeq &r) { return kv_blocks(r); }, s, q, blk)) return;
    const int pos_q = q.len - q.n;                                   // the first row's position
    const int pos = max(pos_q, (pos_q / 32 + blk) * 32);             // this block's first row
    const int off = pos % 32;
    const int m = min(32 - off, q.len - pos);                        // rows here
    const int row = q.q0 + (pos - pos_q);
    const int end = off + m;
    const int page = kv_page(a.b, a.c, s, pos);

    // cos and sin of position * base^(-2 i / rd): the angle in turns, reduced
    // to half a turn exactly
    for (int i = threadIdx.x; i < m * half; i += KA_WAVES * 64) {
        const int t = i / half, p = i % half;
        double turns = (double)(pos + t) * (exp2(a.log2_step * (double)p) * 0.15915494309189533577);
        turns -= rint(turns);
        double sn, cs;
        sincospi(2.0 * turns, &sn, &cs);
        s_rot[i] = make_double2(cs, sn);
    }
    __syncthreads();

    const int share = m <= 8 ? 1 : m <= 16 ? 2 : 4;                  // wavefronts of a head
    const int rg = w & (share - 1), r0 = 8 * rg;
    uint8_t *tile = s_tile + (w / share) * share * 8 * LROW;         // rows of this wavefront's head
    const int sub = lane / (HD / 2), d0 = 2 * (lane % (HD / 2));
    // the rotation's partner of each of the lane's dims
    auto partner = [&](int d) { return d < half ? d + half : d < 2 * half ? d - half : d; };
    const int p0 = partner(d0), p1 = partner(d0 + 1);
    const size_t row_floats = (size_t)heads * HD;

    for (int pass = 0; pass < share; pass++) {
        const int hh = (blockIdx.y * KA_WAVES) + pass * (KA_WAVES / share) + w / share;
        const bool rotated = hh < a.nh + a.nkv, cached = hh >= a.nh && hh < heads && page >= 0;
        const bool is_v = !rotated;
        float v[STEPS][2];
        float amax = 0.0f;
        if (hh < heads) {
            const float *src = a.qkv + (size_t)row * row_floats + (size_t)hh * HD + d0;
#pragma unroll
            for (int u = 0; u < STEPS; u++) {
                const int t = r0 + u * TPW + sub;
                float2 x = make_float2(0.0f, 0.0f);
                if (t < m) {
                    x = *reinterpret_cast<const float2 *>(src + (size_t)t * row_floats);
                    for (int k = 1; k < a.ks; k++) {   // the projection's reduction slices, in order
                        const float2 y = *reinterpret_cast<const float2 *>(src + (size_t)k * a.kstride + (size_t)t * row_floats);
                        x.x = x.x + y.x;
                        x.y = x.y + y.y;
                    }
                }
                v[u][0] = x.x;
                v[u][1] = x.y;
            }
            if (rotated) {
                float g0 = 1.0f, g1 = 1.0f;
                if (a.qk_norm) {
                    const float *gain = hh < a.nh ? a.q_norm : a.k_norm;
                    g0 = gain[d0];
                    g1 = gain[d0 + 1];
                }
#pragma unroll
                for (int u = 0; u < STEPS; u++) {
                    const int t = r0 + u * TPW + sub;
                    double y0 = v[u][0], y1 = v[u][1];
                    if (a.qk_norm) {
                        double ss = y0 * y0 + y1 * y1;
#pragma unroll
                        for (int d = HD / 4; d >= 1; d >>= 1) ss += __shfl_xor(ss, d, 64);
                        const double scale = 1.0 / sqrt(ss / (double)HD + (double)a.eps);
                        y0 = y0 * scale * (double)g0;
                        y1 = y1 * scale * (double)g1;
                    }
                    if (half) {
                        const int l0 = sub * (HD / 2) + p0 / 2, l1 = sub * (HD / 2) + p1 / 2;
                        const double a0 = __shfl(y0, l0, 64), b0 = __shfl(y1, l0, 64);
                        const double a1 = __shfl(y0, l1, 64), b1 = __shfl(y1, l1, 64);
                        const double z0 = p0 & 1 ? b0 : a0, z1 = p1 & 1 ? b1 : a1;
                        auto turn = [&](int d, double y, double z) {
                            if (d >= 2 * half || t >= m) return y;
                            const double2 r = s_rot[t * half + (d < half ? d : d - half)];
                            return d < half ? y * r.x - z * r.y : z * r.y + y * r.x;
                        };
                        y0 = turn(d0, y0, z0);
                        y1 = turn(d0 + 1, y1, z1);
                    }
                    v[u][0] = (float)y0;
                    v[u][1] = (float)y1;
                    if (hh < a.nh && t < m)
                        *reinterpret_cast<float2 *>(a.q_out + ((size_t)(row + t) * a.nh + hh) * HD + d0) =
                            make_float2(v[u][0], v[u][1]);
                }
            }
        }
        if (blockIdx.y * KA_WAVES + KA_WAVES <= (unsigned)a.nh) continue;   // only queries here: nothing to exchange

        const int h = hh - a.nh - (is_v ? a.nkv : 0);
        const size_t slot = cached ? ((size_t)page * a.nkv + h) * (a.c.T / 32) + pos % a.c.T / 32 : 0;
        uint8_t *dst = (uint8_t *)(is_v ? a.c.v : a.c.k) + slot * 32 * HD * EB;
        int8_t *exps = is_v ? a.c.v_exp : a.c.k_exp;
        float inv = 1.0f, grown = 1.0f;
        bool regrow = false;
        if (F8) {
            int old = 0;
            if (cached) {
                old = exps[slot];
#pragma unroll
                for (int u = 0; u < STEPS; u++)
                    if (r0 + u * TPW + sub < m)
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            if (fabsf(v[u][e]) <= 3.402823466e38f) amax = fmaxf(amax, fabsf(v[u][e]));
#pragma unroll
                for (int d = 32; d >= 1; d >>= 1) amax = fmaxf(amax, __shfl_xor(amax, d, 64));
            }
            if (lane == 0) s_amax[w] = amax;
            __syncthreads();
            for (int i = 0; i < share; i++) amax = fmaxf(amax, s_amax[w - rg + i]);
            int e = kv_exponent(amax);
            if (off) {
                regrow = e > old;
                e = max(e, old);
                if (regrow) grown = ldexpf(1.0f, old - e);
            }
            inv = ldexpf(1.0f, -e);
            // (every wavefront has read `old` before the barrier)
            if (cached && lane == 0 && rg == 0 && (off == 0 || regrow)) exps[slot] = (int8_t)e;
        }
        // the rows' codes to the tile, [row][dim]
        if (cached) {
#pragma unroll
            for (int u = 0; u < STEPS; u++) {
                const int t = r0 + u * TPW + sub;
                if (t >= m) continue;
                if (F8)
                    *reinterpret_cast<uint16_t *>(tile + t * LROW + d0) = (uint16_t)kv_e4m3x2(v[u][0] * inv, v[u][1] * inv);
                else
                    *reinterpret_cast<kv_h2 *>(tile + t * LROW + 2 * d0) = kv_h2{(_Float16)v[u][0], (_Float16)v[u][1]};
            }
        }
        __syncthreads();
        if (cached) {
            auto regrown = [&](uint32_t x) {                         // four kept codes
                const uint32_t lo = kv_e4m3x2(__builtin_amdgcn_cvt_f32_fp8(x, 0) * grown, __builtin_amdgcn_cvt_f32_fp8(x, 1) * grown);
                const uint32_t hi = kv_e4m3x2(__builtin_amdgcn_cvt_f32_fp8(x, 2) * grown, __builtin_amdgcn_cvt_f32_fp8(x, 3) * grown);
                return lo | hi << 16;
            };
            if (!is_v) {
                constexpr int PR = HD * EB / 16;                     // pieces of a row
                for (int i = lane + 64 * rg + (regrow ? 0 : off * PR); i < end * PR; i += 64 * share) {
                    const int r = i / PR, p = i % PR;
                    uint4 x;
                    if (r >= off) {
                        x = *reinterpret_cast<const uint4 *>(tile + (r - off) * LROW + 16 * p);
                    } else {
                        x = *reinterpret_cast<const uint4 *>(dst + (size_t)i * 16);
                        x = make_uint4(regrown(x.x), regrown(x.y), regrown(x.z), regrown(x.w));
                    }
                    *reinterpret_cast<uint4 *>(dst + (size_t)i * 16) = x;
                }
            } else {
                // 8 tokens of a dim (F16) or of two (E4M3) a piece; a piece that
                // these rows fill in part keeps the others
                constexpr int ND = F8 ? 2 : 1;
                for (int i = lane + 64 * rg; i < 4 * HD / ND; i += 64 * share) {
                    const int d = i / 4 * ND, t0 = i % 4 * 8;
                    const bool fresh = t0 < end && t0 + 8 > off;
                    if (!fresh && !(regrow && t0 < off)) continue;
                    uint8_t x[16];
                    if (t0 < off || t0 + 8 > end) {
                        uint4 o = *reinterpret_cast<const uint4 *>(dst + (size_t)i * 16);
                        __builtin_memcpy(x, &o, 16);
                        if (regrow) {
                            // what lies past these rows is no one's: only kept tokens are rewritten
                            o = make_uint4(regrown(o.x), regrown(o.y), regrown(o.z), regrown(o.w));
                            uint8_t n[16];
                            __builtin_memcpy(n, &o, 16);
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                if (t0 + (j & 7) < off) x[j] = n[j];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < ND; e++)
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (t0 + j >= off && t0 + j < end) {
                                const uint8_t *from = tile + (t0 + j - off) * LROW + (d + e) * EB;
                                if (F8) {
                                    x[8 * e + j] = *from;
                                } else {
                                    x[2 * j] = from[0];
                                    x[2 * j + 1] = from[1];
                                }
                            }
                    uint4 o;
                    __builtin_memcpy(&o, x, 16);
                    *reinterpret_cast<uint4 *>(dst + (size_t)i * 16) = o;
                }
            }
        }
        __syncthreads();                                             // the tile is the next pass's
    }
}

hipError_t launch_kv_append(const KvAppendArgs &args, hipStream_t s)
{
    KvAppendArgs a = args;
    if (a.rd < 0 || a.rd > a.hd || a.rd % 2 || a.ks < 1) return hipErrorInvalidValue;
    a.blocks = (int32_t)kv_blocks_most(a.b.n_seqs, a.b.n_tokens);
    const int heads = a.nh + 2 * a.nkv;
    const dim3 grid((unsigned)a.blocks + (a.rest ? 32 : 0), (heads + KA_WAVES - 1) / KA_WAVES);
    const bool f8 = a.c.type == DMOE_KV_E4M3;
    const size_t lds = (size_t)32 * (a.rd / 2) * sizeof(double2);
    switch (a.hd * (f8 ? -1 : 1)) {
    case 64: hipLaunchKernelGGL((k_kv_append<64, false>), grid, dim3(KA_WAVES * 64), lds, s, a); break;
    case 128: hipLaunchKernelGGL((k_kv_append<128, false>), grid, dim3(KA_WAVES * 64), lds, s, a); break;
    case -64: hipLaunchKernelGGL((k_kv_append<64, true>), grid, dim3(KA_WAVES * 64), lds, s, a); break;
    case -128: hipLaunchKernelGGL((k_kv_append<128, true>), grid, dim3(KA_WAVES * 64), lds, s, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

} // namespace dmoe
