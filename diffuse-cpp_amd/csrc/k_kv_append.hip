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
#include <type_traits>

#include "dmoe_device.h"
#include "dmoe_kv.h"

#pragma clang fp contract(off)

namespace dmoe {

constexpr int KA_WAVES = 4;

struct __attribute__((packed, aligned(4))) Quad {
    float x[4];
};

// f32 -> E4M3 (round to nearest even); what the type does not hold (inf, NaN,
// and values over 448, which only KV_EMAX lets through) becomes its NaN.
__device__ __forceinline__ uint32_t kv_e4m3x2(float a, float b)
{
    const float nan = __builtin_nanf("");
    a = fabsf(a) <= 448.0f ? a : nan;
    b = fabsf(b) <= 448.0f ? b : nan;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

// cos and sin of an angle in turns: reduced exactly to an eighth of a turn and a
// quadrant, then their Taylor series to the 16th and 17th power (the next terms
// are below 2^-58).
__device__ __forceinline__ double2 kv_cos_sin(double turns)
{
    turns -= rint(turns);
    const double k = rint(4.0 * turns);
    const double x = (turns - 0.25 * k) * 6.283185307179586477, z = x * x;
    double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;
    s = __builtin_fma(-s, z, 1.0 / 1307674368000.0);
    c = __builtin_fma(-c, z, 1.0 / 87178291200.0);
    s = __builtin_fma(-s, z, 1.0 / 6227020800.0);
    c = __builtin_fma(-c, z, 1.0 / 479001600.0);
    s = __builtin_fma(-s, z, 1.0 / 39916800.0);
    c = __builtin_fma(-c, z, 1.0 / 3628800.0);
    s = __builtin_fma(-s, z, 1.0 / 362880.0);
    c = __builtin_fma(-c, z, 1.0 / 40320.0);
    s = __builtin_fma(-s, z, 1.0 / 5040.0);
    c = __builtin_fma(-c, z, 1.0 / 720.0);
    s = __builtin_fma(-s, z, 1.0 / 120.0);
    c = __builtin_fma(-c, z, 1.0 / 24.0);
    s = __builtin_fma(-s, z, 1.0 / 6.0);
    c = __builtin_fma(-c, z, 0.5);
    s = __builtin_fma(-s, z, 1.0) * x;
    c = __builtin_fma(-c, z, 1.0);
    const int q = (int)k & 3;
    const double cc = q & 1 ? s : c, ss = q & 1 ? c : s;
    return make_double2(q == 1 || q == 2 ? -cc : cc, q >= 2 ? -ss : ss);
}

// 1 / sqrt(x), x >= 0: two Newton steps from the hardware's estimate.
__device__ __forceinline__ double kv_rsqrt(double x)
{
    double r = __builtin_amdgcn_rsq(x);
    if (!(x > 0.0 && x < __builtin_inf())) return r;
#pragma unroll
    for (int i = 0; i < 2; i++) r = __builtin_fma(0.5 * r, __builtin_fma(-x * r, r, 1.0), r);
    return r;
}

// The sum over a row's 16 lanes, in every one of them.
__device__ __forceinline__ double kv_row_sum(double v)
{
#define KV_ROR(n) \
    v += __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), 0x120 + n, 0xf, 0xf, false), \
                          __builtin_amdgcn_update_dpp(0, __double2loint(v), 0x120 + n, 0xf, 0xf, false))
    KV_ROR(8);
    KV_ROR(4);
    KV_ROR(2);
    KV_ROR(1);
#undef KV_ROR
    return v;
}

// The value 8 lanes on within a row of 16.
__device__ __forceinline__ double kv_ror8(double v)
{
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), 0x128, 0xf, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), 0x128, 0xf, 0xf, false));
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

// One workgroup: one block's rows (up to 32) of `group` heads.  A wavefront
// takes up to eight rows of a head, so 1, 2 or 4 of them share a head by the
// block's rows, and the group's heads take one or more passes; the cosines and
// sines of the rows are formed once for all of them.  16 lanes hold a row, four
// dims of each 64 a lane (16-byte loads; the norm's sum takes four DPP steps for
// four rows at once).
// Bound by its bytes: 4001 rows of 32 + 2 * 4 heads of 128 with an E4M3 cache,
// 152 MB, take 32.9 us, 4.6 TB/s of the 5.15 that a large copy reaches; without
// the norm and the rotation it is no faster.  What that took (at four heads a
// workgroup, 42.2 us without either): a block's head groups next to each other in
// the grid, 40.8, query stores past the caches, 37.3, both, 36.1.
// ROT: rd / 2 where it is 32 or 64 (the partners of a lane's dims are 8 lanes on,
// or its own other vector), else -1.
template <int HD, bool F8, int ROT>
__global__ __launch_bounds__(KA_WAVES * 64) void k_kv_append(KvAppendArgs a)
{
    constexpr int NV = HD / 64;                    // vectors of four dims of a lane
    constexpr int EB = F8 ? 1 : 2;
    constexpr int LROW = HD * EB + 16;             // bytes of a row in the values' tile
    __shared__ __align__(16) uint8_t s_tile[32 * LROW];
    __shared__ __align__(16) double s_x[KA_WAVES][ROT < 0 ? 4 * HD : 1];     // rows of a step, for the rotation's partners
    __shared__ float s_amax[KA_WAVES];
    extern __shared__ __align__(16) double s_rot[];                  // cosines [rows][rd / 2], sines behind 32 rows of them
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int half = ROT < 0 ? a.rd / 2 : ROT, heads = a.nh + 2 * a.nkv;

    // a block's head groups one after the other: what runs at a time covers whole rows
    const uint32_t groups = gridDim.x / (uint32_t)(a.blocks + a.zeros), item = blockIdx.x / groups, hg = blockIdx.x % groups;
    if (item >= (uint32_t)a.blocks) {
        // a layer's padded rows, past the last sequence's: their attention is zero
        const int64_t first = (int64_t)min(max(a.b.q_start[a.b.n_seqs], 0), a.b.n_tokens) * a.nh * HD;
        const int64_t n = (int64_t)a.b.n_tokens * a.nh * HD - first;
        const int64_t step = (int64_t)a.zeros * groups * KA_WAVES * 64 * 4;
        const int64_t i0 = (int64_t)(blockIdx.x - a.blocks * groups) * KA_WAVES * 64 + threadIdx.x;
        for (int64_t i = 4 * i0; i < n; i += step)
            *reinterpret_cast<float4 *>(a.rest + first + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        return;
    }
    int s, blk;
    KvSeq q;
    // Up to 64 sequences: their blocks counted, without gaps between them (16 blocks
    // of 32 rows 7.4 us on end, from their places 9.4).  More: from their places, as
    // counting takes every workgroup a pass over all of them (4096 rows of as many
    // sequences 837 us, so 196).
    if (a.b.n_seqs <= 64 ? !kv_find(a.b, (int)item, [](const KvSeq &r) { return kv_blocks(r); }, s, q, blk)
                         : !kv_find_block(a.b, (int)item, s, q, blk))
        return;
    const int pos_q = q.len - q.n;                                   // the first row's position
    const int pos = max(pos_q, (pos_q / 32 + blk) * 32);             // this block's first row
    const int off = pos % 32;
    const int m = min(32 - off, q.len - pos);                        // rows here
    const int row = q.q0 + (pos - pos_q);
    const int end = off + m;
    const int page = kv_page(a.b, a.c, s, pos);

    const int share = m <= 8 ? 1 : m <= 16 ? 2 : 4;                  // wavefronts of a head
    const int rg = w & (share - 1), r0 = 8 * rg;
    uint8_t *tile = s_tile + (w / share) * share * 8 * LROW;         // rows of this wavefront's head
    const int sub = lane >> 4, d0 = 4 * (lane & 15);                 // row of a step; dims d0 + 64 v ..
    const size_t row_floats = (size_t)heads * HD;
    const int head0 = (int)hg * a.group, head1 = min(head0 + a.group, heads);
    const bool rotates = head0 < a.nh + a.nkv, caches = head1 > a.nh;

    float x[2][NV][4], next[2][NV][4];
    auto load = [&](float (&x)[2][NV][4], int hh) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int t = r0 + 4 * u + sub;
            const float *src = a.qkv + (size_t)(row + t) * row_floats + (size_t)hh * HD + d0;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (t < m && hh < head1) {
                    y = *reinterpret_cast<const float4 *>(src + 64 * v);
                    for (int k = 1; k < a.ks; k++) {   // the projection's reduction slices, in order
                        const float4 z = *reinterpret_cast<const float4 *>(src + 64 * v + (size_t)k * a.kstride);
                        y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
                    }
                }
                x[u][v][0] = y.x;
                x[u][v][1] = y.y;
                x[u][v][2] = y.z;
                x[u][v][3] = y.w;
            }
        }
    };
    load(x, head0 + w / share);

    // cos and sin of position * base^(-2 i / rd).  A thread forms those of one
    // pair's first row and, by rotating on, of every rows_apart-th row after it
    if (rotates && half) {
        const int p = threadIdx.x % half, rows_apart = KA_WAVES * 64 / half;
        const double turn = exp2(a.log2_step * (double)p) * 0.15915494309189533577;
        int t = threadIdx.x / half;
        if (t < min(m, rows_apart)) {
            double2 r = kv_cos_sin((double)(pos + t) * turn), d = make_double2(1.0, 0.0);
            if (m > rows_apart) d = kv_cos_sin((double)rows_apart * turn);
            for (; t < m; t += rows_apart) {
                s_rot[t * half + p] = r.x;
                s_rot[(32 + t) * half + p] = r.y;
                r = make_double2(__builtin_fma(r.x, d.x, -(r.y * d.y)), __builtin_fma(r.x, d.y, r.y * d.x));
            }
        }
    }
    __syncthreads();
    // A lane's dims and rows are the same in every pass, and where the partners'
    // distance is known its dims' angles are those of four pairs
    double c[2][4], sn[2][4];
    if (ROT >= 0) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double *rc = s_rot + min(r0 + 4 * u + sub, m - 1) * half + d0 % half + j;
                c[u][j] = rc[0];
                sn[u][j] = rc[32 * half];
            }
    }

    for (int hb = head0; hb < head1; hb += KA_WAVES / share) {
        const int hh = hb + w / share;
        load(next, hh + KA_WAVES / share);                           // the next pass's rows, in flight from here on
        auto advance = [&]() {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < 4; j++) x[u][v][j] = next[u][v][j];
        };
        const bool mine = hh < head1, is_v = hh >= a.nh + a.nkv, cached = mine && hh >= a.nh && page >= 0;
        if (mine && !is_v) {
            double g[NV][4];
            const float *gain = hh < a.nh ? a.q_norm : a.k_norm;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                Quad c = {{1.0f, 1.0f, 1.0f, 1.0f}};
                if (a.qk_norm) c = *reinterpret_cast<const Quad *>(gain + 64 * v + d0);
#pragma unroll
                for (int j = 0; j < 4; j++) g[v][j] = (double)c.x[j];
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int t = r0 + 4 * u + sub;
                if (r0 + 4 * u >= m) break;
                double y[NV][4];
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < 4; j++) y[v][j] = (double)x[u][v][j];
                if (a.qk_norm) {
                    double ss = 0.0;
#pragma unroll
                    for (int v = 0; v < NV; v++)
#pragma unroll
                        for (int j = 0; j < 4; j++) ss = __builtin_fma(y[v][j], y[v][j], ss);
                    ss = kv_row_sum(ss);
                    const double scale = kv_rsqrt(__builtin_fma(ss, 1.0 / HD, (double)a.eps));
#pragma unroll
                    for (int v = 0; v < NV; v++)
#pragma unroll
                        for (int j = 0; j < 4; j++) y[v][j] *= scale * g[v][j];
                }
                if (half) {
                    // z: the other one of each dim's pair
                    double z[NV][4];
                    if constexpr (ROT == 32) {
#pragma unroll
                        for (int j = 0; j < 4; j++) z[0][j] = kv_ror8(y[0][j]);
                    } else if constexpr (ROT == 64) {
#pragma unroll
                        for (int v = 0; v < NV; v++)
#pragma unroll
                            for (int j = 0; j < 4; j++) z[v][j] = y[NV - 1 - v][j];
                    } else {
                        double *sx = &s_x[w][sub * HD];
                        __builtin_amdgcn_wave_barrier();
                        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
                        for (int v = 0; v < NV; v++)
#pragma unroll
                            for (int j = 0; j < 4; j++) sx[64 * v + d0 + j] = y[v][j];
                        __builtin_amdgcn_wave_barrier();
                        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
                        for (int v = 0; v < NV; v++)
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const int d = 64 * v + d0 + j;
                                z[v][j] = sx[d < half ? d + half : d < 2 * half ? d - half : d];
                            }
                    }
                    const double *rc = s_rot + min(t, m - 1) * half, *rs = rc + 32 * half;
#pragma unroll
                    for (int v = 0; v < NV; v++) {
                        if (64 * v >= 2 * half) break;
                        if (ROT < 0) {
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const int d = 64 * v + d0 + j, at = min(d >= half ? d - half : d, half - 1);
                                c[u][j] = rc[at];
                                sn[u][j] = rs[at];
                            }
                            // (read whether or not the dim is rotated: a branch per dim costs more)
                            asm volatile("" : "+v"(c[u][0]), "+v"(c[u][1]), "+v"(c[u][2]), "+v"(c[u][3]), "+v"(sn[u][0]), "+v"(sn[u][1]), "+v"(sn[u][2]), "+v"(sn[u][3]));
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int d = 64 * v + d0 + j;
                            const double to = __builtin_fma(d >= half ? z[v][j] : -z[v][j], sn[u][j], y[v][j] * c[u][j]);
                            y[v][j] = ROT >= 0 || d < 2 * half ? to : y[v][j];
                        }
                    }
                }
#pragma unroll
                for (int v = 0; v < NV; v++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) x[u][v][j] = (float)y[v][j];
                    if (hh < a.nh && t < m)
                        // (past the caches: written once, and read by other CUs if at all)
                        __builtin_nontemporal_store(kv_f4{x[u][v][0], x[u][v][1], x[u][v][2], x[u][v][3]},
                                                    reinterpret_cast<kv_f4 *>(a.q_out + ((size_t)(row + t) * a.nh + hh) * HD + 64 * v + d0));
                }
            }
        }
        if (!caches) {                                               // only queries here: nothing to exchange
            advance();
            continue;
        }
        const int h = hh - a.nh - (is_v ? a.nkv : 0);
        const size_t slot = cached ? ((size_t)page * a.nkv + h) * (a.c.T / 32) + pos % a.c.T / 32 : 0;
        uint8_t *dst = (uint8_t *)(is_v ? a.c.v : a.c.k) + slot * 32 * HD * EB;
        float inv = 1.0f, grown = 1.0f;
        bool regrow = false;
        if (F8) {
            int8_t *exps = is_v ? a.c.v_exp : a.c.k_exp;
            int old = 0;
            float amax = 0.0f;
            if (cached) {
                old = exps[slot];
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int v = 0; v < NV; v++)
#pragma unroll
                        for (int j = 0; j < 4; j++)      // (rows past m are zeros)
                            if (fabsf(x[u][v][j]) <= 3.402823466e38f) amax = fmaxf(amax, fabsf(x[u][v][j]));
                amax = wave_max_f32(amax, 0.0f);
            }
            if (share > 1) {
                if (lane == 0) s_amax[w] = amax;
                __syncthreads();
                for (int i = 0; i < share; i++) amax = fmaxf(amax, s_amax[w - rg + i]);
            }
            int e = kv_exponent(amax);
            if (off) {
                regrow = e > old;
                e = max(e, old);
                if (regrow) grown = ldexpf(1.0f, old - e);
            }
            inv = ldexpf(1.0f, -e);
            // (every wavefront of the head has read `old` before the barrier)
            if (cached && lane == 0 && rg == 0 && (off == 0 || regrow)) exps[slot] = (int8_t)e;
        }
        // keys straight to their rows, values to the tile, [row][dim]
        if (cached) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int t = r0 + 4 * u + sub;
                if (t >= m) continue;
                uint8_t *to = is_v ? tile + t * LROW : dst + (off + t) * HD * EB;
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    const float *y = x[u][v];
                    if (F8)
                        *reinterpret_cast<uint32_t *>(to + 64 * v + d0) =
                            kv_e4m3x2(y[0] * inv, y[1] * inv) | kv_e4m3x2(y[2] * inv, y[3] * inv) << 16;
                    else
                        *reinterpret_cast<uint2 *>(to + 2 * (64 * v + d0)) =
                            make_uint2(__builtin_bit_cast(uint32_t, kv_h2{(_Float16)y[0], (_Float16)y[1]}),
                                       __builtin_bit_cast(uint32_t, kv_h2{(_Float16)y[2], (_Float16)y[3]}));
                }
            }
        }
        __syncthreads();
        auto regrown = [&](uint32_t c) {                             // four kept codes
            const uint32_t lo = kv_e4m3x2(__builtin_amdgcn_cvt_f32_fp8(c, 0) * grown, __builtin_amdgcn_cvt_f32_fp8(c, 1) * grown);
            const uint32_t hi = kv_e4m3x2(__builtin_amdgcn_cvt_f32_fp8(c, 2) * grown, __builtin_amdgcn_cvt_f32_fp8(c, 3) * grown);
            return lo | hi << 16;
        };
        if (cached && !is_v && regrow) {
            for (int i = lane + 64 * rg; i < off * HD / 16; i += 64 * share) {
                uint4 c = *reinterpret_cast<const uint4 *>(dst + (size_t)i * 16);
                c = make_uint4(regrown(c.x), regrown(c.y), regrown(c.z), regrown(c.w));
                *reinterpret_cast<uint4 *>(dst + (size_t)i * 16) = c;
            }
        }
        if (cached && is_v) {
            // 8 tokens of a dim (F16) or of two (E4M3) a piece; a piece that
            // these rows fill in part keeps the others
            constexpr int ND = F8 ? 2 : 1;
            for (int i = lane + 64 * rg; i < 4 * HD / ND; i += 64 * share) {
                const int d = i / 4 * ND, t0 = i % 4 * 8;
                const bool fresh = t0 < end && t0 + 8 > off;
                if (!fresh && !(regrow && t0 < off)) continue;
                uint8_t y[16];
                const uint8_t *from = tile + (t0 - off) * LROW + d * EB;
                if (t0 >= off && t0 + 8 <= end) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint16_t x2 = *reinterpret_cast<const uint16_t *>(from + j * LROW);
                        y[F8 ? j : 2 * j] = (uint8_t)x2;
                        y[F8 ? 8 + j : 2 * j + 1] = (uint8_t)(x2 >> 8);
                    }
                } else {
                    uint4 c = *reinterpret_cast<const uint4 *>(dst + (size_t)i * 16);
                    __builtin_memcpy(y, &c, 16);
                    if (regrow) {
                        // what lies past these rows is no one's: only kept tokens are rewritten
                        c = make_uint4(regrown(c.x), regrown(c.y), regrown(c.z), regrown(c.w));
                        uint8_t n[16];
                        __builtin_memcpy(n, &c, 16);
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            if (t0 + (j & 7) < off) y[j] = n[j];
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (t0 + j >= off && t0 + j < end) {
                            const uint16_t x2 = *reinterpret_cast<const uint16_t *>(from + j * LROW);
                            y[F8 ? j : 2 * j] = (uint8_t)x2;
                            y[F8 ? 8 + j : 2 * j + 1] = (uint8_t)(x2 >> 8);
                        }
                }
                uint4 c;
                __builtin_memcpy(&c, y, 16);
                *reinterpret_cast<uint4 *>(dst + (size_t)i * 16) = c;
            }
        }
        __syncthreads();                                             // the tile is the next pass's
        advance();
    }
}

hipError_t launch_kv_append(const KvAppendArgs &args, hipStream_t s)
{
    KvAppendArgs a = args;
    if (a.rd < 0 || a.rd > a.hd || a.rd % 2 || a.ks < 1) return hipErrorInvalidValue;
    a.blocks = (int32_t)kv_blocks_most(a.b.n_seqs, a.b.n_tokens);
    const int heads = a.nh + 2 * a.nkv;
    // Heads of a workgroup.  Few rows a sequence: four, which its wavefronts take
    // at once (61 rows of 61 sequences 7.3 us, two heads 9.9).  Many: one where the
    // chip has places for all (16 blocks of 32 rows 8.0, two 10.0), else two, the
    // second's loads in flight during the first (4001 rows 32.9, one 38.9, four
    // 36.1, eight 40.9).
    a.group = a.b.n_tokens < 16 * a.b.n_seqs ? KA_WAVES : (long)a.blocks * heads <= 2048 ? 1 : 2;
    a.zeros = a.rest ? 32 : 0;
    const dim3 grid((unsigned)((a.blocks + a.zeros) * ((heads + a.group - 1) / a.group)));
    const bool f8 = a.c.type == DMOE_KV_E4M3;
    const size_t lds = (size_t)64 * (a.rd / 2) * sizeof(double);
    const dim3 threads(KA_WAVES * 64);
    auto go = [&](auto hd, auto e4m3) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool F8 = decltype(e4m3)::value;
        if (a.rd == 64)
            hipLaunchKernelGGL((k_kv_append<HD, F8, 32>), grid, threads, lds, s, a);
        else if (a.rd == 128 && HD == 128)
            hipLaunchKernelGGL((k_kv_append<HD, F8, HD == 128 ? 64 : -1>), grid, threads, lds, s, a);
        else
            hipLaunchKernelGGL((k_kv_append<HD, F8, -1>), grid, threads, lds, s, a);
    };
    auto with = [&](auto hd) { f8 ? go(hd, std::true_type{}) : go(hd, std::false_type{}); };
    if (a.hd == 64)
        with(std::integral_constant<int, 64>{});
    else if (a.hd == 128)
        with(std::integral_constant<int, 128>{});
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

} // namespace dmoe
