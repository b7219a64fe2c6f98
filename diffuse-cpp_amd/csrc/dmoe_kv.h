// dmoe_kv.h — the paged KV cache as its kernels see it (k_kv_append.hip,
// k_kv_attn.hip) and the device helpers that both use.
//
// Layouts, T tokens a page, blocks of 32 tokens, 16-byte pieces:
//   k  [n_pages][nkv][T][hd]
//   v  [n_pages][nkv][T / 32] blocks, transposed so that a lane's operand of
//      the P V product (8 consecutive tokens of a dim) is one piece (F16) or
//      half of one (E4M3):
//        F16   piece 4 d + t / 8: tokens t .. t + 7 (t % 8 == 0) of dim d
//        E4M3  piece 4 (d / 2) + t / 8: tokens t .. t + 7 of dim d, then of d + 1
//   k_exp, v_exp  int8 [n_pages][nkv][T / 32]: a block's values are code * 2^exp
#pragma once

#include "dmoe_internal.h"
#include "dmoe_kv_plan.h"

namespace dmoe {

typedef _Float16 kv_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t kv_u4 __attribute__((ext_vector_type(4)));
typedef float kv_f2 __attribute__((ext_vector_type(2)));
typedef float kv_f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ KvSeq kv_seq(const KvBatch &b, int s)
{
    return kv_seq_of(b.q_start[s], b.q_start[s + 1], b.kv_len[s], b.n_tokens);
}

// Inclusive scan over the 64 lanes, by DPP (0 is neutral to `op`).
template <class T, class Op>
__device__ __forceinline__ T kv_wave_scan(T v, Op &&op)
{
#define KV_DPP(ctrl, rows) \
    v = op(v, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, false)))
    KV_DPP(0x111, 0xf);                  // row_shr 1, 2, 4, 8
    KV_DPP(0x112, 0xf);
    KV_DPP(0x114, 0xf);
    KV_DPP(0x118, 0xf);
    KV_DPP(0x142, 0xa);                  // lane 15 of rows 0 and 2 to rows 1 and 3
    KV_DPP(0x143, 0xc);                  // lane 31 to rows 2 and 3
#undef KV_DPP
    return v;
}

template <class T>
__device__ __forceinline__ T kv_wave_scan(T v)
{
    return kv_wave_scan(v, [](T x, T y) { return x + y; });
}

// A scan's last value, which is the whole wavefront's.
template <class T>
__device__ __forceinline__ T kv_wave_last(T v)
{
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Sequence base + lane of 64, and which rows are its: `top` is the largest first
// row met so far (0 before the first 64).  In a table that decreases, a sequence
// whose rows could be an earlier one's has none, so that the rows of all of them
// are disjoint and the counts that follow from n_tokens hold for any table.
__device__ __forceinline__ KvSeq kv_seqs(const KvBatch &b, int base, int &top)
{
    const int s = base + (threadIdx.x & 63);
    KvSeq q{0, 0, 0};
    if (s < b.n_seqs) q = kv_seq(b, s);
    const int first = max(top, (unsigned)q.q0 <= (unsigned)b.n_tokens ? q.q0 : 0);
    const int v = kv_wave_scan(first, [](int x, int y) { return max(x, y); });
    top = kv_wave_last(v);
    if (v > q.q0) q.n = 0;
    return q;
}

// Item `item` of a list that holds count(seq) items of each sequence in turn:
// its sequence (and the item's index within it), found by one wavefront in
// steps of 64 sequences; false past the list's end.
template <class Count>
__device__ __forceinline__ bool kv_find(const KvBatch &b, int item, Count &&count, int &seq, KvSeq &info, int &index)
{
    int top = 0;
    for (int base = 0; base < b.n_seqs; base += 64) {
        const KvSeq q = kv_seqs(b, base, top);
        const int c = count(q);
        const int end = kv_wave_scan(c);
        const uint64_t past = __ballot(end > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            seq = base + l;
            info.q0 = __builtin_amdgcn_readlane(q.q0, l);
            info.n = __builtin_amdgcn_readlane(q.n, l);
            info.len = __builtin_amdgcn_readlane(q.len, l);
            index = item - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(c, l));
            return true;
        }
        item -= kv_wave_last(end);
    }
    return false;
}

// Block `blk` of sequence `seq` at place `item` of kv_place's list, found by one
// wavefront, 64 sequences at a time or every 64th part of more; false where a
// place is empty.  (In a table that decreases it may be any sequence's, or none's.)
__device__ __forceinline__ bool kv_find_block(const KvBatch &b, int item, int &seq, KvSeq &info, int &blk)
{
    const int lane = threadIdx.x & 63;
    const bool by_row = kv_by_row(b.n_seqs, b.n_tokens);
    int first = 0, n = b.n_seqs;
    while (n > 64) {
        const int part = (n + 63) / 64, i = lane * part;
        const uint64_t before = __ballot(i < n && kv_place(b.q_start[first + min(i, n - 1)], first + i, by_row) <= item);
        if (!before) return false;
        const int k = 63 - __builtin_clzll(before);
        first += k * part;
        n = min(part, n - k * part);
    }
    KvSeq q{0, 0, 0};
    if (lane < n) q = kv_seq(b, first + lane);
    const uint64_t before = __ballot(lane < n && kv_place(q.q0, first + lane, by_row) <= item);
    if (!before) return false;
    const int l = 63 - __builtin_clzll(before);
    seq = first + l;
    info.q0 = __builtin_amdgcn_readlane(q.q0, l);
    info.n = __builtin_amdgcn_readlane(q.n, l);
    info.len = __builtin_amdgcn_readlane(q.len, l);
    blk = item - kv_place(info.q0, seq, by_row);
    return blk >= 0 && blk < kv_blocks(info);
}

// The page that holds token `pos` of sequence s, or -1.
__device__ __forceinline__ int kv_page(const KvBatch &b, const KvCacheView &c, int s, int pos)
{
    const int i = kv_entry_of(pos, c.T, b.max_pages);
    return i < 0 ? -1 : kv_page_of(b.pages[(size_t)s * b.max_pages + i], c.n_pages);
}

} // namespace dmoe
