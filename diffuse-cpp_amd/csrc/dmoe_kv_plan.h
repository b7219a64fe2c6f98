// dmoe_kv_plan.h — what the paged KV cache's entry points accept, and how its
// kernels read the tables of a batch: pure functions of sizes, addresses and
// table entries, for the host and the GPU.  tests/test_kv_plan.py compiles this
// file for the CPU.
#pragma once

#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/dmoe.h"

#ifdef __HIPCC__
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

namespace dmoe {

// Rows of a sequence in the call's token buffers and its cached tokens, these
// rows included.  Entries that contradict each other (rows outside the buffers,
// more rows than cached tokens, more tokens than KV_TOKENS_MOST) leave the
// sequence without rows, so that no index derived from them leaves a buffer or
// 32 bits.
struct KvSeq {
    int q0, n, len;
};
constexpr int KV_TOKENS_MOST = 1 << 30;
// Rows and sequences of a call, times n_head + 2 n_head_kv.
constexpr int64_t KV_ROWS_MOST = 1 << 27, KV_SEQS_MOST = 1 << 24;

KV_HD KvSeq kv_seq_of(int start, int end, int len, int n_tokens)
{
    const bool ok = start >= 0 && end >= start && end <= n_tokens && len >= end - start &&
                    len <= KV_TOKENS_MOST;
    return KvSeq{start, ok ? end - start : 0, len};
}

// Blocks of 32 tokens that a sequence's rows touch.
KV_HD int kv_blocks(const KvSeq &q)
{
    return q.n ? (q.len - 1) / 32 - (q.len - q.n) / 32 + 1 : 0;
}

// Where a sequence's blocks begin in a list that has room for those of every one,
// found from its first row alone: a sequence of n rows touches at most n blocks,
// and at most n / 32 + 2.  `by_row`: a place for each row, else one for each 32 and
// two for each sequence, whichever is less in all.
KV_HD bool kv_by_row(int n_seqs, int n_tokens)
{
    return n_tokens <= n_tokens / 32 + 2 * (int64_t)n_seqs;
}

KV_HD int kv_place(int start, int s, bool by_row)
{
    return by_row ? start : start / 32 + 2 * s;
}

// Places of that list: no less than the blocks of a batch.
KV_HD int64_t kv_blocks_most(int n_seqs, int n_tokens)
{
    return kv_by_row(n_seqs, n_tokens) ? n_tokens : n_tokens / 32 + 2 * (int64_t)n_seqs;
}

// The entry of a sequence's row of the page table for token `pos`, or -1 past
// the table.
KV_HD int kv_entry_of(int pos, int page_tokens, int max_pages)
{
    const uint32_t i = (uint32_t)pos / (uint32_t)page_tokens;
    return i < (uint32_t)max_pages ? (int)i : -1;
}

// The page of an entry, or -1 for one that is no page of the cache.
KV_HD int kv_page_of(int entry, int n_pages)
{
    return (unsigned)entry < (unsigned)n_pages ? entry : -1;
}

// Tokens of a sequence that the table can hold.
KV_HD int kv_cached(int len, int page_tokens, int max_pages)
{
    const int64_t most = (int64_t)page_tokens * max_pages;
    return len < most ? len : (int)most;
}

// Tokens that the query at position `pos` sees of the `cached` first ones.
KV_HD int kv_visible(int pos, int cached, int block)
{
    if (block <= 0) return cached;
    // (below 2^32: pos is below 2^30, and so is pos / block * block)
    const uint32_t end = ((uint32_t)pos / (uint32_t)block + 1) * (uint32_t)block;
    return end < (uint32_t)cached ? (int)end : cached;
}

// ---------------------------------------------------------------------------
// Refusals: DMOE_OK, or the status with the reason in `why`.
struct KvRefusal {
    int code = DMOE_OK;
    char why[256] = "";
    int set(int status, const char *fmt, ...)
    {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(why, sizeof(why), fmt, ap);
        va_end(ap);
        return code = status;
    }
};

inline bool kv_overlap(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

inline size_t kv_cache_blocks(const dmoe_kv_cache &kv)
{
    return (size_t)kv.n_pages * kv.n_head_kv * (kv.page_tokens / DMOE_KV_BLOCK);
}

inline size_t kv_cache_bytes(const dmoe_kv_cache &kv)
{
    return kv_cache_blocks(kv) * DMOE_KV_BLOCK * kv.head_dim * (kv.type == DMOE_KV_E4M3 ? 1 : 2);
}

// Whether a buffer shares memory with a cache (checked before).
inline bool kv_in_cache(const dmoe_kv_cache &kv, const void *p, size_t n)
{
    const size_t bytes = kv_cache_bytes(kv), blocks = kv.type == DMOE_KV_E4M3 ? kv_cache_blocks(kv) : 0;
    return kv_overlap(p, n, kv.k, bytes) || kv_overlap(p, n, kv.v, bytes) ||
           (blocks && (kv_overlap(p, n, kv.k_exp, blocks) || kv_overlap(p, n, kv.v_exp, blocks)));
}

// A cache, a batch and the attention's sizes; `pointers`: those too.
inline int kv_check(KvRefusal &r, const dmoe_kv_cache *kv, const dmoe_kv_batch *b, const dmoe_attn_hparams *ap,
                    bool pointers)
{
    if (!kv || !b || !ap) return r.set(DMOE_ERR_INVALID_ARG, "kv: cache / batch / hparams is NULL");
    if (kv->type != DMOE_KV_F16 && kv->type != DMOE_KV_E4M3)
        return r.set(DMOE_ERR_UNSUPPORTED_TYPE, "kv: cache type %d (DMOE_KV_F16 or DMOE_KV_E4M3)", kv->type);
    if (kv->head_dim != 64 && kv->head_dim != 128)
        return r.set(DMOE_ERR_SHAPE, "kv: head_dim = %d (64 or 128 supported)", kv->head_dim);
    if (kv->page_tokens <= 0 || kv->page_tokens % DMOE_KV_BLOCK)
        return r.set(DMOE_ERR_SHAPE, "kv: page_tokens = %d must be a positive multiple of %d", kv->page_tokens,
                     DMOE_KV_BLOCK);
    if (kv->n_head_kv <= 0 || kv->n_pages <= 0)
        return r.set(DMOE_ERR_SHAPE, "kv: n_head_kv = %d, n_pages = %d", kv->n_head_kv, kv->n_pages);
    if (ap->n_head <= 0 || ap->n_head_kv != kv->n_head_kv || ap->n_head % ap->n_head_kv)
        return r.set(DMOE_ERR_SHAPE, "kv: n_head = %d, n_head_kv = %d over a cache of %d", ap->n_head, ap->n_head_kv,
                     kv->n_head_kv);
    if (ap->head_dim != kv->head_dim)
        return r.set(DMOE_ERR_SHAPE, "kv: head_dim = %d over a cache of %d", ap->head_dim, kv->head_dim);
    if (b->n_seqs <= 0 || b->n_tokens <= 0 || b->max_pages <= 0)
        return r.set(DMOE_ERR_INVALID_ARG, "kv: n_seqs = %d, n_tokens = %d, max_pages = %d must be positive", b->n_seqs,
                     b->n_tokens, b->max_pages);
    // the indexes of (row, head) pairs are 32 bits wide, and a launch has less
    // than 2^24 workgroups of 256 threads
    const int64_t heads = ap->n_head + 2 * (int64_t)ap->n_head_kv;
    if (heads > KV_SEQS_MOST || b->n_tokens * heads > KV_ROWS_MOST || b->n_seqs * heads > KV_SEQS_MOST || b->n_seqs > (1 << 20))
        return r.set(DMOE_ERR_SHAPE, "kv: %d rows of %d + 2 * %d heads, %d sequences are too many", b->n_tokens,
                     ap->n_head, ap->n_head_kv, b->n_seqs);
    if (!pointers) return DMOE_OK;
    const bool f8 = kv->type == DMOE_KV_E4M3;
    if (!kv->k || !kv->v || (f8 && (!kv->k_exp || !kv->v_exp)))
        return r.set(DMOE_ERR_INVALID_ARG, "kv: a pointer of the cache is NULL");
    if ((uintptr_t)kv->k % 16 || (uintptr_t)kv->v % 16)
        return r.set(DMOE_ERR_INVALID_ARG, "kv: k and v must be 16-byte aligned");
    const size_t blocks = kv_cache_blocks(*kv), bytes = kv_cache_bytes(*kv);
    if (kv_overlap(kv->k, bytes, kv->v, bytes) || (f8 && kv_overlap(kv->k_exp, blocks, kv->v_exp, blocks)))
        return r.set(DMOE_ERR_INVALID_ARG, "kv: keys and values overlap");
    if (!b->q_start || !b->kv_len || !b->pages) return r.set(DMOE_ERR_INVALID_ARG, "kv: a table of the batch is NULL");
    if ((uintptr_t)b->q_start % 4 || (uintptr_t)b->kv_len % 4 || (uintptr_t)b->pages % 4)
        return r.set(DMOE_ERR_INVALID_ARG, "kv: the batch's tables must be 4-byte aligned");
    return DMOE_OK;
}

inline int kv_check_rotary(KvRefusal &r, const dmoe_attn_hparams &a)
{
    if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 2)
        return r.set(DMOE_ERR_SHAPE, "kv: rotary_dim = %d", a.rotary_dim);
    if (!(a.rms_eps >= 0.0f) || isinf(a.rms_eps) || !(a.rope_base > 0.0f) || isinf(a.rope_base))
        return r.set(DMOE_ERR_INVALID_ARG, "kv: rms_eps / rope_base out of range");
    return DMOE_OK;
}

inline int kv_check_append(KvRefusal &r, const dmoe_kv_cache *kv, const dmoe_kv_batch *b, const dmoe_attn_hparams *ap,
                           const void *qkv, const void *q_norm, const void *k_norm, const void *q_out)
{
    if (kv_check(r, kv, b, ap, true) || kv_check_rotary(r, *ap)) return r.code;
    if (!qkv || !q_out || (ap->use_qk_norm && (!q_norm || !k_norm)))
        return r.set(DMOE_ERR_INVALID_ARG, "kv_append: qkv / q_out / q_norm / k_norm is NULL");
    if ((uintptr_t)qkv % 16 || (uintptr_t)q_out % 16)
        return r.set(DMOE_ERR_INVALID_ARG, "kv_append: qkv and q_out must be 16-byte aligned");
    if (ap->use_qk_norm && ((uintptr_t)q_norm % 4 || (uintptr_t)k_norm % 4))
        return r.set(DMOE_ERR_INVALID_ARG, "kv_append: q_norm and k_norm must be 4-byte aligned");
    const size_t head = (size_t)b->n_tokens * ap->head_dim * 4;
    if (kv_overlap(qkv, head * ((size_t)ap->n_head + 2 * (size_t)ap->n_head_kv), q_out, head * ap->n_head))
        return r.set(DMOE_ERR_INVALID_ARG, "kv_append: qkv and q_out overlap");
    if (kv_in_cache(*kv, qkv, head * ((size_t)ap->n_head + 2 * (size_t)ap->n_head_kv)) ||
        kv_in_cache(*kv, q_out, head * ap->n_head))
        return r.set(DMOE_ERR_INVALID_ARG, "kv_append: qkv or q_out overlaps the cache");
    return DMOE_OK;
}

inline int kv_check_attn(KvRefusal &r, const dmoe_kv_cache *kv, const dmoe_kv_batch *b, const dmoe_attn_hparams *ap,
                         const void *q, const void *out)
{
    if (kv_check(r, kv, b, ap, true)) return r.code;
    if (!q || !out) return r.set(DMOE_ERR_INVALID_ARG, "kv_attn: q / out is NULL");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16)
        return r.set(DMOE_ERR_INVALID_ARG, "kv_attn: q and out must be 16-byte aligned");
    const size_t bytes = (size_t)b->n_tokens * ap->n_head * ap->head_dim * 4;
    if (kv_overlap(q, bytes, out, bytes)) return r.set(DMOE_ERR_INVALID_ARG, "kv_attn: q and out overlap");
    if (kv_in_cache(*kv, out, bytes)) return r.set(DMOE_ERR_INVALID_ARG, "kv_attn: out overlaps the cache");
    return DMOE_OK;
}

inline int kv_check_layer(KvRefusal &r, const dmoe_kv_cache *kv, const dmoe_kv_batch *b, const dmoe_attn_hparams *ap,
                          const void *h, const void *h_out, const void *moe_in)
{
    if (kv_check(r, kv, b, ap, true) || kv_check_rotary(r, *ap)) return r.code;
    if (!h || !h_out) return r.set(DMOE_ERR_INVALID_ARG, "attn_cached: h / h_out is NULL");
    if ((uintptr_t)h % 16 || (uintptr_t)h_out % 16 || (uintptr_t)moe_in % 16)
        return r.set(DMOE_ERR_INVALID_ARG, "attn_cached: device buffers must be 16-byte aligned");
    const size_t bytes = (size_t)b->n_tokens * ap->n_embd * 4;
    if ((h_out != h && kv_overlap(h, bytes, h_out, bytes)) ||
        (moe_in && (kv_overlap(moe_in, bytes, h, bytes) || kv_overlap(moe_in, bytes, h_out, bytes))))
        return r.set(DMOE_ERR_INVALID_ARG, "attn_cached: h, h_out and moe_in overlap");
    if (kv_in_cache(*kv, h, bytes) || kv_in_cache(*kv, h_out, bytes) || (moe_in && kv_in_cache(*kv, moe_in, bytes)))
        return r.set(DMOE_ERR_INVALID_ARG, "attn_cached: h, h_out or moe_in overlaps the cache");
    return DMOE_OK;
}

inline int kv_check_workspace(KvRefusal &r, const void *ws, size_t bytes, size_t need)
{
    if (bytes < need)
        return r.set(DMOE_ERR_INVALID_ARG, "kv: a workspace of %zu bytes, %zu are needed", bytes, need);
    if ((uintptr_t)ws % 16) return r.set(DMOE_ERR_INVALID_ARG, "kv: the workspace must be 16-byte aligned");
    return DMOE_OK;
}

} // namespace dmoe
