/*
 * fcci_paged.h — C ABI of the paged KV cache of the B200 (sm_100a) attention path.
 *
 * The arena of fcci_decode.h reserves every sequence's capacity at once and holds fp16. Here
 * the rows of all sequences live in pages of page_size tokens taken from one pool, named by
 * a page table, and a pool may hold e4m3 codes with one power-of-two scale for each page and
 * kv head, which halves the bytes that a decode step reads. There is no counterpart in the
 * reference; the steps are those of its decode drivers and kv_init
 * (scripts/direct_custom_decode_500.py:229-250, case4_graph_generator_server_ipc.py:1241-1262).
 *
 *   fcci_paged_append    RoPE on k_new (and q, when given) at positions T_b + i, and the
 *                        append of (k_rot, v_new) into the pages; no attention
 *   fcci_paged_decode    one new token per sequence: append (when k_new is given) and
 *                        split-KV attention over all keys of its sequence
 *   fcci_paged_prefill   n_b new tokens of every sequence: append and causal attention of
 *                        new token i over keys 0 .. T_b + i
 *   fcci_paged_workspace_bytes / _init, fcci_paged_read_error
 *                        sizing, zeroing and error readback of the caller-owned workspace
 *
 * Status codes, fcci_last_status and fcci_last_error_string are those of fcci_decode.h, and
 * so are the bits of the device error word, with two more:
 */
#ifndef FCCI_PAGED_H
#define FCCI_PAGED_H

#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime.h>

#include "fcci_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FCCI_PAGED_ABI_VERSION 1

#define FCCI_DEV_ERR_PAGE 8u /* a page that a live row needs is not in [0, num_pages): never
                                dereferenced; the sequence's results are not to be used */
#define FCCI_DEV_ERR_SCALE 16u /* a prefill of long chunks read a page of scale above 2^8, which no append
                                  makes and whose values its fp16 rows may not hold: the sequence's
                                  results are not to be used */

/* cache_type */
#define FCCI_PAGED_F16 0
#define FCCI_PAGED_E4M3 1

/*
 * Shapes and layouts (fp16 unless stated; strides in elements; head_dim contiguous;
 * 16-byte aligned bases, strides multiples of 16 bytes; what a call writes may not overlap itself):
 *   new tokens   cu_seqlens_q == NULL: sequence b owns row b (total_q == B, one token each);
 *                else rows cu_seqlens_q[b] .. cu_seqlens_q[b+1]-1, n_b of them, at most
 *                max_seqlen_q; rows behind cu_seqlens_q[B] are neither read nor written.
 *                q [total_q, Hq, D], k_new / v_new [total_q, Hkv, D], out [total_q, Hq, D]
 *   pools        row t of (sequence b, kv head h) at
 *                pages + page*stride_p + h*stride_h + (t % page_size)*stride_t with
 *                page = page_table[b*page_table_stride + t / page_size]; fp16, or e4m3 codes
 *                (cache_type FCCI_PAGED_E4M3, strides then in bytes)
 *   scales       e4m3 only: byte s at scales + page*stride_p + h*stride_h says 2^(s - 127); a
 *                row's values are code * 2^(s - 127). 255 is none; of a page without live rows the
 *                byte may be anything. A prefill of more than 64 query rows of one kv head (max_seqlen_q *
 *                Hq / Hkv) takes those that an append makes, 112 to 135: smaller ones lose what is below
 *                2^-25, larger ones are reported (FCCI_DEV_ERR_SCALE)
 *   T_b          seq_lens[b] (device int32, read on device): rows already cached. T_b + n_b
 *                must not exceed max_pages * page_size
 *   RoPE         rotate-half on the first rotary_dim dims (a multiple of 16, 0 disables it)
 *                at position T_b + i, angle pos * rope_theta^(-2j/rotary_dim) reduced exactly,
 *                fp32 products
 *   append       rows T_b .. T_b + n_b - 1, each value rounded once from fp32: to fp16, or to
 *                e4m3 after the exact product with 2^-e. e of a page is the smallest in
 *                [-15, 8] with max|new rows of the page| (in fp32) <= 448 * 2^e, or the page's present e
 *                if that is larger and the page holds rows below T_b; if e grows, those
 *                rows are rounded to the new scale. Infinities saturate, NaN stays NaN. A page
 *                that gets rows must belong to one sequence alone.
 *   attention    out = softmax_t(q_rot . k_t * scale) v_t, fp32 accumulation; a token that
 *                sees no key gets 0. What pages hold behind a sequence's rows (NaN
 *                among it) has no effect. Among the new tokens of one prefill, a value that is
 *                NaN or infinite may reach tokens before its own (its weight there is 0, and
 *                0 * NaN is NaN); keys that are not finite do not.
 *   advance      when non-zero, seq_lens[b] += n_b after the step
 * rope_theta 1e-6 at least. head_dim 64, 128 or 256 (prefill: 128); page_size 16, 32, 64 or 128 with
 * page_size * D <= 16384; Hq a multiple of Hkv, at most 16 query heads a kv head (8 with
 * head_dim 256).
 *
 * Calls that share a workspace must not overlap on the GPU.
 */
typedef struct fcci_paged_desc {
    int32_t abi_version; /* FCCI_PAGED_ABI_VERSION */
    int32_t B, Hq, Hkv, D;
    int32_t total_q;      /* rows of q / k_new / v_new / out */
    int32_t max_seqlen_q; /* bound on n_b (1 without cu_seqlens_q) */
    const int32_t* cu_seqlens_q;
    const void* q; /* append: nullable */
    int64_t q_stride_t, q_stride_h;
    const void* k_new; /* decode: nullable together with v_new */
    int64_t k_new_stride_t, k_new_stride_h;
    const void* v_new;
    int64_t v_new_stride_t, v_new_stride_h;
    int32_t cache_type; /* FCCI_PAGED_F16 or FCCI_PAGED_E4M3 */
    int32_t page_size, num_pages, max_pages; /* max_pages: entries of one sequence in page_table */
    void* k_pages;
    int64_t k_stride_p, k_stride_h, k_stride_t;
    void* v_pages;
    int64_t v_stride_p, v_stride_h, v_stride_t;
    uint8_t* k_scales; /* NULL with FCCI_PAGED_F16 */
    int64_t k_scales_stride_p, k_scales_stride_h;
    uint8_t* v_scales;
    int64_t v_scales_stride_p, v_scales_stride_h;
    const int32_t* page_table;
    int64_t page_table_stride;
    int32_t* seq_lens;
    void* out; /* decode, prefill */
    int64_t out_stride_t, out_stride_h;
    void* q_rot_out; /* append: required with q; decode: nullable. [total_q, Hq, D] contiguous */
    float scale;
    float rope_theta;
    int32_t rotary_dim;
    int32_t advance;
    int32_t max_kv_tokens; /* prefill: bound on the sum of T_b + n_b; negative: what the workspace has room for */
    void* workspace;       /* fcci_paged_workspace_bytes() bytes, zeroed once with _init */
    size_t workspace_bytes;
    uint32_t flags; /* FCCI_PAGED_PREFETCH_KV (decode only) */
} fcci_paged_desc;

/* Decode: read seq_lens, the page table, scales and the cached rows below T_b before the programmatic-launch wait, so
 * that they overlap the kernel before it on the stream; q, k_new and v_new are still read after it. Set it only when no
 * kernel that can still be running when this one starts writes any of those. Those are the kernel before it and, where that
 * one was launched with this flag too, the ones before that, back to the last ordinary launch or paged call
 * without the flag: everything before that one has ended. So it may be set for example right after the projection that
 * produced q/k/v, or in a chain of layers' steps of which only the last advances and the first has not the flag. */
#define FCCI_PAGED_PREFETCH_KV 1u

int fcci_paged_append(const fcci_paged_desc* desc, cudaStream_t stream);
int fcci_paged_decode(const fcci_paged_desc* desc, cudaStream_t stream);
int fcci_paged_prefill(const fcci_paged_desc* desc, cudaStream_t stream);

/* Workspace for calls of up to total_q new tokens, max_seqlen_q of one sequence; 0 for
 * invalid shapes. max_kv_tokens: 0 without fcci_paged_prefill. A workspace of larger bounds
 * serves smaller calls. */
size_t fcci_paged_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t total_q,
                                  int32_t max_seqlen_q, int32_t max_kv_tokens, int device);
int fcci_paged_workspace_init(void* workspace, size_t bytes, cudaStream_t stream);
/* Copy the device error word to *flags (synchronises `stream`); clear it when clear != 0. After
 * FCCI_DEV_ERR_TIMEOUT run fcci_paged_workspace_init on the workspace before its next use. */
int fcci_paged_read_error(void* workspace, uint32_t* flags, int clear, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FCCI_PAGED_H */
