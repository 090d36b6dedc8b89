// Host side of the paged entry points: checks, workspace layout and dispatch.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <initializer_list>
#include <utility>

#include "paged.cuh"

namespace fcci {
namespace pg {

// ------------------------------------------------------------------ host side

WsLayout ws_layout(int B, int Hq, int Hkv, int D, int total_q, int max_q, int max_kv, int grid) {
    auto up = [](size_t x) { return (x + 1023) & ~size_t(1023); };
    WsLayout w;
    w.part_lse = up(kHeadBytes);
    w.part_o = w.part_lse + up((size_t)2 * grid * kMaxCols * 4);
    w.q_rot = w.part_o + up((size_t)2 * grid * kMaxCols * D * 4);
    w.total = w.q_rot;
    if (max_kv != 0 && long_chunk(Hq, Hkv, max_q)) {
        w.cu_kv = w.q_rot + up((size_t)total_q * Hq * D * 2);
        w.items = w.cu_kv + up((size_t)(B + 1) * 4);
        w.expanded = w.items + up((size_t)max_items(B, Hq, total_q) * 16);
        w.total = w.expanded + (max_kv > 0 ? up((size_t)max_kv * Hkv * D * 4) : 0);
    } else {
        w.cu_kv = w.items = w.expanded = w.total;
    }
    return w;
}

enum class Op { kAppend, kDecode, kPrefill };

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether blocks of `inner` elements, one for each index of all dimensions (extent, stride), may share elements: not when each
// stride, in rising order, reaches past all that the smaller ones span.
static bool overlapping(int64_t inner, std::initializer_list<std::pair<int64_t, int64_t>> dims) {
    std::pair<int64_t, int64_t> d[4];
    int n = 0;
    for (const auto& x : dims)
        if (x.first > 1) d[n++] = {x.second, x.first};
    std::sort(d, d + n);
    __int128 span = inner;
    for (int i = 0; i < n; ++i) {
        if (d[i].first < span) return true;
        span += (__int128)(d[i].second - 1) * d[i].first;
    }
    return false;
}

// Validates a descriptor; on failure records the reason and returns its FCCI_E* code.
static int fill(const fcci_paged_desc* d, Op op, Params& p, Freqs& f, WsLayout& L) {
    auto bad = [](int code, const char* why) { return set_status(code, why); };
    if (!d) return bad(FCCI_EINVAL, "descriptor is NULL");
    if (d->abi_version != FCCI_PAGED_ABI_VERSION) return bad(FCCI_EINVAL, "abi_version mismatch");
    if (d->B <= 0 || d->Hq <= 0 || d->Hkv <= 0 || d->Hq % d->Hkv != 0)
        return bad(FCCI_EINVAL, "B, Hq, Hkv must be positive and Hq a multiple of Hkv");
    if (d->D != 64 && d->D != 128 && d->D != 256) return bad(FCCI_EUNSUPPORTED, "unsupported head_dim (64, 128 or 256)");
    if (op == Op::kPrefill && d->D != 128) return bad(FCCI_EUNSUPPORTED, "prefill: head_dim must be 128");
    if (op != Op::kAppend && d->Hq / d->Hkv > (d->D == 256 ? 8 : 16))
        return bad(FCCI_EUNSUPPORTED, "query group size unsupported");
    if (d->B > 65535 || d->Hq > 65535) return bad(FCCI_EUNSUPPORTED, "batch or head count above 65535");
    if (d->page_size != 16 && d->page_size != 32 && d->page_size != 64 && d->page_size != 128)
        return bad(FCCI_EUNSUPPORTED, "page_size must be 16, 32, 64 or 128");
    if (d->page_size * d->D > 16384) return bad(FCCI_EUNSUPPORTED, "page_size * head_dim above 16384");
    if (d->cache_type != FCCI_PAGED_F16 && d->cache_type != FCCI_PAGED_E4M3)
        return bad(FCCI_EINVAL, "unknown cache_type");
    const bool e4m3 = d->cache_type == FCCI_PAGED_E4M3;
    if (!d->k_pages || !d->v_pages || !d->page_table || !d->seq_lens)
        return bad(FCCI_EINVAL, "k_pages, v_pages, page_table and seq_lens are required");
    if (e4m3 != (d->k_scales != nullptr) || e4m3 != (d->v_scales != nullptr))
        return bad(FCCI_EINVAL, "k_scales and v_scales go with an e4m3 cache, and only with one");
    if (d->num_pages <= 0 || d->max_pages <= 0 || (int64_t)d->max_pages * d->page_size > 0x7fffffff)
        return bad(FCCI_EINVAL, "num_pages and max_pages must be positive and a sequence below 2^31 rows");
    if (d->page_table_stride < 0) return bad(FCCI_EINVAL, "negative page_table stride");
    if ((d->k_new == nullptr) != (d->v_new == nullptr)) return bad(FCCI_EINVAL, "k_new and v_new go together");
    if (op != Op::kDecode && !d->k_new) return bad(FCCI_EINVAL, "k_new and v_new are required");
    if (op != Op::kAppend && (!d->q || !d->out)) return bad(FCCI_EINVAL, "q and out are required");
    if (op == Op::kAppend && (d->q != nullptr) != (d->q_rot_out != nullptr))
        return bad(FCCI_EINVAL, "q and q_rot_out go together");
    if (d->total_q < 0 || d->max_seqlen_q < 0) return bad(FCCI_EINVAL, "negative token count");
    if (op == Op::kPrefill && !d->cu_seqlens_q) return bad(FCCI_EINVAL, "prefill: cu_seqlens_q is required");
    if (op == Op::kDecode && d->cu_seqlens_q) return bad(FCCI_EINVAL, "decode: one token per sequence, no cu_seqlens_q");
    if (!d->cu_seqlens_q && d->total_q != d->B) return bad(FCCI_EINVAL, "total_q must be B without cu_seqlens_q");
    if (d->rotary_dim < 0 || d->rotary_dim > d->D || d->rotary_dim % 16)
        return bad(FCCI_EUNSUPPORTED, "rotary_dim must be a multiple of 16 within head_dim");
    if (d->rotary_dim > 0 && !(d->rope_theta >= 1e-6f && d->rope_theta < INFINITY))
        return bad(FCCI_EINVAL, "rope_theta must be positive (1e-6 at least)");
    if (op != Op::kAppend && !(d->scale > 0.f && d->scale < INFINITY)) return bad(FCCI_EINVAL, "scale must be positive");
    if (d->flags & ~(op == Op::kDecode ? FCCI_PAGED_PREFETCH_KV : 0u)) return bad(FCCI_EINVAL, "unknown bits in flags");
    if (d->advance && !d->k_new) return bad(FCCI_EINVAL, "advance needs k_new");
    const int64_t elt = e4m3 ? 1 : 2;
    const void* ptrs[7] = {d->q, d->k_new, d->v_new, d->k_pages, d->v_pages, d->out, d->q_rot_out};
    for (const void* x : ptrs)
        if (!aligned16(x)) return bad(FCCI_EINVAL, "tensors must be 16-byte aligned");
    const int64_t half_st[8] = {d->q_stride_t,     d->q_stride_h,     d->k_new_stride_t, d->k_new_stride_h,
                                d->v_new_stride_t, d->v_new_stride_h, d->out_stride_t,   d->out_stride_h};
    for (int64_t x : half_st)
        if (x < 0 || (x & 7)) return bad(FCCI_EINVAL, "strides must be non-negative multiples of 16 bytes");
    const int64_t pool_st[6] = {d->k_stride_p, d->k_stride_h, d->k_stride_t, d->v_stride_p, d->v_stride_h, d->v_stride_t};
    for (int64_t x : pool_st)
        if (x < 0 || (x * elt & 15)) return bad(FCCI_EINVAL, "strides must be non-negative multiples of 16 bytes");
    if (d->k_stride_t < d->D || d->v_stride_t < d->D) return bad(FCCI_EINVAL, "the rows of a page overlap");
    if (d->k_scales_stride_p < 0 || d->k_scales_stride_h < 0 || d->v_scales_stride_p < 0 || d->v_scales_stride_h < 0)
        return bad(FCCI_EINVAL, "negative scale stride");
    if (d->k_new) {  // rows are written
        const int64_t n = d->num_pages, h = d->Hkv, ps = d->page_size;
        if (overlapping(d->D, {{ps, d->k_stride_t}, {h, d->k_stride_h}, {n, d->k_stride_p}}) ||
            overlapping(d->D, {{ps, d->v_stride_t}, {h, d->v_stride_h}, {n, d->v_stride_p}}))
            return bad(FCCI_EINVAL, "pages, heads or rows of a pool that gets rows overlap");
        if (e4m3 && (overlapping(1, {{h, d->k_scales_stride_h}, {n, d->k_scales_stride_p}}) ||
                     overlapping(1, {{h, d->v_scales_stride_h}, {n, d->v_scales_stride_p}})))
            return bad(FCCI_EINVAL, "scales of a pool that gets rows overlap");
    }
    if (op != Op::kAppend && overlapping(d->D, {{d->Hq, d->out_stride_h}, {d->total_q, d->out_stride_t}}))
        return bad(FCCI_EINVAL, "rows of out overlap");
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_status(cudaGetLastError());
    const int sms = device_sm_count(dev);
    if (sms <= 0) return bad(FCCI_ECUDA, "no device");
    if (op == Op::kPrefill && max_items(d->B, d->Hq, d->total_q) > 0x7fffffff)
        return bad(FCCI_EINVAL, "prefill: too many work items");
    L = ws_layout(d->B, d->Hq, d->Hkv, d->D, d->total_q, d->max_seqlen_q, op == Op::kPrefill ? d->max_kv_tokens : 0,
                  sms * kMaxCtasPerSm);
    if (!d->workspace || d->workspace_bytes < L.total) return bad(FCCI_EWORKSPACE, "workspace missing or too small");
    if (!aligned16(d->workspace)) return bad(FCCI_EINVAL, "workspace must be 16-byte aligned");

    memset(&p, 0, sizeof(p));
    p.B = d->B, p.Hq = d->Hq, p.Hkv = d->Hkv, p.G = d->Hq / d->Hkv, p.D = d->D;
    p.total_q = d->total_q;
    p.max_q = d->cu_seqlens_q ? d->max_seqlen_q : 1;
    p.cu_q = d->cu_seqlens_q;
    p.q = static_cast<const __half*>(d->q), p.q_st = d->q_stride_t, p.q_sh = d->q_stride_h;
    p.k_new = static_cast<const __half*>(d->k_new), p.kn_st = d->k_new_stride_t, p.kn_sh = d->k_new_stride_h;
    p.v_new = static_cast<const __half*>(d->v_new), p.vn_st = d->v_new_stride_t, p.vn_sh = d->v_new_stride_h;
    p.page = d->page_size, p.num_pages = d->num_pages, p.max_pages = d->max_pages;
    p.page_log2 = d->page_size == 16 ? 4 : d->page_size == 32 ? 5 : d->page_size == 64 ? 6 : 7;
    p.k_pages = static_cast<uint8_t*>(d->k_pages);
    p.k_sp = d->k_stride_p * elt, p.k_sh = d->k_stride_h * elt, p.k_st = d->k_stride_t * elt;
    p.v_pages = static_cast<uint8_t*>(d->v_pages);
    p.v_sp = d->v_stride_p * elt, p.v_sh = d->v_stride_h * elt, p.v_st = d->v_stride_t * elt;
    p.k_scales = d->k_scales, p.ks_sp = d->k_scales_stride_p, p.ks_sh = d->k_scales_stride_h;
    p.v_scales = d->v_scales, p.vs_sp = d->v_scales_stride_p, p.vs_sh = d->v_scales_stride_h;
    p.table = d->page_table, p.table_st = d->page_table_stride;
    p.seq_lens = d->seq_lens;
    p.out = static_cast<__half*>(d->out), p.o_st = d->out_stride_t, p.o_sh = d->out_stride_h;
    uint8_t* ws = static_cast<uint8_t*>(d->workspace);
    p.q_rot = static_cast<__half*>(d->q_rot_out);
    p.scale_log2 = d->scale * 1.4426950408889634f;
    p.rot = d->rotary_dim;
    p.append = d->k_new ? 1 : 0;
    p.err = reinterpret_cast<uint32_t*>(ws);
    p.done_cnt = reinterpret_cast<uint32_t*>(ws + 4);
    if (p.rot > 0) {
        // the frequencies of the last (theta, rotary_dim) of this thread: 128 powers a call would cost more than the launch
        static thread_local float theta = -1.f;
        static thread_local int rot = 0;
        static thread_local Freqs kept;
        if (theta != d->rope_theta || rot != p.rot) {
            const int half = p.rot / 2;
            for (int i = 0; i < half; ++i) {
                const long double turns = powl((long double)d->rope_theta, -(long double)i / half) * 0.15915494309189533576888L;
                kept.turn[i] = (uint64_t)ldexpl(turns - floorl(turns), 64);  // whole turns per position change nothing
            }
            theta = d->rope_theta, rot = p.rot;
        }
        f = kept;
    }
    return FCCI_OK;
}

static int paged_step(const fcci_paged_desc* d, Op op, cudaStream_t stream) {
    Params p;
    Freqs f;
    WsLayout L;
    int rc = fill(d, op, p, f, L);
    if (rc) return rc;
    if (p.total_q == 0) return set_status(FCCI_OK, nullptr);
    const bool e4m3 = d->cache_type == FCCI_PAGED_E4M3;
    if (op == Op::kAppend) {
        p.advance = d->advance;
        return launch_append(p, f, e4m3, stream);
    }
    uint8_t* ws = static_cast<uint8_t*>(d->workspace);
    if (op == Op::kPrefill && long_chunk(p.Hq, p.Hkv, p.max_q)) {
        p.q_rot = reinterpret_cast<__half*>(ws + L.q_rot);
        int64_t kv = d->max_kv_tokens;
        if (kv < 0) kv = (int64_t)((d->workspace_bytes - L.expanded) / ((size_t)p.Hkv * p.D * 4));
        return launch_prefill(p, f, e4m3, ws, L, (int)(kv < 0x7fffffff ? kv : 0x7fffffff), p.scale_log2, d->advance, stream);
    }
    Params rows = p;  // a prefill's append of its rows
    rows.q = nullptr;
    p.advance = d->advance;
    return launch_split(p, f, op == Op::kPrefill ? &rows : nullptr, e4m3, op == Op::kDecode && p.append, d->flags & FCCI_PAGED_PREFETCH_KV, ws, L, stream);
}

}  // namespace pg
}  // namespace fcci

extern "C" int fcci_paged_append(const fcci_paged_desc* desc, cudaStream_t stream) {
    return fcci::pg::paged_step(desc, fcci::pg::Op::kAppend, stream);
}

extern "C" int fcci_paged_decode(const fcci_paged_desc* desc, cudaStream_t stream) {
    return fcci::pg::paged_step(desc, fcci::pg::Op::kDecode, stream);
}

extern "C" int fcci_paged_prefill(const fcci_paged_desc* desc, cudaStream_t stream) {
    return fcci::pg::paged_step(desc, fcci::pg::Op::kPrefill, stream);
}

extern "C" size_t fcci_paged_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t total_q,
                                             int32_t max_seqlen_q, int32_t max_kv_tokens, int device) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128 && D != 256) || total_q < 0 ||
        max_seqlen_q < 0 || max_kv_tokens < 0)
        return 0;
    const int sms = fcci::device_sm_count(device);
    if (sms <= 0) return 0;
    return fcci::pg::ws_layout(B, Hq, Hkv, D, total_q, max_seqlen_q, max_kv_tokens, sms * fcci::kMaxCtasPerSm).total;
}

extern "C" int fcci_paged_workspace_init(void* workspace, size_t bytes, cudaStream_t stream) {
    if (!workspace || bytes < fcci::pg::kHeadBytes)
        return fcci::set_status(FCCI_EWORKSPACE, "fcci_paged_workspace_init: workspace too small");
    return fcci::set_cuda_status(cudaMemsetAsync(workspace, 0, fcci::pg::kHeadBytes, stream));
}

extern "C" int fcci_paged_read_error(void* workspace, uint32_t* flags, int clear, cudaStream_t stream) {
    return fcci_decode_read_error(workspace, flags, clear, stream);
}
