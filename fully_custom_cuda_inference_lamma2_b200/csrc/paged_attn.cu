// Attention over the paged KV cache, and the host side of the paged entry points.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "paged.cuh"

namespace fcci {
namespace pg {

constexpr int kAttnThreads = 128;

// One CTA per (new token, query head, sequence): warp w takes keys w, w + 4, ... with a running
// maximum and sum, and the four states are joined at the end.
template <int D, bool E4M3>
__global__ void __launch_bounds__(kAttnThreads) paged_attn_kernel(const __grid_constant__ Params p) {
    constexpr int E = D / 32, kWarps = kAttnThreads / 32;
    __shared__ float acc_sm[kWarps][D], m_sm[kWarps], l_sm[kWarps];
    __shared__ int flag;
    griddep_launch_dependents();
    griddep_wait();
    const int i = blockIdx.x, hq = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d0 = lane * E;
    const Seq s = seq_of(p, b);
    const int n = s.ok ? s.n : 0;
    if (!s.ok && i == 0 && hq == 0 && threadIdx.x == 0) set_error(p, FCCI_DEV_ERR_CAPACITY);
    const bool row_there = i < n || (!s.ok && !p.cu_q);
    if (row_there) {
        const int keys = s.ok ? s.T + (p.append ? i + 1 : 0) : 0;
        const int64_t row = p.cu_q ? s.tok0 + i : b;
        const int h = hq / p.G;
        float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            q[e] = __half2float(p.q[row * p.q_st + hq * p.q_sh + d0 + e]);
            acc[e] = 0.f;
        }
        for (int t = warp; t < keys; t += kWarps) {
            const int id = page_of(p, b, t);
            if (id < 0) continue;
            const uint8_t* kr = p.k_pages + id * p.k_sp + h * p.k_sh + (t & (p.page - 1)) * p.k_st;
            const uint8_t* vr = p.v_pages + id * p.v_sp + h * p.v_sh + (t & (p.page - 1)) * p.v_st;
            float ks = 1.f, vs = 1.f, x = 0.f, k[E], v[E];
            if constexpr (E4M3) {
                ks = exp2_int((int)p.k_scales[id * p.ks_sp + h * p.ks_sh] - 127);
                vs = exp2_int((int)p.v_scales[id * p.vs_sp + h * p.vs_sh] - 127);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint32_t a = half2_of_e4m3x2(kr[d0 + e]), c = half2_of_e4m3x2(vr[d0 + e]);
                    k[e] = __low2float(*reinterpret_cast<const __half2*>(&a));
                    v[e] = __low2float(*reinterpret_cast<const __half2*>(&c));
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    k[e] = __half2float(reinterpret_cast<const __half*>(kr)[d0 + e]);
                    v[e] = __half2float(reinterpret_cast<const __half*>(vr)[d0 + e]);
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) x = fmaf(q[e], k[e], x);
#pragma unroll
            for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            x *= ks * p.scale_log2;
            const float mn = fmaxf(m, x), al = ex2(m - mn), pr = ex2(x - mn);
            l = l * al + pr;
            m = mn;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = acc[e] * al + pr * vs * v[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) acc_sm[warp][d0 + e] = acc[e];
        if (lane == 0) m_sm[warp] = m, l_sm[warp] = l;
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kAttnThreads) {
            float M = -INFINITY, L = 0.f, o = 0.f;
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, m_sm[w]);
            for (int w = 0; w < kWarps && M != -INFINITY; ++w) {
                const float a = ex2(m_sm[w] - M);
                L += l_sm[w] * a;
                o += acc_sm[w][d] * a;
            }
            p.out[row * p.o_st + hq * p.o_sh + d] = __float2half_rn(L > 0.f ? o / L : 0.f);
        }
    }
    advance_lengths(p, &flag);
}

template <int D, bool E4M3>
static int launch_attn_t(const Params& p, cudaStream_t st) {
    return launch_pdl(paged_attn_kernel<D, E4M3>, dim3(p.max_q, p.Hq, p.B), dim3(kAttnThreads), 0, st, p);
}

static int launch_attn(const Params& p, bool e4m3, cudaStream_t st) {
    switch (p.D) {
        case 64: return e4m3 ? launch_attn_t<64, true>(p, st) : launch_attn_t<64, false>(p, st);
        case 128: return e4m3 ? launch_attn_t<128, true>(p, st) : launch_attn_t<128, false>(p, st);
        default: return e4m3 ? launch_attn_t<256, true>(p, st) : launch_attn_t<256, false>(p, st);
    }
}

// ------------------------------------------------------------------ host side

WsLayout ws_layout(int Hq, int Hkv, int D, int total_q, int max_q, int max_kv, int grid) {
    auto up = [](size_t x) { return (x + 1023) & ~size_t(1023); };
    WsLayout w;
    w.part_lse = up(kHeadBytes);
    w.part_o = w.part_lse + up((size_t)2 * grid * kMaxCols * 4);
    w.q_rot = w.part_o + up((size_t)2 * grid * kMaxCols * D * 4);
    w.total = w.q_rot + up((size_t)total_q * Hq * D * 2);
    return w;
}

enum class Op { kAppend, kDecode, kPrefill };

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

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
    if (d->rotary_dim > 0 && !(d->rope_theta > 0.f && d->rope_theta < INFINITY))
        return bad(FCCI_EINVAL, "rope_theta must be positive");
    if (op != Op::kAppend && !(d->scale > 0.f && d->scale < INFINITY)) return bad(FCCI_EINVAL, "scale must be positive");
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
    if (d->k_stride_t * elt < d->D || d->v_stride_t * elt < d->D) return bad(FCCI_EINVAL, "the rows of a page overlap");
    if (d->k_scales_stride_p < 0 || d->k_scales_stride_h < 0 || d->v_scales_stride_p < 0 || d->v_scales_stride_h < 0)
        return bad(FCCI_EINVAL, "negative scale stride");
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_status(cudaGetLastError());
    const int sms = device_sm_count(dev);
    if (sms <= 0) return bad(FCCI_ECUDA, "no device");
    L = ws_layout(d->Hq, d->Hkv, d->D, d->total_q, d->max_seqlen_q, op == Op::kPrefill ? d->max_kv_tokens : 0,
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
    p.q_rot = d->q_rot_out ? static_cast<__half*>(d->q_rot_out) : reinterpret_cast<__half*>(ws + L.q_rot);
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
            for (int i = 0; i < half; ++i)
                kept.turn[i] = (uint64_t)(powl((long double)d->rope_theta, -(long double)i / half) *
                                              0.15915494309189533576888L * 18446744073709551616.0L + 0.5L);
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
    // the append writes the rotated queries to q_rot, where the attention reads them
    if (p.append || p.rot > 0 || d->q_rot_out) {
        rc = launch_append(p, f, e4m3, stream);
        if (rc) return rc;
        p.q = p.q_rot, p.q_st = (int64_t)p.Hq * p.D, p.q_sh = p.D;
    }
    p.advance = d->advance;
    return launch_attn(p, e4m3, stream);
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
    return fcci::pg::ws_layout(Hq, Hkv, D, total_q, max_seqlen_q, max_kv_tokens, sms * fcci::kMaxCtasPerSm).total;
}

extern "C" int fcci_paged_workspace_init(void* workspace, size_t bytes, cudaStream_t stream) {
    if (!workspace || bytes < fcci::pg::kHeadBytes)
        return fcci::set_status(FCCI_EWORKSPACE, "fcci_paged_workspace_init: workspace too small");
    return fcci::set_cuda_status(cudaMemsetAsync(workspace, 0, fcci::pg::kHeadBytes, stream));
}

extern "C" int fcci_paged_read_error(void* workspace, uint32_t* flags, int clear, cudaStream_t stream) {
    return fcci_decode_read_error(workspace, flags, clear, stream);
}
