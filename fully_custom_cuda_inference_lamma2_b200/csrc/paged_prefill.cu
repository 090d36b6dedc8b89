// Prompts and long chunks over the paged cache: the keys and values of a call's sequences are expanded to fp16 rows
// [Hkv, rows, 128] in the workspace and go through the library's causal prefill attention.
//
// Expanding costs 1 byte in and 2 bytes out for each cached value, and the attention then reads 2; that is
// small beside its products once a chunk has some dozens of query rows per kv head (shorter
// ones take the split-KV kernels, which read the pages in place). code * 2^e is exact in fp16 for every scale that an
// append makes, but for a value's 256 * 2^8, which becomes 65504 (2^-11 of itself, an fp16 rounding); rotated keys go up to
// 352 * 2^8 and are expanded at half their size (paged.cuh: kLongKeyExp). The rotated queries and the weights are rounded once
// to fp16, as in the attention over an arena (the queries halved, so that none passes its range): holding the queries in
// two parts, as the split kernels do, would add half to the products of a kernel that the products bound, and take shared
// memory for two more tiles (results are off by 3.5e-4 to 4.2e-4 in the 2-norm, 2.1e-4 of it their own rounding).
//
// Measured: 2 x 2048 new tokens after 12000 to 14000, 64 / 8 heads: attention 1456 us, append 61, expansion 45 (3.6 TB/s
// in and out); 16 prompts of 256 to 4096, 32 heads: attention 659 us, append 335 (one pass; in a loop, under the power cap,
// the attention takes up to 1600 and 720).
//
// Launches: the plan (row ranges, work list), the append (which also writes its own rows expanded, while it has
// them), the expansion of the rows cached before, the attention.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <mutex>

#include "paged.cuh"
#include "prefill_list.cuh"

namespace fcci {
namespace pg {

constexpr int kPlanThreads = 256, kExpandThreads = 256;

// One CTA: rows [cu_kv[b], cu_kv[b + 1]) of the expanded arrays for every sequence with new tokens, and the work list.
// A sequence for which no rows are left gets none, is reported and not served.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const __grid_constant__ Params p,
                                                               const __grid_constant__ pf::Params a, int32_t* cu_kv,
                                                               int64_t max_items) {
    extern __shared__ int plan_sm[];
    __shared__ int64_t need;
    griddep_launch_dependents();
    griddep_wait();
    for (int b = threadIdx.x; b < p.B; b += kPlanThreads) {
        const Seq s = seq_of(p, b);
        if (!s.ok) set_error(p, FCCI_DEV_ERR_CAPACITY);
        plan_sm[b] = s.ok && s.n > 0 ? s.T + s.n : 0;
        plan_sm[p.B + b] = s.n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int at = 0;
        int64_t items = 0;
        cu_kv[0] = 0;
        for (int b = 0; b < p.B; ++b) {
            if (plan_sm[b] > a.capacity - at) {
                set_error(p, FCCI_DEV_ERR_CAPACITY);
            } else {
                at += plan_sm[b];
                if (plan_sm[b] > 0) items += (int64_t)((plan_sm[p.B + b] + 255) / 256) * p.Hq;
            }
            cu_kv[b + 1] = at;
        }
        need = items;
    }
    __syncthreads();
    if (need > max_items) {
        // only offsets that run backwards, so that sequences share rows, can ask for so many: nothing is served
        for (int b = threadIdx.x; b <= p.B; b += kPlanThreads) cu_kv[b] = 0;
        if (threadIdx.x == 0) {
            set_error(p, FCCI_DEV_ERR_CAPACITY);
            *a.n_items = 0;
            *a.item_cnt = 0u;
            *a.exit_cnt = 0u;
        }
        return;
    }
    pf::build_work_list(a, plan_sm);
}

// Rows [0, T_b) of every sequence with new tokens. A warp takes (page, kv head, K or V): 16 bytes a lane, four or two rows
// a step, four steps' loads under way at once.
template <bool E4M3>
__global__ void __launch_bounds__(kExpandThreads) paged_expand_kernel(const __grid_constant__ Params p) {
    constexpr int D = 128, LPR = E4M3 ? 8 : 16, RPS = 32 / LPR;  // lanes per row, rows per step
    extern __shared__ int pages_before[];                       // [B + 1]
    __shared__ int warp_sum[kExpandThreads / 32];
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int chunk = (p.B + kExpandThreads - 1) / kExpandThreads, lo = tid * chunk, hi = min(p.B, lo + chunk);
    int local = 0;
    for (int b = lo; b < hi; ++b) {
        const bool served = p.cu_kv[b + 1] > p.cu_kv[b];
        const int n = served ? (p.seq_lens[b] + p.page - 1) >> p.page_log2 : 0;
        pages_before[b + 1] = n;
        local += n;
    }
    int incl = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    if (tid == 0) pages_before[0] = 0;
    __syncthreads();
    int run = incl - local;
    for (int w = 0; w < warp; ++w) run += warp_sum[w];
    for (int b = lo; b < hi; ++b) pages_before[b + 1] = run += pages_before[b + 1];
    __syncthreads();

    const int64_t tasks = (int64_t)pages_before[p.B] * p.Hkv * 2;
    const int r0 = lane / LPR, ch = lane % LPR;
    for (int64_t t = (int64_t)blockIdx.x * (kExpandThreads / 32) + warp; t < tasks; t += (int64_t)gridDim.x * (kExpandThreads / 32)) {
        const bool is_v = t & 1;
        const int64_t u = t >> 1;
        const int h = (int)(u % p.Hkv), page_i = (int)(u / p.Hkv);
        int b = 0, r = p.B - 1;  // last sequence with pages_before[b] <= page_i
        while (b < r) {
            const int mid = (b + r + 1) >> 1;
            if (pages_before[mid] <= page_i) b = mid;
            else r = mid - 1;
        }
        const int j = page_i - pages_before[b];
        const int T = p.seq_lens[b], first = j << p.page_log2, rows = min(p.page, T - first);
        const int id = page_of(p, b, first);
        if (id < 0) continue;
        const uint8_t* src = (is_v ? p.v_pages + id * p.v_sp + h * p.v_sh : p.k_pages + id * p.k_sp + h * p.k_sh) + ch * 16;
        const int64_t st = is_v ? p.v_st : p.k_st;
        __half* dst = (is_v ? p.exp_v : p.exp_k) + h * p.exp_sh + (int64_t)(p.cu_kv[b] + first) * D;
        __half2 scale;
        bool clamp = false;
        if constexpr (E4M3) {
            const int e = (int)(is_v ? p.v_scales[id * p.vs_sp + h * p.vs_sh] : p.k_scales[id * p.ks_sp + h * p.ks_sh]) - 127;
            const int xe = is_v ? e : e + kLongKeyExp;
            scale = expansion_scale(p, e, xe);
            clamp = xe >= kScaleMax;
        }
        for (int row = r0; row < rows; row += 4 * RPS) {
            uint4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (row + k * RPS < rows) x[k] = *reinterpret_cast<const uint4*>(src + (row + k * RPS) * st);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (row + k * RPS >= rows) continue;
                __half* d = dst + (int64_t)(row + k * RPS) * D;
                if constexpr (E4M3) {
                    *reinterpret_cast<uint4*>(d + ch * 16) = expanded(make_uint2(x[k].x, x[k].y), scale, clamp);
                    *reinterpret_cast<uint4*>(d + ch * 16 + 8) = expanded(make_uint2(x[k].z, x[k].w), scale, clamp);
                } else {
                    *reinterpret_cast<uint4*>(d + ch * 8) = x[k];
                }
            }
        }
    }
}

int launch_prefill(const Params& base, const Freqs& f, bool e4m3, uint8_t* ws, const WsLayout& L, int max_kv, float scale_log2,
                   int advance, cudaStream_t st) {
    Params p = base;
    if (max_kv <= 0) return set_status(FCCI_EWORKSPACE, "paged prefill: workspace has no room for the expanded keys");
    const size_t plan_smem = (size_t)(4 * p.B + 1) * sizeof(int);
    if (p.B > 12000) return set_status(FCCI_EUNSUPPORTED, "paged prefill: batch too large");
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_status(cudaGetLastError());
    if (dev < 0 || dev >= 128) return set_status(FCCI_EINVAL, "device index");
    static std::once_flag once[128];
    static cudaError_t attr[128];
    std::call_once(once[dev], [dev]() {
        attr[dev] = cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    });
    if (attr[dev] != cudaSuccess) return set_cuda_status(attr[dev]);
    const int sms = device_sm_count(dev);
    int32_t* cu_kv = reinterpret_cast<int32_t*>(ws + L.cu_kv);
    p.cu_kv = cu_kv;
    p.exp_k = reinterpret_cast<__half*>(ws + L.expanded);
    p.exp_sh = (int64_t)max_kv * p.D;
    p.exp_v = p.exp_k + p.Hkv * p.exp_sh;
    p.advance = 0;
    const int64_t items = max_items(p.B, p.Hq, p.total_q);

    pf::Params a;
    memset(&a, 0, sizeof(a));
    a.B = p.B, a.Hq = p.Hq, a.Hkv = p.Hkv, a.G = p.G, a.total_q = p.total_q, a.max_q = p.max_q;
    a.cu_q = p.cu_q, a.cu_kv = cu_kv, a.seq_lens = p.seq_lens;
    a.capacity = max_kv;
    a.k_cache = p.exp_k, a.k_sh = p.exp_sh, a.k_st = p.D;
    a.v_cache = p.exp_v, a.v_sh = p.exp_sh, a.v_st = p.D;
    a.out = p.out, a.o_st = p.o_st, a.o_sh = p.o_sh;
    a.scale_log2 = scale_log2 / (kLongQuery * (e4m3 ? ldexpf(1.f, kLongKeyExp) : 1.f));
    a.weight_log2 = 7.f;  // keys down to 2^-31 of a row's largest weight count (2^-24 with 0), and thousands may share it
    a.advance = advance;
    a.err = p.err;
    uint32_t* head = reinterpret_cast<uint32_t*>(ws + 32);
    a.item_cnt = head, a.exit_cnt = head + 1, a.n_items = reinterpret_cast<int32_t*>(head + 2);
    a.items = reinterpret_cast<int4*>(ws + L.items);
    a.q_rot = p.q_rot;

    int rc = launch_pdl(paged_plan_kernel, dim3(1), dim3(kPlanThreads), plan_smem, st, p, a, cu_kv, items);
    if (!rc) rc = launch_append(p, f, e4m3, st);
    if (!rc) rc = launch_pdl(e4m3 ? paged_expand_kernel<true> : paged_expand_kernel<false>, dim3(8 * sms), dim3(kExpandThreads),
                             (size_t)(p.B + 1) * sizeof(int), st, p);
    if (!rc) rc = pf::launch_attend(a, items, st);
    return rc;
}

}  // namespace pg
}  // namespace fcci
