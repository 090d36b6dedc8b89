// Append of new keys and values to the paged cache, with the position rotation on the way.
//
// What a call must move: k_new, v_new and q in (fp16), q rotated out (fp16), the rows out
// (fp16, or one byte and a scale per page): it is bound by memory, or by launch and load
// latency when there are few tokens. Each value is rounded once, from the fp32 rotation.
//
// An e4m3 page has one scale 2^e for each kv head. Powers of two make the product with 2^-e
// exact, and an e that grows later re-rounds only the codes that become subnormal.
//
// Measured: 16 prompts of 256 to 4096 tokens, 32 q and 32 kv heads, 328 us (5.0 TB/s of what must move); 256 sequences
// of one token, 64 q and 8 kv heads, 7.1 us (4.5 in a graph); one sequence 2.4 us in a graph.
#include <initializer_list>
#include <mutex>

#include "paged.cuh"

namespace fcci {
namespace pg {

constexpr int kTokenWarps = 16, kTokenThreads = kTokenWarps * 32;
constexpr int kTokenTasks = 4;  // rows of a warp, at most

// 2^(from - to), from what a page had to what it takes; at least the least normal number, which leaves a code nothing either.
// (A page that no append has filled may have any scale byte.)
__device__ __forceinline__ float rescale(int from, int to) { return exp2_int(max(from - to, -126)); }

// One token per sequence. A warp takes `tasks` rows (query heads, or the key or value of a kv head): one when there are few
// sequences, so that the rows spread over as many warps as there are, else up to four, whose loads are
// under way together while the CTA gets through the chain length -> page -> scale and the angles, which all rows share.
template <int D, bool E4M3>
__global__ void __launch_bounds__(kTokenThreads) paged_append_token_kernel(const __grid_constant__ Params p,
                                                                         const __grid_constant__ Freqs f, int tasks) {
    constexpr int E = D / 32;  // elements of a row per lane
    __shared__ int flag;
    __shared__ float2 cs[D / 2];
    const int half = p.rot >> 1;
    const uint64_t turn = threadIdx.x < half ? f.turn[threadIdx.x] : 0;  // a launch constant: read before the wait
    griddep_wait();
    griddep_launch_dependents();  // behind the wait (paged.cuh)
    const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nkv = 2 * p.Hkv, all = nkv + (p.q ? p.Hq : 0);
    const int d0 = lane * E;
    const bool first = d0 < half;
    __align__(16) __half raw[kTokenTasks][E], other[kTokenTasks][E];
    auto load = [](__half(&dst)[E], const __half* a) {
        if constexpr (E == 8) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(a);
        else if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(a);
        else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(a);
    };
    const int task0 = blockIdx.y * tasks * kTokenWarps + warp;  // task k: + k * kTokenWarps
#pragma unroll
    for (int k = 0; k < kTokenTasks; ++k) {
        const int task = task0 + k * kTokenWarps;
        if (k >= tasks || task >= all) continue;
        const bool is_q = task >= nkv, is_v = !is_q && task >= p.Hkv;
        const int h = is_q ? task - nkv : (is_v ? task - p.Hkv : task);
        const __half* src = is_q ? p.q + b * p.q_st + h * p.q_sh
                                 : (is_v ? p.v_new + b * p.vn_st + h * p.vn_sh : p.k_new + b * p.kn_st + h * p.kn_sh);
        load(raw[k], src + d0);
        if (!is_v && d0 < p.rot) load(other[k], src + (first ? d0 + half : d0 - half));
    }
    const Seq s = seq_of(p, b);
    if (!s.ok) {
        if (blockIdx.y == 0 && threadIdx.x == 0) set_error(p, FCCI_DEV_ERR_CAPACITY);
    } else {
        const bool kv_here = blockIdx.y * tasks * kTokenWarps < nkv;  // the CTA has a key or a value
        const int id = kv_here ? page_of(p, b, s.T) : -1;
        if (threadIdx.x < half) cs[threadIdx.x] = rope_cs(turn, s.T);
        const int off = s.T & (p.page - 1);
        int had[kTokenTasks];
        uint8_t* sp[kTokenTasks];
#pragma unroll
        for (int k = 0; k < kTokenTasks; ++k) {
            const int task = task0 + k * kTokenWarps;
            had[k] = -1000;  // a fresh page has no scale yet
            sp[k] = nullptr;
            if (!E4M3 || k >= tasks || task >= nkv || id < 0) continue;
            const int h = task >= p.Hkv ? task - p.Hkv : task;
            sp[k] = task >= p.Hkv ? p.v_scales + id * p.vs_sp + h * p.vs_sh : p.k_scales + id * p.ks_sp + h * p.ks_sh;
            if (off) had[k] = (int)*sp[k] - 127;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kTokenTasks; ++k) {
            const int task = task0 + k * kTokenWarps;
            if (k >= tasks || task >= all) continue;
            const bool is_q = task >= nkv, is_v = !is_q && task >= p.Hkv;
            const int h = is_q ? task - nkv : (is_v ? task - p.Hkv : task);
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = __half2float(raw[k][e]);
                if (!is_v && d0 < p.rot)
                    x[e] = rotated(x[e], __half2float(other[k][e]), cs[(first ? d0 : d0 - half) + e], first);
            }
            auto store16 = [&](__half* dst) {
#pragma unroll
                for (int e = 0; e < E; e += 2)
                    *reinterpret_cast<uint32_t*>(dst + d0 + e) = pack_half2(x[e], x[e + 1]);
            };
            if (is_q) {
                store16(p.q_rot + ((int64_t)b * p.Hq + h) * D);
                continue;
            }
            if (id < 0) continue;
            uint8_t* page = is_v ? p.v_pages + id * p.v_sp + h * p.v_sh : p.k_pages + id * p.k_sp + h * p.k_sh;
            const int64_t st = is_v ? p.v_st : p.k_st;
            if constexpr (!E4M3) {
                store16(reinterpret_cast<__half*>(page + off * st));
            } else {
                float amax = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) amax = fmaxf(amax, fabsf(x[e]));
#pragma unroll
                for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                int ex = scale_exponent(amax);
                if (off && ex > had[k]) {
                    // the rows before this one take the larger scale (rare: the page's largest value grew past a power of two)
                    const float down = rescale(had[k], ex);
                    for (int i = lane; i < off * (D / 4); i += 32) {
                        uint32_t* w = reinterpret_cast<uint32_t*>(page + (i / (D / 4)) * st + (i % (D / 4)) * 4);
                        const uint32_t c = *w;
                        const uint32_t lo = half2_of_e4m3x2(c & 0xffffu), hi = half2_of_e4m3x2(c >> 16);
                        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        *w = e4m3x2(a.x * down, a.y * down) | (e4m3x2(g.x * down, g.y * down) << 16);
                    }
                }
                ex = max(ex, had[k]);
                const float up = rescale(0, ex);
                if constexpr (E == 2) {
                    *reinterpret_cast<uint16_t*>(page + off * st + d0) = (uint16_t)e4m3x2(x[0] * up, x[1] * up);
                } else {
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *reinterpret_cast<uint32_t*>(page + off * st + d0 + e) =
                            e4m3x2(x[e] * up, x[e + 1] * up) | (e4m3x2(x[e + 2] * up, x[e + 3] * up) << 16);
                }
                if (lane == 0) *sp[k] = (uint8_t)(ex + 127);
            }
        }
    }
    advance_lengths(p, &flag);
}

// Many tokens per sequence. A CTA takes one page's worth of positions of one sequence (page
// blockIdx.x behind the first page that the call touches) and a share of the heads: it
// builds the cos/sin table of its positions once in shared memory, and its warps then run over the
// heads. A warp holds R = 2048 / D rows of one head in registers (64 values a lane, as 4
// rows of two 8-element chunks, a chunk of the first half and the one it is rotated with),
// so a page is 1 to 8 warps, which agree on the largest value through shared memory
// before they round.
constexpr int kRowsThreads = 256;

// LONG: for a long chunk's attention, which takes halved queries and the new rows expanded to fp16 as well.
// STRIDE: a CTA also takes every gridDim.x-th page behind its first (16 prompts: 370 us, 342 without the loop).
template <int D, bool E4M3, bool LONG, bool STRIDE>
__global__ void __launch_bounds__(kRowsThreads, 2) paged_append_rows_kernel(const __grid_constant__ Params p,
                                                                         const __grid_constant__ Freqs f) {
    constexpr int R = 2048 / D;      // rows per warp
    constexpr int PL = D / 16;       // lanes per row
    constexpr int RP = 32 / PL;      // rows per pass
    constexpr int kWarps = kRowsThreads / 32;
    // [page][4][rot / 16]: (cos, cos, sin, sin) of angles 8 j + 2 m and 8 j + 2 m + 1 of a row at [row][m][j], so that the
    // lanes of a row, which have neighbouring j, read 16 neighbouring bytes each
    extern __shared__ float4 cs_table[];
    __shared__ int flag;
    __shared__ float amax_sm[2][kWarps];
    griddep_wait();
    griddep_launch_dependents();  // behind the wait (paged.cuh)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.y;
    const Seq s = seq_of(p, b);
    // a long chunk's plan has given rows to every sequence that is served
    const bool served = s.ok && s.n > 0 && (!LONG || p.cu_kv[b + 1] - p.cu_kv[b] == s.T + s.n);
    if (!s.ok && blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) set_error(p, FCCI_DEV_ERR_CAPACITY);
    // (a sequence that is not served may have any length, a negative one too: no page of it is looked at)
    const int pages = served ? (s.T + s.n - 1 >> p.page_log2) + 1 : 0;
    for (int page_i = served ? (s.T >> p.page_log2) + (int)blockIdx.x : 0; page_i < pages; page_i += gridDim.x) {
        const int p0 = page_i << p.page_log2;  // first position of the page
        const int half = p.rot >> 1;
        for (int i = tid; i < p.page * half; i += kRowsThreads) {
            const int r = i / half, k = i - r * half;
            if (p0 + r >= s.T && p0 + r < s.T + s.n) {
                const float2 cs = rope_cs(f.turn[k], p0 + r);
                float* at = reinterpret_cast<float*>(&cs_table[r * (half >> 1) + ((k >> 1) & 3) * (half >> 3) + (k >> 3)]);
                at[k & 1] = cs.x;
                at[2 + (k & 1)] = cs.y;
            }
        }
        const int id = page_of(p, b, p0);
        __syncthreads();
        const int W = max(1, p.page / R);      // warps of one page
        const int groups = kWarps / W;         // heads in flight
        const int grp = warp / W, part = warp % W;
        const int row0 = part * R + lane / PL;  // row of pass 0; pass i: + i * RP
        const int j = lane % PL;
        // chunk pair j: two 8-element chunks rotated with one another, then the plain ones
        const bool turn_j = j < (p.rot >> 4);
        const int dlo = turn_j ? 8 * j : p.rot + 16 * (j - (p.rot >> 4));
        const int dhi = turn_j ? dlo + half : dlo + 8;
        const int heads = (p.q ? p.Hq : 0) + 2 * p.Hkv;
        const int per = (heads + gridDim.z - 1) / gridDim.z;
        const int h_end = min(heads, (int)(blockIdx.z + 1) * per);
        // a long chunk's attention reads fp16 rows: write these while they are here
        const int64_t exp_row = LONG ? p.cu_kv[b] : 0;
        // passes whose row is new, and those whose row the page held before
        uint32_t is_new = 0, is_old = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row0 + i * RP, pos = p0 + r;
            if (r < p.page && pos >= s.T && pos < s.T + s.n) is_new |= 1u << i;
            if (r < p.page && pos < s.T) is_old |= 1u << i;
        }
        const int64_t src_row = s.tok0 + p0 + row0 - s.T;
        const int ahead_pos = p0 + part * R + lane / (D / 64);
        const int64_t ahead_row = s.tok0 + ahead_pos - s.T;
        const bool ahead = ahead_pos >= s.T && ahead_pos < s.T + s.n && ahead_pos < p0 + p.page;
        int buf = 0;
        for (int hb = blockIdx.z * per; hb < h_end; hb += groups, buf ^= 1) {
            const int item = hb + grp;
            const bool live = item < h_end;
            const bool is_k = item < p.Hkv, is_v = !is_k && item < 2 * p.Hkv, is_q = !is_k && !is_v;
            const int h = is_k ? item : (is_v ? item - p.Hkv : item - 2 * p.Hkv);
            const __half* src = is_q ? p.q + h * p.q_sh : (is_v ? p.v_new + h * p.vn_sh : p.k_new + h * p.kn_sh);
            const int64_t sst = is_q ? p.q_st : (is_v ? p.vn_st : p.kn_st);
            uint8_t* page = nullptr;
            uint8_t* sp = nullptr;
            const int64_t st = is_v ? p.v_st : p.k_st;
            if (live && !is_q && id >= 0) {
                page = is_v ? p.v_pages + id * p.v_sp + h * p.v_sh : p.k_pages + id * p.k_sp + h * p.k_sh;
                if constexpr (E4M3)
                    sp = is_v ? p.v_scales + id * p.vs_sp + h * p.vs_sh : p.k_scales + id * p.ks_sp + h * p.ks_sh;
            }
            const bool work = live && (is_q || page);
            float2 x[4][8];
            float amax = 0.f;
            uint4 lo[4], hi[4];
            src += src_row * sst;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
                if (work && (is_new >> i & 1)) {
                    lo[i] = *reinterpret_cast<const uint4*>(src + i * RP * sst + dlo);
                    hi[i] = *reinterpret_cast<const uint4*>(src + i * RP * sst + dhi);
                }
            }
            // the warp's next item on its way into L2 (its rows are 32 lines of 128 bytes, one a lane): the registers are full
            if (item + groups < h_end && ahead) {
                const int nx = item + groups;
                const bool nq = nx >= 2 * p.Hkv, nv = !nq && nx >= p.Hkv;
                const int nh = nq ? nx - 2 * p.Hkv : (nv ? nx - p.Hkv : nx);
                const __half* a = nq ? p.q + nh * p.q_sh : (nv ? p.v_new + nh * p.vn_sh : p.k_new + nh * p.kn_sh);
                a += ahead_row * (nq ? p.q_st : (nv ? p.vn_st : p.kn_st)) + (lane % (D / 64)) * 64;
                asm volatile("prefetch.global.L2 [%0];" ::"l"(a));
            }
            const bool turn = turn_j && !is_v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2* a = reinterpret_cast<const __half2*>(&lo[i]);
                const __half2* c = reinterpret_cast<const __half2*>(&hi[i]);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    float2 u = __half22float2(a[m]), w = __half22float2(c[m]);
                    if (turn && (is_new >> i & 1)) {
                        const float4 cs = cs_table[(row0 + i * RP) * (half >> 1) + m * (half >> 3) + j];
                        const float2 co = make_float2(cs.x, cs.y), si = make_float2(cs.z, cs.w);
                        const float2 y = __fmul2_rn(w, si), z = __fmul2_rn(u, si);
                        u = __ffma2_rn(u, co, make_float2(-y.x, -y.y));
                        w = __ffma2_rn(w, co, z);
                    }
                    x[i][m] = u;
                    x[i][4 + m] = w;
                    if (E4M3) amax = fmaxf(fmaxf(amax, fmaxf(fabsf(u.x), fabsf(u.y))), fmaxf(fabsf(w.x), fabsf(w.y)));
                }
            }
            auto store16 = [&](__half* row, int i) {
                const float factor = E4M3 || is_q ? kLongQuery : 1.f;  // (e4m3: queries alone come here)
                auto two = [&](float2 v) {
                    if (LONG) v = __fmul2_rn(v, make_float2(factor, factor));
                    return pack_half2(v.x, v.y);
                };
                *reinterpret_cast<uint4*>(row + dlo) = make_uint4(two(x[i][0]), two(x[i][1]), two(x[i][2]), two(x[i][3]));
                *reinterpret_cast<uint4*>(row + dhi) = make_uint4(two(x[i][4]), two(x[i][5]), two(x[i][6]), two(x[i][7]));
            };
            if constexpr (E4M3) {
#pragma unroll
                for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                // old rows of the call's first page keep (or grow) the page's scale
                const bool old = p0 < s.T;
                const int had = old && sp ? (int)*sp - 127 : -1000;
                if (W > 1 && work && !is_q) {
                    // every warp of the page has read the old scale before this barrier;
                    // two buffers: a warp may be one head ahead of another's reads
                    if (lane == 0) amax_sm[buf][warp] = amax;
                    named_bar_sync(1 + grp, 32 * W);
                    for (int w = 0; w < W; ++w) amax = fmaxf(amax, amax_sm[buf][grp * W + w]);
                } else {
                    __syncwarp();  // every lane has read the old scale
                }
                if (work && !is_q) {
                    int ex = scale_exponent(amax);
                    const bool grows = old && ex > had;
                    ex = max(ex, had);
                    const float up = rescale(0, ex), down = grows ? rescale(had, ex) : 1.f;
                    const float2 up2 = make_float2(up, up);
                    const int xe = is_k ? ex + kLongKeyExp : ex;
                    const __half2 s2 = LONG ? expansion_scale(p, ex, xe) : __half2();
                    const bool clamp = xe >= kScaleMax;
                    auto four = [&](float2 u, float2 w) {
                        u = __fmul2_rn(u, up2), w = __fmul2_rn(w, up2);
                        return e4m3x2(u.x, u.y) | (e4m3x2(w.x, w.y) << 16);
                    };
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint8_t* row = page + (row0 + i * RP) * st;
                        if (is_new >> i & 1) {
                            const int pos = p0 + row0 + i * RP;
                            const uint2 u = make_uint2(four(x[i][0], x[i][1]), four(x[i][2], x[i][3]));
                            const uint2 w = make_uint2(four(x[i][4], x[i][5]), four(x[i][6], x[i][7]));
                            *reinterpret_cast<uint2*>(row + dlo) = u;
                            *reinterpret_cast<uint2*>(row + dhi) = w;
                            if (LONG) {
                                __half* er = (is_v ? p.exp_v : p.exp_k) + h * p.exp_sh + (exp_row + pos) * D;
                                *reinterpret_cast<uint4*>(er + dlo) = expanded(u, s2, clamp);
                                *reinterpret_cast<uint4*>(er + dhi) = expanded(w, s2, clamp);
                            }
                        } else if (grows && (is_old >> i & 1)) {
                            for (int k = 0; k < 4; ++k) {
                                uint32_t* w = reinterpret_cast<uint32_t*>(row + (k < 2 ? dlo : dhi) + (k & 1) * 4);
                                const uint32_t c = *w;
                                const uint32_t c0 = half2_of_e4m3x2(c & 0xffffu), c1 = half2_of_e4m3x2(c >> 16);
                                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&c0));
                                const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&c1));
                                *w = e4m3x2(a.x * down, a.y * down) | (e4m3x2(g.x * down, g.y * down) << 16);
                            }
                        }
                    }
                    if (part == 0 && lane == 0) *sp = (uint8_t)(ex + 127);
                }
            }
            if (work && (is_q || !E4M3)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!(is_new >> i & 1)) continue;
                    const int pos = p0 + row0 + i * RP;
                    __half* row = is_q ? p.q_rot + ((src_row + i * RP) * p.Hq + h) * D
                                       : reinterpret_cast<__half*>(page + (row0 + i * RP) * st);
                    store16(row, i);
                    if (LONG && !is_q)
                        store16((is_v ? p.exp_v : p.exp_k) + h * p.exp_sh + (exp_row + pos) * D, i);
                }
            }
        }
        if constexpr (!STRIDE) break;
        __syncthreads();  // the angles of this page have been read
    }
    advance_lengths(p, &flag);
}

template <int D, bool E4M3, bool LONG = false>
static int launch_append_t(const Params& p, const Freqs& f, cudaStream_t st) {
    const int heads = (p.q ? p.Hq : 0) + 2 * p.Hkv;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_status(cudaGetLastError());
    if (dev < 0 || dev >= 128) return set_status(FCCI_EINVAL, "device index");
    const int sms = device_sm_count(dev);
    if (!p.cu_q) {
        // one row a warp while that fits the GPU at once (4 CTAs an SM), else as many as it takes, up to four
        int tasks = 1;
        while (tasks < kTokenTasks && (int64_t)p.B * ((heads + tasks * kTokenWarps - 1) / (tasks * kTokenWarps)) > 4 * sms) ++tasks;
        const int y = (heads + tasks * kTokenWarps - 1) / (tasks * kTokenWarps);
        return launch_pdl(paged_append_token_kernel<D, E4M3>, dim3(p.B, y), dim3(kTokenThreads), 0, st, p, f, tasks);
    }
    // pages that the longest run of new tokens can touch, and a head split that fills the GPU
    // when there are few pages
    int64_t slots = ((int64_t)(p.max_q < p.total_q ? p.max_q : p.total_q) + p.page - 2) / p.page + 1;
    const int64_t pages = (int64_t)p.total_q / p.page + p.B;
    int64_t z = (8 * sms + pages - 1) / pages;
    const int64_t most = (heads + 7) / 8;
    if (z > most) z = most;
    if (z < 1) z = 1;
    // max_q is a bound on any sequence, total_q on all: where their product is far above the pages that there can be, the
    // CTAs of a sequence take several pages each
    const int64_t ctas = 16 * pages * z > 65536 ? 16 * pages * z : 65536;
    const bool stride = slots > ctas / (p.B * z);
    if (stride) slots = ctas / (p.B * z) > 1 ? ctas / (p.B * z) : 1;
    const auto kernel = stride ? paged_append_rows_kernel<D, E4M3, LONG, true> : paged_append_rows_kernel<D, E4M3, LONG, false>;
    const size_t smem = (size_t)p.page * (p.rot / 2) * sizeof(float2);
    static std::once_flag once[128];
    static cudaError_t attr[128];
    std::call_once(once[dev], [&]() {
        for (auto k : {paged_append_rows_kernel<D, E4M3, LONG, false>, paged_append_rows_kernel<D, E4M3, LONG, true>}) {
            attr[dev] = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
            if (attr[dev] != cudaSuccess) return;
        }
    });
    if (attr[dev] != cudaSuccess) return set_cuda_status(attr[dev]);
    return launch_pdl(kernel, dim3((unsigned)slots, p.B, (unsigned)z), dim3(kRowsThreads), smem, st, p, f);
}

int launch_append(const Params& p, const Freqs& f, bool e4m3, cudaStream_t st) {
    if (p.exp_k) return e4m3 ? launch_append_t<128, true, true>(p, f, st) : launch_append_t<128, false, true>(p, f, st);
    switch (p.D) {
        case 64: return e4m3 ? launch_append_t<64, true>(p, f, st) : launch_append_t<64, false>(p, f, st);
        case 128: return e4m3 ? launch_append_t<128, true>(p, f, st) : launch_append_t<128, false>(p, f, st);
        case 256: return e4m3 ? launch_append_t<256, true>(p, f, st) : launch_append_t<256, false>(p, f, st);
        default: return set_status(FCCI_EUNSUPPORTED, "paged append: unsupported head_dim");
    }
}

}  // namespace pg
}  // namespace fcci
