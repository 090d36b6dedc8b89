// Split-KV attention over e4m3 pages of head_dim 128 on the 5th-generation tensor cores: one new token per
// sequence (its append fused in), or a few of them whose rows an append has written already.
// Work and fetching: paged_tiles.cuh, tiles of 128 keys.
//
// The e4m3 codes go into tcgen05 (kind::f8f6f4, fp32 sums) as they lie in shared memory. With mma.sync they would
// have to become fp16 in registers first, and that conversion unit (16 lanes a cycle and SM, for 2 codes each)
// bound that kernel at 59 % of the memory rate. The other operand keeps its precision as a sum of 8-bit parts, rows of the
// same product:
// S^T[key, (part, row)] = K Q^T     A = the K tile (128 keys), B = 3 * COLS rows of query parts, e4m3
// O^T[dim, (part, row)] += V^T P^T  A = the V tile read dim-major, B = the weight parts, e5m2, 4 * COLS bytes of each
//                                   key side by side (N-major), which is what the key's thread has
// The parts are summed where S is read, and where O is read at a unit's end.
//   - A query is p0 + p1 / 16 + p2 / 256, each part the e4m3 rounding of what the ones before left, times 16: within 2^-12
//     of it, or 2^-18 absolute (of 448, the row's largest).
//   - A weight is rounded to fp16 and then is p0 + p1 / 8 + p2 / 64 + p3 / 512 exactly: e5m2 is fp16's upper byte, so a
//     part is cut off, not rounded, and takes three bits. With the largest at 2^13 or more, all of fp16's 11 bits are there
//     down to 2^-27 of the largest, and one bit down to 2^-37. (Three e4m3 parts, rounded, held 2^-24 of it and nothing
//     below: 16384 keys of 2^-20 beside one lost 0.4 %. 32 x 4096 keys: group 8 48.6 us a layer with either, group 16
//     63.4 with three parts, 65.3 with four, 66.8 with four that are rounded.)
//   - A query row is rotated in fp32 and scaled by a power of two to at most 448 before it is split.
//   - Thread t of the softmax owns key t of the tile: its scales are its own numbers. The exponent of V's scale
//     joins the score, x = s + log2 vs, so the weight that multiplies the codes is 2^(x - m), and no scale can push it out
//     of range (the bits that it keeps count from the largest weight times scale); the sum l takes 2^(x - m) / vs, the
//     weight of the value itself.
//   - m moves only when a weight would exceed 2^15.75 (e5m2 ends at 57344), to leave the largest at 2^13: O in
//     tensor memory is scaled rarely, and four warps agree on it with one barrier a tile.
//
// Measured: 32 x 4096 keys, 8 kv heads 51.2 us (5.3 TB/s; 6.4 in the loop, the rest is the start: lengths, queries, first
// tiles, and the end); 64 sequences of 128 to 8192 keys, 32 kv heads 384 us (5.8 TB/s). A tile takes the softmax some 1900
// cycles of latency, less than the memory needs for it with two CTAs an SM.
//
// 224 threads: warps 0..3 softmax (TMEM lane t = key t, then dim t), warps 4 and 6 fetch K and V, warp 5 issues the
// products.
// TMEM: two S tiles of 3 * COLS columns and O of 4 * COLS, in strides of 32 or 64.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "paged_tiles.cuh"
#include "tcgen05.cuh"

namespace fcci {
namespace pg {

constexpr int kTcThreads = kCompute + 96;
constexpr int kTcD = 128, kTcKeys = 128;
constexpr float kWeightTop = 13.f, kWeightMost = 15.75f;  // log2 of the largest weight after a move of m, and at most
constexpr float kNoMax = -1e30f;                         // m before a row has seen a key

template <int NB>
struct TcCfg {
    using TL = Tile<kTcKeys, kTcD>;
    static constexpr int COLS = 8 * NB;
    static constexpr int N = NB == 1 ? 32 : 48;         // rows of query parts: 3 * COLS, a multiple of 16
    static constexpr int NO = 4 * COLS;                 // rows of weight parts
    static constexpr int STRIDE = NB == 1 ? 32 : 64;    // TMEM columns of one accumulator
    static constexpr int TMEM = NB == 1 ? 128 : 256;
    static constexpr int QB = N * 128;                  // bytes of the query parts
    static constexpr int PW = NO;                       // bytes of a key's weight parts (the swizzle's width)
    static constexpr int PB = kTcKeys * PW;             // bytes of a weight buffer
    // shared memory behind the stages
    static constexpr int kP = QB, kSmall = QB + 2 * PB;  // queries, two weight buffers, the rest
    static_assert(2 * PB >= COLS * (kTcD / 2) * 8, "angles of COLS tokens in the weight buffers");
    static size_t smem(int stages, int B) {
        return 1024 + (size_t)stages * 2 * TL::BYTES + kSmall + 64 * 8 /* cos, sin */ + 8 * COLS * 4 /* maxima, sums */ +
               COLS * 4 /* query scales */ + kMaxStages * 64 /* page scales */ + 256 /* barriers */ + 64 +
               Line<kTcKeys, COLS>::ints(B) * 4;
    }
};

struct Bars {  // mbarriers: fetched / freed stages; S written / read; P written / consumed; queries ready; row appended
    uint64_t full[kMaxStages], empty[kMaxStages], s_full[2], s_free[2], p_full[2], p_free[2], q_full, row_done, drain;
};
static_assert(sizeof(Bars) <= 256, "barrier area");

__device__ __forceinline__ float redux_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float of_query_parts(uint32_t a, uint32_t b, uint32_t c) {
    return fmaf(__uint_as_float(c), 1.f / 256.f, fmaf(__uint_as_float(b), 1.f / 16.f, __uint_as_float(a)));
}

__device__ __forceinline__ float of_weight_parts(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return fmaf(__uint_as_float(d), 1.f / 512.f,
                fmaf(__uint_as_float(c), 1.f / 64.f, fmaf(__uint_as_float(b), 1.f / 8.f, __uint_as_float(a))));
}

// Whether any of the computing threads says so (all of them take part).
__device__ __forceinline__ bool any_of_compute(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x), "n"(kBar), "n"(kCompute)
        : "memory");
    return r != 0;
}

template <int NB>
__global__ void __launch_bounds__(kTcThreads, 2) paged_split_tc_kernel(const __grid_constant__ CUtensorMap mk,
                                                                   const __grid_constant__ CUtensorMap mv,
                                                                   const __grid_constant__ CUtensorMap mk16,
                                                                   const __grid_constant__ CUtensorMap mv16,
                                                                   const __grid_constant__ TileParams tp,
                                                                   const __grid_constant__ Freqs f) {
    using C = TcCfg<NB>;
    using TL = typename C::TL;
    constexpr int D = kTcD, KEYS = kTcKeys, COLS = C::COLS;
    const Params& p = tp.p;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const int S = tp.stages, G = p.G;
    uint8_t* rest = sm + (size_t)S * 2 * TL::BYTES;
    uint8_t* q_sm = rest;             // [N rows][128 dims], 128-byte swizzle
    uint8_t* p_sm = rest + C::kP;     // two of [128 keys][PW], swizzled over PW bytes
    float2* cs = reinterpret_cast<float2*>(rest + C::kSmall);  // decode: cos and sin of position T
    float* mx_sm = reinterpret_cast<float*>(cs + 64);          // [4][COLS] maxima, then sums
    float* l_sm = mx_sm + 4 * COLS;
    float* qs_sm = l_sm + 4 * COLS;
    float* scale_sm = qs_sm + COLS;                            // [stage][K, V][8]
    Bars* bar = reinterpret_cast<Bars*>(scale_sm + kMaxStages * 16);
    int* misc = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bar) + 256);
    volatile int* abort_flag = misc;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 3);
    Line<KEYS, COLS> line(tp, misc + 16);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&bar->full[s], 4);  // the fetched bytes and the scales, of K and of V
            mbar_init(&bar->empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar->s_full[i], 1);
            mbar_init(&bar->s_free[i], kComputeWarps);
            mbar_init(&bar->p_full[i], kComputeWarps);
            mbar_init(&bar->p_free[i], 1);
        }
        mbar_init(&bar->q_full, kComputeWarps);
        mbar_init(&bar->row_done, kComputeWarps);
        mbar_init(&bar->drain, 1);
        misc[0] = 0;
        fence_mbar_init();
    }
    if (warp == 4 && lane == 0) {
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
        prefetch_tmap(&mk16);
        prefetch_tmap(&mv16);
    }
    if (warp == 5) {
        tc::tmem_alloc(tmem_slot, C::TMEM);
        tc::tmem_relinquish();
    }
    const uint64_t turn = tid < p.rot / 2 ? f.turn[tid] : 0;  // a launch constant: its cold read is over before the wait is
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (!tp.early) griddep_wait();
    griddep_launch_dependents();  // behind the wait (paged.cuh)
    At at = line.template build<kTcThreads>(reinterpret_cast<int*>(mx_sm));
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_o = tmem + 2 * C::STRIDE;
    const int ntiles = line.ntiles;
    auto fail = [&]() {
        *abort_flag = 1;
        set_error(p, FCCI_DEV_ERR_TIMEOUT);
    };
    auto wait = [&](uint64_t* b, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_wait_sparing(b, parity & 1u, abort_flag, kWaitLimitNs))) return true;
        if (!*abort_flag) fail();
        return false;
    };
    // the append of row T happens in the tile that holds it
    auto appends = [&](const At& x) { return tp.fused && x.T >= 0 && x.T / KEYS == x.j; };

    if (warp == 4 || warp == 6) {
        const bool is_v = warp == 6;
        fetch_tiles<TL, true, COLS>(line, at, is_v, is_v ? &mv : &mk, is_v ? &mv16 : &mk16, sm, bar->full, bar->empty, scale_sm,
                                    abort_flag);
    } else if (warp == 5) {
        // ============================================================ products, by one thread
        if (elect_one()) {
            auto wait1 = [&](uint64_t* b, uint32_t parity) {
                if (mbar_wait_sparing(b, parity & 1u, abort_flag, kWaitLimitNs)) return true;
                if (!*abort_flag) fail();
                return false;
            };
            constexpr uint32_t id_s = tc::idesc_e4m3_f32(128, C::N, 0, 0);
            constexpr uint32_t id_o = tc::idesc_e4m3_f32(128, C::NO, 1, 1, 1);
            const uint64_t qd = tc::smem_desc_sw128(smem_u32(q_sm), 16, 1024);
            const uint64_t kd0 = tc::smem_desc_sw128(smem_u32(sm), 16, 1024);
            const uint64_t vd0 = tc::smem_desc_sw128(smem_u32(sm) + TL::BYTES, TL::BYTES, 1024);
            const uint64_t pd0 = tc::smem_desc_sw<C::PW>(smem_u32(p_sm), C::PB, 8 * C::PW);
            int nrow = 0, nq = 0;
            bool begins_prev = false;  // tile it - 1 is its unit's first here
            // O += V^T P of tile i in stage st (begins: O = V^T P)
            auto issue_o = [&](int i, int st, bool begins) {
                if (!wait1(&bar->p_full[i & 1], i >> 1)) return false;
                tc::fence_after_sync();
                const uint64_t vd = vd0 + (uint64_t)(st * (2 * TL::BYTES >> 4)), pd = pd0 + (uint64_t)((i & 1) * (C::PB >> 4));
#pragma unroll
                for (int k = 0; k < KEYS / 32; ++k)  // 32 keys: 4 groups of 8 rows of V and of P
                    tc::mma_ss_f8(tmem_o, vd + (uint64_t)(k * 4096 >> 4), pd + (uint64_t)(k * 32 * C::PW >> 4), id_o, !begins || k > 0);
                tc::commit(&bar->p_free[i & 1]);
                tc::commit(&bar->empty[st]);
                return true;
            };
            bool ok = true;
            Ring ring(S);
            int st_prev = 0;  // stage of tile it - 1
            for (int it = 0; it < ntiles; ++it) {
                // S of this tile first, so that the softmax has it when it is through with the last one; but not
                // when the tile is still on its way (the last one's stage would come free late), and not
                // over a unit's end (the new queries come after the old O was read)
                const int st = ring.s;
                const bool begins = it == 0 || at.j == 0;
                const bool o_first = it > 0 && (begins || !mbar_test_wait(&bar->full[st], ring.round & 1u));
                if (o_first && !(ok = issue_o(it - 1, st_prev, begins_prev))) break;
                if (begins && !(ok = wait1(&bar->q_full, nq++))) break;
                if (!(ok = wait1(&bar->full[st], ring.round))) break;
                if (appends(at) && !(ok = wait1(&bar->row_done, nrow++))) break;
                if (it >= 2 && !(ok = wait1(&bar->s_free[it & 1], (it >> 1) - 1))) break;
                tc::fence_after_sync();
                const uint64_t kd = kd0 + (uint64_t)(st * (2 * TL::BYTES >> 4));
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
                    tc::mma_ss_f8(tmem + (it & 1) * C::STRIDE, kd + (uint64_t)(k * 32 >> 4), qd + (uint64_t)(k * 32 >> 4), id_s, k > 0);
                tc::commit(&bar->s_full[it & 1]);
                if (it > 0 && !o_first && !(ok = issue_o(it - 1, st_prev, begins_prev))) break;
                begins_prev = begins;
                st_prev = st;
                ring.next();
                line.step(at);
            }
            if (ok && ntiles > 0) issue_o(ntiles - 1, st_prev, begins_prev);
            // every product has completed before TMEM is released
            tc::commit(&bar->drain);
            volatile int never = 0;
            mbar_wait_sparing(&bar->drain, 0, &never, kDrainLimitNs);
        }
        __syncwarp();
    } else {
        // ============================================================ softmax
        // A wait that fails leaves garbage behind, never a barrier that some warps skip: the loop runs on, its
        // waits return at once, and the error word says so.
        if (tp.early) griddep_wait();  // before the queries, the new rows and everything that is written
        const uint32_t lane_row = (uint32_t)warp * 32;
        const int rot = p.rot, half = rot >> 1;
        const int box_log2 = min(p.page_log2, 7);
        float mm[COLS], l[COLS], qf[COLS];  // m - kWeightTop, sum, factor of a score
        bool fresh = true;
        int first_tile = 0;
        Ring ring(S);
        for (int it = 0; it < ntiles; ++it) {
            const int T = at.T, n = at.n, L = at.L;
            const int r0 = at.c * COLS, rows = min(COLS, n * G - r0);
            if (fresh) {
                first_tile = at.j;
                // ---- queries: warp w takes rows w, w + 4, ...; a lane 4 neighbouring dims
                const int64_t tok0 = p.cu_q ? p.cu_q[at.b] : at.b;
                const int d = 4 * lane;
                uint2 xr[COLS / 4], yr[COLS / 4];
#pragma unroll
                for (int k = 0; k < COLS / 4; ++k) {
                    const int c = 4 * k + warp, i = (r0 + c) / G;
                    xr[k] = yr[k] = make_uint2(0, 0);
                    if (c < rows) {
                        const __half* q = p.q + (tok0 + i) * p.q_st + (at.h * G + (r0 + c) - i * G) * p.q_sh;
                        xr[k] = *reinterpret_cast<const uint2*>(q + d);
                        if (d < rot) yr[k] = *reinterpret_cast<const uint2*>(q + (d < half ? d + half : d - half));
                    }
                }
                // ---- angles, while the loads are under way: of position T, or of each of the unit's tokens (the weight
                // buffers hold them: the last product that read those has completed)
                const int i0 = r0 / G;
                const float2* angles = cs;
                if (rot > 0) {
                    if (!p.cu_q) {
                        if (tid < half) cs[tid] = rope_cs(turn, max(T, 0));
                    } else {
                        float2* table = reinterpret_cast<float2*>(p_sm);
                        const int ntok = (r0 + rows - 1) / G - i0 + 1;
                        for (int x = warp; x < ntok; x += kComputeWarps)
                            for (int k = lane; k < half; k += 32) table[x * half + k] = rope_cs(f.turn[k], T + i0 + x);
                        angles = table;
                    }
                    named_bar_sync(kBar, kCompute);
                }
#pragma unroll
                for (int k = 0; k < COLS / 4; ++k) {
                    const int c = 4 * k + warp, i = (r0 + c) / G;
                    const __half* a = reinterpret_cast<const __half*>(&xr[k]);
                    const __half* y = reinterpret_cast<const __half*>(&yr[k]);
                    float x[4], amax = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = __half2float(a[e]);
                        if (d < rot && c < rows) {
                            const int t = (d < half ? d : d - half) + e;
                            x[e] = rotated(x[e], __half2float(y[e]), angles[(i - i0) * half + t], d < half);
                        }
                        amax = fmaxf(amax, fabsf(x[e]));
                    }
                    if (p.q_rot && at.j == 0 && c < rows && T >= 0)
                        *reinterpret_cast<uint2*>(p.q_rot + ((tok0 + i) * p.Hq + at.h * G + (r0 + c) - i * G) * D + d) =
                            make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
                    const float largest = redux_max(amax);
                    const int e = exponent_448(largest, -100, 100);
                    const float up = exp2_int(-e);
                    if (lane == 0) qs_sm[c] = largest < INFINITY ? exp2_int(e) * p.scale_log2 : NAN;  // codes would saturate
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] *= up;
#pragma unroll
                    for (int part = 0; part < 3; ++part) {
                        const uint32_t lo = e4m3x2(x[0], x[1]), hi = e4m3x2(x[2], x[3]);
                        const int r = part * COLS + c;
                        *reinterpret_cast<uint32_t*>(q_sm + r * 128 + ((lane >> 2) ^ (r & 7)) * 16 + (d & 15)) = lo | (hi << 16);
                        const uint32_t bl = half2_of_e4m3x2(lo), bh = half2_of_e4m3x2(hi);
                        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&bl));
                        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&bh));
                        x[0] = (x[0] - u.x) * 16.f, x[1] = (x[1] - u.y) * 16.f;
                        x[2] = (x[2] - v.x) * 16.f, x[3] = (x[3] - v.y) * 16.f;
                    }
                }
                fence_proxy_async_smem();
                tc::fence_before_sync();  // O of the unit before was read
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->q_full);
                named_bar_sync(kBar, kCompute);  // the scales of the query rows
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    mm[c] = kNoMax;
                    l[c] = 0.f;
                    qf[c] = qs_sm[c];
                }
            }
            const int s = ring.s;
            uint8_t* kt = sm + (size_t)s * 2 * TL::BYTES;
            float* scales = scale_sm + s * 16;
            const bool ready = wait(&bar->full[s], ring.round);
            if (appends(at)) {
                // ---- warp 0 the key, warp 1 the value, before the tile's first product
                const int bx = (T & (KEYS - 1)) >> box_log2;
                if (ready && warp < 2 && scales[bx] >= 0.f)
                    append_in_tile<TL, D, true>(p, at.b, at.h, T, warp == 1, cs, kt + (warp ? TL::BYTES : 0), scales + 8 * warp + bx);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->row_done);
                named_bar_sync(kBar, kCompute);  // the scales that it changed
            }
            // ---- this thread's key: its scales, whether it is there; values that are not are zeroed, since 0 * NaN
            const int t = at.j * KEYS + tid, bx = tid >> box_log2;
            const float ks = scales[bx], vs = scales[8 + bx];
            const bool live = t < L && ks >= 0.f;
            if (!live) {
                const uint32_t v32 = smem_u32(kt + TL::BYTES);
#pragma unroll
                for (int ch = 0; ch < 8; ++ch)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(TL::cell(v32, tid, ch)), "r"(0) : "memory");
            }
            // (values of 448 * 2^-60 are 0 in the result; without that bound a zeroed cache's scales of 2^-127 make the sum infinite)
            const int ev = max(-60, min(126, (int)(__float_as_uint(vs) >> 23) - 127));
            const float lv = (float)ev;
            const float inv_vs = live ? exp2_int(-ev) : 0.f;
            // ---- scores of this key, in the log2 domain, with V's exponent
            wait(&bar->s_full[it & 1], it >> 1);
            tc::fence_after_sync();
            float x[COLS];
            {
                uint32_t a[C::N];
                tc::ld32(tc::taddr(tmem, lane_row, (it & 1) * C::STRIDE), *reinterpret_cast<uint32_t(*)[32]>(a));
                if constexpr (C::N == 48) tc::ld16(tc::taddr(tmem, lane_row, (it & 1) * C::STRIDE + 32), *reinterpret_cast<uint32_t(*)[16]>(a + 32));
                tc::wait_ld();
                tc::fence_before_sync();
                if (lane == 0) mbar_arrive(&bar->s_free[it & 1]);
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    const float sum = of_query_parts(a[c], a[COLS + c], a[2 * COLS + c]);
                    x[c] = fmaf(sum * ks, qf[c], lv);
                }
            }
            if (!live) {
#pragma unroll
                for (int c = 0; c < COLS; ++c) x[c] = -INFINITY;
            }
            if (p.cu_q && (at.j + 1) * KEYS > T) {  // a row sees the keys up to its own position
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if (t > T + (r0 + c) / G) x[c] = -INFINITY;
            }
            // ---- move m when a weight would leave e4m3's range
            float most = x[0] - mm[0];
#pragma unroll
            for (int c = 1; c < COLS; ++c) most = fmaxf(most, x[c] - mm[c]);
            const bool over = most > kWeightMost;
            if (any_of_compute(over)) {
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    const float top = redux_max(x[c]);
                    if (lane == 0) mx_sm[warp * COLS + c] = top;
                }
                named_bar_sync(kBar, kCompute);
                float alpha[COLS];
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    const float top = fmaxf(fmaxf(mx_sm[c], mx_sm[COLS + c]), fmaxf(mx_sm[2 * COLS + c], mx_sm[3 * COLS + c]));
                    alpha[c] = 1.f;
                    if (top - mm[c] > kWeightMost) {
                        alpha[c] = ex2(mm[c] - (top - kWeightTop));
                        mm[c] = top - kWeightTop;
                        l[c] *= alpha[c];
                    }
                }
                if (!fresh) {
                    // O's rows of this thread: the product before must have completed
                    wait(&bar->p_free[(it - 1) & 1], (it - 1) >> 1);
                    tc::fence_after_sync();
#pragma unroll
                    for (int part = 0; part < 4; ++part)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            uint32_t o[8];
                            const uint32_t a = tc::taddr(tmem_o, lane_row, part * COLS + 8 * nb);
                            tc::ld8(a, o);
                            tc::wait_ld();
#pragma unroll
                            for (int c = 0; c < 8; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha[8 * nb + c]);
                            tc::st8(a, o);
                        }
                    tc::wait_st();
                }
            }
            fresh = false;
            // ---- weights, their sum, and their parts (of the weight in fp16): bytes part * COLS + c of this key
            uint32_t w[COLS];
#pragma unroll
            for (int c = 0; c < COLS; c += 4) {
                float u[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    u[k] = ex2(x[c + k] - mm[c + k]);
                    l[c + k] = fmaf(u[k], inv_vs, l[c + k]);
                }
                uint32_t h0 = pack_half2(u[0], u[1]), h1 = pack_half2(u[2], u[3]);
#pragma unroll
                for (int part = 0; part < 4; ++part) {
                    w[(part * COLS + c) / 4] = e5m2x4_of_half4(h0, h1);
                    if (part < 3) h0 = half2_rest8(h0), h1 = half2_rest8(h1);
                }
            }
            if (it >= 2) wait(&bar->p_free[it & 1], (it >> 1) - 1);
            {
                // 16-byte chunk ch of key t lies at ch ^ (t >> 2 & 1) of 32 bytes, ch ^ (t >> 1 & 3) of 64
                const uint32_t row = smem_u32(p_sm + (it & 1) * C::PB) + tid * C::PW;
                const int sw = NB == 1 ? (tid >> 2) & 1 : (tid >> 1) & 3;
#pragma unroll
                for (int ch = 0; ch < 2 * NB; ++ch)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + (ch ^ sw) * 16), "r"(w[4 * ch]),
                                 "r"(w[4 * ch + 1]), "r"(w[4 * ch + 2]), "r"(w[4 * ch + 3]) : "memory");
            }
            fence_proxy_async_smem();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->p_full[it & 1]);

            if (at.j == at.tiles - 1 || it == ntiles - 1) {
                // ---- the unit's (or its part's) end: sums over the keys, then O, of which thread t has dim t
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    float v = l[c];
#pragma unroll
                    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    if (lane == 0) l_sm[warp * COLS + c] = v;
                }
                named_bar_sync(kBar, kCompute);
                const int2 ctas = line.ctas_of(at);
                const bool whole = ctas.x == ctas.y;
                const size_t part = part_slot(blockIdx.x, first_tile == 0);
                wait(&bar->p_free[it & 1], it >> 1);
                tc::fence_after_sync();
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    uint32_t a[4][8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) tc::ld8(tc::taddr(tmem_o, lane_row, i * COLS + 8 * nb), a[i]);
                    tc::wait_ld();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int c = 8 * nb + k;
                        if (c >= rows) continue;
                        const float sum = (l_sm[c] + l_sm[COLS + c]) + (l_sm[2 * COLS + c] + l_sm[3 * COLS + c]);
                        const float o = of_weight_parts(a[0][k], a[1][k], a[2][k], a[3][k]);
                        const float y = sum == 0.f ? 0.f : o / sum;  // no key; a NaN stays one
                        if (whole) {
                            out_row(p, at, r0, c)[tid] = __float2half_rn(y);
                        } else {
                            tp.part_o[(part * kMaxCols + c) * D + tid] = y;
                            if (tid == 0) tp.part_lse[part * kMaxCols + c] = sum > 0.f ? mm[c] + __log2f(sum) : -INFINITY;
                        }
                    }
                }
                if (!whole) join_parts<D>(tp, at, r0, rows, ctas.x, ctas.y, misc + 1);
                fresh = true;
            }
            line.step(at);
            ring.next();
        }
    }
    // ---- teardown
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 5) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, C::TMEM);
    }
    if (line.N > 0) advance_lengths(p, misc + 2);  // no place on the line: no new token, or nothing is served
}

template <int NB>
static int launch_tc(TileParams& tp, const Freqs& f, const Params* rows, int sms, int dev, cudaStream_t st) {
    using C = TcCfg<NB>;
    static std::once_flag once[128];
    static cudaError_t attr[128];
    if (dev < 0 || dev >= 128) return set_status(FCCI_EINVAL, "device index");
    std::call_once(once[dev], [&]() {
        attr[dev] = cudaFuncSetAttribute(paged_split_tc_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    });
    if (attr[dev] != cudaSuccess) return set_cuda_status(attr[dev]);
    int stages = 0, per_sm = 0;
    for (int ctas = kMaxCtasPerSm; ctas >= 1 && !stages; --ctas)
        for (int s = kMaxStages; s >= 2 && !stages; --s)
            if (C::smem(s, tp.p.B) <= (size_t)(228 * 1024 / ctas - 1024)) stages = s, per_sm = ctas;
    if (!stages) return set_status(FCCI_EUNSUPPORTED, "paged attention: batch too large for shared memory");
    tp.stages = stages;
    CUtensorMap m[4];
    int rc = encode_pages<typename C::TL, true>(tp.p, m);
    if (!rc) rc = append_before(rows, f, true, st);
    if (rc) return rc;
    return launch_pdl(paged_split_tc_kernel<NB>, dim3(sms * per_sm), dim3(kTcThreads), C::smem(stages, tp.p.B), st, m[0], m[1],
                      m[2], m[3], tp, f);
}

int launch_split_tc(TileParams& tp, const Freqs& f, const Params* rows, int sms, int dev, cudaStream_t st) {
    return tp.p.cu_q || tp.p.G <= 8 ? launch_tc<1>(tp, f, rows, sms, dev, st) : launch_tc<2>(tp, f, rows, sms, dev, st);
}

}  // namespace pg
}  // namespace fcci
