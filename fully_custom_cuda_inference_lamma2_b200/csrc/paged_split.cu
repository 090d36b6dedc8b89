// Split-KV attention over the paged cache: one new token per sequence (decode, with its append
// fused in), or a few of them (a short chunk whose rows an append has written already).
//
// Work: paged_tiles.cuh.
//
// Inside a CTA warps 4 and 5 fetch and warps 0..3 compute. A stage holds the K and the V tile, in
// rows of 128 bytes (64 for e4m3 with head_dim 64) in the tensor-map swizzle; the pages of a tile
// are fetched side by side, one lane and one box each, the page that ends a sequence in boxes
// of 16 rows. The page table is read one tile ahead and the scales arrive behind the tile
// that they belong to, so neither latency is on the path. Warp w owns keys [16 MT w, 16 MT (w+1)):
//   S^T = K Q^T      A = 16 keys, B = 8 query rows (mma m16n8k16, fp32 sums)
//   O^T += V^T P^T   A = 16 dims, B = P^T by movmatrix
// e4m3 codes become fp16 in registers, exactly, and the power-of-two scales go onto S and onto
// the product of each 16 keys, in fp32, so no scale can leave fp16's range. The queries are
// rotated here in fp32 and split in two fp16 parts (hi + lo): one rounding of them to fp16 would
// be the largest error of the whole step (3.6e-4 instead of 2.4e-4 of the result, 2.1e-4 of it its own rounding).
// P is rounded to fp16 (relative 2^-11), times 2^14, so that fp16's least numbers are 2^-38 of the largest weight: with the
// largest at 1 the keys below 2^-25 of it were lost, a quarter of what 16384 keys of 2^-26 beside one share.
//
// Measured: fp16 pages, 17 sequences of 1 to 5000 keys, 8 kv heads, group 3: 40 us (4.7 TB/s).
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "paged_tiles.cuh"

namespace fcci {
namespace pg {

constexpr int kThreads = kCompute + 64;
constexpr float kSplitTop = 14.f;  // log2 of the weight of the largest score

template <int D, int NB, bool E4M3>
struct Cfg {
    static constexpr int ROWB = E4M3 ? D : 2 * D;             // bytes of a row
    // keys of a tile; an e4m3 page always lies in one tile (page * D <= 16384), because an append
    // that grows its scale rewrites the page's rows where the tile holds them
    static constexpr int KEYS = ROWB <= 128 && (E4M3 || NB == 1) ? 128 : 64;
    static constexpr int MT = KEYS / 64;                      // 16-key groups of a warp
    using TL = Tile<KEYS, ROWB>;
    static constexpr int TILE = TL::BYTES;
    static constexpr int COLS = 8 * NB;
    static constexpr int RP = D + 4;                          // fp32 pitch of the joining rows
    static constexpr int QP = D + 16;                         // fp16 pitch of the query rows
    // query fragments in registers where they fit beside two CTAs' accumulators, else in shared memory
    static constexpr bool QREG = NB == 1 && D <= 128;
    static constexpr int RED = 2 * COLS * RP * 4;             // bytes; with QREG the query rows pass through it
    static constexpr int QB = QREG ? 0 : 2 * COLS * QP * 2;   // bytes of their own buffer
    static_assert(!QREG || 2 * COLS * QP * 2 <= RED, "queries in the joining buffer");
    static size_t smem(int stages, int B, int rope_rows, int rot) {
        return 1024 + (size_t)stages * 2 * TILE + RED + QB + (size_t)rope_rows * (rot / 2) * 8 + 2 * kComputeWarps * COLS * 4 +
               kMaxStages * (2 * 8 * 4 + 16) + 64 + (4 * (size_t)B + 2) * 4;
    }
};

template <int D, int NB, bool E4M3>
__global__ void __launch_bounds__(kThreads, 2) paged_split_kernel(const __grid_constant__ CUtensorMap mk,
                                                            const __grid_constant__ CUtensorMap mv,
                                                            const __grid_constant__ CUtensorMap mk16,
                                                            const __grid_constant__ CUtensorMap mv16,
                                                            const __grid_constant__ TileParams sp,
                                                            const __grid_constant__ Freqs f) {
    using C = Cfg<D, NB, E4M3>;
    using TL = typename C::TL;
    constexpr int KEYS = C::KEYS, MT = C::MT, COLS = C::COLS, RP = C::RP, QP = C::QP;
    constexpr int KSTEPS = D / 16;
    const Params& p = sp.p;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const int S = sp.stages, B = p.B, G = p.G;
    uint8_t* tiles_sm = sm;
    float* red = reinterpret_cast<float*>(sm + (size_t)S * 2 * C::TILE);
    __half* q_hi = reinterpret_cast<__half*>(C::QREG ? red : red + C::RED / 4);
    __half* q_lo = q_hi + COLS * QP;
    float* red_ml = red + (C::RED + C::QB) / 4;              // [4 warps][COLS][2]
    uint64_t* full = reinterpret_cast<uint64_t*>(red_ml + 2 * kComputeWarps * COLS);
    uint64_t* empty = full + kMaxStages;
    float* scale_sm = reinterpret_cast<float*>(empty + kMaxStages);  // [stage][K, V][8 page boxes]; K -1: no such page
    int* misc = reinterpret_cast<int*>(scale_sm + kMaxStages * 16);
    volatile int* abort_flag = misc;
    Line<KEYS, COLS> line(sp, misc + 16);
    float2* cs = reinterpret_cast<float2*>(misc + 16 + 4 * B + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 4);  // the fetched bytes and the scales, of K and of V
            mbar_init(&empty[s], kComputeWarps);
        }
        misc[0] = 0;
        fence_mbar_init();
    }
    if (tid == kCompute) {
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
        prefetch_tmap(&mk16);
        prefetch_tmap(&mv16);
    }
    __syncthreads();
    if (!sp.early) griddep_wait();
    griddep_launch_dependents();  // behind the wait (paged.cuh)

    At at = line.template build<kThreads>(reinterpret_cast<int*>(red_ml));
    const int ntiles = line.ntiles;
    const int box = min(p.page, KEYS);  // rows of one page in a tile
    if (warp >= kComputeWarps) {
        const bool is_v = warp > kComputeWarps;
        fetch_tiles<TL, E4M3, COLS>(line, at, is_v, is_v ? &mv : &mk, is_v ? &mv16 : &mk16, tiles_sm, full, empty, scale_sm, abort_flag);
    } else {
        // ============================================================ computing warps
        if (sp.early) griddep_wait();  // before the queries, the new rows and everything that is written
        const int w = warp, g = lane >> 2, t4 = lane & 3;
        const int rot = p.rot, half = rot >> 1;
        float m[NB][2], l[NB][2];
        float2 acc[NB][KSTEPS][2];
        uint32_t qreg[2][NB][C::QREG ? KSTEPS : 1][2] = {};  // hi, lo
        int lim[NB][2];
        int cs_b = -1, cs_c = -1;
        bool fresh = true;
        int first_tile = at.j;
        auto cell = [](uint32_t tile, int r, int ch) { return TL::cell(tile, r, ch); };
        // B fragment of k step kk: e4m3 lanes hold 4 neighbouring dims of a chunk, and k follows them
        auto q_fragment = [&](int part, int nb, int kk, uint32_t(&r)[2]) {
            const __half* q = (part ? q_lo : q_hi) + (nb * 8 + g) * QP + 16 * kk + (E4M3 ? 4 * t4 : 2 * t4);
            if constexpr (E4M3) {
                const uint2 v = *reinterpret_cast<const uint2*>(q);
                r[0] = v.x, r[1] = v.y;
            } else {
                r[0] = *reinterpret_cast<const uint32_t*>(q);
                r[1] = *reinterpret_cast<const uint32_t*>(q + 8);
            }
        };

        auto q_of = [&](int part, int nb, int kk, uint32_t(&r)[2]) {
            if constexpr (C::QREG) r[0] = qreg[part][nb][kk][0], r[1] = qreg[part][nb][kk][1];
            else q_fragment(part, nb, kk, r);
        };

        Ring ring(S);
        for (int it = 0; it < ntiles; ++it) {
            const int T = at.T, n = at.n, L = at.L;
            const int r0 = at.c * COLS, rows = min(COLS, n * G - r0);  // query rows of this unit
            if (fresh) {
                fresh = false;
                first_tile = at.j;
                const int i0 = r0 / G;  // first token of the unit
                if (rot > 0 && (cs_b != at.b || cs_c != at.c)) {
                    const int ntok = (r0 + rows - 1) / G - i0 + 1;
                    for (int x = tid; x < ntok * half; x += kCompute)
                        cs[x] = rope_cs(f.turn[x % half], max(T, 0) + i0 + x / half);
                    cs_b = at.b, cs_c = at.c;
                    named_bar_sync(kBar, kCompute);
                }
                // rotated queries, fp32, as hi + lo
                const int64_t tok0 = p.cu_q ? p.cu_q[at.b] : at.b;
#pragma unroll 4
                for (int e = tid * 2; e < COLS * D; e += 2 * kCompute) {
                    const int c = e / D, d = e - c * D;
                    float x0 = 0.f, x1 = 0.f;
                    if (c < rows) {
                        const int i = (r0 + c) / G, hq = at.h * G + (r0 + c) - i * G;
                        const __half* q = p.q + (tok0 + i) * p.q_st + hq * p.q_sh;
                        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(q + d));
                        x0 = x.x, x1 = x.y;
                        if (d < rot) {
                            const bool lowhalf = d < half;
                            const int k = lowhalf ? d : d - half;
                            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(q + (lowhalf ? d + half : k)));
                            x0 = rotated(x0, y.x, cs[(i - i0) * half + k], lowhalf);
                            x1 = rotated(x1, y.y, cs[(i - i0) * half + k + 1], lowhalf);
                        }
                        if (p.q_rot && at.j == 0 && T >= 0)
                            *reinterpret_cast<uint32_t*>(p.q_rot + ((tok0 + i) * p.Hq + hq) * D + d) = pack_half2(x0, x1);
                    }
                    // (a rotation of the largest fp16 values passes fp16's range: the low part takes the rest)
                    const __half2 hi = __floats2half2_rn(fmaxf(-65504.f, fminf(x0, 65504.f)), fmaxf(-65504.f, fminf(x1, 65504.f)));
                    const float2 back = __half22float2(hi);
                    *reinterpret_cast<__half2*>(q_hi + c * QP + d) = hi;
                    *reinterpret_cast<__half2*>(q_lo + c * QP + d) = __floats2half2_rn(x0 - back.x, x1 - back.y);
                }
                named_bar_sync(kBar, kCompute);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int kk = 0; kk < KSTEPS; ++kk) {
                        if constexpr (C::QREG) {
                            q_fragment(0, nb, kk, qreg[0][nb][kk]);
                            q_fragment(1, nb, kk, qreg[1][nb][kk]);
                        }
                        acc[nb][kk][0] = acc[nb][kk][1] = make_float2(0.f, 0.f);
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        m[nb][c] = -INFINITY;
                        l[nb][c] = 0.f;
                        const int col = nb * 8 + 2 * t4 + c;
                        // keys a row sees: all of them, or up to its own position
                        lim[nb][c] = col >= rows ? 0 : p.cu_q ? T + (r0 + col) / G + 1 : L;
                    }
                }
                // the query rows may lie in the joining buffer, which a faster warp writes next
                if (C::QREG) named_bar_sync(kBar, kCompute);
            }

            const int s = ring.s;
            const bool ready =
                __all_sync(0xffffffffu, mbar_wait_sparing(&full[s], ring.round & 1u, abort_flag, kWaitLimitNs));
            if (!ready && !*abort_flag) {
                *abort_flag = 1;
                set_error(p, FCCI_DEV_ERR_TIMEOUT);
            }
            const uint32_t kt = smem_u32(tiles_sm + (size_t)s * 2 * C::TILE), vt = kt + C::TILE;
            float* ksc = scale_sm + s * 16;
            bool wrote = false;
            if (sp.fused && T >= 0 && T / KEYS == at.j) {
                // ---- append: warp 0 the key, warp 1 the value, into the tile and the page
                named_bar_sync(kBar, kCompute);
                const int bx = (T % KEYS) / box;
                if (ready && w < 2 && ksc[bx] >= 0.f)
                    append_in_tile<TL, D, E4M3>(p, at.b, at.h, T, w == 1, cs, tiles_sm + (size_t)s * 2 * C::TILE + (w ? C::TILE : 0),
                                                ksc + 8 * w + bx);
                wrote = true;
                named_bar_sync(kBar, kCompute);
            }
            const int key0 = KEYS * at.j + 16 * MT * w;
            if (ready && key0 < L) {
                // ---- rows behind the last key: zero their values, so that 0 * NaN cannot be
                const int nv = L - key0;
                if (nv < 16 * MT) {
                    const int end = min((nv + 15) & ~15, 16 * MT);
                    for (int i = lane; i < (end - nv) * (C::ROWB / 16); i += 32) {
                        const int r = 16 * MT * w + nv + i / (C::ROWB / 16);
                        const uint32_t a = cell(vt, r, i % (C::ROWB / 16));
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0) : "memory");
                    }
                    wrote = true;
                    __syncwarp();
                }
                // ---- S^T, 16 keys at a time
                const int lrow = 16 * MT * w + (lane & 7) + (((lane >> 3) & 1) << 3);
                float x[MT][NB][4];
                bool live[MT];
                float vs[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int bx = (16 * (MT * w + mt)) / box;
                    const float ks = ksc[bx];
                    vs[mt] = ksc[8 + bx];
                    live[mt] = ks >= 0.f && key0 + 16 * mt < L;
                    float s0[NB][4], s1[NB][4];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s0[nb][c] = s1[nb][c] = 0.f;
                    if (live[mt]) {
                        if constexpr (E4M3) {
#pragma unroll
                            for (int kk = 0; kk < KSTEPS; kk += 2) {
                                uint32_t r0_, r1_, r2_, r3_;
                                ldsm_x4(cell(kt, lrow + 16 * mt, kk + (lane >> 4)), r0_, r1_, r2_, r3_);
                                const uint32_t a0 = half2_of_e4m3x2(r0_ & 0xffffu), a2 = half2_of_e4m3x2(r0_ >> 16);
                                const uint32_t a1 = half2_of_e4m3x2(r1_ & 0xffffu), a3 = half2_of_e4m3x2(r1_ >> 16);
                                const uint32_t b0 = half2_of_e4m3x2(r2_ & 0xffffu), b2 = half2_of_e4m3x2(r2_ >> 16);
                                const uint32_t b1 = half2_of_e4m3x2(r3_ & 0xffffu), b3 = half2_of_e4m3x2(r3_ >> 16);
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                    for (int part = 0; part < 2; ++part) {
                                        uint32_t u[2], v[2];
                                        q_of(part, nb, kk, u);
                                        q_of(part, nb, kk + 1, v);
                                        mma_16816(s0[nb], a0, a1, a2, a3, u[0], u[1]);
                                        mma_16816(s1[nb], b0, b1, b2, b3, v[0], v[1]);
                                    }
                            }
                        } else {
#pragma unroll
                            for (int kk = 0; kk < KSTEPS; ++kk) {
                                uint32_t a0, a1, a2, a3;
                                ldsm_x4(cell(kt, lrow + 16 * mt, 2 * kk + (lane >> 4)), a0, a1, a2, a3);
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb) {
                                    uint32_t u[2], v[2];
                                    q_of(0, nb, kk, u);
                                    q_of(1, nb, kk, v);
                                    mma_16816(s0[nb], a0, a1, a2, a3, u[0], u[1]);
                                    mma_16816(s1[nb], a0, a1, a2, a3, v[0], v[1]);
                                }
                            }
                        }
                    }
                    const int k0 = key0 + 16 * mt + g;
                    const float f2 = E4M3 ? ks * p.scale_log2 : p.scale_log2;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            x[mt][nb][c] = live[mt] && k0 + 8 * (c >> 1) < lim[nb][c & 1] ? (s0[nb][c] + s1[nb][c]) * f2 : -INFINITY;
                }
                // ---- running maximum and sum of each query row (log2 domain)
                uint32_t pb[MT][NB][2];
                float2 alpha[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float al[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = fmaxf(x[0][nb][c], x[0][nb][c + 2]);
#pragma unroll
                        for (int mt = 1; mt < MT; ++mt) mx = fmaxf(mx, fmaxf(x[mt][nb][c], x[mt][nb][c + 2]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float mn = fmaxf(m[nb][c], mx);
                        const float mu = mn == -INFINITY ? 0.f : mn;  // a row that has seen no key yet
                        al[c] = ex2(m[nb][c] - mu);
                        m[nb][c] = mn;
                        const float zero = mu - kSplitTop;  // the score of weight 1
                        float sum = 0.f;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            x[mt][nb][c] = ex2(x[mt][nb][c] - zero);
                            x[mt][nb][c + 2] = ex2(x[mt][nb][c + 2] - zero);
                            sum += x[mt][nb][c] + x[mt][nb][c + 2];
                        }
                        l[nb][c] = l[nb][c] * al[c] + sum;
                    }
                    alpha[nb] = make_float2(al[0], al[1]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        pb[mt][nb][0] = movmatrix_t(pack_half2(x[mt][nb][0], x[mt][nb][1]));
                        pb[mt][nb][1] = movmatrix_t(pack_half2(x[mt][nb][2], x[mt][nb][3]));
                    }
                }
                // ---- O^T = alpha O^T + sum over 16-key groups of scale * V^T P^T
                if constexpr (E4M3) {
#pragma unroll
                    for (int mb = 0; mb < KSTEPS; ++mb)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            acc[nb][mb][0] = __fmul2_rn(acc[nb][mb][0], alpha[nb]);
                            acc[nb][mb][1] = __fmul2_rn(acc[nb][mb][1], alpha[nb]);
                        }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        if (!live[mt]) continue;
                        const float2 v2 = make_float2(vs[mt], vs[mt]);
#pragma unroll
                        for (int mb = 0; mb < KSTEPS; mb += 2) {
                            uint32_t r[4];
                            ldsm_x4_t(cell(vt, lrow + 16 * mt, mb + (lane >> 4)), r[0], r[1], r[2], r[3]);
                            uint32_t a[8];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t y = __byte_perm(r[i], 0, 0x3120);  // (even dim: 2 keys, odd dim: 2 keys)
                                a[2 * i] = half2_of_e4m3x2(y & 0xffffu);
                                a[2 * i + 1] = half2_of_e4m3x2(y >> 16);
                            }
#pragma unroll
                            for (int k = 0; k < 2; ++k)
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb) {
                                    float o[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma_16816(o, a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3], pb[mt][nb][0], pb[mt][nb][1]);
                                    acc[nb][mb + k][0] = __ffma2_rn(make_float2(o[0], o[1]), v2, acc[nb][mb + k][0]);
                                    acc[nb][mb + k][1] = __ffma2_rn(make_float2(o[2], o[3]), v2, acc[nb][mb + k][1]);
                                }
                        }
                    }
                } else {
                    const int vrow = 16 * MT * w + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                    for (int mb = 0; mb < KSTEPS; ++mb) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            acc[nb][mb][0] = __fmul2_rn(acc[nb][mb][0], alpha[nb]);
                            acc[nb][mb][1] = __fmul2_rn(acc[nb][mb][1], alpha[nb]);
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            if (!live[mt]) continue;
                            uint32_t a0, a1, a2, a3;
                            ldsm_x4_t(cell(vt, vrow + 16 * mt, 2 * mb + ((lane >> 3) & 1)), a0, a1, a2, a3);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                float o[4] = {acc[nb][mb][0].x, acc[nb][mb][0].y, acc[nb][mb][1].x, acc[nb][mb][1].y};
                                mma_16816(o, a0, a1, a2, a3, pb[mt][nb][0], pb[mt][nb][1]);
                                acc[nb][mb][0] = make_float2(o[0], o[1]);
                                acc[nb][mb][1] = make_float2(o[2], o[3]);
                            }
                        }
                    }
                }
            }
            if (wrote) fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);

            if (at.j == at.tiles - 1 || it == ntiles - 1) {
                // ---- the unit's (or its part's) end: join the four warps, halving them twice
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float v = l[nb][c];
                        v += __shfl_xor_sync(0xffffffffu, v, 4);
                        v += __shfl_xor_sync(0xffffffffu, v, 8);
                        v += __shfl_xor_sync(0xffffffffu, v, 16);
                        l[nb][c] = v;
                    }
                // dims of accumulator element (mb, k): e4m3 16 mb + 2 g + k, fp16 16 mb + g + 8 k
                auto dim = [&](int mb, int k) { return 16 * mb + (E4M3 ? 2 * g + k : g + 8 * k); };
#pragma unroll
                for (int far = 2; far >= 1; far >>= 1) {
                    if (w >= far && w < 2 * far) {
                        float* dst = red + (w - far) * COLS * RP;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const int c = nb * 8 + 2 * t4;
#pragma unroll
                            for (int mb = 0; mb < KSTEPS; ++mb)
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    dst[c * RP + dim(mb, k)] = acc[nb][mb][k].x;
                                    dst[(c + 1) * RP + dim(mb, k)] = acc[nb][mb][k].y;
                                }
                            if (g == 0)
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    red_ml[((w - far) * COLS + c + k) * 2] = m[nb][k];
                                    red_ml[((w - far) * COLS + c + k) * 2 + 1] = l[nb][k];
                                }
                        }
                    }
                    named_bar_sync(kBar, kCompute);
                    if (w < far) {
                        const float* src = red + w * COLS * RP;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const int c = nb * 8 + 2 * t4;
                            float a[2], o[2];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const float om = red_ml[(w * COLS + c + k) * 2], ol = red_ml[(w * COLS + c + k) * 2 + 1];
                                const float mn = fmaxf(m[nb][k], om), mu = mn == -INFINITY ? 0.f : mn;
                                a[k] = ex2(m[nb][k] - mu);
                                o[k] = ex2(om - mu);
                                l[nb][k] = l[nb][k] * a[k] + ol * o[k];
                                m[nb][k] = mn;
                            }
#pragma unroll
                            for (int mb = 0; mb < KSTEPS; ++mb)
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    acc[nb][mb][k].x = acc[nb][mb][k].x * a[0] + src[c * RP + dim(mb, k)] * o[0];
                                    acc[nb][mb][k].y = acc[nb][mb][k].y * a[1] + src[(c + 1) * RP + dim(mb, k)] * o[1];
                                }
                        }
                    }
                    if (far == 2) named_bar_sync(kBar, kCompute);
                }
                // warp 0 holds the joined state: the result, or this CTA's part of it
                const int2 ctas = line.ctas_of(at);
                const bool whole = ctas.x == ctas.y;
                if (w == 0) {
                    const size_t part = part_slot(blockIdx.x, first_tile == 0);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int c = nb * 8 + 2 * t4 + k;
                            if (c >= rows) continue;
                            const float inv = l[nb][k] > 0.f ? 1.f / l[nb][k] : 0.f;
                            __half* o16 = out_row(p, at, r0, c);
                            float* o32 = sp.part_o + (part * kMaxCols + c) * D;
                            if (!whole && g == 0)
                                sp.part_lse[part * kMaxCols + c] = l[nb][k] > 0.f ? m[nb][k] - kSplitTop + __log2f(l[nb][k]) : -INFINITY;
#pragma unroll
                            for (int mb = 0; mb < KSTEPS; ++mb) {
                                const float y0 = (k ? acc[nb][mb][0].y : acc[nb][mb][0].x) * inv;
                                const float y1 = (k ? acc[nb][mb][1].y : acc[nb][mb][1].x) * inv;
                                if (whole) {
                                    if constexpr (E4M3) {
                                        *reinterpret_cast<uint32_t*>(o16 + dim(mb, 0)) = pack_half2(y0, y1);
                                    } else {
                                        o16[dim(mb, 0)] = __float2half_rn(y0);
                                        o16[dim(mb, 1)] = __float2half_rn(y1);
                                    }
                                } else {
                                    o32[dim(mb, 0)] = y0;
                                    o32[dim(mb, 1)] = y1;
                                }
                            }
                        }
                }
                if (!whole) join_parts<D>(sp, at, r0, rows, ctas.x, ctas.y, misc + 1);
                named_bar_sync(kBar, kCompute);  // the joining buffer becomes the next unit's queries
                fresh = true;
            }
            line.step(at);
            ring.next();
        }
    }
    if (line.N > 0) advance_lengths(p, misc + 2);  // no place on the line: no new token, or nothing is served
}

int append_before(const Params* rows, const Freqs& f, bool e4m3, cudaStream_t st) {
    return rows ? launch_append(*rows, f, e4m3, st) : FCCI_OK;
}

template <int D, int NB, bool E4M3>
static int launch_split_t(TileParams& sp, const Freqs& f, const Params* rows, int sms, int dev, cudaStream_t st) {
    using C = Cfg<D, NB, E4M3>;
    const Params& p = sp.p;
    static std::once_flag once[128];
    static cudaError_t attr[128];
    if (dev < 0 || dev >= 128) return set_status(FCCI_EINVAL, "device index");
    std::call_once(once[dev], [&]() {
        attr[dev] = cudaFuncSetAttribute(paged_split_kernel<D, NB, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    });
    if (attr[dev] != cudaSuccess) return set_cuda_status(attr[dev]);
    // tokens whose angles a unit needs at once
    const int rope_rows = p.cu_q ? (C::COLS + p.G - 1) / p.G + 1 : 1;
    int stages = 0, per_sm = 0;
    for (int ctas = kMaxCtasPerSm; ctas >= 1 && !stages; --ctas)
        for (int s = kMaxStages; s >= 2 && !stages; --s)
            if (C::smem(s, p.B, rope_rows, p.rot) <= (size_t)(228 * 1024 / ctas - 1024)) stages = s, per_sm = ctas;
    if (!stages) return set_status(FCCI_EUNSUPPORTED, "paged attention: batch too large for shared memory");
    sp.stages = stages;
    CUtensorMap m[4];
    int rc = encode_pages<typename C::TL, E4M3>(p, m);
    if (!rc) rc = append_before(rows, f, E4M3, st);
    if (rc) return rc;
    const size_t smem = C::smem(stages, p.B, rope_rows, p.rot);
    return launch_pdl(paged_split_kernel<D, NB, E4M3>, dim3(sms * per_sm), dim3(kThreads), smem, st, m[0], m[1], m[2], m[3], sp, f);
}

int launch_split(const Params& p, const Freqs& f, const Params* rows, bool e4m3, bool fused, bool early, uint8_t* ws,
                 const WsLayout& L, cudaStream_t st) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_status(cudaGetLastError());
    const int sms = device_sm_count(dev);
    TileParams sp;
    sp.p = p;
    sp.fused = fused;
    sp.early = early;
    sp.stages = 0;
    sp.cut_cnt = reinterpret_cast<uint32_t*>(ws + 256);
    sp.part_lse = reinterpret_cast<float*>(ws + L.part_lse);
    sp.part_o = reinterpret_cast<float*>(ws + L.part_o);
    if (sms * kMaxCtasPerSm > kMaxGrid) return set_status(FCCI_EUNSUPPORTED, "paged attention: too many SMs");
    // e4m3 pages of head_dim 128 go to the tensor memory kernel: 51 against 69 us at batch 32 x 4096 keys
    if (e4m3 && p.D == 128) return launch_split_tc(sp, f, rows, sms, dev, st);
    const int nb = (int64_t)p.max_q * p.G <= 8 || p.D == 256 ? 1 : 2;
    switch ((p.D * 10 + nb) * 2 + (e4m3 ? 1 : 0)) {
        case 1282: return launch_split_t<64, 1, false>(sp, f, rows, sms, dev, st);
        case 1283: return launch_split_t<64, 1, true>(sp, f, rows, sms, dev, st);
        case 1284: return launch_split_t<64, 2, false>(sp, f, rows, sms, dev, st);
        case 1285: return launch_split_t<64, 2, true>(sp, f, rows, sms, dev, st);
        case 2562: return launch_split_t<128, 1, false>(sp, f, rows, sms, dev, st);
        case 2564: return launch_split_t<128, 2, false>(sp, f, rows, sms, dev, st);
        case 5122: return launch_split_t<256, 1, false>(sp, f, rows, sms, dev, st);
        case 5123: return launch_split_t<256, 1, true>(sp, f, rows, sms, dev, st);
        default: return set_status(FCCI_EUNSUPPORTED, "paged attention: unsupported head_dim");
    }
}

}  // namespace pg
}  // namespace fcci
