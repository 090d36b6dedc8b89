// The line of key tiles that the split-KV kernels of the paged cache share: where a CTA's stretch lies, the
// warp that fetches its tiles, the append of the new row inside a tile, and the joining of a unit
// that several CTAs worked on.
//
// A unit is (sequence b, kv head h, column group c): up to COLS query rows of the group, rows being
// (token, query head) pairs, so a cached key is read once for all of them. A unit's keys are cut into tiles
// of KEYS rows; all tiles of all units form one line, of which every CTA of a persistent grid takes an
// equal stretch, whatever the lengths are. On the line a unit begins with kHead places that hold no tile: what its queries and
// its end cost. With 0, 2, 4 and 8 places (us, a CTA with many short units held up all): e4m3, D 128, 64 sequences of 128 to
// 8192 keys x 32 kv heads 529, 350, 332, 337; 17 of 1 to 5000 x 8 kv heads 40.0, 29.0, 27.5, 28.3; e4m3, D 64, the same
// 472, 311, 295, 308 and 32.6, 23.9, 23.0, 24.4; fp16, D 128, 64 x 8 kv heads 203, 169, 167, 167 and 17 50.9, 42.6, 38.7, 37.0.
// A unit that lies in one stretch is finished there; of a cut
// one, every CTA leaves its part (o, log-sum-exp) in the workspace and the last to arrive joins them. No
// CTA waits for another.
#pragma once
#include <cuda.h>

#include "paged.cuh"

namespace fcci {
namespace pg {

constexpr int kComputeWarps = 4, kCompute = kComputeWarps * 32;  // threads that compute
constexpr int kMaxStages = 6;
constexpr uint64_t kWaitLimitNs = 4000000000ull;  // 4 s: far beyond any healthy wait
constexpr uint64_t kDrainLimitNs = 500000000ull;
constexpr int kBar = 1;
constexpr int kHead = 4;  // places of a unit's head on the line

struct TileParams {
    Params p;
    int32_t fused;   // the kernel appends row T itself (decode)
    int32_t early;   // lengths, page table, scales and cached rows may be read before the programmatic-launch wait
    int32_t stages;
    float* part_lse;    // [2 * grid][kMaxCols]
    float* part_o;      // [2 * grid][kMaxCols][D]
    uint32_t* cut_cnt;  // [grid], zero between calls
};

// Tiles of KEYS rows of ROWB bytes, in blocks of PITCH bytes a row (the tensor-map swizzle's width).
template <int KEYS_, int ROWB_>
struct Tile {
    static constexpr int KEYS = KEYS_, ROWB = ROWB_;
    static constexpr int PITCH = ROWB < 128 ? ROWB : 128;
    static constexpr int BLOCKS = ROWB / PITCH;
    static constexpr int BYTES = KEYS * ROWB;
    // address of 16-byte chunk ch of row r of the tile at `tile`
    static __device__ __forceinline__ uint32_t cell(uint32_t tile, int r, int ch) {
        constexpr int CHUNKS = PITCH / 16;
        const int blk = ch / CHUNKS, c = ch % CHUNKS;
        const int sw = PITCH == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
        return tile + blk * KEYS * PITCH + r * PITCH + sw * 16;
    }
};

// Ring of S stages: the stage of the present tile and the times the ring has been gone round (a division by S
// would cost more than the rest of a loop's bookkeeping).
struct Ring {
    int S, s = 0;
    uint32_t round = 0;
    __device__ explicit Ring(int n) : S(n) {}
    __device__ __forceinline__ void next() {
        if (++s == S) s = 0, ++round;
    }
};

// A place on the line.
struct At {
    int b, h, c, j;     // sequence, kv head, column group, tile
    int tiles, groups;  // of sequence b
    int T, n, L;        // its cached rows (-1: not served), new tokens, keys
};

template <int KEYS, int COLS>
struct Line {
    const TileParams& tp;
    // shared: [B + 1] places and units before a sequence; its cached rows (-1: not served) and new tokens
    int *base, *units, *T, *n;
    unsigned N, CT;     // places in all, CTAs that take some
    unsigned per, more;  // N / CT and N % CT
    int ntiles;         // of this CTA

    static size_t ints(int B) { return 4 * (size_t)B + 2; }
    __device__ Line(const TileParams& tp_, int* sm)
        : tp(tp_), base(sm), units(sm + tp_.p.B + 1), T(units + tp_.p.B + 1), n(T + tp_.p.B) {}

    __device__ __forceinline__ int keys(int t, int m) const { return t + (tp.fused || tp.p.cu_q ? m : 0); }
    __device__ __forceinline__ int groups(int m) const { return (m * tp.p.G + COLS - 1) / COLS; }
    __device__ __forceinline__ int tiles(int t, int m) const { return max(1, (keys(t, m) + KEYS - 1) / KEYS); }

    __device__ __forceinline__ void enter(At& x) const {
        x.T = T[x.b], x.n = n[x.b];
        x.L = x.T < 0 ? 0 : keys(x.T, x.n);
        x.groups = groups(x.n);
        x.tiles = x.T < 0 ? 1 : tiles(x.T, x.n);
    }

    __device__ __forceinline__ void step(At& x) const {
        if (++x.j < x.tiles) return;
        x.j = 0;
        if (++x.c < x.groups) return;
        x.c = 0;
        if (++x.h < tp.p.Hkv) return;
        x.h = 0;
        do ++x.b;
        while (x.b < tp.p.B && base[x.b + 1] == base[x.b]);
        if (x.b < tp.p.B) enter(x);
    }

    // Lengths, prefixes of places and units, and this CTA's stretch. All threads; scratch: 32 shared ints.
    template <int THREADS>
    __device__ At build(int* scratch) {
        const Params& p = tp.p;
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = p.B;
        bool uniform = true, too_many = false;
        constexpr long long kMostPlaces = 1 << 23;  // of a thread: the line stays below 2^31 (8 M tiles are 10^9 keys)
        static_assert(THREADS <= 256, "places in 31 bits");
        // (places, units) of sequence b; writes its T and n
        auto count = [&](int b, long long& places) {
            const Seq s = seq_of(p, b);
            if (!s.ok && blockIdx.x == 0) set_error(p, FCCI_DEV_ERR_CAPACITY);
            // a sequence that is not served: its one row gets zeros in decode, none are touched otherwise
            const int m = s.ok ? s.n : (p.cu_q ? 0 : 1);
            T[b] = s.ok ? s.T : -1;
            n[b] = m;
            const int u = p.Hkv * groups(m);
            places = (long long)((s.ok ? tiles(s.T, m) : 1) + kHead) * u;
            return u;
        };
        if (B <= 32) {
            // every warp does the same by itself: no barrier between the lengths' arrival and the first copy
            long long places = 0;
            const int u = lane < B ? count(lane, places) : 0;
            too_many = __any_sync(0xffffffffu, places > kMostPlaces);
            const int cnt = (int)min(places, kMostPlaces);
            int incl = cnt, incl_u = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o), w = __shfl_up_sync(0xffffffffu, incl_u, o);
                if (lane >= o) incl += v, incl_u += w;
            }
            if (lane == 0) base[0] = 0, units[0] = 0;
            if (lane < B) base[lane + 1] = incl, units[lane + 1] = incl_u;
            const int cnt0 = __shfl_sync(0xffffffffu, cnt, 0);
            uniform = __all_sync(0xffffffffu, lane >= B || cnt == cnt0);
            __syncwarp();
        } else {
            const int chunk = (B + THREADS - 1) / THREADS, lo = tid * chunk, hi = min(B, lo + chunk);
            int local = 0, local_u = 0, first = -1;
            for (int b = lo; b < hi; ++b) {
                long long places;
                const int u = count(b, places), cnt = (int)min(places, kMostPlaces);
                too_many = too_many || local + places > kMostPlaces;
                base[b + 1] = cnt;
                units[b + 1] = u;
                local = (int)min(local + places, kMostPlaces);
                local_u += u;
                if (first < 0) first = cnt;
                if (cnt != first) uniform = false;
            }
            int incl = local, incl_u = local_u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o), u = __shfl_up_sync(0xffffffffu, incl_u, o);
                if (lane >= o) incl += v, incl_u += u;
            }
            if (lane == 31) scratch[warp] = incl, scratch[16 + warp] = incl_u;
            if (tid == 0) base[0] = 0, units[0] = 0, scratch[8] = first;
            __syncthreads();
            if (first >= 0 && first != scratch[8]) uniform = false;
            int run = incl - local, run_u = incl_u - local_u;
            for (int w = 0; w < warp; ++w) run += scratch[w], run_u += scratch[16 + w];
            for (int b = lo; b < hi; ++b) {
                base[b + 1] = run += base[b + 1];
                units[b + 1] = run_u += units[b + 1];
            }
            too_many = __syncthreads_or(too_many) != 0;
            uniform = __syncthreads_and(uniform) != 0;
        }

        N = (unsigned)base[B];
        if (too_many) {
            if (blockIdx.x == 0 && tid == 0) set_error(p, FCCI_DEV_ERR_CAPACITY);
            N = 0;  // nothing is served
        }
        CT = min(N, gridDim.x);
        if (uniform && N > 0) {
            // equal units: a number of CTAs that is a multiple of the units keeps every cut at the same places of each,
            // unless that leaves more than 15 % of the grid idle. Us, with the rule and without, 8 kv heads, e4m3 D 128,
            // e4m3 D 64, fp16 D 128: 32 x 4096 keys (14 % idle) 50.0 / 55.5, 45.1 / 45.9, 88.7 / 93.2; 35 x 2000 (5 %)
            // 32.3 / 41.4, 26.9 / 32.6, 53.4 / 57.1; beyond it 30 x 4096 (19 %) 48.0 / 52.9, 45.1 / 43.7, 81.7 / 87.5 and
            // 25 x 4096 (32 %) 44.3 / 46.8, 44.7 / 38.2, 75.3 / 76.4: there it depends on the kernel.
            const unsigned all = (unsigned)units[B];
            if (all <= gridDim.x) {
                const unsigned k = min(gridDim.x / all, N / all);
                if (20 * all * k >= 17 * CT) CT = all * k;
            }
        }
        per = CT ? N / CT : 0;
        more = N - per * CT;
        At at = {0, 0, 0, 0, 1, 1, -1, 0, 0};
        ntiles = 0;
        if (blockIdx.x < CT) {
            At end = at;
            const int first_tile = place(start(blockIdx.x), at);
            ntiles = place(start(blockIdx.x + 1), end) - first_tile;
        }
        return at;
    }

    // The first tile at or behind place t: where it is, and the tiles before it on the line.
    __device__ int place(unsigned t, At& x) const {
        const int B = tp.p.B;
        if (t >= N) return base[B] - kHead * units[B];
        int l = 0, r = B - 1;
        while (l < r) {
            const int mid = (l + r + 1) >> 1;
            if ((unsigned)base[mid] <= t) l = mid;
            else r = mid - 1;
        }
        x.b = l;
        enter(x);
        const int rem = (int)t - base[l], unit = rem / (x.tiles + kHead);
        x.j = max(0, rem - unit * (x.tiles + kHead) - kHead);
        x.h = x.groups == 1 ? unit : unit / x.groups;
        x.c = unit - x.h * x.groups;
        return base[l] - kHead * units[l] + unit * x.tiles + x.j;
    }

    // First place of CTA c: floor(c N / CT), in 32 bits (c * more < CT^2).
    __device__ __forceinline__ unsigned start(unsigned c) const { return c * per + (more ? c * more / CT : 0); }

    // CTA that has place t: a guess in fp32 (off by one at most), put right.
    __device__ __forceinline__ int cta_of(unsigned t) const {
        int c = (int)(((float)t + 0.5f) * ((float)CT / (float)N));
        c = max(0, min((int)CT - 1, c));
        while (start(c) > t) --c;
        while (start(c + 1) <= t) ++c;
        return c;
    }

    // First and last CTA of the unit at x.
    __device__ __forceinline__ int2 ctas_of(const At& x) const {
        const unsigned u = base[x.b] + ((unsigned)x.h * x.groups + x.c) * (x.tiles + kHead) + kHead;  // of its first tile
        return make_int2(cta_of(u), cta_of(u + x.tiles - 1));
    }
};

// Slot of this CTA's part of a cut unit: it has at most two parts, one that begins a unit and one that does not.
__device__ __forceinline__ size_t part_slot(int cta, bool begins) { return 2 * (size_t)cta + (begins ? 1 : 0); }

// A fetching warp: that of K or of V (an issue of a copy takes the thread some 90 cycles, and a tile of 16-row pages
// has 8 boxes of each). A lane has one page box of the tile. The page table is read a tile ahead, and a tile's
// scales are published (the warp's second arrival on `full`) after the next tile's copies are under way,
// so neither latency delays a copy.
// scales: [stage][K, V][8]: 2^e of the box's page (fp16 pages: 1); -1 where there is none.
template <class TL, bool E4M3, int COLS>
__device__ void fetch_tiles(const Line<TL::KEYS, COLS>& line, At at, bool is_v, const CUtensorMap* map,
                            const CUtensorMap* map16, uint8_t* tiles, uint64_t* full, uint64_t* empty, float* scales,
                            volatile int* abort_flag) {
    constexpr int KEYS = TL::KEYS, PITCH = TL::PITCH;
    const TileParams& tp = line.tp;
    const Params& p = tp.p;
    const int lane = threadIdx.x & 31, ntiles = line.ntiles;
    Ring ring(tp.stages);
    const int box = min(p.page, KEYS), boxes = KEYS / box;
    const uint64_t pol = l2_policy_evict_first();
    const int32_t* table = p.table;
    const int64_t table_st = p.table_st;
    const int page_log2 = p.page_log2, row_mask = p.page - 1, first_row = lane * box;
    const unsigned num_pages = (unsigned)p.num_pages;
    const uint8_t* scale_bytes = is_v ? p.v_scales : p.k_scales;
    const int64_t ssp = is_v ? p.vs_sp : p.ks_sp, ssh = is_v ? p.vs_sh : p.ks_sh;
    if (is_v) tiles += TL::BYTES, scales += 8;
    auto rows_at = [&](const At& x) { return lane < boxes ? max(0, min(box, x.L - x.j * KEYS - first_row)) : 0; };
    auto page_at = [&](const At& x) {
        return rows_at(x) > 0 ? table[x.b * table_st + ((x.j * KEYS + first_row) >> page_log2)] : -1;
    };
    // byte: the scale byte as loaded (turned into a number here, a tile later, so that the load has had its time)
    auto publish = [&](int st, int byte) {
        if (lane < boxes) scales[st * 16 + lane] = byte < 0 ? -1.f : exp2_int(byte - 127);
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
    };
    int pid = ntiles > 0 ? page_at(at) : -1;
    int byte = -1, it = 0, s_prev = 0;
    bool published = false;  // tile it - 1 has had its second arrival when the loop ends early
    for (; it < ntiles; ++it) {
        const int s = ring.s;
        const int rows = rows_at(at), h = at.h;
        const int row0 = (at.j * KEYS + first_row) & row_mask;
        const bool there = rows > 0 && (unsigned)pid < num_pages;
        if (rows > 0 && !there) set_error(p, FCCI_DEV_ERR_PAGE);
        const int id = there ? pid : 0;
        line.step(at);
        if (it + 1 < ntiles) pid = page_at(at);
        // when no stage is free, whoever frees one may need the tile before whole first
        const uint32_t parity = (ring.round & 1u) ^ 1u;
        const bool early = !__all_sync(0xffffffffu, mbar_test_wait(&empty[s], parity));
        if (early && it > 0) publish(s_prev, byte);
        if (!__all_sync(0xffffffffu, mbar_wait_sparing(&empty[s], parity, abort_flag, kWaitLimitNs))) {
            if (lane == 0) {
                *abort_flag = 1;
                set_error(p, FCCI_DEV_ERR_TIMEOUT);
            }
            published = early;
            break;
        }
        const int fetched = !there ? 0 : rows == box ? box : (rows + 15) & ~15;
        const uint32_t bytes = __reduce_add_sync(0xffffffffu, (unsigned)(fetched * TL::ROWB));
        if (lane == 0) mbar_arrive_expect_tx(&full[s], bytes);
        __syncwarp();
        if (there) {
            uint8_t* dst = tiles + (size_t)s * 2 * TL::BYTES + first_row * PITCH;
#pragma unroll
            for (int k = 0; k < TL::BLOCKS; ++k) {
                const int col = k * PITCH / (E4M3 ? 1 : 2);
                if (rows == box) {
                    tma_load_4d(dst + k * KEYS * PITCH, map, col, row0, h, id, &full[s], pol);
                } else {  // the page that ends the sequence: only the 16-row boxes that hold rows of it
                    for (int r = 0; r < fetched; r += 16)
                        tma_load_4d(dst + k * KEYS * PITCH + r * PITCH, map16, col, row0 + r, h, id, &full[s], pol);
                }
            }
        }
        if (it > 0 && !early) publish(s_prev, byte);
        byte = there ? 127 : -1;
        if (E4M3 && there) byte = scale_bytes[id * ssp + h * ssh];
        s_prev = s;
        ring.next();
    }
    if (it > 0 && !published) publish(s_prev, byte);
    if (*abort_flag) {
        // let copies still in flight land before the CTA can exit
        volatile int never = 0;
        for (int i = max(0, it - ring.S); i < it; ++i)
            mbar_wait_sparing(&full[i % ring.S], (uint32_t)(i / ring.S) & 1u, &never, kDrainLimitNs);
    }
}

// Append of row T of (b, h) by one warp, into the fetched tile and into the page: is_v the value, else the key,
// rotated by cs (cos and sin of position T). scale: the box's entry in shared memory.
template <class TL, int D, bool E4M3>
__device__ void append_in_tile(const Params& p, int b, int h, int T, bool is_v, const float2* cs, uint8_t* tile, float* scale_slot) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, half = p.rot >> 1;
    const int d0 = lane * E, r = T % TL::KEYS, off = T & (p.page - 1);
    const __half* src = is_v ? p.v_new + b * p.vn_st + h * p.vn_sh : p.k_new + b * p.kn_st + h * p.kn_sh;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        x[e] = __half2float(src[d0 + e]);
        if (!is_v && d0 < p.rot) {
            const bool lowhalf = d0 < half;
            const int k = (lowhalf ? d0 : d0 - half) + e;
            x[e] = rotated(x[e], __half2float(src[lowhalf ? k + half : k]), cs[k], lowhalf);
        }
    }
    const int id = p.table[(int64_t)b * p.table_st + (T >> p.page_log2)];
    uint8_t* page = is_v ? p.v_pages + id * p.v_sp + h * p.v_sh : p.k_pages + id * p.k_sp + h * p.k_sh;
    const int64_t st = is_v ? p.v_st : p.k_st;
    const uint32_t t32 = smem_u32(tile);
    auto in_tile = [&](int row, int byte) { return tile + (TL::cell(t32, row, byte >> 4) - t32) + (byte & 15); };
    if constexpr (!E4M3) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const uint32_t v = pack_half2(x[e], x[e + 1]);
            *reinterpret_cast<uint32_t*>(page + off * st + (d0 + e) * 2) = v;
            *reinterpret_cast<uint32_t*>(in_tile(r, (d0 + e) * 2)) = v;
        }
    } else {
        const float had = *scale_slot;
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) amax = fmaxf(amax, fabsf(x[e]));
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        float scale = exp2_int(scale_exponent(amax));
        if (off && had >= scale) {
            scale = had;
        } else if (off) {
            // the rows before take the larger scale, in the tile and in the page
            const float down = had / scale;
            for (int i = lane; i < off * (D / 4); i += 32) {
                const int row = i / (D / 4), byte = (i % (D / 4)) * 4;
                uint32_t* a = reinterpret_cast<uint32_t*>(in_tile(r - off + row, byte));
                const uint32_t lo2 = half2_of_e4m3x2(*a & 0xffffu), hi2 = half2_of_e4m3x2(*a >> 16);
                const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&lo2));
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hi2));
                *a = e4m3x2(u.x * down, u.y * down) | (e4m3x2(v.x * down, v.y * down) << 16);
                *reinterpret_cast<uint32_t*>(page + row * st + byte) = *a;
            }
        }
        const float up = 1.f / scale;  // a power of two: exact
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const uint16_t v = (uint16_t)e4m3x2(x[e] * up, x[e + 1] * up);
            *reinterpret_cast<uint16_t*>(page + off * st + d0 + e) = v;
            *reinterpret_cast<uint16_t*>(in_tile(r, d0 + e)) = v;
        }
        __syncwarp();
        if (lane == 0) {
            *scale_slot = scale;
            uint8_t* s8 = is_v ? p.v_scales + id * p.vs_sp + h * p.vs_sh : p.k_scales + id * p.ks_sp + h * p.ks_sh;
            *s8 = (uint8_t)(__float_as_uint(scale) >> 23);
        }
    }
}

// Output row of query row c of a unit whose rows begin at r0.
__device__ __forceinline__ __half* out_row(const Params& p, const At& at, int r0, int c) {
    const int64_t tok0 = p.cu_q ? p.cu_q[at.b] : at.b;
    const int i = (r0 + c) / p.G;
    return p.out + (tok0 + i) * p.o_st + (int64_t)(at.h * p.G + (r0 + c) - i * p.G) * p.o_sh;
}

// The last part of a cut unit to arrive joins all of them; called by the computing threads, after their
// stores of this part. Release: the barrier orders those before thread 0's fence and count; acquire:
// its fence after the count. The counter is that of the unit's first CTA, where no other cut unit begins.
template <int D>
__device__ void join_parts(const TileParams& tp, const At& at, int r0, int rows, int ca, int cb, int* flag) {
    const int tid = threadIdx.x;
    named_bar_sync(kBar, kCompute);
    if (tid == 0) {
        __threadfence();
        *flag = atomicAdd(&tp.cut_cnt[ca], 1u) == (unsigned)(cb - ca);
        if (*flag) __threadfence();
    }
    named_bar_sync(kBar, kCompute);
    if (!*flag) return;
    const int parts = cb - ca + 1;
    for (int e = tid * 4; e < rows * D; e += 4 * kCompute) {
        const int c = e / D, d = e - c * D;
        float M = -INFINITY, W = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {
            const size_t part = part_slot(ca + i, i == 0);
            const float lse = __ldcg(tp.part_lse + part * kMaxCols + c);
            const float4 y = __ldcg(reinterpret_cast<const float4*>(tp.part_o + (part * kMaxCols + c) * D + d));
            const float mn = fmaxf(M, lse), mu = mn == -INFINITY ? 0.f : mn;
            const float a = ex2(M - mu), u = ex2(lse - mu);
            W = W * a + u;
            o.x = o.x * a + y.x * u, o.y = o.y * a + y.y * u;
            o.z = o.z * a + y.z * u, o.w = o.w * a + y.w * u;
            M = mn;
        }
        const float inv = W > 0.f ? 1.f / W : 0.f;
        uint2 v;
        v.x = pack_half2(o.x * inv, o.y * inv);
        v.y = pack_half2(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(out_row(tp.p, at, r0, c) + d) = v;
    }
    if (tid == 0) atomicExch(&tp.cut_cnt[ca], 0u);
}

// Tensor maps (dims, row of a page, kv head, page) of both pools: boxes of a whole page (or tile) and of 16 rows.
template <class TL, bool E4M3>
int encode_pages(const Params& p, CUtensorMap (&m)[4]) {
    const int elt = E4M3 ? 1 : 2;
    for (int i = 0; i < 4; ++i) {
        const bool v = i & 1;
        const uint64_t dims[4] = {(uint64_t)p.D, (uint64_t)p.page, (uint64_t)p.Hkv, (uint64_t)p.num_pages};
        const int64_t sb[3] = {v ? p.v_st : p.k_st, v ? p.v_sh : p.k_sh, v ? p.v_sp : p.k_sp};
        const uint32_t box[4] = {(uint32_t)(TL::PITCH / elt), (uint32_t)(i >= 2 ? 16 : p.page < TL::KEYS ? p.page : TL::KEYS), 1, 1};
        const int rc = encode_tiled(&m[i], E4M3, TL::PITCH == 64, v ? p.v_pages : p.k_pages, 4, dims, sb, box);
        if (rc) return set_status(rc, "paged attention: cuTensorMapEncodeTiled rejected the page layout");
    }
    return FCCI_OK;
}

}  // namespace pg
}  // namespace fcci
