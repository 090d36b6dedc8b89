// What the kernels of the paged KV cache share: the launch parameters, a sequence's ranges,
// the e4m3 / power-of-two scale arithmetic and the position rotation.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "fcci_internal.h"
#include "fcci_paged.h"
#include "ptx.cuh"

// The append and the split attention let the next kernel start (griddep_launch_dependents) only after their own wait, unless
// they read early: the next one may read lengths and rows before its wait, and must not do so while a kernel before
// this one, a step that moves the lengths for instance, is still running. (A token append in a chain takes 2.44 us
// instead of 2.37, a decode step over 512 keys 11.2 instead of 11.0.)
namespace fcci {
namespace pg {

constexpr int kMaxRot = 256;
constexpr int kScaleMin = -15, kScaleMax = 8;  // exponents of a page's scale

// Long chunks hold their rotated queries in fp16 times this: a rotation of the largest fp16 values reaches 92637, past
// fp16's 65504. Their scale takes it back. (Halving is exact but for elements below 2^-13, then off by 2^-24.)
constexpr float kLongQuery = 0.5f;
// The same for the keys of e4m3 pages, as an exponent: a page of scale 2^8 may hold rotated keys up to 352 * 2^8 = 90112.
// (Exact but for codes below 2^-6 at scale 2^-15, then off by 2^-25 before the scale takes it back.)
constexpr int kLongKeyExp = -1;

struct Params {
    int32_t B, Hq, Hkv, G, D;
    int32_t total_q, max_q;
    const int32_t* cu_q;
    const __half* q;
    int64_t q_st, q_sh;
    const __half* k_new;
    int64_t kn_st, kn_sh;
    const __half* v_new;
    int64_t vn_st, vn_sh;
    int32_t page, page_log2, num_pages, max_pages;
    uint8_t* k_pages;  // strides in bytes
    int64_t k_sp, k_sh, k_st;
    uint8_t* v_pages;
    int64_t v_sp, v_sh, v_st;
    uint8_t* k_scales;
    int64_t ks_sp, ks_sh;
    uint8_t* v_scales;
    int64_t vs_sp, vs_sh;
    const int32_t* table;
    int64_t table_st;
    int32_t* seq_lens;
    __half* out;
    int64_t o_st, o_sh;
    __half* q_rot;  // [total_q, Hq, D] contiguous
    // long chunks: rows [cu_kv[b], cu_kv[b + 1]) of the expanded fp16 keys and values are sequence b's
    const int32_t* cu_kv;
    __half* exp_k;
    __half* exp_v;
    int64_t exp_sh;
    float scale_log2;
    int32_t rot;
    int32_t advance;
    int32_t append;
    uint32_t* err;
    uint32_t* done_cnt;
};

// Frequencies theta^(-2i/rot) / 2 pi in turns per position, as 64-bit fixed-point fractions:
// pos * freq wraps modulo one turn by itself, so the angle of a far position loses nothing.
struct Freqs {
    uint64_t turn[kMaxRot / 2];
};

struct Seq {
    int T, n, tok0;  // cached rows, new tokens, first row of the new tokens
    bool ok;
};

__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
    Seq s;
    s.T = p.seq_lens[b];
    s.tok0 = p.cu_q ? p.cu_q[b] : b;
    s.n = p.cu_q ? p.cu_q[b + 1] - s.tok0 : 1;
    const long long cap = (long long)p.max_pages << p.page_log2;
    s.ok = s.T >= 0 && s.n >= 0 && s.n <= p.max_q && s.tok0 >= 0 && (long long)s.tok0 + s.n <= p.total_q &&
           (long long)s.T + (p.append ? s.n : 0) <= cap;
    return s;
}

__device__ __forceinline__ void set_error(const Params& p, uint32_t bit) { atomicOr(p.err, bit); }

// Page of row t of sequence b; -1 (and the error bit) when the table names none of the pool.
__device__ __forceinline__ int page_of(const Params& p, int b, int t) {
    const int id = p.table[(int64_t)b * p.table_st + (t >> p.page_log2)];
    if ((unsigned)id < (unsigned)p.num_pages) return id;
    set_error(p, FCCI_DEV_ERR_PAGE);
    return -1;
}

// Smallest e in [lo, hi] with amax <= 448 * 2^e: 448 = 1.75 * 2^8, so with amax = m * 2^E it is
// E - 8, one more when m > 1.75 (mantissa bits above 0x600000).
__device__ __forceinline__ int exponent_448(float amax, int lo, int hi) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(lo, min(hi, e));
}

__device__ __forceinline__ int scale_exponent(float amax) { return exponent_448(amax, kScaleMin, kScaleMax); }

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two values to e4m3 codes (round to nearest even, saturating; the first in the low byte).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// e5m2 is fp16's upper byte. The codes of four fp16 values, cut (not rounded) to three bits each, and 8 times what that
// leaves of two of them, which is exact.
__device__ __forceinline__ uint32_t e5m2x4_of_half4(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7531); }
__device__ __forceinline__ uint32_t half2_rest8(uint32_t a) {
    const uint32_t cut = a & 0xff00ff00u;
    const __half2 r = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&cut)),
                              __float2half2_rn(8.f));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Two e4m3 codes to fp16 (exact).
__device__ __forceinline__ uint32_t half2_of_e4m3x2(uint32_t codes) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
    return h;
}

// fp16's 2^xe of a page with scale 2^e. A scale above those that an append makes may hold values that fp16 cannot: it is
// reported, and cut so that zeros stay zeros. Below 2^-25 it is 0.
__device__ __forceinline__ __half2 expansion_scale(const Params& p, int e, int xe) {
    if (e > kScaleMax) set_error(p, FCCI_DEV_ERR_SCALE);
    return __float2half2_rn(exp2_int(max(-126, min(xe, 15))));
}

// Eight e4m3 codes times the scale, as fp16; clamp: the product may pass 65504.
__device__ __forceinline__ uint4 expanded(uint2 codes, __half2 scale, bool clamp) {
    uint32_t h[4] = {half2_of_e4m3x2(codes.x & 0xffffu), half2_of_e4m3x2(codes.x >> 16),
                     half2_of_e4m3x2(codes.y & 0xffffu), half2_of_e4m3x2(codes.y >> 16)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), scale);
        if (clamp) v = __hmin2_nan(__hmax2_nan(v, __float2half2_rn(-65504.f)), __float2half2_rn(65504.f));
        h[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(h[0], h[1], h[2], h[3]);
}

// cos and sin of pos * freq. The top 32 bits of the wrapped product are the angle in units of
// 2^-32 turns; the nearest quarter turn is taken off as an integer, so what is rounded to fp32 is at
// most an eighth of a turn, what that rounding leaves off is put on to first order, and the quarters go back as
// a swap and signs.
__device__ __forceinline__ float2 rope_cs(uint64_t turn, int pos) {
    const uint32_t a = (uint32_t)(((uint64_t)(uint32_t)pos * turn) >> 32);
    const uint32_t quarter = (a + 0x20000000u) >> 30;
    const int32_t rest = (int32_t)(a - (quarter << 30));
    const float x32 = (float)rest;
    float s, c;
    sincospif(x32 * 4.656612873077393e-10f, &s, &c);
    const float off = (float)(rest - (int32_t)x32) * 1.4629180792671596e-9f;  // pi * 2^-31 each
    const float s0 = s;
    s = fmaf(c, off, s);
    c = fmaf(-s0, off, c);
    const bool odd = quarter & 1;
    const float x = odd ? s : c, y = odd ? c : s;
    // quarter 0: (c, s), 1: (-s, c), 2: (-c, -s), 3: (s, -c)
    return make_float2(((quarter + 1) & 2) ? -x : x, (quarter & 2) ? -y : y);
}

// x1' = x1 cos - x2 sin, x2' = x2 cos + x1 sin
__device__ __forceinline__ float rotated(float x, float partner, float2 cs, bool first_half) {
    return first_half ? fmaf(x, cs.x, -(partner * cs.y)) : fmaf(x, cs.x, partner * cs.y);
}

// The last CTA of the grid moves seq_lens: every CTA has read them by then. Called by all
// threads at the kernel's end; `flag` is a shared word.
__device__ __forceinline__ void advance_lengths(const Params& p, int* flag) {
    if (!p.advance) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        const unsigned total = gridDim.x * gridDim.y * gridDim.z;
        *flag = atomicAdd(p.done_cnt, 1u) == total - 1;
    }
    __syncthreads();
    if (!*flag) return;
    __threadfence();
    for (int b = threadIdx.x; b < p.B; b += blockDim.x) {
        const Seq s = seq_of(p, b);
        if (s.ok) p.seq_lens[b] = s.T + (p.append ? s.n : 0);
    }
    if (threadIdx.x == 0) atomicExch(p.done_cnt, 0u);
}

// Workspace: a fixed head (error word, counters that are zero between calls) and per-call
// regions behind it, so that one workspace serves calls of different shapes.
constexpr int kMaxGrid = 1024;  // CTAs of the split attention launch, at most
constexpr size_t kHeadBytes = 256 + kMaxGrid * 4;
constexpr int kMaxCols = 16;  // query rows of one attention unit
struct WsLayout {
    size_t part_lse, part_o, q_rot, cu_kv, items, expanded, total;
};
// Work items of a prefill, at most: 256 new tokens of one sequence and query head each.
inline int64_t max_items(int B, int Hq, int total_q) { return ((int64_t)total_q / 256 + B) * Hq; }
// Query rows of one kv head (new tokens x group) up to which a chunk takes the split-KV kernels. Split against expanding,
// us, e4m3: 8 sequences of 2000 keys, 8 kv heads, 64 rows 76 against 107, 128 rows 122 against 108; one of 8000, 128
// rows 59 against 140; 32 of 4000, 128 rows 646 against 948, 256 rows 1312 against 952; 16 of 500, 32 kv heads, 16 rows
// 86 against 123, 32 rows 142 against 126. Where they cross depends on lengths that only the device knows; max_q is the
// caller's bound on them, so a loose one sends short chunks the long way.
constexpr int kSplitRows = 64;
inline bool long_chunk(int Hq, int Hkv, int max_q) { return (int64_t)max_q * (Hq / Hkv) > kSplitRows; }
WsLayout ws_layout(int B, int Hq, int Hkv, int D, int total_q, int max_q, int max_kv, int grid);

int launch_append(const Params& p, const Freqs& f, bool e4m3, cudaStream_t st);
// Split-KV attention; `fused`: the launch appends the one new row of each sequence itself.
// early: FCCI_PAGED_PREFETCH_KV. rows: what an append launched before it writes (or NULL), once every check has passed.
int launch_split(const Params& p, const Freqs& f, const Params* rows, bool e4m3, bool fused, bool early, uint8_t* ws,
                 const WsLayout& L, cudaStream_t st);
int append_before(const Params* rows, const Freqs& f, bool e4m3, cudaStream_t st);
int launch_prefill(const Params& p, const Freqs& f, bool e4m3, uint8_t* ws, const WsLayout& L, int max_kv, float scale_log2,
                   int advance, cudaStream_t st);
struct TileParams;
// The same on the 5th-generation tensor cores, for e4m3 pages of head_dim 128.
int launch_split_tc(TileParams& tp, const Freqs& f, const Params* rows, int sms, int dev, cudaStream_t st);

}  // namespace pg
}  // namespace fcci
