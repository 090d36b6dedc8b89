// What the causal prefill attention shares with the callers that prepare its inputs: its launch parameters and the
// work list.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "fcci_decode.h"
#include "fcci_internal.h"

namespace fcci {
namespace pf {

constexpr int D = 128;
constexpr int kPairRows = 256;   // new tokens of one work item: two query tiles of 128
constexpr int kMaxSortB = 1024;  // sequences ranked by length up to this batch size

struct Params {
    const __half* q;
    int64_t q_st, q_sh;
    const __half* k_new;
    int64_t kn_st, kn_sh;
    const __half* v_new;
    int64_t vn_st, vn_sh;
    __half* k_cache;
    int64_t k_sb, k_sh, k_st;
    __half* v_cache;
    int64_t v_sb, v_sh, v_st;
    int32_t capacity;
    const int32_t* cu_q;
    const int32_t* cu_kv;
    int32_t* seq_lens;
    int32_t fixed_len;
    __half* out;
    int64_t o_st, o_sh;
    float scale_log2;
    float weight_log2;  // log2 of the weight of a row's maximum when that moves, at most 7 (it may then grow by 2^8)
    float rope_theta;
    int32_t rotary_dim;
    int32_t advance;
    int32_t B, Hq, Hkv, G, total_q, max_q;
    int32_t table_pos;  // positions covered by the table (= capacity)
    // workspace
    uint32_t* err;
    uint32_t* item_cnt;
    uint32_t* exit_cnt;
    int32_t* n_items;
    uint32_t* table_hdr;  // magic, theta bits, rotary_dim, positions
    uint32_t* table_cnt;
    int4* items;
    __half* q_rot;
    float2* table;
};

__device__ __forceinline__ void set_error(const Params& p, uint32_t bit) {
    if (p.err) atomicOr(p.err, bit);
}

struct SeqRange {
    int T, n, tok0, kvrow0, kvb;
    bool ok;
};

__device__ __forceinline__ SeqRange seq_range(const Params& p, int b) {
    SeqRange s;
    s.tok0 = p.cu_q[b];
    s.n = p.cu_q[b + 1] - s.tok0;
    s.T = p.seq_lens ? p.seq_lens[b] : p.fixed_len;
    int cap = p.capacity;
    bool ok = true;
    if (p.cu_kv) {
        const int lo = p.cu_kv[b], hi = p.cu_kv[b + 1];
        s.kvrow0 = lo;
        s.kvb = 0;
        cap = hi - lo;
        ok = lo >= 0 && hi >= lo && hi <= p.capacity;
    } else {
        s.kvrow0 = 0;
        s.kvb = b;
    }
    ok = ok && s.T >= 0 && s.n >= 0 && s.n <= p.max_q && s.tok0 >= 0 && s.tok0 + s.n <= p.total_q &&
         (long long)s.T + s.n <= cap;
    s.ok = ok;
    return s;
}

// Work list: items (b, h, pair) sequence-major with sequences ranked by T_b + n_b
// (longest first), then head, then pair from last to first. Also resets the
// attention kernel's counters. One CTA.
inline __device__ void build_work_list(const Params& p, int* sm) {
    const int tid = threadIdx.x;
    const int B = p.B;
    int* np = sm;              // [B] pairs of sequence b (0 when invalid)
    int* key = np + B;         // [B] ranking key
    int* order = key + B;      // [B] rank -> b
    int* off = order + B;      // [B+1] first item of rank r
    for (int b = tid; b < B; b += blockDim.x) {
        const SeqRange s = seq_range(p, b);
        np[b] = s.ok ? (s.n + kPairRows - 1) / kPairRows : 0;
        key[b] = s.ok ? s.T + s.n : -1;
        order[b] = b;
    }
    __syncthreads();
    if (B <= kMaxSortB) {
        for (int b = tid; b < B; b += blockDim.x) {
            const int kb = key[b];
            int r = 0;
            for (int o = 0; o < B; ++o) {
                const int ko = key[o];
                r += (ko > kb) || (ko == kb && o < b);
            }
            order[r] = b;
        }
        __syncthreads();
    }
    if (tid == 0) {
        int acc = 0;
        for (int r = 0; r < B; ++r) {
            off[r] = acc;
            acc += np[order[r]] * p.Hq;
        }
        off[B] = acc;
        *p.n_items = acc;
        *p.item_cnt = 0u;
        *p.exit_cnt = 0u;
    }
    __syncthreads();
    const int total = off[B];
    for (int v = tid; v < total; v += blockDim.x) {
        int lo = 0, hi = B - 1;  // last rank with off[r] <= v
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (off[mid] <= v) lo = mid; else hi = mid - 1;
        }
        const int b = order[lo];
        const int n = np[b];
        const int w = v - off[lo];
        const int h = w / n;
        const int pair = n - 1 - (w % n);
        p.items[v] = make_int4(b, h, pair, 0);
    }
}

// The attention launch over p.items: q_rot [total_q, Hq, D], keys and values through k_cache / v_cache and their
// strides; max_items bounds *p.n_items.
int launch_attend(const Params& p, int64_t max_items, cudaStream_t stream);

}  // namespace pf
}  // namespace fcci
