// vox_paged.cuh -- device helpers of the paged-cache kernels: checked batch
// metadata, the list of key blocks a tile of query rows sees, masks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/vox_decoder.h"
#include "vox_device.cuh"
#include "vox_paged.h"

namespace vox {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

constexpr float kNegInf = -__builtin_huge_valf();

// 2^x on the special-function unit (relative error about 2^-22); 0 for -inf.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct PagedSeq {
    int q0, nq, len;  // first token, tokens of the call, cached tokens
    bool ok;          // false: bad lengths, the sequence is skipped (nq 0)
};

// A sequence's lengths, checked against the host's bounds (A: either argument struct).
template <class A>
__device__ __forceinline__ PagedSeq paged_seq(const A& a, int s) {
    const int q0 = a.q_start[s], q1 = a.q_start[s + 1], len = a.kv_len[s];
    PagedSeq r;
    r.ok = q0 >= 0 && q1 >= q0 && q1 <= a.n_tokens && q1 - q0 <= a.max_q && len >= 0 && len <= a.max_kv &&
           (len >> a.page_shift) + ((len & ((1 << a.page_shift) - 1)) != 0) <= a.table_width;
    r.q0 = q0;
    r.nq = r.ok ? q1 - q0 : 0;
    r.len = len;
    return r;
}

template <class A>
__device__ __forceinline__ void paged_status(const A& a, uint32_t bit) {
    if (a.status) atomicOr(a.status, bit);
}

// The sequence whose tokens hold token t: the last s with q_start[s] <= t
// (-1: none).  The caller still checks that t lies in it.
template <class A>
__device__ __forceinline__ int paged_seq_of(const A& a, int t) {
    int lo = 0, hi = a.n_seqs;  // first s in [0, n_seqs) with q_start[s] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] > t) hi = mid; else lo = mid + 1;
    }
    return lo - 1;
}

// The prefix's length, or -1 where it is out of its bounds.
__device__ __forceinline__ int paged_prefix_len(const PagedAttnArgs& a) {
    const int n = *a.pfx_len;
    const int pages = (n >> a.page_shift) + ((n & ((1 << a.page_shift) - 1)) != 0);
    return n < 0 || n > a.pfx_max || pages > a.pfx_n_pages ? -1 : n;
}

// Tile `t` of the tiles of `rows` query rows (a sequence's row is token * group
// + head) that cover every sequence in turn; one warp calls it.  Returns the
// sequence (-1: none) and the tile's place in it.
__device__ __forceinline__ int paged_find_tile(const PagedAttnArgs& a, int t, int rows, int* place) {
    const int lane = threadIdx.x & 31;
    if (a.max_q * a.group <= rows) {  // at most one tile a sequence
        *place = 0;
        return t < a.n_seqs ? t : -1;
    }
    int before = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        int n = 0;
        if (s < a.n_seqs) {
            const PagedSeq q = paged_seq(a, s);
            if (!q.ok) paged_status(a, VOX_PAGED_BAD_LENGTH);  // no tile stands for it
            n = (q.nq * a.group + rows - 1) / rows;
        }
        int sum = n;
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned hit = __ballot_sync(~0u, before + sum > t);
        if (hit) {
            const int src = __ffs(hit) - 1;
            *place = t - before - __shfl_sync(~0u, sum - n, src);
            return s0 + src;
        }
        before += __shfl_sync(~0u, sum, 31);
    }
    *place = 0;
    return -1;
}

// The blocks of 2^shift keys that some row with an index in [pmin, pmax] sees,
// among keys 0..len-1: the sinks' blocks, then the window's.
struct KeyBlocks {
    int sink_blocks, first, total;  // total blocks; the window's begin with `first`
    int end, lo, sinks;             // keys [0, min(sinks, end)) and [lo, end) are seen
    __device__ __forceinline__ int block(int i) const { return i < sink_blocks ? i : first + i - sink_blocks; }
    __device__ __forceinline__ bool seen(int j) const { return j < end && (j >= lo || j < sinks); }
    // whether any of the n keys from j on is
    __device__ __forceinline__ bool any_seen(int j, int n) const { return max(j, lo) < min(j + n, end) || j < min(sinks, end); }
};
__device__ __forceinline__ KeyBlocks paged_key_blocks(int pmin, int pmax, int len, int window, int sinks, int shift) {
    KeyBlocks b;
    b.end = min(pmax, len - 1) + 1;
    if (b.end < 0) b.end = 0;
    b.lo = window ? max(0, pmin - window + 1) : 0;
    b.sinks = b.lo ? sinks : 0;
    const int mask = (1 << shift) - 1;
    const int nb = (b.end >> shift) + ((b.end & mask) != 0);
    const int se = min(b.sinks, b.end);
    b.sink_blocks = (se >> shift) + ((se & mask) != 0);
    b.first = max(b.lo >> shift, b.sink_blocks);
    b.total = b.sink_blocks + (b.lo < b.end ? max(0, nb - b.first) : 0);
    return b;
}

// The blocks [begin, end) of part `part` of `parts` equal ones of `total`.
__device__ __forceinline__ void paged_part(int total, int part, int parts, int* begin, int* end) {
    const int each = total / parts, more = total - each * parts;
    *begin = each * part + min(part, more);
    *end = *begin + each + (part < more);
}

// Whether the token with index p sees key j (of keys 0..len-1).
__device__ __forceinline__ bool paged_sees(int p, int j, int len, int window, int sinks) {
    return j <= p && j < len && (window == 0 || j < sinks || j > p - window);
}

// What a tile of rows attends to: keys 0..len-1, of which the first plen are in
// the pages pfx and the others in the pages of a table row; and the sink count.
struct PagedKeys {
    const int32_t* table;
    int len, sinks;
    const int32_t* pfx;
    int plen;
    __device__ __forceinline__ int page(int j, int shift) const {
        return j < plen ? pfx[j >> shift] : table[(j - plen) >> shift];
    }
    __device__ __forceinline__ int slot(int j, int shift) const { return (j < plen ? j : j - plen) & ((1 << shift) - 1); }
};

// Offset of key j's row of kv head h, or -1 where its page id is bad.
__device__ __forceinline__ int64_t paged_row(const PagedAttnArgs& a, const PagedKeys& ks, int j, int h) {
    const int page = ks.page(j, a.page_shift);
    if ((unsigned)page >= (unsigned)a.n_pages) {
        paged_status(a, VOX_PAGED_BAD_PAGE);
        return -1;
    }
    return page * a.page_stride + h * a.head_stride + ks.slot(j, a.page_shift) * a.slot_stride;
}

__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) < __builtin_huge_valf()); }

// ---- rows whose result is not finite ----
//
// A masked weight is 0, but 0 x inf is NaN: a result that is not finite may come from
// a value that the row does not see.  Where a CTA meets one, its warps list the keys
// among its own whose values are not all finite (paged_find_odd).  A row whose every
// such result has a value of a key that it sees behind it has the sum of those
// (paged_explain_row); one with a result that none explains is done again key by key
// (paged_redo_row).  A row whose sum of weights is NaN is NaN, whatever the values (of
// f32 see paged_rescore_row).

// (All inlined: a call anywhere in the tcgen05 kernel costs its loop 2 to 5 %.)

// A CTA's keys: blocks b0..b1-1 of those in kb, of kv head h.
struct PagedShare {
    PagedKeys ks;
    KeyBlocks kb;
    int b0, b1, h;
};
// Those with values that are not finite; more than fit are counted and left out.
constexpr int kPagedOddKeys = 32;
struct PagedOdd {
    int n, key[kPagedOddKeys];
};

// Lists the keys (odd->n is 0 before); blocks are of `keys` keys, and warp `warp` of
// `warps` takes its share.
template <class T, int E>
__device__ __forceinline__ void paged_find_odd(const PagedAttnArgs& a, const PagedShare& c, PagedOdd* odd, int keys, int warp,
                                               int warps) {
    constexpr int U = 4;  // keys at once
    const int lane = threadIdx.x & 31, total = (c.b1 - c.b0) * keys;
#pragma unroll 1
    for (int i0 = warp * U; i0 < total; i0 += warps * U) {
        int j[U];
        bool bad[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u;
            j[u] = c.kb.block(c.b0 + i / keys) * keys + i % keys;
            bad[u] = false;
            if (i < total && c.kb.seen(j[u])) {
                const int64_t off = paged_row(a, c.ks, j[u], c.h);
                if (off >= 0) {
#pragma unroll
                    for (int e = 0; e < E; ++e) bad[u] |= not_finite(to_f32(static_cast<const T*>(a.v)[off + lane + 32 * e]));
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (__any_sync(~0u, bad[u]) && lane == 0) {
                const int at = atomicAdd(&odd->n, 1);
                if (at < kPagedOddKeys) odd->key[at] = j[u];
            }
    }
}

// acc[e]: element lane + 32 e of the result of a row with index p.  Where the row
// sees values there that are not finite it becomes their sum (in any order the
// same).  Whether that explains all of them; one warp calls it.
template <class T, int E>
__device__ __forceinline__ bool paged_explain_row(const PagedAttnArgs& a, const PagedShare& c, const PagedOdd* odd, int p,
                                                  float (&acc)[E]) {
    const int lane = threadIdx.x & 31, n = min(odd->n, kPagedOddKeys);
    float sum[E] = {};
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int j = odd->key[i];
        if (!paged_sees(p, j, c.ks.len, a.window, c.ks.sinks)) continue;
        const int64_t off = paged_row(a, c.ks, j, c.h);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = to_f32(static_cast<const T*>(a.v)[off + lane + 32 * e]);
            if (not_finite(v)) sum[e] += v;
        }
        bool more = false;  // (NaN stays NaN)
#pragma unroll
        for (int e = 0; e < E; ++e) more |= not_finite(acc[e]) && sum[e] == sum[e];
        if (!__any_sync(~0u, more)) break;
    }
    bool open = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        // (a key that is not listed could turn an infinity into NaN)
        open |= not_finite(sum[e]) ? odd->n > n && sum[e] == sum[e] : not_finite(acc[e]);
        if (not_finite(sum[e])) acc[e] = sum[e];
    }
    return !__any_sync(~0u, open);
}

// One row again, key by key: acc[e] = sum of 2^(score - m) v[lane + 32 e] over
// the keys that the row sees, in blocks of `keys` keys; one warp calls it.
template <class T, int E>
__device__ __forceinline__ void paged_redo_row(const PagedAttnArgs& a, const PagedShare& c, int keys, int tok, int head, int p,
                                               float m, float (&acc)[E]) {
    const int lane = threadIdx.x & 31;
    float q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = to_f32(static_cast<const T*>(a.q)[tok * a.q_ts + head * a.q_hs + lane + 32 * e]);
        acc[e] = 0.f;
    }
    const float base = m == kNegInf ? 0.f : m;
    constexpr int U = 4;  // keys at once
#pragma unroll 1
    for (int i0 = 0, total = (c.b1 - c.b0) * keys; i0 < total; i0 += U) {
        float s[U], v[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = c.kb.block(c.b0 + (i0 + u) / keys) * keys + (i0 + u) % keys;
            const int64_t off = i0 + u < total && paged_sees(p, j, c.ks.len, a.window, c.ks.sinks) ? paged_row(a, c.ks, j, c.h) : -1;
            s[u] = off < 0 ? kNegInf : 0.f;  // a bad page: zeros, add nothing
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[u][e] = 0.f;
                if (off >= 0) {
                    s[u] = fmaf(q[e], to_f32(static_cast<const T*>(a.k)[off + lane + 32 * e]), s[u]);
                    v[u][e] = to_f32(static_cast<const T*>(a.v)[off + lane + 32 * e]);
                }
            }
        }
        for (int o = 16; o; o >>= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] += __shfl_xor_sync(~0u, s[u], o);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = fast_exp2(s[u] * a.scale_log2 - base);
            if (w == 0.f) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(w, v[u][e], acc[e]);
        }
    }
}

// One f32 row again with its scores: the halves of a key's or a query's infinity
// multiply to NaN where the score itself is an infinity (one that is -inf has no
// weight).  Sets the reference m, the sum l and acc; NaN where a score is.
template <int E>
__device__ __forceinline__ void paged_rescore_row(const PagedAttnArgs& a, const PagedShare& c, int keys, int tok, int head, int p,
                                                  float* m, float* l, float (&acc)[E]) {
    const int lane = threadIdx.x & 31;
    float q[E], top = kNegInf, sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = static_cast<const float*>(a.q)[tok * a.q_ts + head * a.q_hs + lane + 32 * e];
        acc[e] = 0.f;
    }
#pragma unroll 1
    for (int i = 0, total = (c.b1 - c.b0) * keys; i < total && sum == sum; ++i) {
        const int j = c.kb.block(c.b0 + i / keys) * keys + i % keys;
        if (!paged_sees(p, j, c.ks.len, a.window, c.ks.sinks)) continue;
        const int64_t off = paged_row(a, c.ks, j, c.h);
        float s = 0.f;
        if (off >= 0)
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(q[e], static_cast<const float*>(a.k)[off + lane + 32 * e], s);
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        s *= a.scale_log2;
        if (s == kNegInf) continue;
        const float now = fmaxf(top, s), f = fast_exp2(top - now), w = fast_exp2(s - now);
        sum = sum * f + w;
        top = now;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = off >= 0 ? static_cast<const float*>(a.v)[off + lane + 32 * e] : 0.f;
            acc[e] = w == 0.f ? acc[e] * f : fmaf(w, v, acc[e] * f);
        }
    }
    *m = top;
    *l = sum;
}

// A tile's query rows, up to 32: lane r of every warp has row r's token (-1: no
// such row), index in the keys' numbering and head within the kv head's group;
// pmin and pmax are the smallest and largest index.  Every warp finds them for
// itself, so that its first keys are asked for before any block-wide barrier.
struct PagedTileRows {
    int tok, p, g, pmin, pmax;
};
template <int ROWS>
__device__ __forceinline__ bool paged_tile_rows(const PagedAttnArgs& a, int tile, PagedTileRows& rows, PagedKeys* ks) {
    const int lane = threadIdx.x & 31;
    const int plen = a.pfx_len ? paged_prefix_len(a) : 0;
    if (plen < 0) {
        if (threadIdx.x == 0) paged_status(a, VOX_PAGED_BAD_LENGTH);
        return false;
    }
    rows.tok = rows.p = -1;
    int row;  // (the host has checked that tokens x heads fit 32 bits)
    ks->pfx = nullptr;
    ks->plen = 0;
    if (a.keys_of != PagedKeysOf::PREFIX) {
        int place;
        const int s = paged_find_tile(a, tile, ROWS, &place);
        if (s < 0) return false;
        const PagedSeq q = paged_seq(a, s);
        if (!q.ok && threadIdx.x == 0) paged_status(a, VOX_PAGED_BAD_LENGTH);
        if (q.nq == 0) return false;
        row = place * ROWS + lane;
        if (lane < ROWS && row < q.nq * a.group) {
            const int i = row / a.group;
            rows.tok = q.q0 + i;
            rows.p = q.len - q.nq + i;
        }
        ks->table = a.table + s * a.table_stride;
        if (a.keys_of == PagedKeysOf::JOINED) {
            ks->pfx = a.pfx_pages;
            ks->plen = plen;
            ks->len = plen + q.len;
            ks->sinks = a.sinks;
            if (rows.tok >= 0) rows.p += plen;
        } else {
            ks->len = q.len;
            ks->sinks = max(0, a.sinks - plen);
        }
    } else {
        row = tile * ROWS + lane;
        if (lane < ROWS && row < a.n_tokens * a.group) {
            const int t = row / a.group;
            const int s = paged_seq_of(a, t);
            if (s >= 0) {
                const PagedSeq q = paged_seq(a, s);
                if (!q.ok) paged_status(a, VOX_PAGED_BAD_LENGTH);
                if (t - q.q0 < q.nq) rows.tok = t, rows.p = plen + q.len - q.nq + (t - q.q0);
            }
        }
        ks->table = a.pfx_pages;
        ks->len = plen;
        ks->sinks = a.sinks;
    }
    rows.g = row % a.group;
    rows.pmin = __reduce_min_sync(~0u, rows.tok >= 0 ? rows.p : 0x7FFFFFFF);
    rows.pmax = __reduce_max_sync(~0u, rows.tok >= 0 ? rows.p : -0x7FFFFFFF);
    return rows.pmin <= rows.pmax;
}

// paged_seq_of for a whole warp: 32 probes at a time.
template <class A>
__device__ __forceinline__ int paged_seq_of_warp(const A& a, int t) {
    int lo = 0, n = a.n_seqs;  // the first s with q_start[s] > t lies in [lo, lo + n]
    const int lane = threadIdx.x & 31;
    while (n > 0) {
        const int step = (n + 31) >> 5;
        const int i = lane * step + step - 1;  // last of this lane's share
        const bool past = i >= n || a.q_start[lo + i] > t;
        const unsigned hit = __ballot_sync(~0u, past);
        const int c = hit ? __ffs(hit) - 1 : 32;
        if (c * step >= n) {
            lo += n;
            break;
        }
        lo += c * step;
        // a probe inside the range found its share's last entry past t already
        n = c * step + step <= n ? step - 1 : n - c * step;
    }
    return lo - 1;
}

}  // namespace vox
