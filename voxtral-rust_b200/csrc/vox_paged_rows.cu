// vox_paged_rows.cu -- paged attention for few query rows per key: decode steps,
// drafted tokens, small batches behind a shared prefix, and f32 of any length.
//
// With G = n_heads / n_kv_heads rows per token, a decode step does 4 G flops
// per element of K and V: the bytes of the cache bound it, so the kernel is a
// stream of K and V rows with just enough arithmetic behind it.  A CTA takes
// 8 NT query rows (token x head of one kv head's group) and a share of the
// 16-key blocks they see.  Its warps work on blocks of their own, each with a
// private ring of cp.async units (no block-wide barrier in the loop), and
// hold the running maximum and sum of the softmax in f32:
//
//   S^T [16 keys x rows] = K Q^T      keys on the M side, so that 4..8 rows fill
//   O^T [dims x rows]   += V^T P^T    N = 8 of mma.sync instead of wasting M = 16
//
// tcgen05 has no use here: its smallest tile has 64 rows.  f16 and bf16 take
// mma.m16n8k16 with the weights rounded to the type (half a step of 2^-11 or
// 2^-8, the size of the result's own rounding; the sums are not rounded).  bf16 has
// the exponents of f32; f16 weights are taken as 2^15 times what they are beside the
// maximum, so that they keep all their bits down to 2^-29 of it (18 nats below a key
// of value 0: without, these were lost) and are off by at most 2^-40 below.  f32 takes
// mma.m16n8k8 on tf32 halves, x = hi + lo with hi rounded to 11 bits: hi hi + hi lo +
// lo hi drops lo lo, 2^-22 of the product.  The tensor core cuts its f32 sums instead
// of rounding them, so f32 sums over the keys are kept outside it: with them inside,
// results over 2400 keys were 1.7e-6 off instead of 4.7e-7.
//
// Work is split over a cluster of up to 16 CTAs per tile, whose partial results
// meet in distributed shared memory: each CTA joins a slice of the output, in
// the order of the ranks (no atomics, nothing in global memory, one launch).
// Where a cluster is not enough, clusters write parts that the merge kernel
// joins.
#include <cooperative_groups.h>

#include <type_traits>
#include <utility>

#include "vox_paged.cuh"

namespace cg = cooperative_groups;

namespace vox {

namespace {

constexpr int kKeys = 16;

// The ring of a warp holds units of one block's K or V rows, in turn; 4 warps.
// With 8 rows three CTAs share an SM, so that one's start and end lie under the
// others' copies (in a CUDA graph, 96 ragged f16 sequences 417 us with two CTAs of 6 units a warp,
// 402 us with three of 4; eight f32 streams 43 us with two of 3, 38 us with three of
// 2); with more rows the registers allow two.
template <class T, int HD, int NT>
struct RowsCfg {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int ROWS = 8 * NT;
    static constexpr int ROW_BYTES = HD * (int)sizeof(T);
    static constexpr int CHUNKS = ROW_BYTES / 16;
    static constexpr int UNIT = kKeys * ROW_BYTES;
    static constexpr int WARPS = 4;
    static constexpr int UNITS = F32 ? (HD == 128 ? 2 : 4) : (HD == 128 ? (NT == 1 ? 4 : 6) : 8);
    static constexpr int RING = WARPS * UNITS * UNIT;
    static constexpr int OS = HD + 4;  // row stride of the partial results
    static constexpr float TOP = std::is_same<T, __half>::value ? 15.f : 0.f;  // log2 of the weight at the maximum
    static constexpr int QF = F32 ? HD / 8 * NT * 512 : HD / 32 * NT * 512;
    static constexpr int BODY = RING > WARPS * ROWS * OS * 4 ? RING : WARPS * ROWS * OS * 4;
    static constexpr int SMEM = BODY + QF;
    static constexpr int PER_SM = SMEM <= 72 * 1024 && NT == 1 ? 3 : SMEM <= 108 * 1024 ? 2 : 1;
    static_assert(SMEM <= 216 * 1024, "shared memory");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;  // 0 bytes read: 16 zeros written
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int OFF>
__device__ __forceinline__ float lds32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1 + %2];" : "=f"(v) : "r"(addr), "n"(OFF) : "memory");
    return v;
}

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo with hi rounded to tf32's 11 bits (half a unit added, the rest
// cut) and lo the exact rest, at most 12 bits that begin 2^-12 below x: the tensor
// core, which ignores the low 13 bits of a word, takes 11 of them, off by at most
// 2^-23 of x.  Three full-rate instructions: the conversion instruction runs at a
// quarter of that.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
template <class F, int... I>
__device__ __forceinline__ void static_for_each(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F f) {
    static_for_each(f, std::make_integer_sequence<int, N>{});
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <class T>
__device__ __forceinline__ void store4(T* p, float4 v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = v;
    } else {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, T{}), pack2(v.z, v.w, T{}));
    }
}

template <class T, int HD, int NT>
__global__ void __launch_bounds__(32 * RowsCfg<T, HD, NT>::WARPS, RowsCfg<T, HD, NT>::PER_SM)
    paged_attn_rows_kernel(const __grid_constant__ PagedAttnArgs a) {
    using Cfg = RowsCfg<T, HD, NT>;
    constexpr bool F32 = Cfg::F32;
    constexpr int ROWS = Cfg::ROWS, U = Cfg::UNITS, UNIT = Cfg::UNIT, C = Cfg::CHUNKS, OS = Cfg::OS;
    constexpr int kWarps = Cfg::WARPS, kThreads = 32 * kWarps;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int tok_s[ROWS], head_s[ROWS], p_s[ROWS];
    __shared__ float m_s[kWarps][ROWS], l_s[kWarps][ROWS], cm_s[ROWS], cl_s[ROWS];
    __shared__ float wc_s[16][ROWS], tot_s[ROWS];
    __shared__ int odd_s[ROWS];
    __shared__ PagedOdd odd_keys;
    float* body = reinterpret_cast<float*>(smem);
    uint4* qf = reinterpret_cast<uint4*>(smem + Cfg::BODY);

    const cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_allow_dependents();
    const int unit = blockIdx.x / cs;
    const int z = unit % a.splits, h = (unit / a.splits) % a.n_kv;
    // last tiles first: a sequence's later tokens see more keys
    const int tile = (int)(gridDim.x / cs / a.splits / a.n_kv) - 1 - unit / a.splits / a.n_kv;
    PagedKeys ks;
    PagedTileRows rows;
    if (!paged_tile_rows<ROWS>(a, tile, rows, &ks)) {  // the whole cluster alike
        pdl_wait_prior_grids();
        return;
    }

    const KeyBlocks kb = paged_key_blocks(rows.pmin, rows.pmax, ks.len, a.window, ks.sinks, 4);
    int b0, b1;
    paged_part(kb.total, z * cs + rank, a.splits * cs, &b0, &b1);

    const uint32_t ring = smem_addr(smem) + warp * (U * UNIT);
    const T* const kg = static_cast<const T*>(a.k) + h * a.head_stride;
    const T* const vg = static_cast<const T*>(a.v) + h * a.head_stride;
    // this lane's key (lanes 0..15) of block i, where some row sees it
    auto wanted = [&](int i, int& j) {
        if (i >= b1 || lane >= kKeys) return false;
        j = kb.block(i) * kKeys + lane;
        return kb.seen(j);
    };
    auto page_of = [&](int i) {
        int j;
        return wanted(i, j) ? ks.page(j, a.page_shift) : 0;
    };
    // where the key begins; -1: zeros
    auto offset_of = [&](int i, int page) -> int64_t {
        int j;
        if (!wanted(i, j)) return -1;
        if ((unsigned)page >= (unsigned)a.n_pages) {
            paged_status(a, VOX_PAGED_BAD_PAGE);
            return -1;
        }
        return page * a.page_stride + ks.slot(j, a.page_shift) * a.slot_stride;
    };
    // Units go out in the order K, V of the warp's first block, K, V of the next, ...
    // A block's rows mostly follow one another (one page, all seen): their
    // addresses are then steps from the first one's, not 16 of their own.
    constexpr int E = 16 / (int)sizeof(T), RP = 32 / C;  // elements of a copy, rows of one pass of the warp
    const int cc = lane % C, cr = lane / C;
    int nxt = b0 + warp, page = page_of(nxt), out_slot = 0;
    int64_t off = -1, first = 0;
    bool out_v = false, steps = false;
    auto issue = [&](const T* base, bool is_v) {
        const uint32_t dst = ring + out_slot * UNIT;
        auto to = [&](int r) { return dst + r * Cfg::ROW_BYTES + ((cc ^ (F32 && is_v ? (r & 3) << 1 : r & 7)) << 4); };
        if (steps) {
            const T* src = base + first + cr * a.slot_stride + cc * E;
#pragma unroll
            for (int n = 0; n < kKeys / RP; ++n, src += RP * a.slot_stride) cp16(to(n * RP + cr), src, true);
        } else {
#pragma unroll
            for (int n = 0; n < kKeys / RP; ++n) {
                const int64_t o = __shfl_sync(~0u, off, n * RP + cr);
                cp16(to(n * RP + cr), base + (o >= 0 ? o : 0) + cc * E, o >= 0);
            }
        }
    };
    auto issue_next = [&]() {
        if (nxt < b1) {
            if (!out_v) {
                off = offset_of(nxt, page);
                page = page_of(nxt + kWarps);
                first = __shfl_sync(~0u, off, 0);
                steps = __all_sync(~0u, lane >= kKeys || (off >= 0 && off == first + lane * a.slot_stride));
                issue(kg, false);
            } else {
                issue(vg, true);
            }
        }
        if (out_v) nxt += kWarps;
        out_v = !out_v;
        out_slot = out_slot == U - 1 ? 0 : out_slot + 1;
        cp_commit();
    };

    // the first keys and values are on their way before the queries are asked for
#pragma unroll 1
    for (int u = 0; u < U - 1; ++u) issue_next();

    // Q^T fragments: one 16-byte word per lane and two k steps (f32: hi and lo of one)
    {
        uint32_t* w = reinterpret_cast<uint32_t*>(qf);
        for (int i = tid; i < ROWS * C; i += kThreads) {
            const int r = i / C, c = i % C;
            uint4 v = make_uint4(0, 0, 0, 0);
            const int tok = __shfl_sync(~0u, rows.tok, r), head = h * a.group + __shfl_sync(~0u, rows.g, r);
            if (tok >= 0) v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + tok * a.q_ts + head * a.q_hs + c * E);
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (F32) {
                    const int at = (((c >> 1) * NT + (r >> 3)) * 32 + (r & 7) * 4 + j) * 4 + (c & 1);
                    uint32_t hi, lo;
                    split_tf32(__uint_as_float(x[j]), hi, lo);
                    w[at] = hi;
                    w[at + 2] = lo;
                } else {
                    w[(((c >> 2) * NT + (r >> 3)) * 32 + (r & 7) * 4 + j) * 4 + (c & 3)] = x[j];
                }
            }
        }
    }
    if (tid < ROWS) tok_s[tid] = rows.tok, head_s[tid] = h * a.group + rows.g, p_s[tid] = rows.p;

    __syncthreads();

    float o[HD / 16][NT][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = kNegInf, l[n][0] = l[n][1] = 0.f;

    int slot = 0;
    for (int i = b0 + warp; i < b1; i += kWarps) {
        const int j0 = kb.block(i) * kKeys;
        issue_next();
        cp_wait<U - 1>();
        __syncwarp();
        const uint32_t kt = ring + slot * UNIT;
        slot = slot == U - 1 ? 0 : slot + 1;

        // f32 with one 8-row group: four sums, so that the products do not queue up
        float s[NT][4] = {}, s2[NT][4] = {}, s3[4] = {}, s4[4] = {};
        if constexpr (F32) {
            // chunk 2k (+ 1) ^ g: its low 3 bits are one of 8 per lane, the rest a constant
            const uint32_t at = kt + g * Cfg::ROW_BYTES + t * 4;
            uint32_t low[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) low[x] = at + ((x ^ g) << 4);
            static_for<HD / 8>([&](auto kc) {
                constexpr int k = decltype(kc)::value, far = k / 4 * 128, below = 8 * Cfg::ROW_BYTES;
                const uint32_t c0 = low[2 * k % 8], c1 = low[2 * k % 8 + 1];
                uint32_t hi[4], lo[4];
                split_tf32(lds32<far>(c0), hi[0], lo[0]);
                split_tf32(lds32<far + below>(c0), hi[1], lo[1]);
                split_tf32(lds32<far>(c1), hi[2], lo[2]);
                split_tf32(lds32<far + below>(c1), hi[3], lo[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 q = qf[(k * NT + n) * 32 + lane];
                    mma8(NT == 1 ? s3 : s2[n], lo, q.x, q.y);
                    mma8(s2[n], hi, q.z, q.w);
                    mma8(NT == 1 && k % 2 ? s4 : s[n], hi, q.x, q.y);
                }
            });
        } else {
#pragma unroll
            for (int k = 0; k < HD / 32; ++k) {
                uint32_t x[4], y[4];
                const int r = lane & 15, c = 4 * k + (lane >> 4);
                ldsm4(kt + r * Cfg::ROW_BYTES + ((c ^ (r & 7)) << 4), x);
                ldsm4(kt + r * Cfg::ROW_BYTES + (((c + 2) ^ (r & 7)) << 4), y);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 q = qf[(k * NT + n) * 32 + lane];
                    mma16(s[n], x, q.x, q.y, T{});
                    mma16(s2[n], y, q.z, q.w, T{});
                }
            }
        }
        __syncwarp();  // the unit is free
        issue_next();

        // keys j0 + g and j0 + g + 8; rows 2t and 2t + 1 of each 8
        const bool all = j0 + kKeys - 1 <= rows.pmin && j0 + kKeys <= ks.len &&
                         (a.window == 0 || j0 > rows.pmax - a.window || j0 + kKeys <= ks.sinks);
        float top[NT][2];
        bool rise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[n][x] = ((s[n][x] + s4[x]) + (s2[n][x] + s3[x])) * a.scale_log2;
                if (!all && !paged_sees(p_s[n * 8 + 2 * t + (x & 1)], j0 + g + (x >> 1) * 8, ks.len, a.window, ks.sinks))
                    s[n][x] = kNegInf;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v = fmaxf(s[n][e], s[n][e + 2]);
                v = fmaxf(v, __shfl_xor_sync(~0u, v, 4));
                v = fmaxf(v, __shfl_xor_sync(~0u, v, 8));
                v = fmaxf(v, __shfl_xor_sync(~0u, v, 16));
                top[n][e] = fmaxf(m[n][e], v);
                rise |= top[n][e] > m[n][e];
            }
        }
        if (__any_sync(~0u, rise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float f = top[n][e] == kNegInf ? 1.f : fast_exp2(m[n][e] - top[n][e]);
                    l[n][e] *= f;
                    m[n][e] = top[n][e];
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) o[d][n][e] *= f, o[d][n][e + 2] *= f;
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float base = m[n][x & 1] == kNegInf ? 0.f : m[n][x & 1] - Cfg::TOP;
                s[n][x] = fast_exp2(s[n][x] - base);
                l[n][x & 1] += s[n][x];
            }
        cp_wait<U - 1>();
        __syncwarp();
        const uint32_t vt = ring + slot * UNIT;
        slot = slot == U - 1 ? 0 : slot + 1;
        if constexpr (F32) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {  // weight of key t (+ 4) of this half, row g
                        const int src = (t + 4 * x) * 4 + (g >> 1);
                        const float w0 = __shfl_sync(~0u, s[n][2 * k], src), w1 = __shfl_sync(~0u, s[n][2 * k + 1], src);
                        split_tf32(g & 1 ? w1 : w0, bh[n][x], bl[n][x]);
                    }
                // chunk (4 d + g / 4, + 2) ^ 2t: its low 3 bits are one of 4 per lane
                const uint32_t at = vt + (k * 8 + t) * Cfg::ROW_BYTES + (g & 3) * 4;
                uint32_t low[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) low[x] = at + (((2 * x + (g >> 2)) ^ (t << 1)) << 4);
                static_for<HD / 16>([&](auto dc) {
                    constexpr int d = decltype(dc)::value, far = d / 2 * 128, below = 4 * Cfg::ROW_BYTES;
                    const uint32_t c0 = low[2 * (d & 1)], c1 = low[2 * (d & 1) + 1];
                    uint32_t hi[4], lo[4];
                    split_tf32(lds32<far>(c0), hi[0], lo[0]);
                    split_tf32(lds32<far>(c1), hi[1], lo[1]);
                    split_tf32(lds32<far + below>(c0), hi[2], lo[2]);
                    split_tf32(lds32<far + below>(c1), hi[3], lo[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float part[4] = {};
                        mma8(part, lo, bh[n][0], bh[n][1]);
                        mma8(part, hi, bl[n][0], bl[n][1]);
                        mma8(part, hi, bh[n][0], bh[n][1]);
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[d][n][x] += part[x];
                    }
                });
            }
        } else {
            uint32_t b[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                b[n][0] = transpose8x8(pack2(s[n][0], s[n][1], T{}));
                b[n][1] = transpose8x8(pack2(s[n][2], s[n][3], T{}));
            }
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                uint32_t v[4];
                const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * d + ((lane >> 3) & 1);
                ldsm4t(vt + r * Cfg::ROW_BYTES + ((c ^ (r & 7)) << 4), v);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16(o[d][n], v, b[n][0], b[n][1], T{});
            }
        }
        __syncwarp();  // the unit is free
    }
    cp_wait<0>();

    // ---- the warps' results ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[n][e] += __shfl_xor_sync(~0u, l[n][e], 4);
            l[n][e] += __shfl_xor_sync(~0u, l[n][e], 8);
            l[n][e] += __shfl_xor_sync(~0u, l[n][e], 16);
            if (g == 0) m_s[warp][n * 8 + 2 * t + e] = m[n][e] - Cfg::TOP, l_s[warp][n * 8 + 2 * t + e] = l[n][e];
        }
    __syncthreads();  // every warp's ring is used up
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                body[(warp * ROWS + n * 8 + 2 * t + (x & 1)) * OS + d * 16 + g + (x >> 1) * 8] = o[d][n][x];
    if (tid < ROWS) {
        float top = kNegInf, sum = 0.f, w[kWarps];
        for (int i = 0; i < kWarps; ++i) top = fmaxf(top, m_s[i][tid]);
        for (int i = 0; i < kWarps; ++i) {
            w[i] = top == kNegInf ? 0.f : fast_exp2(m_s[i][tid] - top);
            sum += w[i] * l_s[i][tid];
        }
        for (int i = 0; i < kWarps; ++i) m_s[i][tid] = w[i];
        cm_s[tid] = top;
        cl_s[tid] = sum;
        odd_s[tid] = 0;
    }
    if (tid == 0) odd_keys.n = 0;
    __syncthreads();
    constexpr int V4 = HD / 4;
    bool odd = false;
    for (int i = tid; i < ROWS * V4; i += kThreads) {
        const int r = i / V4, d = (i % V4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < kWarps; ++w) {
            const float f = m_s[w][r];
            const float4 x = *reinterpret_cast<const float4*>(body + (w * ROWS + r) * OS + d);
            v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
        }
        *reinterpret_cast<float4*>(body + r * OS + d) = v;
        if (not_finite((v.x + v.y) + (v.z + v.w)) && tok_s[r] >= 0 && (F32 || cl_s[r] == cl_s[r])) odd_s[r] = odd = true;
    }
    if (__syncthreads_or(odd)) {
        const PagedShare mine{ks, kb, b0, b1, h};
        paged_find_odd<T, HD / 32>(a, mine, &odd_keys, kKeys, warp, kWarps);
        __syncthreads();
#pragma unroll 1
        for (int r = warp; r < ROWS; r += kWarps) {
            if (!odd_s[r]) continue;
            float acc[HD / 32];
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) acc[e] = body[r * OS + lane + 32 * e];
            if (F32 && cl_s[r] != cl_s[r]) {
                float m_new, l_new;
                paged_rescore_row<HD / 32>(a, mine, kKeys, tok_s[r], head_s[r], p_s[r], &m_new, &l_new, acc);
                __syncwarp();
                if (lane == 0) cm_s[r] = m_new, cl_s[r] = l_new;
            } else if (!paged_explain_row<T, HD / 32>(a, mine, &odd_keys, p_s[r], acc))
                paged_redo_row<T, HD / 32>(a, mine, kKeys, tok_s[r], head_s[r], p_s[r], cm_s[r], acc);
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) body[r * OS + lane + 32 * e] = acc[e];
        }
        __syncthreads();
    }

    // ---- the cluster's, or this CTA's, result ----
    if (cs > 1) {
        cluster.sync();
        for (int i = tid; i < cs * ROWS; i += kThreads) {
            const int c = i / ROWS, r = i % ROWS;
            wc_s[c][r] = *cluster.map_shared_rank(&cm_s[r], c);
        }
        __syncthreads();
        float top = kNegInf, sum = 0.f;
        if (tid < ROWS) {
            for (int c = 0; c < cs; ++c) top = fmaxf(top, wc_s[c][tid]);
            for (int c = 0; c < cs; ++c) {
                const float f = top == kNegInf ? 0.f : fast_exp2(wc_s[c][tid] - top);
                wc_s[c][tid] = f;
                sum += f * *cluster.map_shared_rank(&cl_s[tid], c);
            }
            tot_s[tid] = sum;
            m_s[0][tid] = top;
        }
    } else if (tid < ROWS) {
        wc_s[0][tid] = 1.f;
        tot_s[tid] = cl_s[tid];
        m_s[0][tid] = cm_s[tid];
    }
    __syncthreads();
    const int i0 = ROWS * V4 * rank / cs, i1 = ROWS * V4 * (rank + 1) / cs;
    for (int i = i0 + tid; i < i1; i += kThreads) {
        const int r = i / V4, d = (i % V4) * 4, tok = tok_s[r];
        if (tok < 0) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = 0; c < cs; ++c) {
            const float f = wc_s[c][r];
            const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(body + r * OS + d, c));
            v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
        }
        const int head = head_s[r];
        const float total = tot_s[r];
        if (a.part_o) {
            const int64_t at = ((int64_t)(a.part0 + z) * a.n_tokens + tok) * a.n_heads + head;
            if (d == 0) a.part_ml[at] = make_float2(m_s[0][r], total);
            *reinterpret_cast<float4*>(a.part_o + at * HD + d) = v;
        } else {
            const float f = total == 0.f ? 0.f : 1.f / total;
            v.x *= f, v.y *= f, v.z *= f, v.w *= f;
            store4(static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + d, v);
        }
    }
    if (cs > 1) cluster.sync();  // the others may still read this CTA's results
    pdl_wait_prior_grids();      // the launch before this one ends first (PagedAttnArgs::follows)
}

template <class T, int HD, int NT>
cudaError_t launch_rows(const PagedAttnArgs& a, int cs, cudaStream_t st) {
    using Cfg = RowsCfg<T, HD, NT>;
    auto* k = paged_attn_rows_kernel<T, HD, NT>;
    static PagedKernelSetup setup;
    cudaError_t e = setup(reinterpret_cast<const void*>(k), Cfg::SMEM, true);
    if (e != cudaSuccess) return e;
    const int64_t grid = paged_tiles_bound(a, Cfg::ROWS) * a.n_kv * a.splits * cs;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(32 * Cfg::WARPS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.follows ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, a);
}

template <class T, int HD>
cudaError_t launch_rows_nt(const PagedAttnArgs& a, int nt, int cs, cudaStream_t st) {
    if (nt == 1) return launch_rows<T, HD, 1>(a, cs, st);
    if (nt == 2) return launch_rows<T, HD, 2>(a, cs, st);
    return launch_rows<T, HD, 4>(a, cs, st);
}

template <class T>
cudaError_t launch_rows_hd(const PagedAttnArgs& a, int nt, int cs, cudaStream_t st) {
    return a.hd == 128 ? launch_rows_nt<T, 128>(a, nt, cs, st) : launch_rows_nt<T, 64>(a, nt, cs, st);
}

}  // namespace

cudaError_t launch_paged_attn_rows(PagedType t, const PagedAttnArgs& a, int nt, int cluster, cudaStream_t st) {
    switch (t) {
        case PagedType::F32: return launch_rows_hd<float>(a, nt, cluster, st);
        case PagedType::F16: return launch_rows_hd<__half>(a, nt, cluster, st);
        case PagedType::BF16: return launch_rows_hd<__nv_bfloat16>(a, nt, cluster, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace vox
