// vox_paged_tiles.cu -- paged attention for many query rows per key, on tcgen05:
// prompts, chunks of long prompts, and batches behind a shared prefix.
//
// 4 D flops per (row, key) pair and nothing re-read per row: bound by the tensor
// cores' products and, close behind, by the exponentials (128 x 128 scores take
// 1024 cycles of special-function throughput and 1024 of products at D = 128).
// A CTA has two tiles of 128 query rows (token x head of one kv head's group)
// that share every K and V tile, so that one tile's softmax runs while the
// other's products do:
//
//   warp 10      K and V tiles of 128 keys from their pages, TMA into a ring
//   warps 8, 9   S_t = Q_t K^T and O_t += P_t V of tile 0 and 1, one thread each
//                issuing tcgen05.mma (from one thread for both, a tile's products
//                wait behind the other tile's softmax)
//   warps 0-3    softmax of tile 0: one thread per row
//   warps 4-7    softmax of tile 1
//
// S, P and O stay in tensor memory: O_t up to 128 columns, and for each tile two
// score buffers of 64 keys, their 16-bit weights over the first 32 columns.  A
// softmax works on one buffer while the other is filled again:
//
//   P_t V(k), then Q_t K(k + 2) into the same columns (one thread's products
//   execute in order, so no wait lies between the two)
//
// What this avoids: with one buffer of 128 keys per tile, a tile's softmax, P V
// and Q K follow one another, and each hand-over through an mbarrier takes 150 to
// 250 cycles: 3800 cycles per block of 128 keys against 2048 of products.  The
// price: at 64 keys (N = 64) Q K reads 6 KB of shared memory per 32 cycles of
// product and takes 48, so that a block's products are 2560 cycles at D = 128.
// Measured: 3200 to 3400 cycles per block of 128 keys and pair of tiles, of which
// a softmax step's exponentials are 590 alone and 1040 beside the other tile's;
// 9000 cycles before a CTA's first scores and 5000 after its last products.  In a CUDA
// graph two 2048-token chunks over 24 k and 32 k tokens (window 8192, 551 GFLOP) take
// 499 us, 1.10 PFLOP/s (a call among others 582: the card's power bounds it), and six
// prompts of 300 to 2500 tokens (151 GFLOP) 203 us.
//
// Measured and not kept: 1 to 3 of 8 pairs of exponentials as polynomials on the
// FMA pipe (2 % faster to 5 % slower at D = 64, up to 8 % slower at 128); one score
// buffer of 128 keys that both tiles use in turn (5 % slower).
//
// A row's weights are 2^(score - m).  Its reference m, the running maximum once,
// moves up only when 64 new weights add up to more than 2^8: until then each is at
// most 2^8, sums are f32, and O needs no rescaling; the final division by the sum
// takes any such factor out again.  So a step of the common kind costs one FMA, one
// exponential, one addition and half a conversion per score, and looks for no
// maximum.  Weights are rounded to the tensors' type (the sums are not): half a
// step of 2^-8 or 2^-11 of each.  bf16 has the exponents of f32.  f16 has not: below
// 2^-14 its steps stay 2^-24, so there m is the maximum less 2^8, weights add up to at
// most 65504, and where a step's add up to less than 2^-4 (keys far below one with
// nearly all of the weight, whose own value may be 0) m moves down to that step's
// maximum.  What is still rounded more coarsely is a key beside one that is over 2^22
// times its weight in the same 64: by up to 2^-33 of that one's.  (The long chunk
// takes 499 us in a CUDA graph, 496 without the step down, which loses keys 18 nats
// below a sink.)
#include <cuda.h>

#include <type_traits>

#include "vox_paged.cuh"
#include "vox_tcgen05.cuh"

namespace vox {

namespace {

constexpr int kTile = 128;  // query rows of a tile, keys of a block
constexpr int kTileThreads = 352;
constexpr int kStep = 64;         // keys of a softmax step
constexpr int kStageBytes = 32 * 128;  // a softmax warp's results on their way out
// Log2 of the weight at a row's maximum when the reference is set by it, and the
// sums of a step's weights above and (f16) below which the reference moves.
template <class T>
struct TilesRange {
    static constexpr bool F16 = std::is_same<T, __half>::value;
    static constexpr float TOP = F16 ? 8.f : 0.f, RISE = F16 ? 65504.f : 256.f, FALL = 0x1p-4f;
    static constexpr uint32_t LEAST = (127u - 60u) << 23;  // 2^-60's bits: sums below are not looked at
};
constexpr uint32_t kTmemO = 0, kTmemS = 256, kTmemCols = 512;  // S_t buffer b at kTmemS + (2 t + b) 64

template <int HD>
struct TilesCfg {
    static constexpr int UNITS = HD == 128 ? 4 : 6;          // K or V tiles in the ring
    static constexpr int TILE_BYTES = kTile * HD * 2;        // a Q, K or V tile
    static constexpr int HALF = kTile * 128;                 // 64 dims of a tile: rows of 128 bytes
    static constexpr int SMEM = (2 + UNITS) * TILE_BYTES + 1024;
};

// Tensor maps of the pool: (dim, slot, head, page).
struct alignas(64) TileMaps {
    CUtensorMap k, v;
};

// K-major or MN-major operand in 128-byte-swizzled rows.  Moving on by o bytes
// adds o >> 4 (the address field is 14 bits, shared memory ends below 2^18): the
// issuing thread builds a descriptor once per tile, since at 64 cycles a product
// a dozen instructions in front of each would set the pace.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Instruction descriptor of kind::f16 (f32 accumulators): A and B f16 or bf16,
// b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t tiles_idesc(bool bf16, int m, int n, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

// Products and commits of one thread of a converged warp (`leader` is 1 in that
// thread): predicated, not branched to, so that the warp's descriptors stay in
// uniform registers.  Behind a branch every product waits for its operands to be
// moved there, about 110 cycles instead of the 64 it takes to execute.
__device__ __forceinline__ uint32_t elect_leader() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r));
    return r;
}
// D (TMEM) (+)= A (smem) x B (smem)
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
// D (TMEM) (+)= A (TMEM) x B (smem)
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
        "r"(leader)
        : "memory");
}
// Waits are bounded by their number of polls (each up to the hardware's own
// suspension of a few microseconds): no clock is read on the way.  The first poll
// comes before the limit is looked at (2 % of the long chunk).
__device__ __forceinline__ bool tiles_wait(uint64_t* bar, uint32_t parity, int polls) {
    if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
    for (int i = 1; i < polls; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}

__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page,
                                              uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

#define R8(a, o) "=r"(a[o]), "=r"(a[o + 1]), "=r"(a[o + 2]), "=r"(a[o + 3]), "=r"(a[o + 4]), "=r"(a[o + 5]), "=r"(a[o + 6]), "=r"(a[o + 7])
#define I8(a, o) "r"(a[o]), "r"(a[o + 1]), "r"(a[o + 2]), "r"(a[o + 3]), "r"(a[o + 4]), "r"(a[o + 5]), "r"(a[o + 6]), "r"(a[o + 7])

// 32 consecutive columns of this thread's lane (the outputs exist after the wait inside).
__device__ __forceinline__ void tmem_ld32(uint32_t ta, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24)
        : "r"(ta)
        : "memory");
}
// 64 columns, likewise.
__device__ __forceinline__ void tmem_ld64(uint32_t ta, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
        : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24), R8(r, 32), R8(r, 40), R8(r, 48), R8(r, 56)
        : "r"(ta)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t ta, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(ta),
        I8(r, 0), I8(r, 8), I8(r, 16), I8(r, 24)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <class T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint64_t pack_f2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Scores of 64 keys that a row does not see become -inf.  p, len, window and
// sinks are counted from the first of them.
__device__ __forceinline__ void tiles_mask(uint32_t* s, int p, int len, int window, int sinks) {
    const int hi = min(p, len - 1), lo = window ? p - window : -1;
#pragma unroll
    for (int c = 0; c < 64; ++c)
        if (c > hi || (c <= lo && c >= sinks)) s[c] = 0xFF800000u;
}

// Weights 2^(scale s + off) of the 64 scores s, packed into w.  Returns their
// sum.  In groups of G: a group's exponentials go out before the last group's
// results are used, so that their latency is covered without a second warp.
template <class T>
__device__ __forceinline__ float tiles_weights(const uint32_t* s, uint32_t* w, float scale, float off) {
    constexpr int G = 16, N = 64 / G;
    const uint64_t sc = pack_f2(scale, scale), of = pack_f2(off, off);
    uint64_t sum[2] = {0, 0};
    float x[N][G];
#pragma unroll
    for (int g = 0; g <= N; ++g) {
        if (g < N) {
#pragma unroll
            for (int c = 0; c < G; c += 2)
                unpack_f2(fma_f2(pack_f2(__uint_as_float(s[g * G + c]), __uint_as_float(s[g * G + c + 1])), sc, of), x[g][c], x[g][c + 1]);
#pragma unroll
            for (int c = 0; c < G; ++c) asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(x[g][c]));
        }
        if (g > 0) {
#pragma unroll
            for (int c = 0; c < G; c += 2) {
                const float a = x[g - 1][c], b = x[g - 1][c + 1];
                sum[(c >> 1) & 1] = add_f2(sum[(c >> 1) & 1], pack_f2(a, b));
                w[((g - 1) * G + c) >> 1] = pack16<T>(a, b);
            }
        }
    }
    float s0, s1, s2, s3;
    unpack_f2(sum[0], s0, s1);
    unpack_f2(sum[1], s2, s3);
    return (s0 + s1) + (s2 + s3);
}

struct TilesShared {
    uint64_t q_full[2], kv_full[6], kv_empty[6], s_full[2][2], p_full[2][2], pv_done[2][2], tail, drained[2];
    uint32_t tmem;
    int lo[8], hi[8];  // smallest and largest index of a warp's rows
    int failed;
    // for rows that are not finite (here, so that no register holds it meanwhile)
    PagedShare share;
    PagedOdd odd;
    unsigned odd_lanes[8];
};

// A row whose result, already written, is not finite (paged_find_odd).
struct OddRow {
    int64_t at;  // where the result begins
    int tok, head, p;
    float m, inv;
};
// The CTA's odd rows; all its warps call it.  Softmax warp w has left those of its
// lanes in `lanes[w]` where it staged its results, in the memory of its tile's queries.
template <class T, int HD>
__device__ __forceinline__ void tiles_mend_rows(const PagedAttnArgs& a, const PagedShare& share, PagedOdd* list,
                                                const unsigned* lanes, const unsigned char* queries, bool to_part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    paged_find_odd<T, HD / 32>(a, share, list, kTile, warp, kTileThreads / 32);
    __syncthreads();
    if (warp >= 8) return;
    const OddRow* rows = reinterpret_cast<const OddRow*>(queries + (warp >> 2) * TilesCfg<HD>::TILE_BYTES + (warp & 3) * kStageBytes);
#pragma unroll 1
    for (unsigned todo = lanes[warp]; todo; todo &= todo - 1) {
        const OddRow r = rows[__ffs(todo) - 1];
        float acc[HD / 32];
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) {
            const int64_t at = r.at + lane + 32 * e;
            acc[e] = to_part ? a.part_o[at] : to_f32(static_cast<T*>(a.out)[at]);
        }
        if (!paged_explain_row<T, HD / 32>(a, share, list, r.p, acc)) {
            paged_redo_row<T, HD / 32>(a, share, kTile, r.tok, r.head, r.p, r.m, acc);
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) acc[e] *= to_part ? 1.f : r.inv;
        }
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) {
            const int64_t at = r.at + lane + 32 * e;
            if (to_part)
                a.part_o[at] = acc[e];
            else
                static_cast<T*>(a.out)[at] = from_f32<T>(acc[e]);
        }
    }
}

template <class T, int HD>
__global__ void __launch_bounds__(kTileThreads, 1)
    paged_attn_tiles_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ TileMaps maps) {
    using Cfg = TilesCfg<HD>;
    constexpr int U = Cfg::UNITS;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    using Range = TilesRange<T>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ TilesShared sh;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_sm = base, ring = base + 2 * Cfg::TILE_BYTES;

    const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;
    // unit: (tile, kv head), the last tiles first: a sequence's later tokens see more keys
    int z, unit, splits = a.splits, units;
    if (a.whole < 0) {
        unit = blockIdx.x / splits;
        z = blockIdx.x - unit * splits;
        units = gridDim.x / splits;
    } else {
        const int behind = (int)blockIdx.x - a.whole;
        units = a.whole + ((int)gridDim.x - a.whole) / splits;
        unit = behind < 0 ? blockIdx.x : a.whole + behind / splits;
        z = behind < 0 ? 0 : behind % splits;
        if (behind < 0) splits = 1;
    }
    const int h = unit % a.n_kv, tile = units / a.n_kv - 1 - unit / a.n_kv;
    const bool to_part = a.part_o && (a.whole < 0 || unit >= a.whole);

    // ---- which rows and keys ----
    pdl_allow_dependents();
    const int plen = a.pfx_len ? paged_prefix_len(a) : 0;
    if (plen < 0) {
        if (tid == 0) paged_status(a, VOX_PAGED_BAD_LENGTH);
        pdl_wait_prior_grids();
        return;
    }
    // every warp looks for itself: one block-wide barrier in the whole prologue
    int place = tile, seq = 0;
    if (a.keys_of == PagedKeysOf::OWN) seq = paged_find_tile(a, tile, 2 * kTile, &place);
    if (seq < 0) {
        pdl_wait_prior_grids();
        return;
    }
    PagedKeys ks{a.pfx_pages, plen, a.sinks, nullptr, 0};
    int tok = -1, p = -1, head = 0;
    if (a.keys_of == PagedKeysOf::OWN) {
        const PagedSeq q = paged_seq(a, seq);
        if (!q.ok && tid == 0) paged_status(a, VOX_PAGED_BAD_LENGTH);
        ks.table = a.table + seq * a.table_stride;
        ks.len = q.len;
        ks.sinks = max(0, a.sinks - plen);
        const int row = place * (2 * kTile) + tid;
        if (tid < 2 * kTile && row < q.nq * a.group) {
            const int i = row / a.group;
            tok = q.q0 + i;
            p = q.len - q.nq + i;
            head = h * a.group + row - i * a.group;
        }
    } else {
        const int row = tile * (2 * kTile) + tid;
        if (tid < 2 * kTile && row < a.n_tokens * a.group) {
            const int t = row / a.group, s = paged_seq_of(a, t);
            if (s >= 0) {
                const PagedSeq q = paged_seq(a, s);
                if (!q.ok) paged_status(a, VOX_PAGED_BAD_LENGTH);
                if (t - q.q0 < q.nq) {
                    tok = t;
                    p = plen + q.len - q.nq + (t - q.q0);
                    head = h * a.group + row - t * a.group;
                }
            }
        }
    }
    // The queries are asked for before anything is set up: a warp's 32 rows, each
    // 16-byte column by a lane (a thread reading its own row would touch 32 lines
    // at a time: 7000 cycles instead of 2000).
    constexpr int QC = HD / 8, QR = 32 / QC;  // columns of a row, rows at once
    uint4 qv[32 / QR];
    if (warp < 8) {
#pragma unroll
        for (int i = 0; i < 32 / QR; ++i) {
            const int r = i * QR + lane / QC;
            const int rt = __shfl_sync(~0u, tok, r), rh = __shfl_sync(~0u, head, r);
            qv[i] = make_uint4(0, 0, 0, 0);
            if (rt >= 0)
                qv[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + rt * a.q_ts + rh * a.q_hs + (lane % QC) * 8);
        }
        const int lo = __reduce_min_sync(~0u, tok >= 0 ? p : 0x7FFFFFFF);
        const int hi = __reduce_max_sync(~0u, tok >= 0 ? p : -0x7FFFFFFF);
        if (lane == 0) sh.lo[warp] = lo, sh.hi[warp] = hi;
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 10 * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
        sh.failed = 0;
        mbar_init(&sh.q_full[0], 4);  // one arrival a warp
        mbar_init(&sh.q_full[1], 4);
        for (int i = 0; i < U; ++i) mbar_init(&sh.kv_full[i], 1), mbar_init(&sh.kv_empty[i], 2);  // both tiles are done with it
        for (int t = 0; t < 2; ++t)
            for (int b = 0; b < 2; ++b) {
                mbar_init(&sh.s_full[t][b], 1);
                mbar_init(&sh.p_full[t][b], 4);  // one arrival a warp
                mbar_init(&sh.pv_done[t][b], 1);
            }
        mbar_init(&sh.tail, 1);
        mbar_init(&sh.drained[0], 1);
        mbar_init(&sh.drained[1], 1);
        fence_barrier_init();
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, sh.tmem, 0);
    int pmin = 0x7FFFFFFF, pmax = -0x7FFFFFFF;
    bool two = false;  // tile 1 has rows (tile 0 then has some, or counts as zeros)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        pmin = min(pmin, sh.lo[i]);
        pmax = max(pmax, sh.hi[i]);
        two |= i >= 4 && sh.lo[i] <= sh.hi[i];
    }
    const bool any = pmin <= pmax;
    const KeyBlocks kb = paged_key_blocks(pmin, pmax, ks.len, a.window, ks.sinks, 7);
    int b0 = 0, n = 0;
    if (any) {
        paged_part(kb.total, z, splits, &b0, &n);
        n -= b0;
    }

    if (tid == 0) sh.share = PagedShare{ks, kb, b0, b0 + n, h}, sh.odd.n = 0;

    // Bounded waits: of a thread, and of a whole warp with one answer.
    auto wait = [&](uint64_t* bar, uint32_t parity) { return tiles_wait(bar, parity, a.wait_polls); };
    auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(~0u, wait(bar, parity)); };
    bool odd = false;
    if (warp == 10) {
        // ---- K and V tiles ----
        const int ps = 1 << a.page_shift;
        const int box = min(ps, kTile), boxes = kTile / box;
        bool ok = true;
        const int units = min(2 * n, a.copy_units);
        int issued = 0;
        for (int i = 0; i < units && ok; ++i) {
            const int slot = i % U, blk = kb.block(b0 + (i >> 1));
            if (i >= U) ok = warp_wait(&sh.kv_empty[slot], (i / U - 1) & 1);
            if (!ok) break;
            const int j0 = blk * kTile;
            // a page that ends the keys: what lies behind them in it must not reach P V
            const bool ragged = (i & 1) && j0 + kTile > kb.end && (kb.end & (box - 1));
            uint64_t* bar = ragged ? &sh.tail : &sh.kv_full[slot];
            if (lane == 0) mbar_arrive_expect_tx(bar, Cfg::TILE_BYTES);
            __syncwarp();
            if (lane < boxes) {
                const int j = j0 + lane * box;
                bool seen = kb.any_seen(j, box);
                int page = seen ? ks.table[j >> a.page_shift] : -1;
                if (seen && (unsigned)page >= (unsigned)a.n_pages) {
                    paged_status(a, VOX_PAGED_BAD_PAGE);
                    seen = false;
                }
                if (!seen) page = a.n_pages;  // outside the tensor: zeros
                const uint32_t dst = ring + slot * Cfg::TILE_BYTES + lane * box * 128;
#pragma unroll
                for (int x = 0; x < HD / 64; ++x)
                    tma_load_page(dst + x * Cfg::HALF, (i & 1) ? &maps.v : &maps.k, x * 64, j & (ps - 1), h, page, bar);
            }
            issued = i + 1;
            if (ragged) {
                ok = warp_wait(&sh.tail, 0);
                if (!ok) {
                    tiles_wait(&sh.tail, 0, kPagedWaitPolls);
                    issued = i;
                    break;
                }
                const int r0 = kb.end - j0, r1 = (r0 + box - 1) & ~(box - 1);
                for (int e = lane; e < (r1 - r0) * (HD / 8); e += 32) {
                    const int r = r0 + e / (HD / 8), c = e % (HD / 8);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + slot * Cfg::TILE_BYTES +
                                                                                 (c >> 3) * Cfg::HALF + r * 128 + (c & 7) * 16),
                                 "r"(0)
                                 : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.kv_full[slot]);
            }
        }
        if (!ok && lane == 0) atomicOr(&sh.failed, 1);
        // Nothing may still be on its way into this CTA's memory when it ends, whichever
        // wait it was that expired (a unit that `tail` stood for has been waited for).
        for (int i = max(0, issued - U); i < issued; ++i) tiles_wait(&sh.kv_full[i % U], (i / U) & 1, kPagedWaitPolls);
    } else if (warp >= 8) {
        // ---- products of tile t ----
        const int t = warp - 8, steps = t == 0 || two ? n : 0;
        constexpr uint32_t id_qk = tiles_idesc(BF16, kTile, kStep, false), id_pv = tiles_idesc(BF16, kTile, HD, true);
        const uint32_t leader = elect_leader();
        bool ok = steps > 0 && warp_wait(&sh.q_full[t], 0);
        auto wait_kv = [&](int i) { return warp_wait(&sh.kv_full[i % U], (i / U) & 1); };
        const uint64_t q_desc = sw128_desc(q_sm, 16, 1024), k_desc = sw128_desc(ring, 16, 1024),
                       v_desc = sw128_desc(ring, Cfg::HALF, 1024);
        const uint64_t qd = q_desc + t * (Cfg::TILE_BYTES >> 4);
        const uint32_t t_o = tmem + kTmemO + t * HD, t_s = tmem + kTmemS + t * (2 * kStep);
        auto qk = [&](int half, uint64_t kd) {
#pragma unroll
            for (int x = 0; x < HD / 16; ++x) {
                const uint32_t o = ((x >> 2) * Cfg::HALF + (x & 3) * 32) >> 4;
                umma_ss(leader, t_s + half * kStep, qd + o, kd + half * (kStep * 128 >> 4) + o, id_qk, x > 0);
            }
            umma_commit_if(leader, &sh.s_full[t][half]);
        };
        auto pv = [&](int half, uint64_t vd, uint32_t more) {
#pragma unroll
            for (int x = 0; x < kStep / 16; ++x)
                umma_ts(leader, t_o, t_s + half * kStep + x * 8, vd + (((half * kStep + x * 16) * 128) >> 4), id_pv, x > 0 ? 1u : more);
            umma_commit_if(leader, &sh.pv_done[t][half]);
        };
        auto unit = [&](uint64_t desc, int i) { return desc + (i % U) * (Cfg::TILE_BYTES >> 4); };
        // only where a later tile waits for it: no arrival may outlive the CTA
        auto free_unit = [&](int i) {
            if (i + U >= 2 * n) return;
            umma_commit_if(leader, &sh.kv_empty[i % U]);
            if (!two) umma_commit_if(leader, &sh.kv_empty[i % U]);
        };
        if (ok && (ok = wait_kv(0))) {
            tmem_fence_after();
            qk(0, k_desc);
            qk(1, k_desc);
            free_unit(0);
        }
#pragma unroll 1
        for (int i = 0; i < steps && ok; ++i) {
            const bool next = i + 1 < n;
            const uint64_t vd = unit(v_desc, 2 * i + 1), kd = unit(k_desc, 2 * i + 2);
            ok = wait_kv(2 * i + 1) && (!next || wait_kv(2 * i + 2));
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                ok = ok && warp_wait(&sh.p_full[t][half], i & 1);
                if (!ok) break;
                tmem_fence_after();
                pv(half, vd, i > 0 || half > 0);
                if (next) qk(half, kd);
            }
            free_unit(2 * i + 1);
            free_unit(2 * i + 2);
        }
        if (!ok && steps > 0 && lane == 0) atomicOr(&sh.failed, 1);
        // No product may be in flight when its memory goes, whichever wait expired: the
        // thread that issued them commits them.
        umma_commit_if(leader, &sh.drained[t]);
        tiles_wait(&sh.drained[t], 0, kPagedWaitPolls);
    } else {
        // ---- softmax ----
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t t_s = tmem + kTmemS + t * (2 * kStep) + lanes, t_o = tmem + kTmemO + t * HD + lanes;
#pragma unroll
        for (int i = 0; i < 32 / QR; ++i) {
            const int r = (warp & 3) * 32 + i * QR + lane / QC, c = lane % QC;
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_sm + t * Cfg::TILE_BYTES + (c >> 3) * Cfg::HALF +
                                                                         r * 128 + (((c & 7) ^ (r & 7)) << 4)),
                         "r"(qv[i].x), "r"(qv[i].y), "r"(qv[i].z), "r"(qv[i].w)
                         : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full[t]);
        float m = tok >= 0 ? kNegInf : 0.f, l = 0.f;
        bool ok = true;
        const int steps = t == 0 || two ? 2 * n : 0;
#pragma unroll 1
        for (int k = 0; k < steps; ++k) {
            ok = warp_wait(&sh.s_full[t][k & 1], (k >> 1) & 1);
            if (!ok) break;
            tmem_fence_after();
            const uint32_t buf = t_s + (k & 1) * kStep;
            uint32_t s[kStep], w[kStep / 2];
            const int j0 = kb.block(b0 + (k >> 1)) * kTile + (k & 1) * kStep;
            const bool all = j0 + kStep - 1 <= pmin && j0 + kStep <= ks.len &&
                             (a.window == 0 || j0 > pmax - a.window || j0 + kStep <= ks.sinks);
            tmem_ld64(buf, s);
            if (!all) tiles_mask(s, p - j0, ks.len - j0, a.window, ks.sinks - j0);
            // The weights are taken with the reference so far, and are on their way before
            // it is known whether that was right.  Only where their sum says that a score
            // may have risen far above it (the first steps, mostly), or for f16 that all are
            // far below it (2^-60 of it and more: the sums' range is f32's), is the maximum
            // looked for and the weights taken again.
            float l_new = 0.f;
            if (k > 0) {
                l_new = tiles_weights<T>(s, w, a.scale_log2, m == kNegInf ? 0.f : -m);
                tmem_st32(buf, w);
            }
            bool fell = Range::F16 && __float_as_uint(l_new) - Range::LEAST < __float_as_uint(Range::FALL) - Range::LEAST;
            if (k == 0 || __any_sync(~0u, l_new > Range::RISE || m == kNegInf || fell)) {
                tmem_wait_st();
                float mx = kNegInf;
#pragma unroll
                for (int c = 0; c < kStep; c += 2) mx = max3(mx, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                const float want = mx * a.scale_log2 - Range::TOP;
                if constexpr (Range::F16) fell = fell && l * fast_exp2(m - want) < 0x1p90f;
                const float m_new = fell ? want : fmaxf(m, want);
                const float f = m_new == kNegInf ? 1.f : fast_exp2(m - m_new);
                m = m_new;
                l *= f;
                if (k > 0) {
                    ok = warp_wait(&sh.pv_done[t][(k - 1) & 1], ((k - 1) >> 1) & 1);
                    if (!ok) break;
                    tmem_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(t_o + c, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(t_o + c, o);
                    }
                }
                l_new = tiles_weights<T>(s, w, a.scale_log2, m == kNegInf ? 0.f : -m);
                tmem_st32(buf, w);
            }
            l += l_new;
            tmem_wait_st();
            tmem_fence_before();
            __syncwarp();
            // 128 arrivals on one barrier would queue up for about 200 cycles
            if (lane == 0) mbar_arrive(&sh.p_full[t][k & 1]);
        }
        // ---- the result ----
        if (ok && steps > 0) ok = warp_wait(&sh.pv_done[t][1], (n - 1) & 1);
        if (!ok && lane == 0) atomicOr(&sh.failed, 1);
        tmem_fence_after();
        const int64_t at = a.whole < 0 ? ((int64_t)(a.part0 + z) * a.n_tokens + tok) * a.n_heads + head
                                       : ((int64_t)(unit - a.whole) * splits + z) * (2 * kTile) + tid;
        const bool write = ok && tok >= 0;
        if (to_part && write) a.part_ml[at] = make_float2(m, l);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        // The rows go through the tile's queries' memory (all products with them are
        // done), 32 floats or 64 results of a row at a time, so that a store covers
        // 128 bytes of a row; the 16-byte columns are swizzled by the row.
        const uint32_t stage = q_sm + t * Cfg::TILE_BYTES + (warp & 3) * kStageBytes;
        const int64_t row_at = to_part ? at * HD : tok * a.o_ts + head * a.o_hs;
        const int width = to_part ? 32 : 64;  // elements of 128 bytes
        if (ok) {
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += width) {
#pragma unroll 1
                for (int c = c0; c < c0 + width; c += 32) {
                    uint32_t o[32];
                    if (steps > 0) {
                        tmem_ld32(t_o + c, o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
                    float check = 0.f;
#pragma unroll
                    for (int e = 0; e < 32; ++e) check += fabsf(__uint_as_float(o[e]));
                    odd |= not_finite(check);
                    if (!to_part) {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = pack16<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (to_part || e < 4)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 +
                                                                                         ((((c - c0) / 8 + e) ^ (lane & 7)) << 4)),
                                         "r"(o[4 * e]), "r"(o[4 * e + 1]), "r"(o[4 * e + 2]), "r"(o[4 * e + 3])
                                         : "memory");
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = i * 4 + lane / 8, e = lane % 8;
                    const int64_t ra = __shfl_sync(~0u, row_at, r);
                    const bool rw = __shfl_sync(~0u, write, r);
                    uint4 v;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                 : "r"(stage + r * 128 + ((e ^ (r & 7)) << 4))
                                 : "memory");
                    if (rw) {
                        if (to_part)
                            *reinterpret_cast<uint4*>(a.part_o + ra + c0 + e * 4) = v;
                        else
                            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + ra + c0 + e * 8) = v;
                    }
                }
                __syncwarp();
            }
        }
        // (what is left of a row is kept where its warp staged the results)
        odd = odd && write && l == l;
        const unsigned lanes_odd = __ballot_sync(~0u, odd);
        if (lane == 0) sh.odd_lanes[warp] = lanes_odd;
        if (odd) reinterpret_cast<OddRow*>(smem_raw + (stage - smem_addr(smem_raw)))[lane] = OddRow{row_at, tok, head, p, m, inv};
        tmem_fence_before();
    }
    if (__syncthreads_or(odd))
        tiles_mend_rows<T, HD>(a, sh.share, &sh.odd, sh.odd_lanes, smem_raw + (q_sm - smem_addr(smem_raw)), to_part);
    if (tid == 0 && sh.failed) paged_status(a, VOX_PAGED_TIMEOUT);
    if (warp == 8) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
    pdl_wait_prior_grids();  // the launch before this one ends first (PagedAttnArgs::follows)
}

// Joins the parts of a split unit; one warp per row of its tile.
template <class T, int HD>
__global__ void __launch_bounds__(128) paged_tail_merge_kernel(const __grid_constant__ PagedAttnArgs a, int units) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31, per = 2 * kTile / 4;
    const int behind = blockIdx.x / per, unit = a.whole + behind, r = (blockIdx.x - behind * per) * 4 + (threadIdx.x >> 5);
    const int h = unit % a.n_kv, tile = units / a.n_kv - 1 - unit / a.n_kv;
    int place, tok = -1, head = 0;
    const int s = paged_find_tile(a, tile, 2 * kTile, &place);
    if (s >= 0) {
        const PagedSeq q = paged_seq(a, s);
        const int row = place * (2 * kTile) + r;
        if (row < q.nq * a.group) {
            tok = q.q0 + row / a.group;
            head = h * a.group + row % a.group;
        }
    }
    pdl_wait_prior_grids();
    if (tok < 0) return;
    const int64_t at = (int64_t)behind * a.splits * (2 * kTile) + r;
    float top = kNegInf;
    for (int z = 0; z < a.splits; ++z) top = fmaxf(top, a.part_ml[at + z * (2 * kTile)].x);
    const float base = top == kNegInf ? 0.f : top;
    float total = 0.f, acc[E] = {};
#pragma unroll 4
    for (int z = 0; z < a.splits; ++z) {
        const float2 ml = a.part_ml[at + z * (2 * kTile)];
        const float f = ml.y == 0.f ? 0.f : fast_exp2(ml.x - base);
        if (ml.y == 0.f) continue;
        total = fmaf(f, ml.y, total);
        const float* o = a.part_o + (at + z * (2 * kTile)) * HD + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(f, o[e], acc[e]);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    T* out = static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = from_f32<T>(acc[e] * inv);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn tensor_map_encoder() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

template <class T, int HD>
cudaError_t launch_tiles(const PagedAttnArgs& a, const TileMaps& maps, cudaStream_t st) {
    auto* k = paged_attn_tiles_kernel<T, HD>;
    static PagedKernelSetup setup;
    cudaError_t e = setup(reinterpret_cast<const void*>(k), TilesCfg<HD>::SMEM, false);
    if (e != cudaSuccess) return e;
    const int64_t units = paged_tiles_bound(a, 2 * kTile) * a.n_kv;
    const int64_t grid = a.whole < 0 ? units * a.splits : a.whole + (units - a.whole) * a.splits;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = TilesCfg<HD>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = a.follows ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k, a, maps);
}

}  // namespace

cudaError_t launch_paged_attn_tiles(PagedType t, const PagedAttnArgs& a, cudaStream_t st) {
    EncodeFn encode = tensor_map_encoder();
    if (!encode) return cudaErrorNotSupported;
    TileMaps maps;
    const int ps = 1 << a.page_shift;
    const cuuint64_t dims[4] = {(cuuint64_t)a.hd, (cuuint64_t)ps, (cuuint64_t)a.n_kv, (cuuint64_t)a.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)a.slot_stride * 2, (cuuint64_t)a.head_stride * 2, (cuuint64_t)a.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(ps < kTile ? ps : kTile), 1, 1}, ones[4] = {1, 1, 1, 1};
    const CUtensorMapDataType dt = t == PagedType::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = 0; i < 2; ++i)
        if (encode(i ? &maps.v : &maps.k, dt, 4, const_cast<void*>(i ? a.v : a.k), dims, strides, box, ones,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    if (t == PagedType::F16)
        return a.hd == 128 ? launch_tiles<__half, 128>(a, maps, st) : launch_tiles<__half, 64>(a, maps, st);
    return a.hd == 128 ? launch_tiles<__nv_bfloat16, 128>(a, maps, st) : launch_tiles<__nv_bfloat16, 64>(a, maps, st);
}

cudaError_t launch_paged_tail_merge(PagedType t, const PagedAttnArgs& a, int units, cudaStream_t st) {
    const int64_t grid = (int64_t)(units - a.whole) * (2 * kTile / 4);
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (t == PagedType::F16)
        return a.hd == 128 ? cudaLaunchKernelEx(&cfg, paged_tail_merge_kernel<__half, 128>, a, units)
                           : cudaLaunchKernelEx(&cfg, paged_tail_merge_kernel<__half, 64>, a, units);
    return a.hd == 128 ? cudaLaunchKernelEx(&cfg, paged_tail_merge_kernel<__nv_bfloat16, 128>, a, units)
                       : cudaLaunchKernelEx(&cfg, paged_tail_merge_kernel<__nv_bfloat16, 64>, a, units);
}

}  // namespace vox
