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
//   warp 9     K and V tiles of 128 keys from their pages, TMA into a ring
//   warp 8     S_t = Q_t K^T and O_t += P_t V, one thread issuing tcgen05.mma
//   warps 0-3  softmax of tile 0: one thread per row
//   warps 4-7  softmax of tile 1
//
// S, P and O stay in tensor memory (S_t 128 columns, its weights P_t in 16 bits
// over the first 64 of them, O_t up to 128).  The products run in the order
// P0 V(i), Q0 K(i+1), P1 V(i), Q1 K(i+1): the tensor core executes one thread's
// products in order, so Q_t K(i+1) may overwrite P_t(i) without a wait.
//
// The running maximum of a row moves only when it rises by more than 2^8: until
// then weights are at most 2^8 (f16 holds 2^15), sums are f32, and O needs no
// rescaling; the final division by the sum takes any such factor out again.
#include <cuda.h>

#include <type_traits>

#include "vox_paged.cuh"
#include "vox_tcgen05.cuh"

namespace vox {

namespace {

constexpr int kTile = 128;  // query rows of a tile, keys of a block
constexpr int kTileThreads = 320;
constexpr uint32_t kTmemS = 0, kTmemO = 256, kTmemCols = 512;

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

// K-major or MN-major operand in 128-byte-swizzled rows.
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

// D (TMEM) (+)= A (TMEM) x B (smem)
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
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
// 128 columns: four loads in flight, one wait.
__device__ __forceinline__ void tmem_ld128(uint32_t ta, uint32_t (&r)[128]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
        "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
        "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127"
        "}, [%128];\n\ttcgen05.wait::ld.sync.aligned;"
        : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24), R8(r, 32), R8(r, 40), R8(r, 48), R8(r, 56), R8(r, 64), R8(r, 72),
          R8(r, 80), R8(r, 88), R8(r, 96), R8(r, 104), R8(r, 112), R8(r, 120)
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

struct TilesShared {
    uint64_t q_full, kv_full[6], kv_empty[6], s_full[2], p_full[2], pv_done[2], tail;
    uint32_t tmem;
    int seq, place, pmin, pmax, rows[2], failed;
};

template <class T, int HD>
__global__ void __launch_bounds__(kTileThreads, 1)
    paged_attn_tiles_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ TileMaps maps) {
    using Cfg = TilesCfg<HD>;
    constexpr int U = Cfg::UNITS;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    __shared__ TilesShared sh;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_sm = base, ring = base + 2 * Cfg::TILE_BYTES;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int z = blockIdx.x % a.splits, h = (blockIdx.x / a.splits) % a.n_kv;
    const int tile = (int)(gridDim.x / a.splits / a.n_kv) - 1 - blockIdx.x / a.splits / a.n_kv;

    // ---- which rows and keys ----
    const int plen = a.pfx_len ? paged_prefix_len(a) : 0;
    if (plen < 0) {
        if (tid == 0) paged_status(a, VOX_PAGED_BAD_LENGTH);
        return;
    }
    if (tid < 32) {
        int place = tile, s = 0;
        if (!a.in_prefix) s = paged_find_tile(a, tile, 2 * kTile, &place);
        if (tid == 0) {
            sh.seq = s;
            sh.place = place;
            sh.pmin = 0x7FFFFFFF;
            sh.pmax = -0x7FFFFFFF;
            sh.rows[0] = sh.rows[1] = sh.failed = 0;
        }
    }
    __syncthreads();
    if (sh.seq < 0) return;
    PagedKeys ks{a.pfx_pages, plen, a.sinks};
    int tok = -1, p = -1, head = 0;
    if (!a.in_prefix) {
        const PagedSeq q = paged_seq(a, sh.seq);
        if (!q.ok && tid == 0) paged_status(a, VOX_PAGED_BAD_LENGTH);
        ks.table = a.table + sh.seq * a.table_stride;
        ks.len = q.len;
        ks.sinks = max(0, a.sinks - plen);
        const int64_t row = (int64_t)sh.place * (2 * kTile) + tid;
        if (tid < 2 * kTile && row < (int64_t)q.nq * a.group) {
            const int i = (int)(row / a.group);
            tok = q.q0 + i;
            p = q.len - q.nq + i;
            head = h * a.group + (int)(row - (int64_t)i * a.group);
        }
    } else {
        const int64_t row = (int64_t)tile * (2 * kTile) + tid;
        if (tid < 2 * kTile && row < (int64_t)a.n_tokens * a.group) {
            const int t = (int)(row / a.group), s = paged_seq_of(a, t);
            if (s >= 0) {
                const PagedSeq q = paged_seq(a, s);
                if (!q.ok) paged_status(a, VOX_PAGED_BAD_LENGTH);
                if (t - q.q0 < q.nq) {
                    tok = t;
                    p = plen + q.len - q.nq + (t - q.q0);
                    head = h * a.group + (int)(row - (int64_t)t * a.group);
                }
            }
        }
    }
    {
        const int lo = __reduce_min_sync(~0u, tok >= 0 ? p : 0x7FFFFFFF);
        const int hi = __reduce_max_sync(~0u, tok >= 0 ? p : -0x7FFFFFFF);
        if (lane == 0 && lo <= hi) {
            atomicMin(&sh.pmin, lo);
            atomicMax(&sh.pmax, hi);
            sh.rows[warp >> 2] = 1;
        }
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        mbar_init(&sh.q_full, 2 * kTile);
        for (int i = 0; i < U; ++i) mbar_init(&sh.kv_full[i], 1), mbar_init(&sh.kv_empty[i], 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], kTile);
            mbar_init(&sh.pv_done[i], 1);
        }
        mbar_init(&sh.tail, 1);
        fence_barrier_init();
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = sh.tmem;
    const int pmin = sh.pmin, pmax = sh.pmax;
    const bool any = pmin <= pmax;
    const bool two = sh.rows[1];  // rows of tile 1 (tile 0 then has some, or is skipped over as zeros)
    const KeyBlocks kb = paged_key_blocks(pmin, pmax, ks.len, a.window, ks.sinks, 7);
    const int b0 = any ? (int)((int64_t)kb.total * z / a.splits) : 0;
    const int n = any ? (int)((int64_t)kb.total * (z + 1) / a.splits) - b0 : 0;

    if (warp == 9) {
        // ---- K and V tiles ----
        const int ps = 1 << a.page_shift;
        const int box = min(ps, kTile), boxes = kTile / box;
        bool ok = true;
        int issued = 0;
        for (int i = 0; i < 2 * n && ok; ++i) {
            const int slot = i % U, blk = kb.block(b0 + (i >> 1));
            if (i >= U) ok = mbar_wait(&sh.kv_empty[slot], (i / U - 1) & 1);
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            const int j0 = blk * kTile;
            // a page that ends the keys: what lies behind them in it must not reach P V
            const bool ragged = (i & 1) && j0 + kTile > kb.end && (kb.end & (box - 1));
            uint64_t* bar = ragged ? &sh.tail : &sh.kv_full[slot];
            if (lane == 0) mbar_arrive_expect_tx(bar, Cfg::TILE_BYTES);
            __syncwarp();
            if (lane < boxes) {
                const int j = j0 + lane * box;
                bool seen = j < kb.end && (j + box > kb.lo || j < kb.sinks);
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
                ok = __all_sync(~0u, mbar_wait(&sh.tail, 0));
                if (!ok) break;
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
        if (!ok) {
            // nothing may still be on its way into this CTA's memory when it ends
            if (lane == 0) atomicOr(&sh.failed, 1);
            for (int i = max(0, issued - U); i < issued; ++i) mbar_wait(&sh.kv_full[i % U], (i / U) & 1);
        }
    } else if (warp == 8) {
        // ---- products ----
        constexpr uint32_t id_qk = tiles_idesc(BF16, kTile, kTile, false), id_pv = tiles_idesc(BF16, kTile, HD, true);
        bool ok = n > 0 && mbar_wait(&sh.q_full, 0);
        auto wait_kv = [&](int i) { return mbar_wait(&sh.kv_full[i % U], (i / U) & 1); };
        auto qk = [&](int t, int i) {
            if (lane == 0) {
                const uint32_t k0 = ring + ((2 * i) % U) * Cfg::TILE_BYTES, q0 = q_sm + t * Cfg::TILE_BYTES;
#pragma unroll
                for (int x = 0; x < HD / 16; ++x) {
                    const uint32_t o = (x >> 2) * Cfg::HALF + (x & 3) * 32;
                    umma_f16(tmem + kTmemS + t * kTile, sw128_desc(q0 + o, 16, 1024), sw128_desc(k0 + o, 16, 1024), id_qk, x > 0);
                }
                umma_commit(&sh.s_full[t]);
            }
            __syncwarp();
        };
        auto pv = [&](int t, int i) {
            if (lane == 0) {
                const uint32_t v0 = ring + ((2 * i + 1) % U) * Cfg::TILE_BYTES;
#pragma unroll
                for (int x = 0; x < kTile / 16; ++x)
                    umma_f16_ts(tmem + kTmemO + t * HD, tmem + kTmemS + t * kTile + x * 8, sw128_desc(v0 + x * 2048, Cfg::HALF, 1024),
                                id_pv, i > 0 || x > 0);
                umma_commit(&sh.pv_done[t]);
            }
            __syncwarp();
        };
        auto free_unit = [&](int i) {
            // only where a later tile waits for it: no arrival may outlive the CTA
            if (lane == 0 && i + U < 2 * n) umma_commit(&sh.kv_empty[i % U]);
            __syncwarp();
        };
        if (ok && (ok = wait_kv(0))) {
            tmem_fence_after();
            qk(0, 0);
            if (two) qk(1, 0);
            free_unit(0);
        }
        for (int i = 0; i < n && ok; ++i) {
            const bool more = i + 1 < n;
            ok = wait_kv(2 * i + 1) && mbar_wait(&sh.p_full[0], i & 1);
            if (!ok) break;
            tmem_fence_after();
            pv(0, i);
            if (more) {
                ok = wait_kv(2 * i + 2);
                if (!ok) break;
                qk(0, i + 1);
            }
            if (two) {
                ok = mbar_wait(&sh.p_full[1], i & 1);
                if (!ok) break;
                tmem_fence_after();
                pv(1, i);
            }
            free_unit(2 * i + 1);
            if (more) {
                if (two) qk(1, i + 1);
                free_unit(2 * i + 2);
            }
        }
        if (!ok && n > 0 && lane == 0) atomicOr(&sh.failed, 1);
    } else {
        // ---- softmax ----
        const int t = warp >> 2, r = tid & (kTile - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t t_s = tmem + kTmemS + t * kTile + lanes, t_o = tmem + kTmemO + t * HD + lanes;
        {
            const uint32_t dst = q_sm + t * Cfg::TILE_BYTES + r * 128;
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (tok >= 0 ? tok * a.q_ts + head * a.q_hs : 0));
            uint4 v[HD / 8];
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) v[c] = tok >= 0 ? src[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < HD / 8; ++c)
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (c >> 3) * Cfg::HALF + (((c & 7) ^ (r & 7)) << 4)),
                             "r"(v[c].x), "r"(v[c].y), "r"(v[c].z), "r"(v[c].w)
                             : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&sh.q_full);
        }
        float m = kNegInf, l = 0.f;
        bool ok = true;
        const int steps = t == 0 || two ? n : 0;
        for (int i = 0; i < steps; ++i) {
            ok = mbar_wait(&sh.s_full[t], i & 1);
            if (!__all_sync(~0u, ok)) break;
            tmem_fence_after();
            uint32_t s[kTile];
            tmem_ld128(t_s, s);
            const int j0 = kb.block(b0 + i) * kTile;
            const bool all = j0 + kTile - 1 <= pmin && j0 + kTile <= ks.len &&
                             (a.window == 0 || j0 > pmax - a.window || j0 + kTile <= ks.sinks);
            if (!all) {
#pragma unroll
                for (int c = 0; c < kTile; ++c)
                    if (!paged_sees(p, j0 + c, ks.len, a.window, ks.sinks)) s[c] = 0xFF800000u;
            }
            float top[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
            for (int c = 0; c < kTile; c += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    top[e] = fmaxf(fmaxf(top[e], __uint_as_float(s[c + 2 * e])), __uint_as_float(s[c + 2 * e + 1]));
            const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2;
            const bool rise = mx > m + 8.f;
            if (i == 0) {
                m = mx;
            } else if (__any_sync(~0u, rise)) {
                const float m_new = rise ? mx : m;
                const float f = m_new == kNegInf ? 1.f : fast_exp2(m - m_new);
                l *= f;
                m = m_new;
                ok = mbar_wait(&sh.pv_done[t], (i - 1) & 1);
                if (!__all_sync(~0u, ok)) break;
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
            const float off = m == kNegInf ? 0.f : -m;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < kTile; c += 2) {
                const float x = fast_exp2(fmaf(__uint_as_float(s[c]), a.scale_log2, off));
                const float y = fast_exp2(fmaf(__uint_as_float(s[c + 1]), a.scale_log2, off));
                sum[(c >> 1) & 3] += x + y;
                s[c >> 1] = pack16<T>(x, y);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st32(t_s, s);
            tmem_st32(t_s + 32, s + 32);
            tmem_wait_st();
            tmem_fence_before();
            mbar_arrive(&sh.p_full[t]);
        }
        // ---- the result ----
        if (ok && steps > 0) ok = mbar_wait(&sh.pv_done[t], (steps - 1) & 1);
        ok = __all_sync(~0u, ok);
        if (!ok && lane == 0) atomicOr(&sh.failed, 1);
        tmem_fence_after();
        const int64_t at = ((int64_t)(a.part0 + z) * a.n_tokens + tok) * a.n_heads + head;
        const bool write = ok && tok >= 0;
        if (a.part_o && write) a.part_ml[at] = make_float2(m, l);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bool odd = false;
        if (ok) {
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
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
                odd |= !(check < __builtin_huge_valf());
                if (!write) continue;
                if (a.part_o) {
                    float4* dst = reinterpret_cast<float4*>(a.part_o + at * HD + c);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                             __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
                } else {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + c);
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        w[e] = pack16<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dst[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                }
            }
        }
        // A value that is not finite may have come from a key that the row does
        // not see (0 x inf): such rows are done again key by key.
        for (unsigned todo = __ballot_sync(~0u, odd && write); todo; todo &= todo - 1) {
            const int src = __ffs(todo) - 1;
            const int rt = __shfl_sync(~0u, tok, src), rh = __shfl_sync(~0u, head, src), rp = __shfl_sync(~0u, p, src);
            const float rm = __shfl_sync(~0u, m, src), ri = __shfl_sync(~0u, inv, src);
            float acc[HD / 32];
            paged_redo_row<T, HD / 32>(a, ks, kb, kTile, b0, b0 + n, h, rt, rh, rp, rm, acc);
            const int64_t ra = ((int64_t)(a.part0 + z) * a.n_tokens + rt) * a.n_heads + rh;
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) {
                if (a.part_o)
                    a.part_o[ra * HD + lane + 32 * e] = acc[e];
                else
                    static_cast<T*>(a.out)[rt * a.o_ts + rh * a.o_hs + lane + 32 * e] = from_f32<T>(acc[e] * ri);
            }
        }
        tmem_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        if (sh.failed) {
            // products may be in flight: let them end before their memory goes
            if (lane == 0) {
                paged_status(a, VOX_PAGED_TIMEOUT);
                mbar_init(&sh.q_full, 1);
                fence_barrier_init();
                umma_commit(&sh.q_full);
                mbar_wait(&sh.q_full, 0);
            }
            __syncwarp();
        }
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
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
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, TilesCfg<HD>::SMEM);
    if (e != cudaSuccess) return e;
    const int64_t grid = paged_tiles_bound(a, 2 * kTile) * a.n_kv * a.splits;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    k<<<(unsigned)grid, kTileThreads, TilesCfg<HD>::SMEM, st>>>(a, maps);
    return cudaGetLastError();
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

}  // namespace vox
