// vox_paged.cu -- paged key/value cache: the append with the position rotation
// on the way, attention for any head dimension and alignment, and the joining
// of partial results.
#include "vox_paged.cuh"

namespace vox {

namespace {

// ---- append -------------------------------------------------------------------
//
// Bound by bytes (every element is read once and written once), and for a few
// tokens by latency.  A thread owns one 16-byte column of a token's rows: its
// pairs' sines and cosines are computed once, then it walks over the heads of k, v
// and q with up to 6 rows in flight, loaded before it is known where the token
// goes.  A CTA of 256 threads takes 2 tokens where there are many (fewer sines; one
// round of loads for 32 + 16 heads of 128: 8.8k tokens 58 us, 4.3 TB/s, against 62
// with 4 tokens and two rounds, 81 with one), and one where there are few (all
// heads at once: a single token 3.3 us; all in a CUDA graph).
//
// The angle a * theta^(-2c/D) matters modulo a turn only.  turns[c] is the turn
// fraction per position as a 64-bit binary fraction, so the 64-bit product with
// the position wraps exactly: the error is the position times 2^-64 of a turn,
// whatever the position, without 64-bit floating point.  sincospif takes the
// wrapped product as a signed 32-bit float (error 2^-25 of a half turn).

template <class T, bool WIDE>
struct alignas(WIDE ? 16 : sizeof(T)) AppendUnit {
    static constexpr int N = WIDE ? 16 / (int)sizeof(T) : 2;
    T v[N];
};

template <class T, bool WIDE>
__device__ __forceinline__ AppendUnit<T, WIDE> append_load(const T* p) {
    AppendUnit<T, WIDE> u;
    if constexpr (WIDE) {
        *reinterpret_cast<uint4*>(&u) = *reinterpret_cast<const uint4*>(p);
    } else {
        u.v[0] = p[0];
        u.v[1] = p[1];
    }
    return u;
}

template <class T, bool WIDE>
__device__ __forceinline__ void append_store(T* p, const AppendUnit<T, WIDE>& u) {
    if constexpr (WIDE) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&u);
    } else {
        p[0] = u.v[0];
        p[1] = u.v[1];
    }
}

// Where token t goes; one warp calls it.  For up to 32 sequences every lane
// takes one, so that all their numbers arrive together.  (More sequences are
// checked by the first CTA, whether a token belongs to them or not.)
struct AppendPlace {
    int seq, p;
    int64_t first;
    bool stored_seq;  // part of a sequence with good lengths
};
__device__ __forceinline__ AppendPlace append_place(const PagedAppendArgs& a, int t) {
    AppendPlace r{-1, 0, 0, false};
    const int lane = threadIdx.x & 31;
    PagedSeq q{};
    if (a.n_seqs <= 32) {
        if (lane < a.n_seqs) {
            q = paged_seq(a, lane);
            if (!q.ok) paged_status(a, VOX_PAGED_BAD_LENGTH);
            r.first = a.first_pos ? a.first_pos[lane] : 0;
        }
        const unsigned before = __ballot_sync(~0u, lane < a.n_seqs && q.q0 <= t);
        if (!before) return r;
        r.seq = 31 - __clz(before);
        q.q0 = __shfl_sync(~0u, q.q0, r.seq);
        q.nq = __shfl_sync(~0u, q.nq, r.seq);
        q.len = __shfl_sync(~0u, q.len, r.seq);
        q.ok = __shfl_sync(~0u, q.ok, r.seq);
        r.first = __shfl_sync(~0u, r.first, r.seq);
    } else {
        r.seq = paged_seq_of_warp(a, t);
        if (r.seq < 0) return r;
        q = paged_seq(a, r.seq);
        r.first = a.first_pos ? a.first_pos[r.seq] : 0;
    }
    r.stored_seq = q.ok && t - q.q0 < q.nq;  // else behind the last sequence, or skipped
    r.p = q.len - q.nq + (t - q.q0);
    return r;
}

template <class T, bool WIDE, int TOKENS>
__global__ void __launch_bounds__(256, 4) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
    constexpr int N = AppendUnit<T, WIDE>::N, P = N / 2, U = TOKENS > 1 ? 6 : 4, TT = 256 / TOKENS;
    const int chunks = a.hd / N, heads_at_once = TT / chunks;
    const int tid = threadIdx.x % TT;
    const int c = tid % chunks, h0 = tid / chunks;
    const int t = blockIdx.x * TOKENS + threadIdx.x / TT;
    if (TOKENS > 1 && t >= a.n_tokens) return;  // whole warps
    const int rows = 2 * a.n_kv + (a.q ? a.n_heads : 0);  // k heads, v heads, q heads
    const bool active = h0 < heads_at_once;

    AppendUnit<T, WIDE> u[U];
    const T* const kn = static_cast<const T*>(a.k_new) + t * a.kn_ts + c * N;
    const T* const vn = static_cast<const T*>(a.v_new) + t * a.vn_ts + c * N;
    const T* const qn = static_cast<const T*>(a.q) + t * a.q_ts + c * N;
    auto load = [&](int r0) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int r = r0 + i * heads_at_once;
            if (active && r < rows)
                u[i] = append_load<T, WIDE>(r < a.n_kv ? kn + r * a.kn_hs
                                                       : r < 2 * a.n_kv ? vn + (r - a.n_kv) * a.vn_hs : qn + (r - 2 * a.n_kv) * a.q_hs);
        }
    };
    load(h0);
    if (blockIdx.x == 0 && a.n_seqs > 32) {
        bool bad = false;
        for (int s = threadIdx.x; s < a.n_seqs; s += 256) bad |= !paged_seq(a, s).ok;
        if (bad) paged_status(a, VOX_PAGED_BAD_LENGTH);
    }

    const AppendPlace at = append_place(a, t);
    if (!at.stored_seq) return;
    const int p = at.p;
    int64_t slot = -1;
    if (p >= 0) {
        const int page = a.table[at.seq * a.table_stride + (p >> a.page_shift)];
        if ((unsigned)page < (unsigned)a.n_pages)
            slot = page * a.page_stride + (p & ((1 << a.page_shift) - 1)) * a.slot_stride;
        else if (tid == 0)
            paged_status(a, VOX_PAGED_BAD_PAGE);
    }
    float sn[P], cs[P];
    if (a.rotate) {
        const uint64_t pos = (uint64_t)(at.first + p);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (!active) break;
            const int64_t turn = (int64_t)(pos * a.turns[c * P + i]);
            sincospif((float)turn * 0x1p-63f, &sn[i], &cs[i]);
        }
    }
    if (!active) return;
    T* const ko = static_cast<T*>(a.k) + slot + c * N;
    T* const vo = static_cast<T*>(a.v) + slot + c * N;
    T* const qo = static_cast<T*>(a.q_out) + t * a.qo_ts + c * N;
    for (int r0 = h0; r0 < rows; r0 += U * heads_at_once) {
        if (r0 != h0) load(r0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int r = r0 + i * heads_at_once;
            if (r >= rows) break;
            const bool is_v = r >= a.n_kv && r < 2 * a.n_kv;
            if (a.rotate && !is_v) {
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const float x0 = to_f32(u[i].v[2 * j]), x1 = to_f32(u[i].v[2 * j + 1]);
                    u[i].v[2 * j] = from_f32<T>(x0 * cs[j] - x1 * sn[j]);
                    u[i].v[2 * j + 1] = from_f32<T>(x0 * sn[j] + x1 * cs[j]);
                }
            }
            T* dst;
            if (r >= 2 * a.n_kv)
                dst = qo + (r - 2 * a.n_kv) * a.qo_hs;
            else if (slot < 0)
                continue;
            else
                dst = (is_v ? vo + (r - a.n_kv) * a.head_stride : ko + r * a.head_stride);
            append_store<T, WIDE>(dst, u[i]);
        }
    }
}

// ---- attention on the CUDA cores -------------------------------------------------
//
// For head dimensions and alignments that the tensor-core kernels do not take.
// A CTA has 8 query rows (token x head of the kv head's group) and walks over
// its share of the 32-key blocks that they see, with the running maximum and
// sum of the softmax: scores by (row, key), values by dimension.  Everything is
// f32 after the load.

constexpr int kGenKeys = 32, kGenThreads = 128;

size_t general_smem(int hd) { return sizeof(float) * ((size_t)kPagedGeneralRows * hd + kGenKeys * (hd + 1) + kGenKeys * hd); }

template <class T>
__global__ void __launch_bounds__(kGenThreads) paged_attn_general_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int R = kPagedGeneralRows;
    extern __shared__ float sm[];
    const int hd = a.hd, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float* q_s = sm;                    // [R][hd]
    float* k_s = q_s + R * hd;          // [32][hd + 1]
    float* v_s = k_s + kGenKeys * (hd + 1);  // [32][hd]
    __shared__ int tok_s[R], head_s[R], p_row_s[R];
    __shared__ float p_s[R][kGenKeys], alpha_s[R], l_s[R], m_s[R];
    __shared__ int64_t off_s[kGenKeys];

    const int z = blockIdx.x % a.splits;
    const int h = (blockIdx.x / a.splits) % a.n_kv;
    const int tile = blockIdx.x / a.splits / a.n_kv;
    PagedKeys ks;
    pdl_allow_dependents();
    PagedTileRows rows;
    if (!paged_tile_rows<R>(a, tile, rows, &ks)) {
        pdl_wait_prior_grids();
        return;
    }
    if (tid < R) tok_s[tid] = rows.tok, head_s[tid] = h * a.group + rows.g, p_row_s[tid] = rows.p;
    __syncthreads();
    for (int i = tid; i < R * hd; i += kGenThreads) {
        const int r = i / hd, d = i % hd;
        float x = 0.f;
        if (tok_s[r] >= 0)
            x = to_f32(static_cast<const T*>(a.q)[tok_s[r] * a.q_ts + head_s[r] * a.q_hs + d]);
        q_s[i] = x;
    }
    const KeyBlocks kb = paged_key_blocks(rows.pmin, rows.pmax, ks.len, a.window, ks.sinks, 5);
    int b0, b1;
    paged_part(kb.total, z, a.splits, &b0, &b1);

    float acc[R][2] = {};
    float m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};  // rows warp and warp + 4
    for (int b = b0; b < b1; ++b) {
        const int j0 = kb.block(b) * kGenKeys;
        __syncthreads();  // the previous block's values are used up
        if (tid < kGenKeys) off_s[tid] = kb.seen(j0 + tid) ? paged_row(a, ks, j0 + tid, h) : -1;
        __syncthreads();
        for (int i = tid; i < kGenKeys * hd; i += kGenThreads) {
            const int j = i / hd, d = i % hd;
            const int64_t o = off_s[j];
            k_s[j * (hd + 1) + d] = o >= 0 ? to_f32(static_cast<const T*>(a.k)[o + d]) : 0.f;
            v_s[i] = o >= 0 ? to_f32(static_cast<const T*>(a.v)[o + d]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = warp + 4 * i;
            float s = 0.f;
            for (int d = 0; d < hd; ++d) s = fmaf(q_s[r * hd + d], k_s[lane * (hd + 1) + d], s);
            const bool seen = tok_s[r] >= 0 && paged_sees(p_row_s[r], j0 + lane, ks.len, a.window, ks.sinks);
            s = seen ? s * a.scale_log2 : kNegInf;
            float top = s;
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            const float m_new = fmaxf(m[i], top), base = m_new == kNegInf ? 0.f : m_new;
            const float pr = seen ? exp2f(s - base) : 0.f;
            float sum = pr;
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            const float alpha = exp2f(m[i] - base);
            l[i] = l[i] * alpha + sum;
            m[i] = m_new;
            p_s[r][lane] = pr;
            if (lane == 0) alpha_s[r] = alpha;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = tid + e * kGenThreads;
            if (d < hd) {
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r][e] *= alpha_s[r];
                for (int j = 0; j < kGenKeys; ++j) {
                    const float x = v_s[j * hd + d];
#pragma unroll
                    for (int r = 0; r < R; ++r) {  // a weight of 0 takes nothing from a value, finite or not
                        const float pr = p_s[r][j];
                        acc[r][e] = pr != 0.f ? fmaf(pr, x, acc[r][e]) : acc[r][e];
                    }
                }
            }
        }
    }
    if (lane == 0) {
        l_s[warp] = l[0], l_s[warp + 4] = l[1];
        m_s[warp] = m[0], m_s[warp + 4] = m[1];
    }
    __syncthreads();
    for (int r = 0; r < R; ++r) {
        const int tok = tok_s[r];
        if (tok < 0) continue;
        const int head = head_s[r];
        const float ls = l_s[r];
        const int64_t at = ((int64_t)(a.part0 + z) * a.n_tokens + tok) * a.n_heads + head;
        if (a.part_o && tid == 0) a.part_ml[at] = make_float2(m_s[r], ls);
        for (int e = 0; e < 2; ++e) {
            const int d = tid + e * kGenThreads;
            if (d >= hd) break;
            if (a.part_o)
                a.part_o[at * hd + d] = acc[r][e];
            else
                static_cast<T*>(a.out)[tok * a.o_ts + head * a.o_hs + d] = from_f32<T>(ls == 0.f ? 0.f : acc[r][e] / ls);
        }
    }
    pdl_wait_prior_grids();  // the launch before this one ends first (PagedAttnArgs::follows)
}

// ---- joining partial results -----------------------------------------------------
//
// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, in the order of the
// parts; one warp per (token, head).  Bound by reading the parts, and for few
// rows by latency: a lane takes one part's (m, l), and the parts' results are
// loaded eight at a time before the first is used.  A part whose sum is 0 is
// not read.  V: head_dim / 32 where that is 2 or 4 (a lane's elements are then
// contiguous), 0 for any other.

template <class T, int V>
__global__ void __launch_bounds__(128) paged_merge_kernel(const __grid_constant__ PagedAttnArgs a, int n_parts) {
    constexpr int E = V ? V : kPagedMaxHeadDim / 32;
    const int64_t n_rows = (int64_t)a.n_tokens * a.n_heads;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int tok = row / a.n_heads, head = row % a.n_heads;
    bool mine = row < n_rows && !(a.pfx_len && paged_prefix_len(a) < 0);
    if (mine) {
        const int s = paged_seq_of_warp(a, tok);
        const PagedSeq q = s >= 0 ? paged_seq(a, s) : PagedSeq{};
        mine = s >= 0 && tok - q.q0 < q.nq;
    }
    pdl_wait_prior_grids();
    if (!mine) return;
    float top = kNegInf;
    for (int i = lane; i < n_parts; i += 32) top = fmaxf(top, a.part_ml[i * n_rows + row].x);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float base = top == kNegInf ? 0.f : top;
    float total = 0.f, acc[E] = {};
    for (int i0 = 0; i0 < n_parts; i0 += 32) {
        float w = 0.f, l = 0.f;
        if (i0 + lane < n_parts) {
            const float2 ml = a.part_ml[(i0 + lane) * n_rows + row];
            l = ml.y;
            w = l == 0.f ? 0.f : exp2f(ml.x - base);
        }
        const unsigned used = __ballot_sync(~0u, l != 0.f);
        const int n = min(32, n_parts - i0);
        for (int i1 = 0; i1 < n; i1 += 8) {
            float x[8][E];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool take = i1 + i < n && (used >> (i1 + i) & 1);
                const float* o = a.part_o + ((i0 + i1 + i) * n_rows + row) * a.hd;
#pragma unroll
                for (int e = 0; e < E; ++e) x[i][e] = 0.f;
                if (V == 4) {
                    if (take) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(o + lane * 4);
                } else if (V == 2) {
                    if (take) *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(o + lane * 2);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (take && lane + 32 * e < a.hd) x[i][e] = o[lane + 32 * e];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = __shfl_sync(~0u, w, (i1 + i) & 31);
                const float g = __shfl_sync(~0u, l, (i1 + i) & 31);
                if (i1 + i >= n) break;
                total = fmaf(f, g, total);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(f, x[i][e], acc[e]);
            }
        }
    }
    T* out = static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs;
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = V ? lane * V + e : lane + 32 * e;
        if (V || d < a.hd) out[d] = from_f32<T>(acc[e] * inv);
    }
}

template <class F>
cudaError_t by_type(PagedType t, F f) {
    switch (t) {
        case PagedType::F32: return f(float{});
        case PagedType::F16: return f(__half{});
        case PagedType::BF16: return f(__nv_bfloat16{});
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_paged_append(PagedType t, const PagedAppendArgs& a, bool wide, cudaStream_t st) {
    return by_type(t, [&](auto x) {
        using T = decltype(x);
        // 2 tokens to a CTA once that still leaves four CTAs to every SM
        if (wide && a.n_tokens >= 2 * 4 * 148)
            paged_append_kernel<T, true, 2><<<(a.n_tokens + 1) / 2, 256, 0, st>>>(a);
        else if (wide)
            paged_append_kernel<T, true, 1><<<a.n_tokens, 256, 0, st>>>(a);
        else
            paged_append_kernel<T, false, 1><<<a.n_tokens, 256, 0, st>>>(a);
        return cudaGetLastError();
    });
}

cudaError_t launch_paged_attn_general(PagedType t, const PagedAttnArgs& a, cudaStream_t st) {
    const int64_t grid = paged_tiles_bound(a, kPagedGeneralRows) * a.n_kv * a.splits;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    const size_t smem = general_smem(a.hd);
    return by_type(t, [&](auto x) {
        auto* k = paged_attn_general_kernel<decltype(x)>;
        static PagedKernelSetup setup;
        cudaError_t e = setup(reinterpret_cast<const void*>(k), (int)general_smem(kPagedMaxHeadDim), false);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3(kGenThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = a.follows ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, k, a);
    });
}

cudaError_t launch_paged_merge(PagedType t, const PagedAttnArgs& a, int n_parts, cudaStream_t st) {
    const int64_t grid = ((int64_t)a.n_tokens * a.n_heads + 3) / 4;
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
    return by_type(t, [&](auto x) {
        using T = decltype(x);
        if (a.hd == 128) return cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, 4>, a, n_parts);
        if (a.hd == 64) return cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, 2>, a, n_parts);
        return cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, 0>, a, n_parts);
    });
}

}  // namespace vox
