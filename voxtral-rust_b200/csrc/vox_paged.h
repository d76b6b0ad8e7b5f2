// vox_paged.h -- what the paged-cache host file (vox_paged.cpp) and its kernels
// (vox_paged*.cu) share: launch arguments and launchers.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include <atomic>
#include <stdint.h>

namespace vox {

enum class PagedType : int { F32, F16, BF16 };

constexpr int kPagedMaxHeadDim = 256;

enum class PagedKeysOf : int { OWN, PREFIX, JOINED };

// Arguments of every paged attention kernel.  Counts and token indices are
// 32 bits (the host checks them); every offset into a tensor is 64 bits.
struct PagedAttnArgs {
    // pool
    const void* k;
    const void* v;
    int64_t page_stride, head_stride, slot_stride;
    int n_pages, page_shift, n_kv, hd;
    // batch
    int n_seqs, n_tokens, max_q, max_kv, table_width;
    int64_t table_stride;
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* table;
    uint32_t* status;
    // shared prefix (pfx_len null: none), and which keys a launch attends to:
    // each sequence's own, the prefix's (the rows are then all tokens of the
    // batch), or for each sequence the prefix's and then its own.
    const int32_t* pfx_pages;
    const int32_t* pfx_len;
    int pfx_n_pages, pfx_max;
    PagedKeysOf keys_of;
    // queries and outputs
    const void* q;
    int64_t q_ts, q_hs;
    void* out;
    int64_t o_ts, o_hs;
    int n_heads, group;
    float scale_log2;   // score scale * log2(e): softmax runs on powers of two
    int window, sinks;  // window 0 = none
    // partial results (part_o null: the kernel writes `out`).  This launch
    // writes the parts part0 .. part0 + splits - 1 of [part][token][head].
    float* part_o;
    float2* part_ml;  // (what weights are taken relative to, in log2 units; their sum)
    int part0, splits;
    // tcgen05 kernel: the first `whole` (tile, kv head) units of the launch are not
    // split and write `out`; where there are others behind them, they write their
    // parts as [unit - whole][part][row of the tile] and launch_paged_tail_merge
    // joins those.  -1: `splits` holds for all.
    int whole;
    // 1: the launch may start before the one in front of it in the stream, an
    // attention kernel over other keys of the same call, has ended (programmatic
    // dependent launch); it reads nothing of that one and waits for it at its
    // end, so that whatever waits for this launch has waited for both.
    int follows;
    // tcgen05 kernel: polls after which a wait gives up (seconds, by default), and K and
    // V tiles that a CTA asks for at most (all, outside tests of the first)
    int wait_polls, copy_units;
};
constexpr int kPagedWaitPolls = 1 << 22;

// Upper bound on the tiles of `rows` query rows, from the host's bounds alone.
inline int64_t paged_tiles_bound(const PagedAttnArgs& a, int rows) {
    if (a.keys_of == PagedKeysOf::PREFIX) return ((int64_t)a.n_tokens * a.group + rows - 1) / rows;
    const int64_t all = (int64_t)a.n_tokens * a.group / rows + a.n_seqs;
    const int64_t each = (int64_t)a.n_seqs * (((int64_t)a.max_q * a.group + rows - 1) / rows);
    return all < each ? all : each;
}

struct PagedAppendArgs {
    void* k;
    void* v;
    int64_t page_stride, head_stride, slot_stride;
    int n_pages, page_shift, n_kv, hd;
    int n_seqs, n_tokens, max_q, max_kv, table_width;
    int64_t table_stride;
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* table;
    const int64_t* first_pos;
    uint32_t* status;
    const void *k_new, *v_new, *q;
    void* q_out;
    int64_t kn_ts, kn_hs, vn_ts, vn_hs, q_ts, q_hs, qo_ts, qo_hs;
    int n_heads, rotate;
    // theta^(-2c/hd) / (2 pi) as a 64-bit binary fraction of a turn
    uint64_t turns[kPagedMaxHeadDim / 2];
};

// A kernel's limits are raised once per device (a call to the runtime for each
// launch costs as much as the launch).  One object per kernel.
class PagedKernelSetup {
  public:
    cudaError_t operator()(const void* kernel, int smem_bytes, bool wide_cluster) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = uint64_t(1) << (dev & 63);
        if (dev < 64 && (done_.load(std::memory_order_acquire) & bit)) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
        if (e == cudaSuccess && wide_cluster) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
        return e;
    }

  private:
    std::atomic<uint64_t> done_{0};
};

cudaError_t launch_paged_append(PagedType t, const PagedAppendArgs& a, bool wide, cudaStream_t st);

// CUDA-core attention: any head_dim and alignment (vox_paged.cu).
cudaError_t launch_paged_attn_general(PagedType t, const PagedAttnArgs& a, cudaStream_t st);
constexpr int kPagedGeneralRows = 8;  // query rows (token x head of a group) of a CTA

// Tensor-core attention for few rows per key (vox_paged_rows.cu): head_dim 64 or
// 128, every row on a 16-byte boundary; nt (1, 2, 4) x 8 query rows per tile,
// `cluster` (1..16) CTAs per tile and part.
cudaError_t launch_paged_attn_rows(PagedType t, const PagedAttnArgs& a, int nt, int cluster, cudaStream_t st);

// tcgen05 attention for many rows per key (vox_paged_tiles.cu): f16 and bf16,
// head_dim 64 or 128, pages of at least 8 slots, every row on a 16-byte boundary.
cudaError_t launch_paged_attn_tiles(PagedType t, const PagedAttnArgs& a, cudaStream_t st);
constexpr int kPagedTileRows = 256;  // query rows of a CTA

// Joins the parts of the units behind the first a.whole of `units` (vox_paged_tiles.cu).
cudaError_t launch_paged_tail_merge(PagedType t, const PagedAttnArgs& a, int units, cudaStream_t st);

// Joins n_parts partial results into `out` (vox_paged.cu).
cudaError_t launch_paged_merge(PagedType t, const PagedAttnArgs& a, int n_parts, cudaStream_t st);

}  // namespace vox
