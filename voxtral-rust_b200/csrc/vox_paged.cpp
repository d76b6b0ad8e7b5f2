// vox_paged.cpp -- host side of the paged key/value cache: checks the
// arguments, plans the launch from the host's bounds (never from device data)
// and launches.  Nothing is allocated and nothing is kept between calls.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>

#include "../../include/vox_decoder.h"
#include "vox_host.h"
#include "vox_paged.h"

using namespace vox;

namespace {

#define TRY(expr)                      \
    do {                               \
        int rc_ = (expr);              \
        if (rc_ != VOX_OK) return rc_; \
    } while (0)

// Makes the cache's device current for the call.
class DeviceGuard {
  public:
    int enter(int device) {
        // An error left by earlier work: reported once, not mistaken for one of this call.
        // (Without a driver every call of the runtime answers so.)
        const cudaError_t earlier = cudaGetLastError();
        if (earlier != cudaSuccess && earlier != cudaErrorInsufficientDriver && earlier != cudaErrorNoDevice)
            return report_errorf(VOX_ERR_CUDA, "an earlier CUDA error was pending on this thread (%s); nothing was launched",
                                 cudaGetErrorString(earlier));
        if (cudaGetDevice(&before_) != cudaSuccess) return no_device(device);
        if (before_ != device) {
            if (cudaSetDevice(device) != cudaSuccess) return no_device(device);
            switched_ = true;
        }
        return VOX_OK;
    }
    ~DeviceGuard() {
        if (switched_) cudaSetDevice(before_);
    }

  private:
    static int no_device(int device) {
        const char* why = cudaGetErrorString(cudaGetLastError());
        return report_errorf(VOX_ERR_CUDA, "cannot use device %d: %s", device, why);
    }
    int before_ = 0;
    bool switched_ = false;
};

int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return VOX_OK;
    (void)cudaGetLastError();
    return report_errorf(VOX_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}

int shift_of(size_t n) {
    int s = 0;
    while ((size_t(1) << s) < n) ++s;
    return s;
}

size_t type_size(PagedType t) { return t == PagedType::F32 ? 4 : 2; }

struct Checked {
    PagedType type;
    int64_t page_stride, head_stride, slot_stride;
    int page_shift;
};

constexpr float kLog2e = 1.4426950408889634f;

constexpr size_t kMaxCount = INT32_MAX / 4;  // tokens, sequences, pages

std::atomic<int> wait_polls{kPagedWaitPolls}, copy_units{INT32_MAX};

int check_cache(const vox_paged_cache* c, Checked* out) {
    if (!c) return report_errorf(VOX_ERR_INVALID_ARG, "null cache");
    switch (c->dtype) {
        case VOX_DT_F32: out->type = PagedType::F32; break;
        case VOX_DT_F16: out->type = PagedType::F16; break;
        case VOX_DT_BF16: out->type = PagedType::BF16; break;
        default: return report_errorf(VOX_ERR_UNSUPPORTED, "cache dtype must be f32, f16 or bf16");
    }
    if (!c->keys || !c->values) return report_errorf(VOX_ERR_INVALID_ARG, "null keys or values");
    if (c->n_pages == 0 || c->n_pages > kMaxCount || c->n_kv_heads == 0 || c->n_kv_heads > 4096)
        return report_errorf(VOX_ERR_INVALID_ARG, "n_pages and n_kv_heads (at most 4096) must be > 0");
    if (c->page_size == 0 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return report_errorf(VOX_ERR_UNSUPPORTED, "page_size must be a power of two in 1..1024");
    if (c->head_dim == 0 || c->head_dim % 2 || c->head_dim > (size_t)kPagedMaxHeadDim)
        return report_errorf(VOX_ERR_UNSUPPORTED, "head_dim must be even and at most %d", kPagedMaxHeadDim);
    out->page_shift = shift_of(c->page_size);
    if (!c->page_stride && !c->head_stride && !c->slot_stride) {
        out->slot_stride = c->head_dim;
        out->head_stride = c->head_dim * c->page_size;
        out->page_stride = out->head_stride * c->n_kv_heads;
    } else {
        if (c->slot_stride < c->head_dim || c->head_stride < c->head_dim ||
            (c->n_pages > 1 && c->page_stride < c->head_dim) ||
            std::max({c->page_stride, c->head_stride, c->slot_stride}) > (size_t(1) << 40))
            return report_errorf(VOX_ERR_SHAPE, "cache strides must be at least head_dim");
        out->page_stride = c->page_stride;
        out->head_stride = c->head_stride;
        out->slot_stride = c->slot_stride;
    }
    const size_t mis = type_size(out->type) - 1;
    if (((uintptr_t)c->keys | (uintptr_t)c->values) & mis)
        return report_errorf(VOX_ERR_INVALID_ARG, "keys or values are not aligned to their type");
    return VOX_OK;
}

int check_batch(const vox_paged_cache* c, const vox_paged_batch* b) {
    if (!b) return report_errorf(VOX_ERR_INVALID_ARG, "null batch");
    if (b->n_seqs > kMaxCount || b->n_tokens > kMaxCount || b->max_kv_len > kMaxCount || b->table_width > kMaxCount ||
        b->table_stride > (size_t(1) << 40))
        return report_errorf(VOX_ERR_UNSUPPORTED, "batch sizes must be at most %d", (int)kMaxCount);
    if (b->n_seqs == 0 || b->n_tokens == 0) return VOX_OK;
    if (!b->q_start || !b->kv_len || (b->table_width && !b->page_table))
        return report_errorf(VOX_ERR_INVALID_ARG, "null q_start, kv_len or page_table");
    if (b->max_q_len == 0 || b->max_q_len > b->n_tokens)
        return report_errorf(VOX_ERR_SHAPE, "max_q_len must be in 1..n_tokens");
    if (b->max_kv_len > b->table_width * c->page_size)
        return report_errorf(VOX_ERR_SHAPE, "max_kv_len needs more pages than the table has columns");
    if (b->n_seqs > 1 && b->table_stride < b->table_width)
        return report_errorf(VOX_ERR_SHAPE, "table_stride must be at least table_width");
    return VOX_OK;
}

// Whether rows of `hd` elements at multiples of the strides are kept apart by them:
// sorted, each stride steps over all that the smaller ones reach.
struct Dim {
    size_t n, stride;
};
bool rows_apart(std::initializer_list<Dim> dims, size_t hd) {
    Dim d[3];
    size_t n = 0;
    for (const Dim& x : dims)
        if (x.n > 1) d[n++] = x;
    std::sort(d, d + n, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    unsigned __int128 reach = hd;
    for (size_t i = 0; i < n; ++i) {
        if (d[i].stride < reach) return false;
        reach += (unsigned __int128)(d[i].n - 1) * d[i].stride;
    }
    return true;
}

// [n_tokens, heads, head_dim] rows: strides, alignment to the type.  Rows that
// are written must not overlap.
int check_rows(const vox_rows* r, const char* name, size_t tokens, size_t heads, size_t hd, PagedType t, bool written,
               int64_t* ts, int64_t* hs) {
    if (!r || !r->ptr) return report_errorf(VOX_ERR_INVALID_ARG, "null %s", name);
    if ((uintptr_t)r->ptr & (type_size(t) - 1))
        return report_errorf(VOX_ERR_INVALID_ARG, "%s is not aligned to its type", name);
    if (!r->token_stride && !r->head_stride) {
        *ts = (int64_t)(heads * hd);
        *hs = (int64_t)hd;
        return VOX_OK;
    }
    if (std::max(r->token_stride, r->head_stride) > (size_t(1) << 40))
        return report_errorf(VOX_ERR_SHAPE, "%s strides out of range", name);
    if (written && !rows_apart({{tokens, r->token_stride}, {heads, r->head_stride}}, hd))
        return report_errorf(VOX_ERR_SHAPE, "%s strides must be at least head_dim and keep its rows apart", name);
    *ts = (int64_t)r->token_stride;
    *hs = (int64_t)r->head_stride;
    return VOX_OK;
}

bool aligned16(const void* p, PagedType t, std::initializer_list<int64_t> strides) {
    if ((uintptr_t)p & 15) return false;
    for (int64_t s : strides)
        if ((s * (int64_t)type_size(t)) & 15) return false;
    return true;
}

template <class A>
void fill_common(A& a, const vox_paged_cache* c, const Checked& k, const vox_paged_batch* b) {
    a.page_stride = k.page_stride;
    a.head_stride = k.head_stride;
    a.slot_stride = k.slot_stride;
    a.n_pages = (int)c->n_pages;
    a.page_shift = k.page_shift;
    a.n_kv = (int)c->n_kv_heads;
    a.hd = (int)c->head_dim;
    a.n_seqs = (int)b->n_seqs;
    a.n_tokens = (int)b->n_tokens;
    a.max_q = (int)b->max_q_len;
    a.max_kv = (int)b->max_kv_len;
    a.table_width = (int)b->table_width;
    a.table_stride = (int64_t)b->table_stride;
    a.q_start = b->q_start;
    a.kv_len = b->kv_len;
    a.table = b->page_table;
    a.status = b->status;
}

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

// How one set of keys (the sequences' own, or the prefix) is attended to.  It
// follows from the host's bounds and the head dimension alone; a call whose
// tensors are not on 16-byte boundaries takes the CUDA-core kernel with the
// same splits.
struct KeysPlan {
    enum Kernel { GENERAL, ROWS, TILES } kernel = GENERAL;
    int nt = 1, cluster = 1, splits = 1;
    int whole = -1, units = 0;  // TILES: see PagedAttnArgs::whole
};

// `rows`: query rows that share their keys (a sequence's, or all); `all_rows`:
// tokens x heads; `tiles(n)`: tiles of n rows; `keys`: keys that a row can see;
// `alike`: no merge follows anyway, and the tiles see about as many keys each.
template <class F>
KeysPlan plan_keys(const vox_paged_cache* c, PagedType t, int64_t rows, int64_t all_rows, int64_t keys, bool alike, F tiles) {
    KeysPlan p;
    const bool fits = c->head_dim == 64 || c->head_dim == 128;
    // tcgen05 tiles have 128 rows: from 32 rows on they win although part of
    // them is empty (the rows' kernel reads K and V again for every 32 rows)
    if (fits && rows > 32 && t != PagedType::F32 && c->page_size >= 8) {
        p.kernel = KeysPlan::TILES;
        const int64_t units = std::max<int64_t>(1, tiles(kPagedTileRows) * (int64_t)c->n_kv_heads);
        // The split that ends first: waves of CTAs (one per SM) times a CTA's blocks
        // of 128 keys, and about 3 blocks' time to start and end one, plus writing
        // and reading a part of every row (a block takes about 2 us, in which the
        // memory moves 13 MB).  Many more tiles than SMs even out by themselves
        // (the longest are first).
        const int64_t blocks = (keys + 127) / 128;
        const double part = 8.0 * (double)all_rows * (double)c->head_dim / 13e6;
        double best = 0;
        for (int64_t z = 1; z <= std::min<int64_t>(64, std::max<int64_t>(1, blocks / 2)); ++z) {
            if (z > 1 && units >= 3 * 148) break;
            const double t = (double)((units * z + 147) / 148) * (double)((blocks + z - 1) / z + 3) + (z > 1 ? part * (double)z : 0.0);
            if (z == 1 || t < best) best = t, p.splits = (int)z;
        }
        // A last wave that leaves at least half of the SMs empty: only its tiles are
        // split, over all SMs (512 tiles of 65 blocks, 3.46 waves: 508 us in a CUDA
        // graph instead of 553); joining them costs about 2 blocks' time.
        const int64_t last = units % 148;
        if (alike && units > 148 && last > 0 && last <= 74) {
            const int64_t z = std::min<int64_t>(148 / last, blocks / 2);
            const double t2 = (double)(units / 148) * (double)(blocks + 3) + (double)((blocks + z - 1) / std::max<int64_t>(z, 1) + 5);
            if (z > 1 && t2 < best) p.splits = (int)z, p.whole = (int)(units - last), p.units = (int)units;
        }
        return p;
    }
    if (fits) p.kernel = KeysPlan::ROWS;
    p.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    const int64_t units = std::max<int64_t>(1, tiles(fits ? 8 * p.nt : kPagedGeneralRows) * (int64_t)c->n_kv_heads);
    // CTAs that run at once.  Fewer tiles than that are split into one wave of
    // equal parts; more, where the bytes bound the call (one decode step's rows),
    // into about eight waves, which evens out ragged lengths: 96 sequences of up
    // to 8192 visible keys 400 us in a CUDA graph, 413 with two CTAs a tile.
    const int64_t slots = 148 * (p.nt == 1 ? 3 : 2);
    const int64_t wanted = units < slots ? slots / units : p.nt == 1 ? (8 * slots + units - 1) / units : 1;
    // At least 64 keys to a CTA of a cluster, 512 where there are enough tiles
    // without, or where the parts go through the merge (one stream of 1536 tokens:
    // 8.5 us in a CUDA graph through clusters alone, 9.6 with a merge behind them).
    int64_t parts = std::max<int64_t>(1, std::min<int64_t>(wanted, keys / (units < slots ? 64 : 512)));
    if (fits)
        while (p.cluster < 16 && 2 * p.cluster <= parts) p.cluster *= 2;
    parts = std::min<int64_t>(parts / p.cluster, keys / 512 / p.cluster);
    p.splits = (int)std::min<int64_t>(std::max<int64_t>(1, parts), 64);
    return p;
}

// What a call launches.
struct AttnPlan {
    KeysPlan own, prefix;
    bool joined = false;   // the prefix as the first part of every sequence's keys
    int parts = 1;         // partial results of a row
    bool partial = false;  // through the workspace
    size_t ml_bytes = 0, bytes = 0;
};

AttnPlan plan_attention(const vox_paged_cache* c, PagedType t, const vox_paged_batch* b, const vox_paged_prefix* p,
                        size_t n_heads, size_t window, size_t sinks) {
    AttnPlan plan;
    const int64_t group = (int64_t)(n_heads / c->n_kv_heads), all_rows = (int64_t)(b->n_tokens * n_heads);
    auto visible = [&](size_t len) {
        return (int64_t)(window && window < len ? std::min(len, window + b->max_q_len + std::min(sinks, len)) : len);
    };
    PagedAttnArgs a{};
    a.n_tokens = (int)b->n_tokens;
    a.n_seqs = (int)b->n_seqs;
    a.max_q = (int)b->max_q_len;
    a.group = (int)group;
    const int64_t rows = (int64_t)b->max_q_len * group;
    // A short prefix is read again for every sequence, out of the L2, as the first
    // part of its keys: one launch where the shared form takes three (8 hypotheses
    // behind 639 tokens: 10 us in a CUDA graph against 19).  32 MB are about 4 us of it.
    plan.joined = p && rows <= 32 &&
                  (double)b->n_seqs * (double)p->max_len * (double)(c->n_kv_heads * c->head_dim * 2 * type_size(t)) <= 32e6;
    const int64_t keys = visible(b->max_kv_len + (plan.joined ? p->max_len : 0));
    // a long past or a window in front of few new tokens
    const bool alike = !p && keys >= 3 * (int64_t)b->max_q_len;
    plan.own = plan_keys(c, t, rows, all_rows, keys, alike, [&](int n) { return paged_tiles_bound(a, n); });
    plan.parts = plan.own.splits;
    if (p && !plan.joined) {
        a.keys_of = PagedKeysOf::PREFIX;
        plan.prefix = plan_keys(c, t, (int64_t)b->n_tokens * group, all_rows, visible(p->max_len), false,
                                [&](int n) { return paged_tiles_bound(a, n); });
        plan.parts += plan.prefix.splits;
    }
    plan.partial = plan.parts > 1;
    if (plan.partial) {
        const size_t n = plan.own.whole >= 0 ? (size_t)(plan.own.units - plan.own.whole) * plan.own.splits * kPagedTileRows
                                             : (size_t)plan.parts * (size_t)all_rows;
        plan.ml_bytes = round256(n * sizeof(float2));
        plan.bytes = plan.ml_bytes + n * c->head_dim * sizeof(float);
    }
    return plan;
}

cudaError_t launch_keys(PagedType t, PagedAttnArgs& a, const KeysPlan& p, bool aligned, cudaStream_t st) {
    a.splits = p.splits;
    a.whole = -1;
    if (p.kernel == KeysPlan::TILES && aligned && std::max({a.page_stride, a.head_stride, a.slot_stride}) < (int64_t(1) << 39)) {
        a.whole = p.whole;
        return launch_paged_attn_tiles(t, a, st);
    }
    // (no room in the workspace for parts of all rows where only the last tiles' was planned)
    if (p.whole >= 0) a.splits = 1, a.part_o = nullptr, a.part_ml = nullptr;
    if (p.kernel == KeysPlan::ROWS && aligned) return launch_paged_attn_rows(t, a, p.nt, p.cluster, st);
    return launch_paged_attn_general(t, a, st);
}

int check_attention(const vox_paged_cache* c, const vox_paged_batch* b, const vox_paged_prefix* p, size_t n_heads,
                    Checked* k) {
    TRY(check_cache(c, k));
    TRY(check_batch(c, b));
    if (n_heads == 0 || n_heads > 65536 || n_heads % c->n_kv_heads)
        return report_errorf(VOX_ERR_INVALID_ARG, "n_heads must be > 0 and divisible by n_kv_heads");
    // the kernels count query rows, rounded up to whole tiles, in 32 bits
    if ((b->n_tokens + 256) * n_heads > kMaxCount * 2)
        return report_errorf(VOX_ERR_UNSUPPORTED, "n_tokens * n_heads must be at most %d", (int)(kMaxCount * 2));
    if (p) {
        if (!p->len || (p->n_pages && !p->pages)) return report_errorf(VOX_ERR_INVALID_ARG, "null prefix pages or length");
        if (p->n_pages > kMaxCount || p->max_len > kMaxCount)
            return report_errorf(VOX_ERR_UNSUPPORTED, "prefix sizes must be at most %d", (int)kMaxCount);
        if (p->max_len > p->n_pages * c->page_size)
            return report_errorf(VOX_ERR_SHAPE, "max_len needs more pages than the prefix has");
    }
    return VOX_OK;
}

int attention_workspace(const vox_paged_cache* c, const vox_paged_batch* b, const vox_paged_prefix* p, size_t n_heads,
                        size_t window, size_t sinks, size_t* bytes) {
    if (!bytes) return report_errorf(VOX_ERR_INVALID_ARG, "null bytes");
    Checked k;
    TRY(check_attention(c, b, p, n_heads, &k));
    *bytes = b->n_seqs && b->n_tokens ? plan_attention(c, k.type, b, p, n_heads, window, sinks).bytes : 0;
    return VOX_OK;
}

int attention(const vox_paged_cache* c, const vox_paged_batch* b, const vox_paged_prefix* p, const vox_rows* q,
              size_t n_heads, size_t window, size_t sinks, float scale, const vox_rows* out, void* ws, size_t ws_bytes,
              void* stream) {
    Checked k;
    TRY(check_attention(c, b, p, n_heads, &k));
    if (!(scale >= 0.f) || !std::isfinite(scale * kLog2e))
        return report_errorf(VOX_ERR_INVALID_ARG, "scale must be >= 0 and, times log2(e), finite");
    if (b->n_seqs == 0 || b->n_tokens == 0) return VOX_OK;
    PagedAttnArgs a{};
    fill_common(a, c, k, b);
    a.k = c->keys;
    a.v = c->values;
    TRY(check_rows(q, "q", b->n_tokens, n_heads, c->head_dim, k.type, false, &a.q_ts, &a.q_hs));
    TRY(check_rows(out, "out", b->n_tokens, n_heads, c->head_dim, k.type, true, &a.o_ts, &a.o_hs));
    if (q->ptr == out->ptr) return report_errorf(VOX_ERR_INVALID_ARG, "out must not be q");
    a.q = q->ptr;
    a.out = out->ptr;
    a.n_heads = (int)n_heads;
    a.group = (int)(n_heads / c->n_kv_heads);
    a.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf((float)c->head_dim)) * kLog2e;
    a.window = window >= kMaxCount * 2 ? 0 : (int)window;
    a.sinks = (int)std::min(sinks, kMaxCount * 2);
    a.wait_polls = wait_polls.load(std::memory_order_relaxed);
    a.copy_units = copy_units.load(std::memory_order_relaxed);
    if (p) {
        a.pfx_pages = p->pages;
        a.pfx_len = p->len;
        a.pfx_n_pages = (int)p->n_pages;
        a.pfx_max = (int)p->max_len;
    }
    const AttnPlan plan = plan_attention(c, k.type, b, p, n_heads, window, sinks);
    if (plan.partial) {
        if (!ws || ws_bytes < plan.bytes || ((uintptr_t)ws & 255))
            return report_errorf(VOX_ERR_INVALID_ARG, "workspace must be %zu bytes, 256-byte aligned", plan.bytes);
        a.part_ml = static_cast<float2*>(ws);
        a.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + plan.ml_bytes);
    }
    DeviceGuard dev;
    TRY(dev.enter(c->device));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool aligned = aligned16(a.k, k.type, {a.page_stride, a.head_stride, a.slot_stride}) &&
                         aligned16(a.v, k.type, {}) && aligned16(a.q, k.type, {a.q_ts, a.q_hs}) &&
                         aligned16(a.out, k.type, {a.o_ts, a.o_hs});
    a.keys_of = plan.joined ? PagedKeysOf::JOINED : PagedKeysOf::OWN;
    const bool shared = p && !plan.joined;
    a.part0 = shared ? plan.prefix.splits : 0;
    TRY(launched(launch_keys(k.type, a, plan.own, aligned, st), "paged attention"));
    if (shared) {
        // its launch starts while the other drains, and waits for it only at its end
        PagedAttnArgs s = a;
        s.keys_of = PagedKeysOf::PREFIX;
        s.part0 = 0;
        s.follows = 1;
        TRY(launched(launch_keys(k.type, s, plan.prefix, aligned, st), "prefix attention"));
    }
    if (a.whole >= 0)
        TRY(launched(launch_paged_tail_merge(k.type, a, plan.own.units, st), "paged merge"));
    else if (plan.partial && a.part_o)
        TRY(launched(launch_paged_merge(k.type, a, plan.parts, st), "paged merge"));
    return VOX_OK;
}

}  // namespace

// For tests of VOX_PAGED_TIMEOUT (not part of the API), from the next call of this
// process on: how many polls a wait of the tcgen05 kernel takes before it gives up,
// and after how many K and V tiles a CTA stops asking for more, so that the products
// wait in vain.  Less than 0 puts the default back.
extern "C" void vox_paged_test_waits(int polls, int units) {
    wait_polls.store(polls < 0 ? kPagedWaitPolls : polls, std::memory_order_relaxed);
    copy_units.store(units < 0 ? INT32_MAX : units, std::memory_order_relaxed);
}

extern "C" int vox_paged_append_rope(const vox_paged_cache* c, const vox_paged_batch* b, const vox_rows* k_new,
                                     const vox_rows* v_new, float theta, size_t n_heads, const vox_rows* q,
                                     const vox_rows* q_out, void* stream) {
    Checked k;
    TRY(check_cache(c, &k));
    TRY(check_batch(c, b));
    if (theta != 0.f && !(theta >= 1.f && std::isfinite(theta)))
        return report_errorf(VOX_ERR_INVALID_ARG, "rope_theta must be 0 or finite and >= 1");
    if (!q && q_out) return report_errorf(VOX_ERR_INVALID_ARG, "null q beside q_out");
    if (q && (n_heads == 0 || n_heads > 65536)) return report_errorf(VOX_ERR_INVALID_ARG, "n_heads must be in 1..65536");
    if (b->n_seqs == 0 || b->n_tokens == 0) return VOX_OK;
    if (!rows_apart({{c->n_pages, (size_t)k.page_stride}, {c->n_kv_heads, (size_t)k.head_stride}, {c->page_size, (size_t)k.slot_stride}},
                    c->head_dim))
        return report_errorf(VOX_ERR_SHAPE, "cache strides must keep the rows of a pool that is written apart");
    PagedAppendArgs a{};
    fill_common(a, c, k, b);
    a.k = c->keys;
    a.v = c->values;
    a.first_pos = b->first_pos;
    TRY(check_rows(k_new, "k_new", b->n_tokens, c->n_kv_heads, c->head_dim, k.type, false, &a.kn_ts, &a.kn_hs));
    TRY(check_rows(v_new, "v_new", b->n_tokens, c->n_kv_heads, c->head_dim, k.type, false, &a.vn_ts, &a.vn_hs));
    a.k_new = k_new->ptr;
    a.v_new = v_new->ptr;
    if (q) {
        TRY(check_rows(q, "q", b->n_tokens, n_heads, c->head_dim, k.type, false, &a.q_ts, &a.q_hs));
        TRY(check_rows(q_out, "q_out", b->n_tokens, n_heads, c->head_dim, k.type, true, &a.qo_ts, &a.qo_hs));
        // in place, every thread writes what it has read itself
        if (q_out->ptr == q->ptr && ((b->n_tokens > 1 && a.q_ts != a.qo_ts) || (n_heads > 1 && a.q_hs != a.qo_hs)))
            return report_errorf(VOX_ERR_SHAPE, "q_out in the place of q must have its strides");
        a.q = q->ptr;
        a.q_out = q_out->ptr;
        a.n_heads = (int)n_heads;
    }
    a.rotate = theta != 0.f;
    if (a.rotate) {
        // theta^(-2c/D) / (2 pi) in units of 2^-64 turn, by repeated products in
        // 64-bit-mantissa arithmetic
        const long double ratio = powl((long double)theta, -2.0L / (long double)c->head_dim);
        long double f = 0.15915494309189533576888376337251436L * 18446744073709551616.0L;
        for (size_t i = 0; i < c->head_dim / 2; ++i, f *= ratio) a.turns[i] = (uint64_t)f;
    }
    // 16-byte columns where every row starts on a 16-byte boundary
    const bool wide = c->head_dim * type_size(k.type) % 16 == 0 &&
                      aligned16(c->keys, k.type, {a.page_stride, a.head_stride, a.slot_stride}) &&
                      aligned16(c->values, k.type, {}) && aligned16(a.k_new, k.type, {a.kn_ts, a.kn_hs}) &&
                      aligned16(a.v_new, k.type, {a.vn_ts, a.vn_hs}) &&
                      (!q || (aligned16(a.q, k.type, {a.q_ts, a.q_hs}) && aligned16(a.q_out, k.type, {a.qo_ts, a.qo_hs})));
    DeviceGuard dev;
    TRY(dev.enter(c->device));
    return launched(launch_paged_append(k.type, a, wide, static_cast<cudaStream_t>(stream)), "paged append");
}

extern "C" int vox_paged_attention_workspace(const vox_paged_cache* c, const vox_paged_batch* b, size_t n_heads,
                                             size_t window, size_t sinks, size_t* bytes) {
    return attention_workspace(c, b, nullptr, n_heads, window, sinks, bytes);
}

extern "C" int vox_paged_attention(const vox_paged_cache* c, const vox_paged_batch* b, const vox_rows* q,
                                   size_t n_heads, size_t window, size_t sinks, float scale, const vox_rows* out,
                                   void* ws, size_t ws_bytes, void* stream) {
    return attention(c, b, nullptr, q, n_heads, window, sinks, scale, out, ws, ws_bytes, stream);
}

extern "C" int vox_paged_prefix_attention_workspace(const vox_paged_cache* c, const vox_paged_batch* b,
                                                    const vox_paged_prefix* p, size_t n_heads, size_t window,
                                                    size_t sinks, size_t* bytes) {
    if (!p) return report_errorf(VOX_ERR_INVALID_ARG, "null prefix");
    return attention_workspace(c, b, p, n_heads, window, sinks, bytes);
}

extern "C" int vox_paged_prefix_attention(const vox_paged_cache* c, const vox_paged_batch* b,
                                          const vox_paged_prefix* p, const vox_rows* q, size_t n_heads, size_t window,
                                          size_t sinks, float scale, const vox_rows* out, void* ws, size_t ws_bytes,
                                          void* stream) {
    if (!p) return report_errorf(VOX_ERR_INVALID_ARG, "null prefix");
    return attention(c, b, p, q, n_heads, window, sinks, scale, out, ws, ws_bytes, stream);
}
