// C entry points of the paged key-value cache: argument checks (all before any CUDA call),
// the choice of the attention kernel, launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <exception>
#include <vector>

#include "../../include/drofell_w4a16.h"
#include "w4a16_host.h"
#include "w4a16_paged.h"

using namespace w4a16;

namespace {

int cuda_error(cudaError_t e, const char* what) {
    return report_error(W4A16_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

constexpr int kMostTokens = (1 << 30) - 1024;

// Rows of a sequence and key-value head (new tokens x heads of the group) from which the
// tensor-core kernel takes the call: the other one reads the keys once for every 16 rows.
// 16 sequences of 4000 tokens, 64 heads on 8: 16 rows 56 us against 74, 24 rows 97 against 74;
// 32 of 200 tokens, 32 heads: 32 rows 56 against 64, 64 rows 89 against 64.
constexpr int kPromptRows = 33, kPromptRowsLong = 17, kLongTokens = 1024;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_pages(const w4a16_pages* p) {
    if (!p || !p->k_dev || !p->v_dev) return report_error(W4A16_ERR_INVALID, "null pages");
    if (p->dtype != W4A16_DTYPE_FP16 && p->dtype != W4A16_DTYPE_BF16)
        return report_error(W4A16_ERR_INVALID, "unknown dtype %d", p->dtype);
    if (p->page_size < 8 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
        return report_error(W4A16_ERR_UNSUPPORTED, "page size %d (a power of two from 8 to 256)", p->page_size);
    if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8)
        return report_error(W4A16_ERR_UNSUPPORTED, "head dim %d (a multiple of 8, at most 128)", p->head_dim);
    if (p->num_pages <= 0 || p->heads_kv <= 0)
        return report_error(W4A16_ERR_INVALID, "num_pages=%d heads_kv=%d", p->num_pages, p->heads_kv);
    if ((p->num_pages > 1 && p->stride_page == 0) || (p->heads_kv > 1 && p->stride_head == 0) || p->stride_token == 0)
        return report_error(W4A16_ERR_INVALID, "page strides of 0");
    if (p->stride_page < 0 || p->stride_head < 0 || p->stride_token < 0 || p->stride_page % 8 || p->stride_head % 8 ||
        p->stride_token % 8)
        return report_error(W4A16_ERR_INVALID, "page strides must be non-negative multiples of 8 elements");
    if (!aligned16(p->k_dev) || !aligned16(p->v_dev))
        return report_error(W4A16_ERR_INVALID, "the pages must be 16-byte aligned");
    return W4A16_OK;
}

int check_seqs(const w4a16_pages* p, const w4a16_seqs* s) {
    if (!s) return report_error(W4A16_ERR_INVALID, "null seqs");
    if (s->batch < 0 || s->tokens < 0 || s->max_q < 0 || s->table_width < 0 || s->table_stride < 0)
        return report_error(W4A16_ERR_INVALID, "batch=%d tokens=%d max_q=%d table_width=%d: none may be negative",
                            s->batch, s->tokens, s->max_q, s->table_width);
    if (s->batch > 0 && (!s->lens_dev || (s->table_width > 0 && !s->tables_dev)))
        return report_error(W4A16_ERR_INVALID, "null tables or lens");
    if (!s->cu_q_dev && s->tokens != s->batch)
        return report_error(W4A16_ERR_INVALID, "%d rows for %d sequences of one new token each", s->tokens, s->batch);
    // sums of a position, a key and a window stay within 32 bits
    if (static_cast<int64_t>(s->table_width) * p->page_size > kMostTokens || s->tokens > kMostTokens)
        return report_error(W4A16_ERR_UNSUPPORTED, "tables of %d pages of %d tokens, %d new tokens: at most %d tokens",
                            s->table_width, p->page_size, s->tokens, kMostTokens);
    return W4A16_OK;
}

int check_rows(const w4a16_rows* r, const char* name) {
    if (!r || !r->dev) return report_error(W4A16_ERR_INVALID, "null %s", name);
    if (r->stride_token < 0 || r->stride_head < 0 || r->stride_token % 8 || r->stride_head % 8 || !aligned16(r->dev))
        return report_error(W4A16_ERR_INVALID, "%s must be 16-byte aligned, its strides non-negative multiples of 8 elements",
                            name);
    return W4A16_OK;
}

// Memory that is written holds no element twice: counts and strides of what lies around rows of `dim`.
struct Extent {
    int64_t count, stride;
};
bool apart(Extent a, Extent b, Extent c, int dim) {
    Extent e[3] = {a, b, c};
    std::sort(e, e + 3, [](const Extent& x, const Extent& y) { return x.stride < y.stride; });
    int64_t taken = dim;
    for (const Extent& x : e) {
        if (x.count <= 1) continue;
        if (x.stride < taken) return false;
        taken += (x.count - 1) * x.stride;
    }
    return true;
}

int check_written(const w4a16_rows* r, int tokens, int heads, int dim, const char* name) {
    const int rc = check_rows(r, name);
    if (rc != W4A16_OK) return rc;
    if (!apart({tokens, r->stride_token}, {heads, r->stride_head}, {1, 0}, dim))
        return report_error(W4A16_ERR_INVALID, "%s's rows overlap", name);
    return W4A16_OK;
}

// Two sets of runs of `size` bytes (or elements), their first runs `delta` apart: a run of the one and
// one of the other lie sum x_i stride_i + delta apart, lo_i <= x_i <= hi_i. Whether any two share
// memory: strides in falling order, and of each only the x that the others can still make up for.
struct Apart {
    int64_t stride, lo, hi;
};
bool share(int64_t delta, const Apart* d, int n, int64_t size) {
    if (n == 0) return delta < size && -delta < size;
    int64_t reach = size - 1;  // of the other strides
    for (int i = 1; i < n; ++i) reach += d[i].stride * std::max(-d[i].lo, d[i].hi);
    if (d->stride == 0) return share(delta, d + 1, n - 1, size);
    const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); };
    const int64_t first = std::max(d->lo, -floor_div(delta + reach, d->stride));
    const int64_t last = std::min(d->hi, floor_div(reach - delta, d->stride));
    for (int64_t x = first; x <= last; ++x)
        if (share(delta + x * d->stride, d + 1, n - 1, size)) return true;
    return false;
}

// Whether two sets of runs with the same strides share memory; addresses and strides in bytes.
bool share_alike(const void* a, const void* b, Extent x, Extent y, Extent z, int64_t size) {
    Extent e[3] = {x, y, z};
    std::sort(e, e + 3, [](const Extent& u, const Extent& w) { return u.stride > w.stride; });
    Apart d[3];
    int n = 0;
    for (const Extent& u : e)
        if (u.count > 1) d[n++] = {u.stride, 1 - u.count, u.count - 1};
    return share(static_cast<int64_t>(reinterpret_cast<intptr_t>(a) - reinterpret_cast<intptr_t>(b)), d, n, size);
}

// Whether rows share memory. Views of one buffer (a q/k/v product, say) have their strides in common.
// Where they do not, and their ranges meet, rows count as sharing it: which of them do would
// have to be searched for.
bool rows_share(const w4a16_rows* a, int heads_a, const w4a16_rows* b, int heads_b, int tokens, int dim) {
    const auto span = [&](const w4a16_rows* r, int heads) {
        return ((tokens - 1) * r->stride_token + (heads - 1) * r->stride_head + dim) * 2;
    };
    const intptr_t pa = reinterpret_cast<intptr_t>(a->dev), pb = reinterpret_cast<intptr_t>(b->dev);
    if (pa + span(a, heads_a) <= pb || pb + span(b, heads_b) <= pa) return false;
    if ((tokens > 1 && a->stride_token != b->stride_token) || (pa - pb) % 2) return true;
    Apart d[3] = {{tokens > 1 ? a->stride_token : 0, 1 - int64_t{tokens}, int64_t{tokens} - 1}};
    int n = 1;
    if (heads_a > 1 && heads_b > 1 && a->stride_head == b->stride_head) {
        d[n++] = {a->stride_head, 1 - int64_t{heads_b}, int64_t{heads_a} - 1};
    } else {
        d[n++] = {heads_a > 1 ? a->stride_head : 0, 0, int64_t{heads_a} - 1};
        d[n++] = {heads_b > 1 ? b->stride_head : 0, 1 - int64_t{heads_b}, 0};
    }
    std::sort(d, d + n, [](const Apart& x, const Apart& y) { return x.stride > y.stride; });
    return share((pa - pb) / 2, d, n, dim);
}

PageView page_view(const w4a16_pages* p) {
    PageView v;
    v.k = static_cast<const uint16_t*>(p->k_dev);
    v.v = static_cast<const uint16_t*>(p->v_dev);
    v.stride_page = p->stride_page;
    v.stride_head = p->stride_head;
    v.stride_token = p->stride_token;
    v.num_pages = p->num_pages;
    v.heads_kv = p->heads_kv;
    v.dim = p->head_dim;
    v.page_shift = 0;
    while ((1 << v.page_shift) < p->page_size) ++v.page_shift;
    return v;
}

SeqView seq_view(const w4a16_seqs* s) {
    SeqView v;
    v.tables = s->tables_dev;
    v.lens = s->lens_dev;
    v.cu_q = s->cu_q_dev;
    v.table_stride = s->table_stride;
    v.width = s->table_width;
    v.batch = s->batch;
    v.tokens = s->tokens;
    v.max_q = s->max_q;
    return v;
}

int sm_count(int device) {
    static std::atomic<int> known[64];
    if (device >= 0 && device < 64) {
        const int n = known[device].load(std::memory_order_relaxed);
        if (n > 0) return n;
    }
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) return 0;
    if (device >= 0 && device < 64) known[device].store(n, std::memory_order_relaxed);
    return n;
}

AttnArgs attn_args(const w4a16_pages* pages, const w4a16_seqs* seqs, int heads, int window, int sinks) {
    AttnArgs a = {};
    a.pages = page_view(pages);
    a.seqs = seq_view(seqs);
    a.seqs.max_q = seqs->cu_q_dev ? seqs->max_q : 1;
    a.heads = heads;
    a.group = heads / pages->heads_kv;
    // a window of all the tables cover hides nothing
    const int covered = seqs->table_width * pages->page_size;
    a.window = window >= covered ? 0 : window;
    a.sinks = a.window == 0 ? 0 : (sinks < covered ? sinks : covered);
    return a;
}

bool takes_prompt(const AttnArgs& a) {
    const bool longer = (static_cast<int64_t>(a.seqs.width) << a.pages.page_shift) >= kLongTokens;
    return static_cast<int64_t>(a.seqs.max_q) * a.group >= (longer ? kPromptRowsLong : kPromptRows) && prompt_fits(a);
}

size_t workspace_bytes_of(const AttnArgs& a, int sms) {
    if (takes_prompt(a)) return prompt_workspace_bytes(a, sms);
    return split_fits(a) ? split_workspace_bytes(plan_split(a, sms), a.pages.dim) : 0;
}

int check_attention(const w4a16_pages* pages, const w4a16_seqs* seqs, int heads, int window, int sinks) {
    int rc = check_pages(pages);
    if (rc == W4A16_OK) rc = check_seqs(pages, seqs);
    if (rc != W4A16_OK) return rc;
    if (heads <= 0 || heads % pages->heads_kv)
        return report_error(W4A16_ERR_INVALID, "%d query heads on %d key-value heads", heads, pages->heads_kv);
    if (window < 0 || sinks < 0) return report_error(W4A16_ERR_INVALID, "window=%d sinks=%d", window, sinks);
    if (sinks > 0 && window == 0) return report_error(W4A16_ERR_INVALID, "sinks without a window");
    if (static_cast<int64_t>(seqs->max_q) * (heads / pages->heads_kv) > INT_MAX / 2)
        return report_error(W4A16_ERR_UNSUPPORTED, "max_q=%d", seqs->max_q);
    return W4A16_OK;
}

}  // namespace

extern "C" {

int w4a16_append_kv(const w4a16_pages* pages, const w4a16_seqs* seqs, const w4a16_rows* k, const w4a16_rows* v,
                    const w4a16_rows* q, const w4a16_rows* q_out, int heads, const float* rope_dev, int rope_positions,
                    int rope_dim, int interleaved, void* stream) {
    int rc = check_pages(pages);
    if (rc == W4A16_OK) rc = check_seqs(pages, seqs);
    if (rc != W4A16_OK) return rc;
    if (seqs->batch == 0 || seqs->tokens == 0) return W4A16_OK;
    rc = check_rows(k, "k");
    if (rc == W4A16_OK) rc = check_rows(v, "v");
    const bool with_q = q && q->dev;
    if (rc == W4A16_OK && with_q) {
        rc = check_rows(q, "q");
        if (rc == W4A16_OK && heads <= 0) rc = report_error(W4A16_ERR_INVALID, "heads=%d", heads);
        if (rc == W4A16_OK) rc = check_written(q_out, seqs->tokens, heads, pages->head_dim, "q_out");
    }
    if (rc == W4A16_OK && !apart({pages->num_pages, pages->stride_page}, {pages->heads_kv, pages->stride_head},
                                 {pages->page_size, pages->stride_token}, pages->head_dim))
        rc = report_error(W4A16_ERR_INVALID, "pages that overlap");
    if (rc != W4A16_OK) return rc;
    if (rope_dev) {
        if (rope_dim <= 0 || rope_dim > pages->head_dim || rope_dim % (interleaved ? 8 : 16))
            return report_error(W4A16_ERR_UNSUPPORTED, "rope dim %d of %d (a multiple of %d)", rope_dim,
                                pages->head_dim, interleaved ? 8 : 16);
        if (!aligned16(rope_dev)) return report_error(W4A16_ERR_INVALID, "the rope table must be 16-byte aligned");
        if (rope_positions < static_cast<int64_t>(seqs->table_width) * pages->page_size)
            return report_error(W4A16_ERR_INVALID, "a rope table of %d positions for tables of %lld tokens", rope_positions,
                                static_cast<long long>(seqs->table_width) * pages->page_size);
    }
    if (share_alike(pages->k_dev, pages->v_dev, {pages->num_pages, pages->stride_page * 2},
                    {pages->heads_kv, pages->stride_head * 2}, {pages->page_size, pages->stride_token * 2},
                    int64_t{pages->head_dim} * 2))
        return report_error(W4A16_ERR_INVALID, "K and V pages that overlap");
    if (with_q) {
        const int hkv = pages->heads_kv, dim = pages->head_dim, n = seqs->tokens;
        const bool in_place = q->dev == q_out->dev && (n == 1 || q->stride_token == q_out->stride_token) &&
                              (heads == 1 || q->stride_head == q_out->stride_head);
        if (!in_place && rows_share(q, heads, q_out, heads, n, dim))
            return report_error(W4A16_ERR_INVALID, "q_out must be q or not overlap it");
        if (rows_share(k, hkv, q_out, heads, n, dim) || rows_share(v, hkv, q_out, heads, n, dim))
            return report_error(W4A16_ERR_INVALID, "q_out must not overlap k or v");
    }
    AppendArgs a = {};
    a.pages = page_view(pages);
    a.seqs = seq_view(seqs);
    a.k_out = static_cast<uint16_t*>(pages->k_dev);
    a.v_out = static_cast<uint16_t*>(pages->v_dev);
    a.k = static_cast<const uint16_t*>(k->dev);
    a.v = static_cast<const uint16_t*>(v->dev);
    a.k_token = k->stride_token, a.k_head = k->stride_head;
    a.v_token = v->stride_token, a.v_head = v->stride_head;
    if (with_q) {
        a.q = static_cast<const uint16_t*>(q->dev);
        a.q_out = static_cast<uint16_t*>(q_out->dev);
        a.q_token = q->stride_token, a.q_head = q->stride_head;
        a.qo_token = q_out->stride_token, a.qo_head = q_out->stride_head;
        a.heads = heads;
    }
    a.rope = rope_dev;
    a.rope_dim = rope_dim;
    a.interleaved = interleaved ? 1 : 0;
    // every new token is stored, whatever max_q says
    a.seqs.max_q = INT_MAX;
    DeviceGuard guard(pages->device);
    if (!guard.ok) return report_error(W4A16_ERR_INVALID, "device %d", pages->device);
    const int sms = sm_count(pages->device);
    if (sms == 0) return report_error(W4A16_ERR_CUDA, "no device %d", pages->device);
    const cudaError_t e = launch_append(a, pages->dtype == W4A16_DTYPE_BF16, sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A16_OK : cuda_error(e, "append_kv launch");
}

size_t w4a16_paged_attention_workspace_size(const w4a16_pages* pages, const w4a16_seqs* seqs, int heads, int window,
                                            int sinks) {
    if (check_attention(pages, seqs, heads, window, sinks) != W4A16_OK) return 0;
    if (seqs->batch == 0 || seqs->tokens == 0 || seqs->max_q == 0) return 0;
    const int sms = sm_count(pages->device);
    return sms == 0 ? 0 : workspace_bytes_of(attn_args(pages, seqs, heads, window, sinks), sms);
}

int w4a16_paged_attention(const w4a16_pages* pages, const w4a16_seqs* seqs, const w4a16_rows* q, const w4a16_rows* out,
                          int heads, float scale, int window, int sinks, void* workspace_dev, size_t workspace_bytes,
                          void* stream) {
    int rc = check_attention(pages, seqs, heads, window, sinks);
    if (rc != W4A16_OK) return rc;
    if (!(scale > 0.f) || !std::isfinite(scale * 1.4426950408889634f))
        return report_error(W4A16_ERR_INVALID, "scale must be positive and finite");
    if (seqs->batch == 0 || seqs->tokens == 0 || seqs->max_q == 0) return W4A16_OK;
    rc = check_rows(q, "q");
    if (rc == W4A16_OK) rc = check_written(out, seqs->tokens, heads, pages->head_dim, "out");
    if (rc != W4A16_OK) return rc;
    if (rows_share(q, heads, out, heads, seqs->tokens, pages->head_dim))
        return report_error(W4A16_ERR_INVALID, "out must not overlap q");
    AttnArgs a = attn_args(pages, seqs, heads, window, sinks);
    a.q = static_cast<const uint16_t*>(q->dev);
    a.q_token = q->stride_token, a.q_head = q->stride_head;
    a.out = static_cast<uint16_t*>(out->dev);
    a.o_token = out->stride_token, a.o_head = out->stride_head;
    a.scale_log2 = scale * 1.4426950408889634f;
    const bool bf16 = pages->dtype == W4A16_DTYPE_BF16;
    const int sms = sm_count(pages->device);
    if (sms == 0) return report_error(W4A16_ERR_CUDA, "no device %d", pages->device);
    DeviceGuard guard(pages->device);
    if (!guard.ok) return report_error(W4A16_ERR_INVALID, "device %d", pages->device);
    const bool prompt = takes_prompt(a);
    if (!prompt && !split_fits(a))
        return report_error(W4A16_ERR_UNSUPPORTED, "tables of %d pages for %d key-value heads", seqs->table_width,
                            pages->heads_kv);
    const size_t need = workspace_bytes_of(a, sms);
    if (workspace_bytes < need || (need > 0 && !workspace_dev))
        return report_error(W4A16_ERR_WORKSPACE, "workspace %zu bytes < %zu needed", workspace_bytes, need);
    // 32: the widest stores
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace_dev) & 31))
        return report_error(W4A16_ERR_INVALID, "the workspace must be 32-byte aligned");
    a.ws = need > 0 ? static_cast<float*>(workspace_dev) : nullptr;
    const cudaError_t e = prompt ? launch_prompt(a, bf16, sms, static_cast<cudaStream_t>(stream))
                                 : launch_split(a, plan_split(a, sms), bf16, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A16_OK : cuda_error(e, "paged attention launch");
}

int w4a16_paged_error(int device, void* stream, int* err_out) {
    if (!err_out) return report_error(W4A16_ERR_INVALID, "null argument");
    DeviceGuard guard(device);
    if (!guard.ok) return report_error(W4A16_ERR_INVALID, "device %d", device);
    const cudaError_t e = read_attention_error(err_out, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A16_OK : cuda_error(e, "paged error read");
}

int w4a16_copy_pages(void* k_dev, void* v_dev, int64_t stride_layer_bytes, int64_t stride_page_bytes, int layers,
                     int num_pages, int64_t page_bytes, const int32_t* src_host, const int32_t* dst_host, int pairs,
                     int device, void* stream) try {
    if (!k_dev || !v_dev) return report_error(W4A16_ERR_INVALID, "null pages");
    if (pairs < 0 || num_pages <= 0 || layers < 0 || layers > 32767 || page_bytes <= 0)
        return report_error(W4A16_ERR_INVALID, "pairs=%d num_pages=%d layers=%d page_bytes=%lld", pairs, num_pages, layers,
                            static_cast<long long>(page_bytes));
    if (page_bytes % 16 || stride_page_bytes % 16 || stride_layer_bytes % 16 || !aligned16(k_dev) || !aligned16(v_dev))
        return report_error(W4A16_ERR_INVALID, "pages and their strides must be multiples of 16 bytes");
    const int64_t in_layer = (num_pages - 1) * stride_page_bytes + page_bytes;
    if (stride_page_bytes < page_bytes || stride_layer_bytes < 0 ||
        (layers > 1 && stride_layer_bytes < in_layer &&
         (num_pages > 1 ? stride_page_bytes < (layers - 1) * stride_layer_bytes + page_bytes : true)) ||
        (layers > 1 && stride_layer_bytes < page_bytes))
        return report_error(W4A16_ERR_INVALID, "pages that overlap");
    // the same memory for both is copied twice to the same effect
    if (k_dev != v_dev && share_alike(k_dev, v_dev, {layers, stride_layer_bytes}, {num_pages, stride_page_bytes}, {1, 0}, page_bytes))
        return report_error(W4A16_ERR_INVALID, "K and V pages that overlap");
    if (pairs == 0 || layers == 0) return W4A16_OK;
    if (!src_host || !dst_host) return report_error(W4A16_ERR_INVALID, "null page ids");
    for (int i = 0; i < pairs; ++i)
        if (src_host[i] < 0 || src_host[i] >= num_pages || dst_host[i] < 0 || dst_host[i] >= num_pages)
            return report_error(W4A16_ERR_INVALID, "copy %d of page %d to %d: %d pages", i, src_host[i], dst_host[i], num_pages);
    // The pages written: a byte for every page of the cache, or a sorted list where the copies are few
    // beside it, so that the cost is that of the copies. 3000 of 8000 pages 136 us a call with bytes,
    // 215 sorted; 1 of 200000 14.8 with bytes, 8.2 sorted; 511 of 2000 34 with either.
    std::vector<uint8_t> is_written;
    std::vector<int32_t> written;
    if (num_pages / 16 <= pairs) {
        is_written.assign(num_pages, 0);
    } else {
        written.assign(dst_host, dst_host + pairs);
        std::sort(written.begin(), written.end());
    }
    for (int i = 0; i < pairs; ++i) {
        const bool twice = written.empty() ? is_written[dst_host[i]] != 0 : i > 0 && written[i] == written[i - 1];
        if (twice) return report_error(W4A16_ERR_INVALID, "page %d written twice", written.empty() ? dst_host[i] : written[i]);
        if (written.empty()) is_written[dst_host[i]] = 1;
    }
    for (int i = 0; i < pairs; ++i)
        if (written.empty() ? is_written[src_host[i]] != 0 : std::binary_search(written.begin(), written.end(), src_host[i]))
            return report_error(W4A16_ERR_INVALID, "copy %d of page %d to %d: a page read and written", i, src_host[i], dst_host[i]);
    DeviceGuard guard(device);
    if (!guard.ok) return report_error(W4A16_ERR_INVALID, "device %d", device);
    CopyArgs a = {};
    a.base[0] = static_cast<uint8_t*>(k_dev);
    a.base[1] = static_cast<uint8_t*>(v_dev);
    a.stride_layer = stride_layer_bytes;
    a.stride_page = stride_page_bytes;
    a.page_bytes = page_bytes;
    a.layers = layers;
    for (int i = 0; i < pairs; i += kCopyPairs) {
        a.pairs = pairs - i < kCopyPairs ? pairs - i : kCopyPairs;
        for (int j = 0; j < a.pairs; ++j) {
            a.src[j] = src_host[i + j];
            a.dst[j] = dst_host[i + j];
        }
        const cudaError_t e = launch_copy(a, static_cast<cudaStream_t>(stream));
        if (e != cudaSuccess) return cuda_error(e, "copy_pages launch");
    }
    return W4A16_OK;
} catch (const std::exception& e) {
    return report_error(W4A16_ERR_INVALID, "copy_pages: %s", e.what());
}

}  // extern "C"
