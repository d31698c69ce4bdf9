// Filling a paged key-value cache (rotary embedding fused) and copying its pages. Both move
// every byte once, 16 bytes a thread, and are bound by HBM (small calls by launch latency).
// Measured, the fills in a graph of calls (from Python: 19.3 and 5.6 us): 5 prompts, 5020 tokens of
// 64 + 8 + 8 heads of 128: 17.5 us, 6.0 TB/s; 8 single tokens of 32 + 32 + 32 heads: 2.2 us. Copies,
// from Python: 8 pages of 32 layers (134 MB moved) 22.3 us, 6.0 TB/s; 511 pages of 16 layers (4.3 GB)
// 650 us, 6.6 TB/s.
#include <algorithm>

#include "w4a16_paged.cuh"
#include "w4a16_ptx.cuh"

namespace w4a16 {
namespace {

constexpr int kAppendHeads = 2;  // read ahead: the same prompts 17.5 us, 18.5 at 1, 18.6 at 3
constexpr int kAppendThreads = 128;  // 5 prompts, 5020 tokens, 64 + 8 + 8 heads: 18.6 us, 21 at 256

// (x_a, x_b) -> (x_a c - x_b s, x_b c + x_a s): one pair of 8-element chunks, or the four
// pairs inside each chunk when interleaved. fp32, rounded once.
template <bool BF16>
__device__ __forceinline__ void rotate_halves(uint4& xa, uint4& xb, const float (&c)[8], const float (&s)[8]) {
    uint32_t* a = reinterpret_cast<uint32_t*>(&xa);
    uint32_t* b = reinterpret_cast<uint32_t*>(&xb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 u = unpack2<BF16>(a[i]), w = unpack2<BF16>(b[i]);
        a[i] = pack2<BF16>(u.x * c[2 * i] - w.x * s[2 * i], u.y * c[2 * i + 1] - w.y * s[2 * i + 1]);
        b[i] = pack2<BF16>(w.x * c[2 * i] + u.x * s[2 * i], w.y * c[2 * i + 1] + u.y * s[2 * i + 1]);
    }
}

template <bool BF16>
__device__ __forceinline__ void rotate_pairs(uint4& x, const float (&c)[8], const float (&s)[8]) {
    uint32_t* a = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 u = unpack2<BF16>(a[i]);
        a[i] = pack2<BF16>(u.x * c[i] - u.y * s[i], u.y * c[i] + u.x * s[i]);
    }
}

// One token per blockIdx.x; its q, k and v heads over blockIdx.y and the thread rows. A
// thread keeps one chunk position (with rotation by halves: the pair of chunks that rotate
// together) over all its heads, so the angles are read once.
template <bool BF16>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a) {
    ptx::grid_dep_wait();
    const int t = blockIdx.x;
    const int dim = a.pages.dim;
    const int half = a.rope && !a.interleaved ? a.rope_dim >> 4 : 0;  // chunk pairs that rotate together
    const int slots = (dim >> 3) - half;
    const int slot = threadIdx.x % slots;
    const int rows = kAppendThreads / slots;
    if (threadIdx.x >= rows * slots) return;
    const bool pair = slot < half;
    const int c0 = (pair ? slot : slot + half) * 8, c1 = (slot + half) * 8;

    // a few heads at a time, read before anything is known of where they go
    const int heads_q = a.q ? a.heads : 0, hkv = a.pages.heads_kv, all = heads_q + 2 * hkv;
    const int stride = rows * gridDim.y;
    uint4 x[kAppendHeads], y[kAppendHeads];
    auto load = [&](int r) {
#pragma unroll
        for (int i = 0; i < kAppendHeads; ++i) {
            const int at = r + i * stride;
            if (at >= all) break;
            const uint16_t* src = at < heads_q ? a.q + t * a.q_token + at * a.q_head
                                  : at < heads_q + hkv ? a.k + t * a.k_token + (at - heads_q) * a.k_head
                                                       : a.v + t * a.v_token + (at - heads_q - hkv) * a.v_head;
            x[i] = *reinterpret_cast<const uint4*>(src + c0);
            if (pair) y[i] = *reinterpret_cast<const uint4*>(src + c1);
        }
    };
    int r = blockIdx.y * rows + threadIdx.x / slots;
    load(r);

    // the token's sequence: the last one that begins at or before row t
    int b = t;
    if (a.seqs.cu_q) {
        int lo = 0, hi = a.seqs.batch;  // cu_q[lo] <= t < cu_q[hi] once the ends are checked
        if (t < a.seqs.cu_q[0] || t >= a.seqs.cu_q[hi]) return;  // rows of no sequence stay as they were
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.seqs.cu_q[mid] <= t) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        b = lo;
    }
    const Seq sq = load_seq(a.seqs, a.pages.page_shift, b);
    if (t < sq.t0 || t - sq.t0 >= sq.nq) return;  // offsets that do not ascend
    const int pos = sq.p0 + (t - sq.t0);
    int page = -1;
    if (pos >= 0) page = a.seqs.tables[b * a.seqs.table_stride + (pos >> a.pages.page_shift)];

    const bool turn = a.rope && pos >= 0 && (pair || (a.interleaved && slot * 8 < a.rope_dim));
    float c[8], s[8];
    if (turn) {
        const float* row = a.rope + static_cast<int64_t>(pos) * a.rope_dim;
        const int n = pair ? 8 : 4, first = pair ? slot * 8 : slot * 4;
        for (int i = 0; i < 8; i += 4) {
            if (i < n) {
                const float4 u = *reinterpret_cast<const float4*>(row + first + i);
                const float4 w = *reinterpret_cast<const float4*>(row + (a.rope_dim >> 1) + first + i);
                c[i] = u.x, c[i + 1] = u.y, c[i + 2] = u.z, c[i + 3] = u.w;
                s[i] = w.x, s[i + 1] = w.y, s[i + 2] = w.z, s[i + 3] = w.w;
            }
        }
    }
    const bool store = page >= 0 && page < a.pages.num_pages;  // a token of no valid page is not stored
    const int64_t cache = store ? page * a.pages.stride_page +
                                      (pos & ((1 << a.pages.page_shift) - 1)) * a.pages.stride_token
                                : 0;
    const int end = store ? all : heads_q;  // the k and v heads come last
    while (r < end) {
#pragma unroll
        for (int i = 0; i < kAppendHeads; ++i) {
            const int at = r + i * stride;
            if (at >= end) break;
            uint16_t* dst = at < heads_q ? a.q_out + t * a.qo_token + at * a.qo_head
                            : at < heads_q + hkv ? a.k_out + cache + (at - heads_q) * a.pages.stride_head
                                                 : a.v_out + cache + (at - heads_q - hkv) * a.pages.stride_head;
            const bool rot = turn && at < heads_q + hkv;
            if (pair) {
                if (rot) rotate_halves<BF16>(x[i], y[i], c, s);
                *reinterpret_cast<uint4*>(dst + c1) = y[i];
            } else if (rot) {
                rotate_pairs<BF16>(x[i], c, s);
            }
            *reinterpret_cast<uint4*>(dst + c0) = x[i];
        }
        r += kAppendHeads * stride;
        if (r < end) load(r);
    }
}

// 16 KB of one page of one layer of K or V per CTA.
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = kCopyThreads * 16 * 4;

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyArgs a) {
    ptx::grid_dep_wait();
    const int pair = blockIdx.y;
    const int layer = blockIdx.z >> 1;
    uint8_t* base = a.base[blockIdx.z & 1] + layer * a.stride_layer;
    const uint8_t* src = base + a.src[pair] * a.stride_page;
    uint8_t* dst = base + a.dst[pair] * a.stride_page;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kCopyBytes + threadIdx.x * 16;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t at = first + i * (kCopyThreads * 16);
        if (at < a.page_bytes) v[i] = *reinterpret_cast<const uint4*>(src + at);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t at = first + i * (kCopyThreads * 16);
        if (at < a.page_bytes) *reinterpret_cast<uint4*>(dst + at) = v[i];
    }
}

template <typename K, typename A>
cudaError_t launch_pdl(K kern, dim3 grid, int threads, const A& a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, bool bf16, int num_sms, cudaStream_t s) {
    if (a.seqs.tokens == 0) return cudaSuccess;
    const int half = a.rope && !a.interleaved ? a.rope_dim >> 4 : 0;
    const int rows = kAppendThreads / ((a.pages.dim >> 3) - half);
    const int all = (a.q ? a.heads : 0) + 2 * a.pages.heads_kv;
    // few tokens: one head per thread row, so that a decode step is one round trip; many:
    // the heads of a token in one CTA, so that the angles are read once. In a graph, us, one head
    // against all: 8 tokens of 32 + 32 + 32 heads 2.2 / 3.5, 148 2.9 / 3.7, 296 4.7 / 4.9, 444 6.0 / 6.1,
    // 592 7.8 / 7.1, 2368 25.7 / 20.0; of 64 + 8 + 8 heads 148 2.8 / 3.5, 296 4.1 / 3.8, 592 6.7 / 5.6
    const int ny = a.seqs.tokens >= 2 * num_sms ? 1 : (all + rows - 1) / rows;
    const dim3 grid(a.seqs.tokens, ny);
    return launch_pdl(bf16 ? append_kernel<true> : append_kernel<false>, grid, kAppendThreads, a, s);
}

cudaError_t launch_copy(const CopyArgs& a, cudaStream_t s) {
    const int64_t nx = (a.page_bytes + kCopyBytes - 1) / kCopyBytes;
    return launch_pdl(copy_kernel, dim3(static_cast<unsigned>(nx), a.pairs, 2 * a.layers), kCopyThreads, a, s);
}

}  // namespace w4a16
