// Internal declarations of the paged key-value cache kernels (not part of the C ABI).
#pragma once
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace w4a16 {

// One layer's pages as the kernels see them: element (page, head, slot, d) of K and of V
// at page * stride_page + head * stride_head + slot * stride_token + d, 64-bit.
struct PageView {
    const uint16_t* k;
    const uint16_t* v;
    int64_t stride_page, stride_head, stride_token;
    int num_pages, heads_kv, page_shift, dim;
};

// The sequences of a call: tables [batch, width] of page ids, lengths with the new tokens
// counted, and where each sequence's new tokens lie among the rows of q (cu_q; null: row b).
struct SeqView {
    const int32_t* tables;
    const int32_t* lens;
    const int32_t* cu_q;
    int64_t table_stride;
    int width, batch, tokens, max_q;
};

struct AppendArgs {
    PageView pages;
    SeqView seqs;
    uint16_t* k_out;  // pages.k / pages.v, written
    uint16_t* v_out;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* q;  // null: no q rows
    uint16_t* q_out;
    const float* rope;  // [positions, rope_dim]: cosines, then sines; null: no rotation
    int64_t k_token, k_head, v_token, v_head, q_token, q_head, qo_token, qo_head;
    int heads, rope_dim, interleaved;
};

struct AttnArgs {
    PageView pages;
    SeqView seqs;
    const uint16_t* q;
    uint16_t* out;
    int64_t q_token, q_head, o_token, o_head;
    int heads, group;   // query heads, query heads per key-value head
    float scale_log2;   // scale * log2(e)
    int window, sinks;  // window 0: none
    float* ws;          // partial results of the split kernel
};

cudaError_t launch_append(const AppendArgs& a, bool bf16, int num_sms, cudaStream_t s);

// Attention split over the cache's length and joined.
struct SplitPlan {
    int ctas;       // CTAs that share the work, four workers each
    int min_units;  // least 16-key tiles per worker
    bool deep;      // one CTA an SM, with deeper rings
};
bool split_fits(const AttnArgs& a);  // the units of a sequence are countable
SplitPlan plan_split(const AttnArgs& a, int num_sms);
size_t split_workspace_bytes(const SplitPlan& p, int dim);
cudaError_t launch_split(const AttnArgs& a, const SplitPlan& p, bool bf16, cudaStream_t s);

// Attention of prompts on the tensor cores (w4a16_attn_sm100.cu).
bool prompt_fits(const AttnArgs& a);
size_t prompt_workspace_bytes(const AttnArgs& a, int num_sms);
cudaError_t launch_prompt(const AttnArgs& a, bool bf16, int num_sms, cudaStream_t s);
// The current device's error word of its bounded waits, then cleared. Synchronises `s`.
cudaError_t read_attention_error(int* out, cudaStream_t s);

constexpr int kCopyPairs = 500;
struct CopyArgs {
    uint8_t* base[2];  // K, V
    int64_t stride_layer, stride_page;  // bytes
    int64_t page_bytes;
    int layers, pairs;
    int32_t src[kCopyPairs], dst[kCopyPairs];
};
cudaError_t launch_copy(const CopyArgs& a, cudaStream_t s);

// Lets `kern` use `bytes` of dynamic shared memory on the current device; the attribute
// belongs to the function on one device, `ready` holds a bit for each that has it.
inline cudaError_t allow_smem(const void* kern, int bytes, std::atomic<uint64_t>& ready) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = uint64_t{1} << (dev & 63);
    if (dev < 64 && (ready.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(bit, std::memory_order_release);
    return e;
}

// Records a message for w4a16_last_error() and returns `code`.
int report_error(int code, const char* fmt, ...);

}  // namespace w4a16
