// Attention of prompts and chunks over a paged cache on the sm_100a tensor cores, causal,
// with an optional sliding window and sinks.
//
// One CTA takes 256 query rows of one sequence and key-value head, as two tiles of 128: a
// row is (token, query head of the group), token-major, so that all heads that share keys
// share their loads. Over tiles of 128 keys, with the running maximum m and sum l of the
// softmax (fp32, base 2):
//   S = Q K^T (tcgen05, fp32 in TMEM), P = 2^(scale S - m) rounded to 16 bits, O += P V.
// P replaces S in TMEM and is the A operand of the second product, read from there; V, whose
// rows are keys, is an MN-major B operand. O stays in TMEM; it is rescaled only when a row's
// maximum grew by more than 2^8 (l and O share the factor; P stays in the type's range), so
// that the usual tile costs no round trip of O.
//
// Rounding P to the 16-bit type (at most half a step each) is what lets the second product
// run on the tensor cores at their 16-bit rate; l sums the unrounded fp32 values. In fp16 P and l
// are taken times 2^7: steps end at 2^-24, so that a weight of less than 2^-21 of the maximum
// at hand loses bits, but n keys lose less than n 2^-32 of the whole.
//
// One persistent CTA per SM goes through its items (256 rows), which all roles learn from the
// loading warp; the next item's rows and keys are loaded behind the current one's.
//
// Warp roles (384 threads): warps 0-3 and 4-7 softmax and epilogue of the two row tiles, one
// row a thread; warp 8 plans the items and loads Q, and K and V page by page (TMA, lane =
// page; a page id that is no page reads zeros behind the cache's end); warp 9 puts zeros into
// V where a tile holds keys that no row sees; warps 10 and 11 issue the MMAs of one row tile
// each: while one is in its softmax, the tensor cores work for the other. One warp for both
// left them idle a third of the time: its waits, slowed to some 300 cycles each by the
// exponentials that share the queue to the shared-memory and special-function units, added up.
// Rows whose sums come out not finite are marked and settled by the softmax warps behind the CTA's
// last item.
//
// What bounds it: the tensor cores and, between them, the chain scores - softmax - product of
// each row tile, at the clock that the power cap leaves. The MMAs of a step (both row tiles,
// 128 keys, 128 dimensions) take 2896 cycles by themselves: 16 of M = N = 128 with both
// operands in shared memory at 107, 16 with P in TMEM at 74. A step takes 3260 of them in a
// long prompt, and 7 thousand go to an item's beginning and end. One prompt of 8192 tokens, 32
// heads, bf16: 474 us while the clock is at 1.8 GHz (1160 TFLOP/s over the visible pairs), 574
// to 592 us (928 to 957) under load for long, at 1.5 GHz.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include <cuda.h>

#include "w4a16_internal.h"
#include "w4a16_paged.cuh"
#include "w4a16_ptx.cuh"

namespace w4a16 {
namespace {

constexpr int kTileKeys = 128;
constexpr int kTileRows = 128;
constexpr int kThreads = 12 * 32;
constexpr int kLoadWarp = 8, kCleanWarp = 9, kMmaWarp = 10;  // kMmaWarp + t: row tile t
// Registers a thread: 168 at launch (65536 / 384); the last four warps give theirs to the
// softmax warps, whose 128 scores a row stay in registers: 2 * 128 * 208 + 128 * 88 of the
// 384 * 168 that the CTA was launched with.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "more registers than launched with");
constexpr int kPostInts = 17;      // of an item and its view
constexpr int kBlock = 128 * 128;  // bytes of a [128 rows x 64] operand block, 128-byte swizzle
constexpr uint32_t kWaitLimit = 1u << 18;  // x at most 10 us of sleep: up to a few seconds
constexpr float kSlack = 8.f;              // log2 of the growth that O tolerates without rescaling
static_assert(kSlack + kWeightBias<false, kTileKeys> < 16.f, "fp16 weights that overflow");

enum : int { kErrLoad = 1, kErrMma = 2, kErrSoftmax = 3, kErrEnd = 4 };
__device__ int g_attention_error;

template <int DP>
struct Cfg {
    static constexpr int kBlocks = DP / 64;
    static constexpr int kTileBytes = kBlocks * kBlock;  // 128 rows of Q, K or V
    static constexpr int kSlots = DP == 128 ? 5 : 8;     // K and V tiles in turn
    static constexpr int kKvOff = 2 * kTileBytes;
    static constexpr int kBarOff = kKvOff + kSlots * kTileBytes;
    static constexpr int kListOff = kBarOff + 512;           // barriers and posted items before it
    static_assert((2 * kSlots + 18) * 8 + 4 + 10 * 4 + 8 * 4 + 2 * kPostInts * 4 <= kListOff - kBarOff, "barriers and posted items");
    static constexpr int kSmem = kListOff + (kThreads + 1) * 4 + 1020;  // and alignment
    static_assert(kSmem <= 227 * 1024, "shared memory budget");
    // TMEM columns: S of both row tiles (P in their first 64), O of both
    static constexpr int kS = 0, kO = 256;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
        "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, "
        "%25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 of_pair(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x of two values on the FMA units, x <= 15: 2^round(x) by the exponent bits, 2^f for f in
// [-1/2, 1/2] by the polynomial of degree 4 of least relative error with value 1 at 0
// (2.8e-6, a hundredth of the 16-bit rounding that follows). Below -126 it runs out through
// the denormals to exactly 0 at -127, where smaller x (and -inf) are held. NaN stays NaN.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
    const uint64_t v = pair_of(x.x, x.y);
    const uint64_t r = add2(v, pair_of(12582912.f, 12582912.f));  // round(x) in the low bits
    const uint64_t f = fma2(add2(r, pair_of(-12582912.f, -12582912.f)), pair_of(-1.f, -1.f), v);
    uint64_t y = fma2(f, pair_of(0.009582700208f, 0.009582700208f), pair_of(0.05590687692f, 0.05590687692f));
    y = fma2(y, f, pair_of(0.2402410358f, 0.2402410358f));
    y = fma2(y, f, pair_of(0.6931241155f, 0.6931241155f));
    y = fma2(y, f, pair_of(1.f, 1.f));
    const float2 a = of_pair(y), b = of_pair(r);
    return make_float2(__int_as_float(__float_as_int(a.x) + (__float_as_int(b.x) << 23)),
                       __int_as_float(__float_as_int(a.y) + (__float_as_int(b.y) << 23)));
}
// Weights are 2^(sc s - base) in one fused operation, base rounded: a factor that the row's weights share,
// but for maxima far beyond what data gives rise to it would take them out of their range. Rows
// that had such a maximum (2^22 in base 2: a factor of 2^(1/4)) are computed anew.
constexpr float kLargeBase = 4194304.f;

// What is taken from a row's scaled scores: its maximum so far, and the weights' factor.
template <bool BF16>
__device__ __forceinline__ float base_of(float m, float sc) {
    return (m == -INFINITY ? 0.f : m * sc) - kWeightBias<BF16, kTileKeys>;
}
// 64 of a row's weights, 2^(sc s - base), packed into the first 32 of s; returns their sum.
// Two pairs of seven are raised on the FMA units, beside the special-function units, which
// both row tiles share: one prompt of 8192 tokens, 32 heads, 512 us with none there, 513 with
// one of eight or of four, 490 with two of seven, 495 with one of three, 538 with half.
template <bool BF16>
__device__ __forceinline__ float weights(uint32_t* s, float sc, float base) {
    const uint64_t sc2 = pair_of(sc, sc), base2 = pair_of(-base, -base);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < 64; c += 2) {
        float2 x = of_pair(fma2(pair_of(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, base2));
        if ((c >> 1) % 7 == 2 || (c >> 1) % 7 == 5) {
            x = exp2_fma(x);
        } else {
            x.x = exp2_approx(x.x);
            x.y = exp2_approx(x.y);
        }
        sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], pair_of(x.x, x.y));
        s[c >> 1] = pack2<BF16>(x.x, x.y);
    }
    const float2 part = of_pair(add2(sum[0], sum[1]));
    return part.x + part.y;
}
// The largest of 64 scores.
__device__ __forceinline__ float largest(const uint32_t* s) {
    float x[2] = {fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])), fmaxf(__uint_as_float(s[2]), __uint_as_float(s[3]))};
#pragma unroll
    for (int c = 4; c < 64; c += 4) {
        x[0] = max3(x[0], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
        x[1] = max3(x[1], __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
    }
    return fmaxf(x[0], x[1]);
}
// Half of P into its columns at `ts`, and the arrival that lets its product start.
__device__ __forceinline__ void put_half(uint32_t ts, const uint32_t* s, uint64_t* pfull) {
    tmem_st32(ts, s);
    ptx::tmem_st_wait();
    ptx::tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(pfull);
}

// Bounded wait that sleeps between polls. Not unrolled, as nothing in this kernel that need
// not be: with everything unrolled it had 180 KB of instructions, and fetching them again for
// every CTA and tile took longer than the work.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* err, int code) {
#pragma unroll 1
    for (uint32_t i = 0; i < kWaitLimit; ++i)
        if (ptx::mbar_try_wait_sleep(bar, parity, 10000u)) return true;
    atomicCAS(err, 0, code);
    return false;
}
// The same answer in every lane of the warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
    return __all_sync(0xffffffffu, wait(bar, parity, err, code));
}

// As warp_wait, for whoever waits until some tile of an item is reached, however many come before
// it: gives up when for kWaitLimit polls no tile was loaded either (*loaded did not change). Only where
// time does not count: the same in every wait cost 4 to 6 % of a prompt.
__device__ __forceinline__ bool warp_wait_long(uint64_t* bar, uint32_t parity, int* err, int code, const volatile int* loaded) {
    bool ok = false;
#pragma unroll 1
    for (int seen = *loaded, now;; seen = now) {
#pragma unroll 1
        for (uint32_t i = 0; i < kWaitLimit && !ok; ++i) ok = ptx::mbar_try_wait_sleep(bar, parity, 10000u);
        now = *loaded;
        if (__all_sync(0xffffffffu, ok)) return true;
        if (__all_sync(0xffffffffu, ok || now == seen)) break;
    }
    atomicCAS(err, 0, code);
    return false;
}

// The lowest n bits, n held to 0 .. 32.
__device__ __forceinline__ uint32_t first_bits(int n) {
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// The most items there can be: batch x row pairs x heads, capped well above what is taken.
int64_t most_items(const AttnArgs& a) {
    const int64_t rows = static_cast<int64_t>(std::min(a.seqs.max_q, a.seqs.tokens)) * a.group;
    const int64_t pairs = (rows + 2 * kTileRows - 1) / (2 * kTileRows) * a.pages.heads_kv;
    return pairs > (int64_t{1} << 31) ? pairs : pairs * a.seqs.batch;
}

// One unit of work: 256 query rows of one sequence and key-value head.
struct Item {
    int b, h, row0;   // sequence, head, first row
    int rows;         // of the sequence
    int t0, p0;       // as Seq
    int j0, j1;       // key tiles: all of them, or a part (the results are then parts too)
};

// What the warps derive from an item: positions, key tiles, which tiles matter to whom.
struct View {
    int p_lo[2], p_hi[2];  // of each row tile's first and last row; p_hi -1: no rows
    int last;              // position of the last row
    int first_seen;        // first key of the earliest window
    int window, sinks;
    KeyTiles<kTileKeys> kt;
    __device__ __forceinline__ View() : kt(0, -1, 0, 0) {}
    __device__ __forceinline__ View(const Item& it, const AttnArgs& a)
        : last(it.p0 + (min(it.rows, it.row0 + 2 * kTileRows) - 1) / a.group),
          first_seen(a.window ? max(0, max(it.p0 + it.row0 / a.group, 0) + 1 - a.window) : 0),
          window(a.window),
          sinks(a.sinks),
          kt(it.p0 + it.row0 / a.group, last, a.window, a.sinks) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r0 = it.row0 + t * kTileRows, r1 = min(it.rows, r0 + kTileRows) - 1;
            p_lo[t] = it.p0 + r0 / a.group;
            p_hi[t] = r0 < it.rows ? it.p0 + r1 / a.group : -1;
        }
    }
    // Whether the 128 keys from k0 hold some that no row sees: behind the length or before the
    // window. What lies there is anybody's, and 0 x NaN would reach every row.
    __device__ __forceinline__ bool cut(int k0) const {
        return k0 + kTileKeys - 1 > last || (k0 < first_seen && k0 + kTileKeys > sinks);
    }
    // Whether any row of row tile t sees any key of the 128 from k0.
    __device__ __forceinline__ bool active(int t, int k0) const {
        return k0 <= p_hi[t] && (window == 0 || k0 + kTileKeys - 1 > max(p_lo[t], 0) - window || k0 < sinks);
    }
};

// Below so many rounds of the CTAs over the items, the last one's are cut along their keys:
// with more, the time lost in it is small beside the others. A piece has at least four tiles.
constexpr int kSplitRounds = 4, kPieceTiles = 4;

// Whether items may be cut: few items, and long enough for two pieces as far as the host knows.
int64_t most_tiles(const AttnArgs& a) {
    const int64_t covered = static_cast<int64_t>(a.seqs.width) << a.pages.page_shift;
    int64_t tiles = (covered + kTileKeys - 1) / kTileKeys;
    if (a.window)
        tiles = std::min<int64_t>(tiles, (int64_t{a.sinks} + kTileKeys - 1) / kTileKeys +
                                             (int64_t{a.window} + 2 * kTileRows / a.group + 2 * kTileKeys) / kTileKeys);
    return tiles;
}
bool prompt_may_split(const AttnArgs& a, int num_sms) {
    return most_items(a) < int64_t{kSplitRounds} * num_sms && most_tiles(a) >= 2 * kPieceTiles;
}
int prompt_ctas(const AttnArgs& a, int num_sms) {
    const int64_t pieces = prompt_may_split(a, num_sms) ? most_tiles(a) / kPieceTiles : 1;
    return static_cast<int>(std::min<int64_t>(num_sms, most_items(a) * pieces));
}

// Workspace of cut items: of each CTA m[256], l[256], o[256][DP] of the one piece it can have,
// then {it has one, first CTA and number of the item's pieces, 0, row0, rows, t0, head}.
constexpr int part_floats(int dp) { return 2 * kTileRows * (dp + 2); }
template <int DP>
__device__ __forceinline__ float* part_slot(const AttnArgs& a, int cta) {
    return a.ws + static_cast<size_t>(cta) * part_floats(DP);
}
template <int DP>
__device__ __forceinline__ int* part_desc(const AttnArgs& a, int ctas, int cta) {
    return reinterpret_cast<int*>(a.ws + static_cast<size_t>(ctas) * part_floats(DP)) + cta * 8;
}

// Items of a sequence: its row pairs, those that see most keys first, over the heads. The host
// has made sure that all of a call fit 31 bits.
__device__ __forceinline__ int items_of(const AttnArgs& a, const Seq& s) {
    return (s.nq * a.group + 2 * kTileRows - 1) / (2 * kTileRows) * a.pages.heads_kv;
}

// Item k of this CTA; false: it has none (x.b is then -1). Rounds of the CTAs run forth and back over
// the items, whose work falls along a sequence: a CTA's shares even out. Where there are few
// rounds, the items of the last, incomplete one are cut along their keys, among all CTAs. `before`
// holds the items before each thread's `per` sequences, `total` of all. A whole warp.
__device__ __forceinline__ bool plan_item(const AttnArgs& a, const int* before, int per, int total, int may_split, int k,
                                          Item& x, View& v, int& piece, int& pieces) {
    const int ctas = gridDim.x, lane = threadIdx.x & 31;
    int64_t at = static_cast<int64_t>(k) * ctas + (k & 1 ? ctas - 1 - static_cast<int>(blockIdx.x) : blockIdx.x);
    pieces = 1, piece = 0;
    const int rounds = total / ctas, rest_items = total - rounds * ctas;
    if (may_split && rounds < kSplitRounds && k >= rounds) {
        pieces = rest_items > 0 ? ctas / rest_items : 1;
        piece = static_cast<int>(blockIdx.x) % pieces;
        at = static_cast<int64_t>(rounds) * ctas + static_cast<int>(blockIdx.x) / pieces;
        if (k > rounds) at = total;
    }
    x.b = -1;
    if (at >= total) return false;
    // the thread whose sequences hold it: how many end at or before it
    int holder = 0;
#pragma unroll 1
    for (int y = 0; y < kThreads && y * per < a.seqs.batch; y += 32)
        holder += __popc(__ballot_sync(0xffffffffu, before[y + lane + 1] <= at));
    int rest = static_cast<int>(at) - before[holder], b = holder * per;
    Seq sq = load_seq(a.seqs, a.pages.page_shift, b);
#pragma unroll 1
    for (int n; rest >= (n = items_of(a, sq));) {
        rest -= n;
        sq = load_seq(a.seqs, a.pages.page_shift, ++b);
    }
    const int pairs = (sq.nq * a.group + 2 * kTileRows - 1) / (2 * kTileRows);
    x.row0 = (pairs - 1 - rest / a.pages.heads_kv) * 2 * kTileRows;
    x.h = rest % a.pages.heads_kv;
    x.rows = sq.nq * a.group;
    x.t0 = sq.t0;
    x.p0 = sq.p0;
    v = View(x, a);
    const int n = v.kt.count;
    pieces = min(pieces, max(1, n / kPieceTiles));
    if (piece >= pieces) return false;
    x.b = b;
    x.j0 = static_cast<int>(static_cast<int64_t>(n) * piece / pieces);
    x.j1 = static_cast<int>(static_cast<int64_t>(n) * (piece + 1) / pieces);
    return true;
}

// A row that has to be settled is marked until then: in the output, all that is not finite becomes a
// NaN that no conversion makes; of a part, the sum of weights gets a minus sign.
template <bool BF16>
constexpr uint32_t kExponent = BF16 ? 0x7f80u : 0x7c00u;
template <bool BF16>
constexpr uint32_t kMark = kExponent<BF16> | 1u;

// Marks the rows of a warp whose bit is set, a lane a row: all of it if it is to be computed anew. A
// row of a part lies at `o`, its sum of weights at `l`. Of item k, which is noted in *items.
template <bool BF16>
__device__ __noinline__ void mark_rows(uint32_t rows, bool all, uint16_t* row, int dim, float* l, float* o,
                                       volatile uint32_t* items, int k) {
    const int lane = threadIdx.x & 31;
    const bool mine = (rows >> lane) & 1u;
    if (lane == 0) *items |= 1u << (k & 31);
    if (mine && l) *l = all ? -1.f : -*l;
#pragma unroll 1
    for (int d = 0; mine && d < dim; d += 2) {
        if (l) {
            if (all) o[d] = o[d + 1] = NAN;
            continue;
        }
        uint32_t x = *reinterpret_cast<uint32_t*>(row + d);
        if (all || (x & kExponent<BF16>) == kExponent<BF16>) x = (x & 0xffff0000u) | kMark<BF16>;
        if (all || ((x >> 16) & kExponent<BF16>) == kExponent<BF16>) x = (x & 0xffffu) | (kMark<BF16> << 16);
        *reinterpret_cast<uint32_t*>(row + d) = x;
    }
    __syncwarp();
}

// Settles the marked rows of the CTA's items k whose bit k % 32 is set in `items`, 16 rows a softmax
// warp. Behind the last item, when nobody waits for a barrier with a limit any more: rows that are
// computed anew can take longer than such a wait lasts (prompts of 2048 tokens, one of them behind
// 198016 others and with a NaN 60 tokens before its end: 2.9 ms without, 129 with it).
template <int DP, bool BF16>
__device__ __noinline__ void settle_marked(const AttnArgs& a, const int* before, int total, int may_split, uint32_t items) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (a.seqs.batch + kThreads - 1) / kThreads;
#pragma unroll 1
    for (int k = 0; k <= total / static_cast<int>(gridDim.x) + 1; ++k) {
        Item it;
        View vw;
        int piece, pieces;
        if (((items >> (k & 31)) & 1u) == 0 || !plan_item(a, before, per, total, may_split, k, it, vw, piece, pieces)) continue;
        float* slot = it.j1 - it.j0 < vw.kt.count ? part_slot<DP>(a, blockIdx.x) : nullptr;
#pragma unroll 1
        for (int first = warp * 16; first < 2 * kTileRows; first += 128) {
            const int row = it.row0 + first + lane, token = row / a.group;
            bool marked = false;
            if (lane < 16 && row < it.rows && slot) {
                float* l = slot + 2 * kTileRows + first + lane;
                marked = __float_as_int(*l) < 0 && *l == *l;
                if (marked) *l = fabsf(*l);
            } else if (lane < 16 && row < it.rows) {
                const uint16_t* x = a.out + static_cast<int64_t>(it.t0 + token) * a.o_token +
                                    (it.h * a.group + row - token * a.group) * a.o_head;
#pragma unroll 1
                for (int d = 0; d < a.pages.dim && !marked; ++d) marked = x[d] == kMark<BF16>;
            }
            const uint32_t bad = __ballot_sync(0xffffffffu, marked);
            if (bad)
                settle_rows<kTileKeys, DP, BF16>(a, it.b, it.h, it.t0, it.p0, it.row0 + first, bad, vw.kt, it.j0, it.j1, slot,
                                                 2 * kTileRows, first);
        }
    }
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ AttnArgs a, const int q_by_tma,
                  const int may_split) {
    using C = Cfg<DP>;
    constexpr int CH = DP / 8;
    constexpr int SL = C::kSlots;
    extern __shared__ __align__(1024) uint8_t smem_dyn[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
    uint64_t* empty = full + SL;
    uint64_t* qfull = empty + SL;   // the query rows are in place
    uint64_t* qempty = qfull + 1;   // and all scores of them are made
    uint64_t* sfull = qempty + 1;   // [2] S of a row tile is complete (and all products before it)
    uint64_t* pfull = sfull + 2;    // [2][2] half of P is written (the first: O rescaled)
    uint64_t* ofull = pfull + 4;    // [2] all products of a row tile are complete, of an item that has some for it
    uint64_t* dirty = ofull + 2;    // V of a tile that the mask cuts is loaded
    uint64_t* clean = dirty + 1;    // and holds zeros where no row sees
    uint64_t* ifull = clean + 1;    // [2] an item is posted
    uint64_t* iempty = ifull + 2;   // [2] and was read by all
    uint64_t* turn = iempty + 2;    // [2] a row tile's turn at the tensor cores
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(turn + 2);
    volatile int* loaded = reinterpret_cast<volatile int*>(tmem_slot + 1);  // tiles of K and V so far
    volatile int* all_items = loaded + 1;                           // of all sequences
    volatile uint32_t* to_settle = tmem_slot + 3;  // [8] of each softmax warp: items with marked rows, a bit each by k % 32
    volatile uint32_t* bad = to_settle + 8;                         // [8] boxes of tile j % 8 whose page id is no page
    volatile int* posted = reinterpret_cast<volatile int*>(bad + 8);  // [2][kPostInts] items; b = -1: no more
    int* before = reinterpret_cast<int*>(smem + C::kListOff);       // [kThreads + 1] items before a thread's sequences

    ptx::grid_dep_wait();
    if (may_split) ptx::grid_dep_launch_dependents();  // the join, which waits for all of this
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- how many items come before each thread's share of the sequences
    const int per = (a.seqs.batch + kThreads - 1) / kThreads;
    {
        const int b0 = min(a.seqs.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.seqs.batch, b0 + per);
        int sum = 0;
#pragma unroll 1
        for (int b = b0; b < b1; ++b) sum += items_of(a, load_seq(a.seqs, a.pages.page_shift, b));
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += o;
        }
        before[threadIdx.x + 1] = sum;
        if (threadIdx.x == 0) before[0] = 0;
    }
    if (threadIdx.x == 0) {
        if (may_split) part_desc<DP>(a, gridDim.x, blockIdx.x)[0] = 0;
        *loaded = 0;
        for (int w = 0; w < 8; ++w) to_settle[w] = 0;
        for (int s = 0; s < SL; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 2);
        }
        ptx::mbar_init(qfull, 1);
        ptx::mbar_init(qempty, 2);
        for (int t = 0; t < 2; ++t) {
            ptx::mbar_init(&ofull[t], 1);
            ptx::mbar_init(&sfull[t], 2);
            ptx::mbar_init(&pfull[2 * t], 4);
            ptx::mbar_init(&pfull[2 * t + 1], 4);
            ptx::mbar_init(&ifull[t], 1);
            ptx::mbar_init(&iempty[t], 11);
            ptx::mbar_init(&turn[t], 1);
        }
        ptx::mbar_init(dirty, 2);
        ptx::mbar_init(clean, 1);
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tm_k);
        ptx::prefetch_tmap(&tm_v);
        if (q_by_tma) ptx::prefetch_tmap(&tm_q);
    }
    if (warp == kMmaWarp) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    int* err = &g_attention_error;

    // Item k of this CTA and its view as the loading warp posted them; false: there is none (or a
    // wait gave up).
    auto next_item = [&](int k, Item& it, View& vw, bool whole_warp) {
        const int s = k & 1, parity = (k >> 1) & 1;
        bool ok = wait(&ifull[s], parity, err, kErrLoad);
        if (whole_warp) ok = __all_sync(0xffffffffu, ok);
        if (!ok) return false;
        volatile int* x = posted + s * kPostInts;
        it.b = x[0], it.h = x[1], it.row0 = x[2], it.rows = x[3], it.t0 = x[4], it.p0 = x[5], it.j0 = x[6], it.j1 = x[7];
        vw.p_lo[0] = x[8], vw.p_lo[1] = x[9], vw.p_hi[0] = x[10], vw.p_hi[1] = x[11];
        vw.last = x[12], vw.first_seen = x[13], vw.window = a.window, vw.sinks = a.sinks;
        vw.kt.sink_tiles = x[14], vw.kt.win_tile = x[15], vw.kt.count = x[16];
        if (whole_warp) __syncwarp();
        if (!whole_warp || lane == 0) ptx::mbar_arrive(&iempty[s]);
        return it.b >= 0;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kLoadWarp) {
            // ------------------------------------------------ items; Q; K and V, page by page
            const int page_size = 1 << a.pages.page_shift;
            const int box = min(page_size, kTileKeys);
            const int boxes = kTileKeys / box;  // per tile, at most 16: one a lane
            int total = 0;  // of all sequences; the warps' sums become one running sum
#pragma unroll 1
            for (int x = 0; x < kThreads && x * per < a.seqs.batch; x += 32) {
                const int y = before[x + lane + 1] + total;
                __syncwarp();
                before[x + lane + 1] = y;
                total = __shfl_sync(0xffffffffu, y, 31);
            }
            __syncwarp();
            if (lane == 0) *all_items = total;
            const int ctas = gridDim.x;
            int i = 0, q_loads = 0;  // tiles of K and V, row pairs of Q so far
            bool ok = true;
            Item it, nx;  // the item whose tiles are loaded, and the next
            View vw, vx;
            it.b = nx.b = -1;
            it.j0 = it.j1 = nx.j0 = nx.j1 = 0;
            auto page_of = [&](const Item& x, const View& v, int j) {  // this lane's page of key tile j
                int page = a.pages.num_pages;  // behind the cache's end: zeros
                if (j < x.j1 && lane < boxes) {
                    const int key = v.kt.first(j) + lane * box;
                    if (key <= v.last) page = a.seqs.tables[x.b * a.seqs.table_stride + (key >> a.pages.page_shift)];
                }
                return page;
            };
            int page = 0, nx_page = 0;
            // item k's tiles; behind its first one and Q, item k + 1 is planned and posted, so that
            // nobody waits for it (k = -1: only that)
#pragma unroll 1
            for (int k = -1; ok; ++k) {
                bool planned = false;
#pragma unroll 1
                for (int j = it.j0; ok;) {
                    if (j < it.j1) {
                        const int key = vw.kt.first(j) + lane * box;
                        const int next = page_of(it, vw, j + 1);
                        const bool none = page < 0 || page >= a.pages.num_pages;
                        const uint32_t none_of = __ballot_sync(0xffffffffu, none && lane < boxes && key <= vw.last);
                        if (none) page = a.pages.num_pages;
#pragma unroll 1
                        for (int w = 0; w < 2; ++w, ++i) {
                            const int sl = i % SL;
                            if (i >= SL) ok = warp_wait(&empty[sl], ((i / SL) - 1) & 1, err, kErrLoad);
                            if (!ok) break;
                            if (lane == 0) {
                                if (w == 0) bad[(i >> 1) & 7] = none_of;
                                ptx::mbar_arrive_expect_tx(&full[sl], C::kTileBytes);
                            }
                            __syncwarp();
                            if (lane < boxes) {
                                const uint32_t dst = ptx::smem_u32(smem + C::kKvOff + sl * C::kTileBytes) + lane * box * 128;
#pragma unroll
                                for (int d = 0; d < C::kBlocks; ++d)
                                    tma_load_4d(dst + d * kBlock, w ? &tm_v : &tm_k, &full[sl], d * 64, key & (page_size - 1), it.h,
                                                page);
                            }
                        }
                        if (lane == 0) *loaded = i;
                        page = next;
                        ++j;
                    }
                    if (planned) {
                        if (j >= it.j1) break;
                        continue;
                    }
                    planned = true;
                    if (k >= 0 && ok && q_by_tma) {
                        // after the first keys: the rows of the last item may still be in use. An item
                        // without keys takes no Q, but its phases pass all the same.
                        if (k > 0) ok = warp_wait(qempty, (k - 1) & 1, err, kErrLoad);
                        if (ok && lane == 0 && it.j0 < it.j1) {
                            ptx::mbar_arrive_expect_tx(qfull, 2 * C::kTileBytes);
                            const int tokens = kTileRows / a.group, token = it.t0 + it.row0 / a.group;
                            for (int x = 0; x < 2 * C::kBlocks; ++x)
                                tma_load_3d(ptx::smem_u32(smem) + x * kBlock, &tm_q, qfull, (x % C::kBlocks) * 64, it.h * a.group,
                                            token + (x / C::kBlocks) * tokens);
                        } else if (ok && lane == 0) {
                            ptx::mbar_arrive(qfull);
                        }
                        if (ok) ++q_loads;
                    }

                    // ---- item k + 1
                    const int k1 = k + 1, s = k1 & 1;
                    int piece = 0, pieces = 1;
                    nx.b = -1;
                    if (plan_item(a, before, per, total, may_split, k1, nx, vx, piece, pieces)) {
                        nx_page = page_of(nx, vx, nx.j0);
                        if (pieces > 1 && lane == 0) {
                            int4* d = reinterpret_cast<int4*>(part_desc<DP>(a, ctas, blockIdx.x));
                            d[1] = make_int4(nx.row0, nx.rows, nx.t0, nx.h);
                            d[0] = make_int4(1, blockIdx.x - piece, pieces, 0);
                        }
                    }
                    if (ok && k1 >= 2) ok = warp_wait(&iempty[s], ((k1 >> 1) - 1) & 1, err, kErrLoad);
                    if (lane == 0) {
                        volatile int* x = posted + s * kPostInts;
                        x[0] = ok ? nx.b : -1, x[1] = nx.h, x[2] = nx.row0, x[3] = nx.rows, x[4] = nx.t0, x[5] = nx.p0;
                        x[6] = nx.j0, x[7] = nx.j1, x[8] = vx.p_lo[0], x[9] = vx.p_lo[1], x[10] = vx.p_hi[0], x[11] = vx.p_hi[1];
                        x[12] = vx.last, x[13] = vx.first_seen;
                        x[14] = vx.kt.sink_tiles, x[15] = vx.kt.win_tile, x[16] = vx.kt.count;
                        ptx::mbar_arrive(&ifull[s]);
                    }
                    if (j >= it.j1) break;
                }
                if (nx.b < 0) break;
                it = nx;
                vw = vx;
                page = nx_page;
            }
            // no copy may be in flight when the CTA ends
#pragma unroll 1
            for (int x = max(0, i - SL); x < i; ++x) warp_wait(&full[x % SL], (x / SL) & 1, err, kErrLoad);
            if (q_loads > 0) warp_wait(qfull, (q_loads - 1) & 1, err, kErrLoad);
        } else if (warp == kCleanWarp) {
            // ------------------------------------------------ zeros into V where no row sees; Q, where a
            // group of heads does not divide a row tile
            int i = 0, asked = 0;
            bool ok = true;
            Item it;
            View vw;
#pragma unroll 1
            for (int k = 0; ok && next_item(k, it, vw, true); ++k) {
                if (!q_by_tma) {
                    if (k > 0) ok = warp_wait_long(qempty, (k - 1) & 1, err, kErrMma, loaded);
                    if (!ok) break;
                    // 16 bytes a lane and copy, into the swizzled operand layout
                    constexpr int kStep = 32 / CH;  // rows between a lane's chunks
                    const uint32_t dst = ptx::smem_u32(smem);
                    const int c = lane % CH, left = it.rows - it.row0;  // rows of this item
                    int r = lane / CH, token = (it.row0 + r) / a.group, g = it.row0 + r - token * a.group;
#pragma unroll 2
                    for (; r < 2 * kTileRows; r += kStep) {
                        const bool in = c * 8 < a.pages.dim && r < left && it.j0 < it.j1;
                        const uint16_t* src =
                            in ? a.q + (it.t0 + token) * a.q_token + (it.h * a.group + g) * a.q_head + c * 8 : a.q;
                        cp_async16(dst + (r >> 7) * C::kTileBytes + (c >> 3) * kBlock + (r & 127) * 128 +
                                       (((c & 7) ^ (r & 7)) << 4),
                                   src, in ? 16u : 0u);
                        g += kStep;
                        while (g >= a.group) {
                            g -= a.group;
                            ++token;
                        }
                    }
                    cp_async_wait_all();
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(qfull);
                }
                // asked for by both MMA threads, one tile at a time (a barrier's parity tells only two
                // phases apart: a warp that skips tiles cannot wait on `full`)
#pragma unroll 1
                for (int j = it.j0; j < it.j1 && ok; ++j, i += 2) {
                    const int k0 = vw.kt.first(j);
                    if (!vw.cut(k0)) continue;
                    ok = warp_wait_long(dirty, asked++ & 1, err, kErrMma, loaded);
                    const uint32_t v = ptx::smem_u32(smem + C::kKvOff + ((i + 1) % SL) * C::kTileBytes);
                    // rows [r, r1) of the tile: behind the last key, then between the sinks and the window
                    auto zero = [&](int r, int r1) {
#pragma unroll 4
                        for (r += lane / CH; r < r1; r += 32 / CH)
                            ptx::st_shared_v4(v + (lane % CH >> 3) * kBlock + r * 128 + (lane & 7) * 16, make_uint4(0, 0, 0, 0));
                    };
                    if (ok) zero(max(0, vw.last + 1 - k0), kTileKeys);
                    if (ok) zero(max(0, a.sinks - k0), min(kTileKeys, vw.first_seen - k0));
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(clean);
                }
            }
        } else if (ptx::elect_one_sync()) {
            // ------------------------------------------------ MMA issuer of row tile t: one elected thread,
            // so that the compiler knows it is one and keeps descriptors uniform (an MMA took 106
            // cycles to issue in a `lane == 0` branch, 74 here: the tensor core's time)
            const int t = warp - kMmaWarp;
            constexpr uint32_t idesc_s = ptx::umma_idesc_f16(kTileRows, kTileKeys, BF16);
            constexpr uint32_t idesc_o = ptx::umma_idesc_f16(kTileRows, DP, BF16) | (1u << 16);  // B = V is MN-major
            const uint32_t ts = tmem + C::kS + t * 128, to = tmem + C::kO + t * 128;
            const uint32_t q = ptx::smem_u32(smem) + t * C::kTileBytes, kv = ptx::smem_u32(smem + C::kKvOff);
            int i = 0, done = 0, cleaned = 0;  // tiles of K and V, products P V, tiles taken from the cleaning warp
            int turns = 0;
            bool ok = true;
            auto my_turn = [&]() {  // row tile 0 has the first
                const int x = turns++ - (t == 0 ? 1 : 0);
                return x < 0 || wait(&turn[t], x & 1, err, kErrMma);
            };
            Item it;
            View vw;
#pragma unroll 1
            for (int k = 0; ok && next_item(k, it, vw, false); ++k) {
                const int n = it.j1 - it.j0;  // j counts from the item's first tile
                ok = wait(qfull, k & 1, err, kErrMma);
                bool first = true, ended = false;
                // step j: P V of tile j - 1, then the scores of tile j
#pragma unroll 1
                for (int j = 0; j <= n && ok; ++j, i += 2) {
                    const int iv = i - 1;                            // of V_{j-1}; K_j is i
                    const int sk = i % SL, sv = (iv + SL) % SL;
                    const int k0 = vw.kt.first(it.j0 + j), v0 = vw.kt.first(it.j0 + j - 1);
                    if (j > 0) {
                        if (vw.cut(v0)) ok = wait(clean, cleaned++ & 1, err, kErrMma);
                        if (ok) ok = wait(&full[sv], (iv / SL) & 1, err, kErrMma);
                    }
                    if (ok && j < n) ok = wait(&full[sk], (i / SL) & 1, err, kErrMma);
                    // the first half of P V whenever P is there; the second half and the next scores in
                    // turn with the other row tile: left to interleave, both end together, and then both
                    // softmaxes run at once while the tensor cores idle (4700 cycles a tile, 3200 in turn)
                    const bool product = j > 0 && vw.active(t, v0);
                    const uint32_t v = kv + sv * C::kTileBytes;
                    auto half_product = [&](int half) {
                        if (half == 1 && ok) ok = my_turn();
                        if (ok) ok = wait(&pfull[2 * t + half], done & 1, err, kErrMma);
                        ptx::tc_fence_after();
#pragma unroll
                        for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                            if (ok)
                                ptx::umma_f16_ts(to, ts + kk * 8, ptx::umma_desc_sw128_mn(v + kk * 2048, kBlock, 1024), idesc_o,
                                                 !first || kk > 0 ? 1u : 0u);
                    };
                    if (ok && product) {
                        half_product(0);
                        half_product(1);
                        ++done;
                        first = false;
                        // the row tile's last product: its epilogue need not wait for the other's
                        if (j < n && k0 > vw.p_hi[t]) {
                            ptx::umma_commit(&ofull[t]);
                            ended = true;
                        }
                    } else if (ok) {
                        ok = my_turn();
                    }
                    if (j > 0) ptx::umma_commit(&empty[sv]);
                    if (ok && j < n) {
                        if (vw.active(t, k0)) {
                            ptx::mbar_arrive(&sfull[t]);  // passes on what the loading warp wrote before `full`
                            const uint32_t kd = kv + sk * C::kTileBytes;
#pragma unroll
                            for (int kk = 0; kk < DP / 16; ++kk) {
                                const uint32_t off = (kk >> 2) * kBlock + (kk & 3) * 32;
                                ptx::umma_f16(ts, ptx::umma_desc_sw128(q + off), ptx::umma_desc_sw128(kd + off), idesc_s,
                                              kk > 0 ? 1u : 0u);
                            }
                            ptx::umma_commit(&sfull[t]);
                        }
                        ptx::umma_commit(&empty[sk]);
                        ptx::mbar_arrive(&turn[t ^ 1]);
                        if (j == n - 1) ptx::umma_commit(qempty);
                        if (vw.cut(k0)) {
                            ok = wait(&full[(i + 1) % SL], ((i + 1) / SL) & 1, err, kErrMma);
                            ptx::mbar_arrive(dirty);
                        }
                    } else if (ok) {
                        ptx::mbar_arrive(&turn[t ^ 1]);
                    }
                }
                i -= 2;  // step n has no K
                if (n == 0) ptx::umma_commit(qempty);
                // only an item that has a product for this row tile is signalled: such a one waits for the
                // softmax warps, others could run two phases ahead of them, which a parity does not tell apart
                if (!ended && !first) ptx::umma_commit(&ofull[t]);
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ------------------------------------------------ softmax of row tile t, a row a thread
        const int t = warp >> 2, tid = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + C::kS + t * 128 + lanes, to = tmem + C::kO + t * 128 + lanes;
        const int step_shift = min(a.pages.page_shift, 7);
        const float sc = a.scale_log2;
        const bool wide = ((reinterpret_cast<uintptr_t>(a.out) & 31) | ((a.o_token | a.o_head | a.pages.dim) & 15)) == 0;
        int i = 0, seen = 0, ends = 0;  // tiles of keys; scores taken; items with any
        bool ok = true;
        Item it;
        View vw;
#pragma unroll 1
        for (int k = 0; ok && next_item(k, it, vw, true); ++k) {
            const bool part = it.j1 - it.j0 < vw.kt.count;
            const int row = it.row0 + t * kTileRows + tid;
            const bool live_row = row < it.rows;
            const int p = live_row ? max(-1, it.p0 + row / a.group) : -1;
            float m = -INFINITY, l = 0.f;  // m in units of the unscaled score
            bool first = true, large = false;
#pragma unroll 1
            for (int j = it.j0; j < it.j1; ++j, ++i) {
                const int k0 = vw.kt.first(j);
                if (!vw.active(t, k0)) continue;
                if (!warp_wait(&sfull[t], seen & 1, err, kErrSoftmax)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
                const uint32_t no_page = bad[i & 7];
                const bool whole = no_page == 0 && k0 + kTileKeys - 1 <= vw.p_lo[t] &&
                                   (a.window == 0 || vw.p_hi[t] - k0 < a.window || k0 + kTileKeys <= a.sinks);
                // The first half's weights are taken against the maximum so far, while this tile's own
                // is still being found; only a row that outgrew it by 2^8 has them taken once more.
                uint32_t s[kTileKeys];
                float part;
                bool masked = false;
                for (;;) {
                    if (__builtin_expect(!whole && !masked, 0)) {
                        // into the scores where they lie, 32 keys at a time: a bit a key, up to the row's own,
                        // in its window or among the sinks, on pages that are pages
                        masked = true;
                        const int hi = p - k0, lo = a.window ? hi - a.window : -1, sink = a.window ? a.sinks - k0 : 0;
#pragma unroll 1
                        for (int c = 0; c < kTileKeys; c += 32) {
                            uint32_t in = first_bits(hi + 1 - c) & (~first_bits(lo + 1 - c) | first_bits(sink - c));
                            if (no_page != 0) {
#pragma unroll 1
                                for (int e = 0; e < 32; e += 8)
                                    if ((no_page >> ((c + e) >> step_shift)) & 1) in &= ~(0xffu << e);
                            }
                            tmem_ld32(ts + c, s);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!((in >> e) & 1)) s[e] = 0xff800000u;
                            tmem_st32(ts + c, s);
                        }
                        ptx::tmem_st_wait();
                    }
                    tmem_ld32(ts, s);
                    tmem_ld32(ts + 32, s + 32);
                    ptx::tmem_ld_wait();
                    tmem_ld32(ts + 64, s + 64);
                    tmem_ld32(ts + 96, s + 96);
                    float top = largest(s);
                    if (__builtin_expect(first, 0)) {
                        ptx::tmem_ld_wait();
                        m = fmaxf(top, largest(s + 64));
                        large = fabsf(base_of<BF16>(m, sc)) > kLargeBase;
                    }
                    part = weights<BF16>(s, sc, base_of<BF16>(m, sc));
                    if (first) break;
                    ptx::tmem_ld_wait();
                    top = fmaxf(top, largest(s + 64));
                    const bool grow = (top - m) * sc > kSlack || (m == -INFINITY && top > m);
                    if (__builtin_expect(!__any_sync(0xffffffffu, grow), 1)) break;
                    const float f = grow ? exp2_approx((m - top) * sc) : 1.f;
                    if (grow) m = top;
                    large |= fabsf(base_of<BF16>(m, sc)) > kLargeBase;
                    l *= f;
#pragma unroll 1
                    for (int c = 0; c < DP; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(to + c, o);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(to + c, o);
                    }
                }
                put_half(ts, s, &pfull[2 * t]);
                part += weights<BF16>(s + 64, sc, base_of<BF16>(m, sc));
                put_half(ts + 32, s + 64, &pfull[2 * t + 1]);
                l += part;
                ++seen;
                first = false;
            }
            // ------------------------------------------------ epilogue
            if (ok && !first) ok = warp_wait(&ofull[t], ends++ & 1, err, kErrEnd);
            if (!ok) break;
            ptx::tc_fence_after();
            const float inv = part ? 1.f : l == 0.f ? 0.f : 1.f / l;
            const int64_t o_off = (it.t0 + row / a.group) * a.o_token + (it.h * a.group + row % a.group) * a.o_head;
            float* slot = part ? part_slot<DP>(a, blockIdx.x) : nullptr;
            const int pr = t * kTileRows + tid;  // row of the part
            if (part) {
                slot[pr] = m == -INFINITY ? m : m * sc;
                slot[2 * kTileRows + pr] = l;
            }
            bool odd = false;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                uint32_t o[32];
                if (!first) {
                    tmem_ld32(to + c, o);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;  // no product was made
                }
                uint64_t nan = 0;  // stays 0 if all are finite
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const uint64_t y = pair_of(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
                    nan = fma2(y, 0, nan);
                    const float2 z = of_pair(mul2(y, pair_of(inv, inv)));
                    w[e >> 1] = pack2<BF16>(z.x, z.y);
                }
                const float2 z = of_pair(nan);
                odd |= !(z.x + z.y == 0.f);
                if (part) {
                    float* dst = slot + 4 * kTileRows + pr * DP + c;
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        if (live_row)
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + e), "r"(o[e]),
                                         "r"(o[e + 1]), "r"(o[e + 2]), "r"(o[e + 3]), "r"(o[e + 4]), "r"(o[e + 5]), "r"(o[e + 6]),
                                         "r"(o[e + 7])
                                         : "memory");
                } else if (live_row) {
                    if (wide) {  // whole 32-byte sectors a thread: half the requests
#pragma unroll
                        for (int e = 0; e < 16; e += 8)
                            if (c + 2 * e < a.pages.dim)
                                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(a.out + o_off + c + 2 * e),
                                             "r"(w[e]), "r"(w[e + 1]), "r"(w[e + 2]), "r"(w[e + 3]), "r"(w[e + 4]), "r"(w[e + 5]),
                                             "r"(w[e + 6]), "r"(w[e + 7])
                                             : "memory");
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            if (c + 2 * e < a.pages.dim)
                                *reinterpret_cast<uint4*>(a.out + o_off + c + 2 * e) =
                                    make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
                    }
                }
            }
            // rows whose sums are not finite while their sums of weights are
            // rows whose sums are not finite while their sums of weights are
            const uint32_t rows = __ballot_sync(0xffffffffu, live_row && ((odd && l == l) || large));
            if (rows)
                mark_rows<BF16>(rows, large, a.out + o_off, a.pages.dim, part ? slot + 2 * kTileRows + pr : nullptr,
                                slot + 4 * kTileRows + pr * DP, to_settle + warp, k);
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the softmax warps alone
        uint32_t items = 0;
        for (int w = 0; w < 8; ++w) items |= to_settle[w];
        if (items) settle_marked<DP, BF16>(a, before, *all_items, may_split, items);
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// The pieces of the cut items, added in key order: of an item's 256 rows every CTA of its
// pieces (and kJoinParts of them) takes a share, a warp a row.
constexpr int kJoinWarps = 8, kJoinParts = 4;

template <int DP, bool BF16>
__global__ void __launch_bounds__(kJoinWarps * 32) prompt_join_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int E = DP / 32;
    ptx::grid_dep_wait();
    const int ctas = gridDim.x;
    const int4* d = reinterpret_cast<const int4*>(part_desc<DP>(a, ctas, blockIdx.x));
    const int4 d0 = d[0];
    if (d0.x == 0) return;
    const int4 d1 = d[1];
    const int first = d0.y, pieces = d0.z, row0 = d1.x, rows = d1.y, t0 = d1.z, h = d1.w;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int share = (static_cast<int>(blockIdx.x) - first) * kJoinParts + blockIdx.y;
    for (int r = share * kJoinWarps + warp; r < min(2 * kTileRows, rows - row0); r += pieces * kJoinParts * kJoinWarps) {
        float m = -INFINITY;
        for (int c = lane; c < pieces; c += 32) m = fmaxf(m, part_slot<DP>(a, first + c)[r]);
#pragma unroll
        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        const float base = m == -INFINITY ? 0.f : m;
        float o[E] = {}, l = 0.f;
#pragma unroll 4
        for (int c = 0; c < pieces; ++c) {
            const float* s = part_slot<DP>(a, first + c);
            const float f = exp2_approx(s[r] - base + kJoinBias);
            l += f * s[2 * kTileRows + r];
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 u = *reinterpret_cast<const float2*>(s + 4 * kTileRows + r * DP + lane * E + e);
                v[e] = u.x, v[e + 1] = u.y;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += share_of(f, v[e]);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int row = row0 + r, token = row / a.group;
        uint16_t* out = a.out + (t0 + token) * a.o_token + (h * a.group + row - token * a.group) * a.o_head + lane * E;
        if (lane * E < a.pages.dim) {
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<BF16>(o[e] * inv, o[e + 1] * inv);
        }
    }
}

template <int DP, bool BF16>
cudaError_t launch_prompt_t(const AttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const CUtensorMap& tm_q,
                            bool q_by_tma, int num_sms, cudaStream_t s) {
    auto kern = prompt_kernel<DP, BF16>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), Cfg<DP>::kSmem, ready);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(prompt_ctas(a, num_sms));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<DP>::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool may_split = prompt_may_split(a, num_sms);
    e = cudaLaunchKernelEx(&cfg, kern, tm_k, tm_v, tm_q, a, q_by_tma ? 1 : 0, may_split ? 1 : 0);
    if (e != cudaSuccess || !may_split) return e;
    cfg.gridDim.y = kJoinParts;
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, prompt_join_kernel<DP, BF16>, a);
}

}  // namespace

bool prompt_fits(const AttnArgs& a) { return most_items(a) <= (1 << 30); }

size_t prompt_workspace_bytes(const AttnArgs& a, int num_sms) {
    if (!prompt_may_split(a, num_sms)) return 0;
    return static_cast<size_t>(prompt_ctas(a, num_sms)) * (part_floats(a.pages.dim <= 64 ? 64 : 128) * sizeof(float) + 32);
}

cudaError_t launch_prompt(const AttnArgs& a, bool bf16, int num_sms, cudaStream_t s) {
    const PageView& p = a.pages;
    const uint64_t size = uint64_t{1} << p.page_shift;
    const uint64_t dims[4] = {static_cast<uint64_t>(p.dim), size, static_cast<uint64_t>(p.heads_kv),
                              static_cast<uint64_t>(p.num_pages)};
    // the stride of a dimension of one is never used, but must be a valid one
    const uint64_t strides[3] = {static_cast<uint64_t>(p.stride_token) * 2,
                                 p.heads_kv > 1 ? static_cast<uint64_t>(p.stride_head) * 2 : 16,
                                 p.num_pages > 1 ? static_cast<uint64_t>(p.stride_page) * 2 : 16};
    const uint32_t box[4] = {64, static_cast<uint32_t>(std::min<uint64_t>(size, kTileKeys)), 1, 1};
    const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap mk, mv;
    if (encode_tmap_4d(&mk, dt, p.k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) != CUDA_SUCCESS ||
        encode_tmap_4d(&mv, dt, p.v, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    // Q rows token-major by heads of a group: a box of the group's heads and 128 / group tokens is
    // a row tile, where the group divides it
    const bool q_by_tma = kTileRows % a.group == 0 && (a.heads == 1 || a.q_head > 0) && (a.seqs.tokens == 1 || a.q_token > 0);
    CUtensorMap mq = mk;
    if (q_by_tma) {
        const uint64_t qdims[3] = {static_cast<uint64_t>(p.dim), static_cast<uint64_t>(a.heads),
                                   static_cast<uint64_t>(a.seqs.tokens)};
        const uint64_t qstrides[2] = {a.heads > 1 ? static_cast<uint64_t>(a.q_head) * 2 : 16,
                                      a.seqs.tokens > 1 ? static_cast<uint64_t>(a.q_token) * 2 : 16};
        const uint32_t qbox[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(kTileRows / a.group)};
        if (encode_tmap_3d(&mq, dt, a.q, qdims, qstrides, qbox, CU_TENSOR_MAP_SWIZZLE_128B) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    if (p.dim <= 64)
        return bf16 ? launch_prompt_t<64, true>(a, mk, mv, mq, q_by_tma, num_sms, s)
                    : launch_prompt_t<64, false>(a, mk, mv, mq, q_by_tma, num_sms, s);
    return bf16 ? launch_prompt_t<128, true>(a, mk, mv, mq, q_by_tma, num_sms, s)
                : launch_prompt_t<128, false>(a, mk, mv, mq, q_by_tma, num_sms, s);
}

cudaError_t read_attention_error(int* out, cudaStream_t s) {
    const int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_attention_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && *out) e = cudaMemcpyToSymbolAsync(g_attention_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    return e;
}

}  // namespace w4a16
