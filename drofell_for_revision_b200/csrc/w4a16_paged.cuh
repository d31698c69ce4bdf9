// Device helpers shared by the kernels of the paged key-value cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "w4a16_paged.h"

namespace w4a16 {

// A sequence of the call: rows [t0, t0 + nq) of q; the first at position p0 (negative when
// there are more new tokens than the length counts).
struct Seq {
    int t0, nq, p0;
};

__device__ __forceinline__ Seq load_seq(const SeqView& s, int page_shift, int b) {
    Seq r;
    int t0 = b, t1 = b + 1;
    if (s.cu_q) {
        t0 = s.cu_q[b];
        t1 = s.cu_q[b + 1];
    }
    t0 = min(max(t0, 0), s.tokens);
    t1 = min(max(t1, t0), s.tokens);
    // lengths are held to what the table covers: no read goes behind it
    const int len = min(max(s.lens[b], 0), s.width << page_shift);
    r.t0 = t0;
    r.nq = min(t1 - t0, s.max_q);
    r.p0 = len - (t1 - t0);
    return r;
}

// Key j is visible to the query at position p: not after it, and within the window or
// among the first `sinks` keys.
__device__ __forceinline__ bool visible(int j, int p, int window, int sinks) {
    return j <= p && (window == 0 || p - j < window || j < sinks);
}

// The keys that the queries at positions [p_lo, p_hi] see, in tiles of TILE keys: the
// tiles of the sinks that lie before the window, then the tiles from the window's start
// to p_hi. Tile i starts at key first(i).
template <int TILE>
struct KeyTiles {
    int sink_tiles, win_tile, count;
    __device__ __forceinline__ KeyTiles(int p_lo, int p_hi, int window, int sinks) {
        sink_tiles = win_tile = count = 0;
        if (p_hi < 0) return;
        const int lo = window ? max(0, max(p_lo, 0) + 1 - window) : 0;
        win_tile = lo / TILE;
        sink_tiles = (min(sinks, lo) + TILE - 1) / TILE;
        win_tile = max(win_tile, sink_tiles);
        count = sink_tiles + max(0, p_hi / TILE + 1 - win_tile);
    }
    __device__ __forceinline__ int first(int i) const {
        return (i < sink_tiles ? i : win_tile + i - sink_tiles) * TILE;
    }
};

// 16 bytes to shared memory, zeros behind the first `bytes` of them.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
    if constexpr (BF16) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
    } else {
        return __half22float2(*reinterpret_cast<const __half2*>(&x));
    }
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Weights enter the value products in 16 bits, taken times 2^kWeightBias; so do the sums of
// weights, and the factor cancels in their quotient. fp16 holds nothing below 2^-24: without a
// factor all weights of less than 2^-25 of the largest would be counted in the sum and missing in the
// product (130000 of them behind a key that outweighs them: an output off by percents). The
// factors fill fp16's range upwards: the split kernel's weights are at most 1 (its maximum is exact),
// the prompt kernel's at most 2^8 (key tiles of 128). bf16 has fp32's exponents and needs none.
template <bool BF16, int TILE>
constexpr float kWeightBias = BF16 ? 0.f : TILE == 16 ? 15.f : 7.f;

// f v of a piece's sum v under a factor f of at most 1 that may have run out to 0. No weight is
// 0, so an infinity or NaN among the values stays one, however small its piece's share.
__device__ __forceinline__ float share_of(float f, float v) {
    return f == 0.f ? (v * 0.f == 0.f ? 0.f : v) : f * v;
}

// A row's maximum, sum of weights and weighted sum of values (four dimensions a lane).
struct RowSum {
    float m, l, o[4];
};

// One row over key tiles [i0, i1) of 16, key by key and each key by selection. A warp a row, lanes
// over the head's dimensions. Slow, but what the split kernel calls takes registers from its loop
// (the form below: 2 to 3 % of a call).
template <int TILE, bool BF16>
__device__ __noinline__ RowSum row_by_keys(const AttnArgs& a, int b, int h, int64_t q_off, int p, const KeyTiles<TILE> kt,
                                           int i0, int i1) {
    const int d = (threadIdx.x & 31) * 4;
    const bool in = d < a.pages.dim;
    auto load4 = [&](const uint16_t* src, float (&x)[4]) {
        x[0] = x[1] = x[2] = x[3] = 0.f;
        if (!in) return;
        const uint2 r = *reinterpret_cast<const uint2*>(src + d);
        const float2 u = unpack2<BF16>(r.x), v = unpack2<BF16>(r.y);
        x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
    };
    RowSum r = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
    float q[4];
    load4(a.q + q_off, q);
    const int32_t* table = a.seqs.tables + b * a.seqs.table_stride;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
#pragma unroll 1
        for (int c = 0; c < TILE; ++c) {
            const int j = kt.first(i) + c;
            if (!visible(j, p, a.window, a.sinks)) continue;
            const int page = table[j >> a.pages.page_shift];
            if (page < 0 || page >= a.pages.num_pages) continue;
            const int64_t at = page * a.pages.stride_page + h * a.pages.stride_head +
                               (j & ((1 << a.pages.page_shift) - 1)) * a.pages.stride_token;
            float k[4], v[4];
            load4(a.pages.k + at, k);
            load4(a.pages.v + at, v);
            float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            s *= a.scale_log2;
            const float m = fmaxf(r.m, s), base = m == -INFINITY ? 0.f : m;
            const float f = r.m == m ? 1.f : exp2_approx(r.m - base), w = exp2_approx(s - base + kWeightBias<BF16, TILE>);
            r.m = m;
            r.l = r.l * f + w;
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[e] = (f == 0.f ? 0.f : r.o[e] * f) + w * v[e];
        }
    }
    return r;
}

// The same, 32 keys at once: a lane a key for the scores, lanes over the head's dimensions for the
// values.
template <int TILE, bool BF16>
__device__ __noinline__ RowSum row_by_32(const AttnArgs& a, int b, int h, int64_t q_off, int p, const KeyTiles<TILE> kt,
                                           int i0, int i1) {
    static_assert(TILE % 32 == 0, "32 keys of a tile at once");
    const int lane = threadIdx.x & 31, d = lane * 4;
    RowSum r = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
    const int32_t* table = a.seqs.tables + b * a.seqs.table_stride;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
#pragma unroll 1
        for (int c = 0; c < TILE; c += 32) {
            const int j = kt.first(i) + c + lane;
            int page = -1;
            if (visible(j, p, a.window, a.sinks)) page = table[j >> a.pages.page_shift];
            const bool seen = page >= 0 && page < a.pages.num_pages;
            const uint32_t keys = __ballot_sync(0xffffffffu, seen);
            if (keys == 0) continue;
            const int64_t at = seen ? page * a.pages.stride_page + h * a.pages.stride_head +
                                          (j & ((1 << a.pages.page_shift) - 1)) * a.pages.stride_token
                                    : 0;
            float s = 0.f;
            if (seen) {
#pragma unroll 4
                for (int x = 0; x < a.pages.dim; x += 8) {
                    const uint4 qv = *reinterpret_cast<const uint4*>(a.q + q_off + x);
                    const uint4 kv = *reinterpret_cast<const uint4*>(a.pages.k + at + x);
                    const uint32_t qw[4] = {qv.x, qv.y, qv.z, qv.w}, kw[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 u = unpack2<BF16>(qw[e]), w = unpack2<BF16>(kw[e]);
                        s += u.x * w.x + u.y * w.y;
                    }
                }
            }
            s = seen ? s * a.scale_log2 : -INFINITY;
            float m = fmaxf(r.m, s);
#pragma unroll
            for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const float base = m == -INFINITY ? 0.f : m;
            const float f = r.m == m ? 1.f : exp2_approx(r.m - base);
            const float w = seen ? exp2_approx(s - base + kWeightBias<BF16, TILE>) : 0.f;
            float sum = w;
#pragma unroll
            for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            r.m = m;
            r.l = r.l * f + sum;
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[e] = f == 0.f ? 0.f : r.o[e] * f;
#pragma unroll 8
            for (int e = 0; e < 32; ++e) {
                const float we = __shfl_sync(0xffffffffu, w, e);
                const int64_t o = __shfl_sync(0xffffffffu, at, e);
                if (((keys >> e) & 1u) == 0 || d >= a.pages.dim) continue;
                const uint2 vv = *reinterpret_cast<const uint2*>(a.pages.v + o + d);
                const float2 u = unpack2<BF16>(vv.x), v = unpack2<BF16>(vv.y);
                r.o[0] += we * u.x;
                r.o[1] += we * u.y;
                r.o[2] += we * v.x;
                r.o[3] += we * v.y;
            }
        }
    }
    return r;
}

// Rows whose weighted sums are not finite although their sums of weights are, a bit each from
// row `first_row` on: either a value that the row sees is not finite, and so the result, or a
// product took one in that it does not see (0 x inf, 0 x NaN), or split an infinite one's
// weight in two parts (inf - inf). The infinities and NaN among the values that the rows see are
// looked for, once for the keys that all of them see; they decide their dimensions. Only a row
// with others that are not finite is computed anew. The rows' results (part: their parts, with
// `part_rows` rows to an array, the first of them `part_row`) are read back and set right.
// This can take long: nobody may wait for it with a limit.
template <int TILE, int DP, bool BF16>
__device__ __noinline__ void settle_rows(const AttnArgs& a, int b, int h, int t0, int p0, int first_row, uint32_t bad,
                                         const KeyTiles<TILE> kt, int i0, int i1, float* part, int part_rows, int part_row) {
    const int lane = threadIdx.x & 31, d = lane * 4;
    const bool in = d < a.pages.dim;
    __syncwarp();
    int p_min = 0x7fffffff, p_max = -1;
    for (uint32_t left = bad; left; left &= left - 1) {
        const int p = max(-1, p0 + (first_row + __ffs(left) - 1) / a.group);
        p_min = min(p_min, p);
        p_max = max(p_max, p);
    }
    auto all_see = [&](int k0, int k1) {  // keys k0 .. k1, by every one of the rows
        return k1 <= p_min && (a.window == 0 || p_max - k0 < a.window || k1 < a.sinks);
    };
    const int32_t* table = a.seqs.tables + b * a.seqs.table_stride;
    // what key j's values are not: bits 0-3 NaN, 4-7 +inf, 8-11 -inf
    auto kinds = [&](int j) {
        const int page = table[j >> a.pages.page_shift];
        if (page < 0 || page >= a.pages.num_pages || !in) return 0u;
        const uint2 r = *reinterpret_cast<const uint2*>(a.pages.v + page * a.pages.stride_page + h * a.pages.stride_head +
                                                        (j & ((1 << a.pages.page_shift) - 1)) * a.pages.stride_token + d);
        const float2 u = unpack2<BF16>(r.x), v = unpack2<BF16>(r.y);
        const float x[4] = {u.x, u.y, v.x, v.y};
        uint32_t f = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) f |= (x[e] != x[e] ? 1u : x[e] == INFINITY ? 16u : x[e] == -INFINITY ? 256u : 0u) << e;
        return f;
    };
    uint32_t shared = 0;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        const int k0 = kt.first(i);
        if (!all_see(k0, k0 + TILE - 1)) continue;
#pragma unroll 4
        for (int c = 0; c < TILE; ++c) shared |= kinds(k0 + c);
    }
#pragma unroll 1
    for (; bad; bad &= bad - 1) {
        const int bit = __ffs(bad) - 1, row = first_row + bit, token = row / a.group;
        const int head = h * a.group + row - token * a.group, p = max(-1, p0 + token);
        uint32_t f = shared;
#pragma unroll 1
        for (int i = i0; i < i1; ++i) {
            const int k0 = kt.first(i);
            if (all_see(k0, k0 + TILE - 1) || k0 > p) continue;
#pragma unroll 4
            for (int c = 0; c < TILE; ++c)
                if (visible(k0 + c, p, a.window, a.sinks)) f |= kinds(k0 + c);
        }
        const int64_t o_off = static_cast<int64_t>(t0 + token) * a.o_token + head * a.o_head + d;
        float* slot = part ? part + 2 * part_rows + (part_row + bit) * DP + d : nullptr;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (in && part) {
            const float4 v = *reinterpret_cast<const float4*>(slot);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else if (in) {
            const uint2 r = *reinterpret_cast<const uint2*>(a.out + o_off);
            const float2 u = unpack2<BF16>(r.x), v = unpack2<BF16>(r.y);
            x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
        }
        bool anew = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) anew |= ((f >> e) & 0x111u) == 0 && !(x[e] * 0.f == 0.f);
        if (__any_sync(0xffffffffu, anew)) {
            const int64_t q_off = static_cast<int64_t>(t0 + token) * a.q_token + head * a.q_head;
            RowSum r;
            if constexpr (TILE % 32 == 0) {
                r = row_by_32<TILE, BF16>(a, b, h, q_off, p, kt, i0, i1);
            } else {
                r = row_by_keys<TILE, BF16>(a, b, h, q_off, p, kt, i0, i1);
            }
            if (part && lane == 0) {
                part[part_row + bit] = r.m;
                part[part_rows + part_row + bit] = r.l;
            }
            const float inv = part ? 1.f : r.l == 0.f ? 0.f : 1.f / r.l;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = r.o[e] * inv;
        }
        // what the row sees of infinities and NaN decides, whichever way the rest was computed
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t k = (f >> e) & 0x111u;
            if (k) x[e] = k == 16u ? INFINITY : k == 256u ? -INFINITY : NAN;
        }
        if (in && part) {
            *reinterpret_cast<float4*>(slot) = make_float4(x[0], x[1], x[2], x[3]);
        } else if (in) {
            *reinterpret_cast<uint2*>(a.out + o_off) = make_uint2(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]));
        }
    }
}

}  // namespace w4a16
