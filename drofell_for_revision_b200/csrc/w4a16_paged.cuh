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

// A row's maximum, sum of weights and weighted sum of values (four dimensions a lane).
struct RowSum {
    float m, l, o[4];
    template <bool BF16>
    __device__ __forceinline__ void store(const AttnArgs& a, int64_t o_off) const {
        const int d = (threadIdx.x & 31) * 4;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (d < a.pages.dim)
            *reinterpret_cast<uint2*>(a.out + o_off + d) =
                make_uint2(pack2<BF16>(o[0] * inv, o[1] * inv), pack2<BF16>(o[2] * inv, o[3] * inv));
    }
};

// One row over key tiles [i0, i1), key by key and each key by selection: for rows whose sums
// are not finite because a product took in a value that the row does not see. A warp a row,
// lanes over the head's dimensions. Slow, and as rare as infinities and NaN are.
template <int TILE, bool BF16>
__device__ __noinline__ RowSum careful_row(const AttnArgs& a, int b, int h, int64_t q_off, int p, const KeyTiles<TILE> kt,
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
            const float f = r.m == m ? 1.f : exp2_approx(r.m - base), w = exp2_approx(s - base);
            r.m = m;
            r.l = r.l * f + w;
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[e] = (f == 0.f ? 0.f : r.o[e] * f) + w * v[e];
        }
    }
    return r;
}

}  // namespace w4a16
