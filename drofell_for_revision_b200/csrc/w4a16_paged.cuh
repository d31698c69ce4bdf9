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

}  // namespace w4a16
