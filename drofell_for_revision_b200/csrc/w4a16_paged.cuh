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

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// The same for rows that are computed anew: bf16 has fp32's range, so that a sum of values may pass
// it where their mean does not. Such a sum comes out not finite and is made anew with weights of
// 2^-24 (fewer than 2^24 keys of equal weight, then); a part's maximum is stored as much higher.
template <bool BF16, int TILE>
constexpr float kAnewBias = BF16 ? -24.f : kWeightBias<BF16, TILE>;
// And for the join of parts, each finite: at most 2^12 of them.
constexpr float kJoinBias = -12.f;

// 2^(scale s - top + bias), top the rounded product of the largest s. Every product is rounded alike
// and none is fused: the largest weight is 2^bias exactly, however large the scores are.
__device__ __forceinline__ float weight_of(float s, float scale, float top, float bias) {
    return exp2_approx((__fmul_rn(s, scale) - top) + bias);
}

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
// (with 32 keys at once, a lane a key, every call took 2 to 3 % longer).
template <int TILE, int DP, bool BF16>
__device__ __noinline__ void row_by_keys(const AttnArgs& a, int b, int h, int t0, int p0, int row, const KeyTiles<TILE> kt, int i0,
                                         int i1, float* part, int part_rows, int part_row) {
    const int token = row / a.group, head = h * a.group + row - token * a.group, p = max(-1, p0 + token);
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
    load4(a.q + static_cast<int64_t>(t0 + token) * a.q_token + head * a.q_head, q);
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
            const float m = fmaxf(r.m, __fmul_rn(s, a.scale_log2)), base = m == -INFINITY ? 0.f : m;
            const float f = r.m == m ? 1.f : exp2_approx(r.m - base);
            const float w = weight_of(s, a.scale_log2, base, kAnewBias<BF16, TILE>);
            r.m = m;
            r.l = r.l * f + w;
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[e] = (f == 0.f ? 0.f : r.o[e] * f) + w * v[e];
        }
    }
    if (part && (threadIdx.x & 31) == 0) {
        part[part_row] = r.m + (kWeightBias<BF16, TILE> - kAnewBias<BF16, TILE>);
        part[part_rows + part_row] = r.l;
    }
    const float inv = part ? 1.f : r.l == 0.f ? 0.f : 1.f / r.l;
    if (in && part) {
        *reinterpret_cast<float4*>(part + 2 * part_rows + part_row * DP + d) = make_float4(r.o[0], r.o[1], r.o[2], r.o[3]);
    } else if (in) {
        *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(t0 + token) * a.o_token + head * a.o_head + d) =
            make_uint2(pack2<BF16>(r.o[0] * inv, r.o[1] * inv), pack2<BF16>(r.o[2] * inv, r.o[3] * inv));
    }
}

// The same for up to 16 rows from row `row0` of the sequence on (a bit each), over key tiles of 128,
// 16 keys at a time on mma.sync; values that are not finite count as 0. Operands come from
// global memory in 16-byte pieces: a product's sum does not care for the order of the dimensions, nor a
// result for which of its columns they are, as long as both sides agree on it. Loads are made
// whether they are wanted or not (then from an address that is one): under conditions they wait for
// one another. 64 dimensions of the values a sweep: what this takes of registers, the prompt
// kernel's loop does without (with 128, 4 bytes spilled there and 5 % of a prompt). The rows' results
// (part: their parts) are written.
template <int DP, bool BF16>
__device__ __noinline__ void rows_by_tiles(const AttnArgs& a, int b, int h, int t0, int p0, int row0, uint32_t rows,
                                           const KeyTiles<128> kt, int i0, int i1, float* part, int part_rows, int part_row) {
    constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
    const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    bool valid[2];
    int p[2];
    int64_t q_off[2];  // rows g and g + 8
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int row = row0 + g + 8 * e, token = row / a.group, head = h * a.group + row - token * a.group;
        valid[e] = (rows >> (g + 8 * e)) & 1u;
        p[e] = valid[e] ? max(-1, p0 + token) : -1;
        q_off[e] = valid[e] ? static_cast<int64_t>(t0 + token) * a.q_token + head * a.q_head : 0;
    }
    const int p_max = __reduce_max_sync(0xffffffffu, max(p[0], p[1]));
    const int32_t* table = a.seqs.tables + b * a.seqs.table_stride;
    auto load = [&](const uint16_t* x, int64_t off, int d, bool there) {
        there = there && d < a.pages.dim;
        const uint4 r = *reinterpret_cast<const uint4*>(x + (there ? off + d : 0));
        return there ? r : make_uint4(0, 0, 0, 0);
    };
#pragma unroll 1
    for (int d0 = 0; d0 < a.pages.dim; d0 += 64) {
        float o[8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll 1
        for (int u = i0 * 8; u < i1 * 8; ++u) {
            const int key0 = kt.first(u >> 3) + (u & 7) * 16;
            if (key0 > p_max) break;
            const int j = min(key0 + (lane & 15), p_max), page = table[j >> a.pages.page_shift];
            const int64_t at = page >= 0 && page < a.pages.num_pages
                                   ? page * a.pages.stride_page + h * a.pages.stride_head +
                                         (j & ((1 << a.pages.page_shift) - 1)) * a.pages.stride_token
                                   : -1;  // of key key0 + lane % 16
            const uint32_t alive = __ballot_sync(0xffffffffu, at >= 0);
            float s[2][4] = {};
            {
                const int64_t k0 = __shfl_sync(0xffffffffu, at, g), k1 = __shfl_sync(0xffffffffu, at, 8 + g);
                // dimensions 8 tq .. 8 tq + 7 of each 32 for two steps
#pragma unroll 2
                for (int d = tq * 8; d < DP; d += 32) {
                    const uint4 q0 = load(a.q, q_off[0], d, valid[0]), q1 = load(a.q, q_off[1], d, valid[1]);
                    const uint4 x0 = load(a.pages.k, k0, d, k0 >= 0), x1 = load(a.pages.k, k1, d, k1 >= 0);
                    const uint32_t u0[4] = {q0.x, q1.x, q0.y, q1.y}, u1[4] = {q0.z, q1.z, q0.w, q1.w};
                    mma16816<BF16>(s[0], u0, x0.x, x0.y);
                    mma16816<BF16>(s[0], u1, x0.z, x0.w);
                    mma16816<BF16>(s[1], u0, x1.x, x1.y);
                    mma16816<BF16>(s[1], u1, x1.z, x1.w);
                }
            }
            // values of keys 2 tq, 2 tq + 1 and 8 further, dimensions d0 + 8 g .. d0 + 8 g + 7: column g of
            // product j has dimension d0 + 8 g + j
            uint32_t v[4][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t key = __shfl_sync(0xffffffffu, at, (e >> 1) * 8 + tq * 2 + (e & 1));
                const uint4 x = load(a.pages.v, key, d0 + g * 8, key >= 0);
                v[e][0] = x.x, v[e][1] = x.y, v[e][2] = x.z, v[e][3] = x.w;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int c = n * 8 + tq * 2 + (e & 1);
                    if (((alive >> c) & 1u) == 0 || !visible(key0 + c, p[e >> 1], a.window, a.sinks)) s[n][e] = -INFINITY;
                }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x = __fmul_rn(fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])), a.scale_log2);
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                x = fmaxf(x, m[r]);
                const float f = x == m[r] ? 1.f : exp2_approx(m[r] - x);
                m[r] = x;
                l[r] *= f;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    o[n][2 * r] *= f;
                    o[n][2 * r + 1] *= f;
                }
                const float base = x == -INFINITY ? 0.f : x;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float y = weight_of(s[n][2 * r], a.scale_log2, base, kAnewBias<BF16, 128>);
                    const float w = weight_of(s[n][2 * r + 1], a.scale_log2, base, kAnewBias<BF16, 128>);
                    l[r] += y + w;
                    hi[2 * n + r] = pack2<BF16>(y, w);
                    const float2 z = unpack2<BF16>(hi[2 * n + r]);
                    lo[2 * n + r] = pack2<BF16>(y - z.x, w - z.y);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if ((v[e][i] & kExp) == kExp) v[e][i] &= 0xffff0000u;
                    if (((v[e][i] >> 16) & kExp) == kExp) v[e][i] &= 0xffffu;
                }
                const uint32_t b0 = __byte_perm(v[0][i], v[1][i], 0x5410), b1 = __byte_perm(v[2][i], v[3][i], 0x5410);
                const uint32_t c0 = __byte_perm(v[0][i], v[1][i], 0x7632), c1 = __byte_perm(v[2][i], v[3][i], 0x7632);
                mma16816<BF16>(o[2 * i], hi, b0, b1);
                mma16816<BF16>(o[2 * i], lo, b0, b1);
                mma16816<BF16>(o[2 * i + 1], hi, c0, c1);
                mma16816<BF16>(o[2 * i + 1], lo, c0, c1);
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (!valid[r]) continue;
            const int row = row0 + g + 8 * r, token = row / a.group, at = part_row + g + 8 * r;
            uint16_t* out = a.out + static_cast<int64_t>(t0 + token) * a.o_token + (h * a.group + row - token * a.group) * a.o_head;
            if (part && tq == 0) {
                part[at] = m[r] + (kWeightBias<BF16, 128> - kAnewBias<BF16, 128>);
                part[part_rows + at] = l[r];
            }
            const float inv = part ? 1.f : l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const int d = d0 + (2 * tq + n) * 8 + i;
                    const float x = o[i][2 * r + n] * inv, y = o[i + 1][2 * r + n] * inv;
                    if (d >= a.pages.dim) continue;
                    if (part) {
                        *reinterpret_cast<float2*>(part + 2 * part_rows + at * DP + d) = make_float2(x, y);
                    } else {
                        *reinterpret_cast<uint32_t*>(out + d) = pack2<BF16>(x, y);
                    }
                }
        }
    }
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
    // What the values of eight keys from j on (of one page) are not, of those whose bit is set: bits 0-3
    // NaN, 4-7 +inf, 8-11 -inf. All of them are looked at for an exponent of ones first.
    auto kinds = [&](int j, uint32_t keys) {
        constexpr uint32_t kCarry = BF16 ? 0x00800080u : 0x04000400u;
        const int page = table[keys ? j >> a.pages.page_shift : 0];
        const bool ok = in && keys && page >= 0 && page < a.pages.num_pages;
        const uint16_t* v = a.pages.v + (ok ? page * a.pages.stride_page + h * a.pages.stride_head +
                                                  (j & ((1 << a.pages.page_shift) - 1)) * a.pages.stride_token + d
                                            : 0);
        const int64_t step = ok ? a.pages.stride_token : 0;
        uint2 r[8];
        uint32_t any = 0, f = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) r[c] = *reinterpret_cast<const uint2*>(v + c * step);
#pragma unroll
        for (int c = 0; c < 8; ++c) any |= ((r[c].x & 0x7fff7fffu) + kCarry) | ((r[c].y & 0x7fff7fffu) + kCarry);
        if (!ok || (any & 0x80008000u) == 0) return 0u;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float2 x = unpack2<BF16>(r[c].x), y = unpack2<BF16>(r[c].y);
            const float z[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((keys >> c) & 1u) f |= (z[e] != z[e] ? 1u : z[e] == INFINITY ? 16u : z[e] == -INFINITY ? 256u : 0u) << e;
        }
        return f;
    };
    uint32_t shared = 0;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        const int k0 = kt.first(i);
        if (!all_see(k0, k0 + TILE - 1)) continue;
#pragma unroll 2
        for (int c = 0; c < TILE; c += 8) shared |= kinds(k0 + c, 0xffu);
        if (__all_sync(0xffffffffu, !in || (shared & 15u) == 15u)) break;  // all NaN already
    }
    // sets a row's result right; whether it has to be computed anew first
    auto settle = [&](int bit, bool may_be_anew) {
        const int row = first_row + bit, token = row / a.group;
        const int head = h * a.group + row - token * a.group, p = max(-1, p0 + token);
        uint32_t f = shared;
#pragma unroll 1
        for (int i = i0; i < i1; ++i) {
            const int k0 = kt.first(i);
            if (all_see(k0, k0 + TILE - 1) || k0 > p) continue;
#pragma unroll 1
            for (int c = k0; c < k0 + TILE; c += 8) {
                uint32_t keys = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) keys |= static_cast<uint32_t>(visible(c + e, p, a.window, a.sinks)) << e;
                f |= kinds(c, keys);
            }
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
        for (int e = 0; e < 4; ++e) {
            const uint32_t k = (f >> e) & 0x111u;
            if (k) x[e] = k == 16u ? INFINITY : k == 256u ? -INFINITY : NAN;
            anew |= k == 0 && !(x[e] * 0.f == 0.f);
        }
        if (may_be_anew && __any_sync(0xffffffffu, anew)) return true;
        if (in && part) {
            *reinterpret_cast<float4*>(slot) = make_float4(x[0], x[1], x[2], x[3]);
        } else if (in) {
            *reinterpret_cast<uint2*>(a.out + o_off) = make_uint2(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]));
        }
        return false;
    };
    uint32_t anew = 0;
#pragma unroll 1
    for (uint32_t left = bad; left; left &= left - 1)
        if (settle(__ffs(left) - 1, true)) anew |= left & -left;
    if (anew == 0) return;
    if constexpr (TILE == 128) {
#pragma unroll 1
        for (int r = 0; r < 32; r += 16)
            if ((anew >> r) & 0xffffu)
                rows_by_tiles<DP, BF16>(a, b, h, t0, p0, first_row + r, (anew >> r) & 0xffffu, kt, i0, i1, part, part_rows,
                                        part_row + r);
    } else {
#pragma unroll 1
        for (uint32_t left = anew; left; left &= left - 1)
            row_by_keys<TILE, DP, BF16>(a, b, h, t0, p0, first_row + __ffs(left) - 1, kt, i0, i1, part, part_rows,
                                        part_row + __ffs(left) - 1);
    }
    __syncwarp();
    // what a row sees of infinities and NaN decides, whichever way the rest was computed
#pragma unroll 1
    for (; anew; anew &= anew - 1) settle(__ffs(anew) - 1, false);
}

}  // namespace w4a16
