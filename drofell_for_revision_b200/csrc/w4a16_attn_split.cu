// Attention of a few new tokens per sequence over a paged cache, split over the cache's
// length and joined. o = sum_j softmax_j(scale q.k_j) v_j in one pass over the keys with
// the running maximum m and sum l of the softmax (fp32, base 2):
//   m' = max(m, max_j s_j), l' = l 2^(m - m') + sum_j 2^(s_j - m'), o' likewise;
// pieces (m_i, l_i, o_i) of one row join as sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m).
//
// What bounds it is HBM: every visible key and value is read once, 4 D bytes a key and
// head for 4 D flops a query head. The dot products run on mma.sync m16n8k16 with the
// query rows that share a key-value head (token-major, so a group of heads of one or a few
// tokens) as the 16 rows: tcgen05 wants 128 rows, and a decode step has 1 to 16.
//
// Work: a unit is a tile of 64 keys of one item (sequence, key-value head, 16 rows). All
// units in item order are cut into equal ranges, one per CTA, so that uneven lengths
// balance and the workspace has a fixed size: at most the first and the last piece of a
// range are parts of an item. Those go to the workspace in fp32 and split_join_kernel adds
// them in range order (the same result for the same lengths, whatever runs when).
#include <algorithm>
#include <atomic>

#include "w4a16_paged.cuh"
#include "w4a16_ptx.cuh"

namespace w4a16 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kWarpKeys = 16;
constexpr int kTile = kWarps * kWarpKeys;  // 64 keys
constexpr int kRows = 16;

template <int DP>
struct SplitCfg {
    static constexpr int kStageBytes = 2 * kWarpKeys * DP * 2;  // K and V rows of one warp
    static constexpr int kStages = DP == 128 ? 3 : 6;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kOPad = DP + 4;
    static_assert(kWarps * kRows * kOPad * 4 <= kRing, "the pieces of the warps are joined in the ring");
    static constexpr int kSmem = kRing;
};

// Workspace of one piece: m[16], l[16], o[16][DP]; two pieces a CTA, then what the CTA's
// first item is: {part of a split item that this range continues first, sequence, head, row
// tile, last CTA}.
constexpr int slot_floats(int dp) { return 2 * kRows + kRows * dp; }
constexpr int kDescInts = 8;

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
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

// Byte offset of 16-byte chunk c of row r: chunks permuted by the row, so that eight rows
// of one chunk column lie in different banks.
template <int DP>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return static_cast<uint32_t>(r * DP * 2 + ((c ^ (r & 7)) << 4));
}

struct Units {
    int tiles, row_tiles;
    int64_t units;
};
__device__ __forceinline__ Units units_of(const AttnArgs& a, const Seq& s) {
    Units u;
    u.tiles = s.nq > 0 ? KeyTiles<kTile>(s.p0, s.p0 + s.nq - 1, a.window, a.sinks).count : 0;
    u.row_tiles = (s.nq * a.group + kRows - 1) / kRows;
    u.units = static_cast<int64_t>(u.tiles) * u.row_tiles * a.pages.heads_kv;
    return u;
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 2) split_kernel(const __grid_constant__ AttnArgs a, const int min_tiles) {
    using C = SplitCfg<DP>;
    constexpr int CH = DP / 8;    // 16-byte chunks of a row
    constexpr int KS = DP / 16;   // k steps of the score product
    constexpr int S = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t sum_warp[kWarps];
    __shared__ int64_t found_off;
    __shared__ int found_b;
    __shared__ float row_m[kWarps][kRows], row_l[kWarps][kRows];
    __shared__ uint32_t live[kWarps][S];  // keys of valid pages of a stage

    ptx::grid_dep_wait();
    ptx::grid_dep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = blockIdx.x;

    // ---- this CTA's range of the units of all sequences
    const int per = (a.seqs.batch + kThreads - 1) / kThreads;
    const int b_lo = min(a.seqs.batch, static_cast<int>(threadIdx.x) * per);
    const int b_hi = min(a.seqs.batch, b_lo + per);
    int64_t mine = 0;
    for (int b = b_lo; b < b_hi; ++b) mine += units_of(a, load_seq(a.seqs, a.pages.page_shift, b)).units;
    int64_t pre = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, pre, d);
        if (lane >= d) pre += o;
    }
    if (lane == 31) sum_warp[warp] = pre;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) pre += sum_warp[w];
        total += sum_warp[w];
    }
    pre -= mine;
    const int64_t share = max(static_cast<int64_t>(min_tiles), (total + gridDim.x - 1) / gridDim.x);
    const int64_t begin = min(total, cta * share), end = min(total, begin + share);
    if (begin >= pre && begin < pre + mine) {
        int64_t at = pre;
        for (int b = b_lo; b < b_hi; ++b) {
            const int64_t n = units_of(a, load_seq(a.seqs, a.pages.page_shift, b)).units;
            if (begin < at + n) {
                found_b = b;
                found_off = begin - at;
                break;
            }
            at += n;
        }
    }
    // rows of sequences without any key are zero
    for (int b = cta; b < a.seqs.batch; b += gridDim.x) {
        const Seq s = load_seq(a.seqs, a.pages.page_shift, b);
        if (s.nq > 0 && units_of(a, s).tiles == 0) {
            const int chunks = a.pages.dim >> 3;
            for (int i = threadIdx.x; i < s.nq * a.heads * chunks; i += kThreads) {
                const int row = i / chunks, c = i % chunks;
                *reinterpret_cast<uint4*>(a.out + (s.t0 + row / a.heads) * a.o_token + (row % a.heads) * a.o_head +
                                          c * 8) = make_uint4(0, 0, 0, 0);
            }
        }
    }
    __syncthreads();
    int* desc = reinterpret_cast<int*>(a.ws + static_cast<size_t>(gridDim.x) * 2 * slot_floats(DP)) + cta * kDescInts;
    if (a.ws && threadIdx.x == 0) desc[0] = 0;
    if (begin >= end) return;

    int b = found_b;
    int64_t off = found_off;  // units of sequence b before the range
    const uint32_t ring = ptx::smem_u32(smem) + warp * (S * C::kStageBytes);
    const int g = lane >> 2, tq = lane & 3;
    const int slot_mask = (1 << a.pages.page_shift) - 1;

    for (int64_t at = begin; at < end; ++b, off = 0) {
        const Seq sq = load_seq(a.seqs, a.pages.page_shift, b);
        const Units un = units_of(a, sq);
        if (un.units == 0) continue;
        const KeyTiles<kTile> kt(sq.p0, sq.p0 + sq.nq - 1, a.window, a.sinks);
        const int p_last = sq.p0 + sq.nq - 1;
        const int lo = a.window ? max(0, max(sq.p0, 0) + 1 - a.window) : 0;  // first key of the earliest window
        int64_t item = off / un.tiles;
        int tile0 = static_cast<int>(off - item * un.tiles);
        const int64_t items = static_cast<int64_t>(un.row_tiles) * a.pages.heads_kv;
        for (; item < items && at < end; ++item, tile0 = 0) {
            const int h = static_cast<int>(item / un.row_tiles), rt = static_cast<int>(item % un.row_tiles);
            const int tile1 = static_cast<int>(min(static_cast<int64_t>(un.tiles), tile0 + (end - at)));
            const int n = tile1 - tile0;
            const int64_t item_start = at - tile0;  // in units of all sequences

            // ---- loads of a tile of this warp: lanes 0..15 find the rows, all copy chunks
            const uint16_t* kbase = a.pages.k + h * a.pages.stride_head;
            const uint16_t* vbase = a.pages.v + h * a.pages.stride_head;
            const int32_t* table = a.seqs.tables + b * a.seqs.table_stride;
            auto find = [&](int i) -> int64_t {  // row offset of this lane's key of tile i, -1: none
                if (i >= tile1) return -1;
                const int key = kt.first(i) + warp * kWarpKeys + (lane & 15);
                if (key > p_last || (key < lo && key >= a.sinks)) return -1;  // seen by no row
                const int page = table[key >> a.pages.page_shift];
                if (page < 0 || page >= a.pages.num_pages) return -1;
                return page * a.pages.stride_page + (key & slot_mask) * a.pages.stride_token;
            };
            auto issue = [&](int i, int64_t row_off) {
                const int st = (i - tile0) % S;
                if (i < tile1) {
                    const uint32_t ok = __ballot_sync(0xffffffffu, row_off >= 0) & 0xffffu;
                    if (lane == 0) live[warp][st] = ok;
                    const uint32_t dst = ring + st * C::kStageBytes;
#pragma unroll
                    for (int j0 = 0; j0 < kWarpKeys * CH; j0 += 32) {
                        const int j = j0 + lane, r = j / CH, c = j % CH;
                        const int64_t ro = __shfl_sync(0xffffffffu, row_off, r);
                        const bool in = ro >= 0 && c * 8 < a.pages.dim;
                        const int64_t o = in ? ro + c * 8 : 0;
                        const uint32_t n16 = in ? 16u : 0u;
                        cp_async16(dst + chunk_at<DP>(r, c), kbase + o, n16);
                        cp_async16(dst + kWarpKeys * DP * 2 + chunk_at<DP>(r, c), vbase + o, n16);
                    }
                }
                cp_async_commit();
            };
            // ---- query rows g and g + 8 of the row tile, as A fragments
            const int r0 = rt * kRows + g, r1 = r0 + 8;
            const int rows = sq.nq * a.group;
            const int i0 = r0 / a.group, i1 = r1 / a.group;
            const int p0 = r0 < rows ? sq.p0 + i0 : -1, p1 = r1 < rows ? sq.p0 + i1 : -1;
            uint32_t qf[KS][4];
            {
                const uint16_t* q0 = a.q + (sq.t0 + i0) * a.q_token + (h * a.group + r0 % a.group) * a.q_head;
                const uint16_t* q1 = a.q + (sq.t0 + i1) * a.q_token + (h * a.group + r1 % a.group) * a.q_head;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int d = ks * 16 + e * 8 + tq * 2;
                        const bool in = d < a.pages.dim;
                        qf[ks][2 * e] = r0 < rows && in ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
                        qf[ks][2 * e + 1] = r1 < rows && in ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
                    }
            }
            // positions of all rows of the tile, for the whole-tile test
            const int row_last = min(rows, rt * kRows + kRows) - 1;
            const int p_min = sq.p0 + (rt * kRows) / a.group, p_max = sq.p0 + row_last / a.group;

            // A value that a row does not see must not reach it as 0 x inf or 0 x NaN, nor an
            // infinite one as (w - rounded w) x inf. Any such product leaves a sum that is not
            // finite: the warp then takes its keys once more, row by row what each sees.
            float o[DP / 8][4], m0, m1, l0, l1;
            bool careful = false;
        again:
#pragma unroll
            for (int j = 0; j < DP / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            m0 = m1 = -INFINITY;
            l0 = l1 = 0.f;
#pragma unroll
            for (int i = 0; i < S - 1; ++i) issue(tile0 + i, find(tile0 + i));
            int64_t next = find(tile0 + S - 1);
            for (int i = tile0; i < tile1; ++i) {
                issue(i + S - 1, next);
                next = find(i + S);
                cp_async_wait<S - 1>();
                __syncwarp();
                const int st = (i - tile0) % S;
                const uint32_t kt_s = ring + st * C::kStageBytes, vt_s = kt_s + kWarpKeys * DP * 2;
                const int key0 = kt.first(i) + warp * kWarpKeys;
                const uint32_t alive = live[warp][st];
                if (alive != 0) {
                    // scores of 16 rows x 16 keys
                    float s[2][4] = {};
                    const int kr = (lane & 7) + ((lane & 16) >> 1), kc = (lane >> 3) & 1;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint32_t kb[4];
                        ldmatrix4(kb, kt_s + chunk_at<DP>(kr, ks * 2 + kc));
                        mma16816<BF16>(s[0], qf[ks], kb[0], kb[1]);
                        mma16816<BF16>(s[1], qf[ks], kb[2], kb[3]);
                    }
                    const bool whole = alive == 0xffffu && key0 + kWarpKeys - 1 <= p_min &&
                                       (a.window == 0 || p_max - key0 < a.window || key0 + kWarpKeys <= a.sinks);
                    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            s[j][e] *= a.scale_log2;
                            s[j][2 + e] *= a.scale_log2;
                            if (!whole) {
                                const int c = j * 8 + tq * 2 + e, key = key0 + c;
                                const bool in = (alive >> c) & 1;
                                if (!in || !visible(key, p0, a.window, a.sinks)) s[j][e] = -INFINITY;
                                if (!in || !visible(key, p1, a.window, a.sinks)) s[j][2 + e] = -INFINITY;
                            }
                            x0 = fmaxf(x0, s[j][e]);
                            x1 = fmaxf(x1, s[j][2 + e]);
                        }
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
                    x0 = fmaxf(x0, m0);
                    x1 = fmaxf(x1, m1);
                    if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
                        const float f0 = x0 > m0 ? exp2f(m0 - x0) : 1.f, f1 = x1 > m1 ? exp2f(m1 - x1) : 1.f;
                        l0 *= f0;
                        l1 *= f1;
#pragma unroll
                        for (int j = 0; j < DP / 8; ++j) {
                            o[j][0] *= f0;
                            o[j][1] *= f0;
                            o[j][2] *= f1;
                            o[j][3] *= f1;
                        }
                        m0 = x0;
                        m1 = x1;
                    }
                    const float c0 = m0 == -INFINITY ? 0.f : m0, c1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            s[j][e] = exp2f(s[j][e] - c0);
                            s[j][2 + e] = exp2f(s[j][2 + e] - c1);
                            l0 += s[j][e];
                            l1 += s[j][2 + e];
                        }
                    // weights as two 16-bit parts, the rounded value and what it leaves: the
                    // product then carries 16 (bf16) or 22 (fp16) bits of them, and the second
                    // mma costs nothing that HBM does not hide
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float u = s[j][2 * e], w = s[j][2 * e + 1];
                            hi[2 * j + e] = pack2<BF16>(u, w);
                            const float2 r = unpack2<BF16>(hi[2 * j + e]);
                            lo[2 * j + e] = pack2<BF16>(u - r.x, w - r.y);
                        }
                    const int vr = (lane & 7) + (lane & 8), vc = lane >> 4;
                    if (!careful) {
#pragma unroll
                        for (int j = 0; j < DP / 16; ++j) {
                            uint32_t vb[4];
                            ldmatrix4_trans(vb, vt_s + chunk_at<DP>(vr, j * 2 + vc));
                            mma16816<BF16>(o[2 * j], hi, vb[0], vb[1]);
                            mma16816<BF16>(o[2 * j + 1], hi, vb[2], vb[3]);
                            mma16816<BF16>(o[2 * j], lo, vb[0], vb[1]);
                            mma16816<BF16>(o[2 * j + 1], lo, vb[2], vb[3]);
                        }
                    } else {  // key by key, each row only what it sees
#pragma unroll 1
                        for (int c = 0; c < kWarpKeys; ++c) {
                            const int from = (lane & ~3) | ((c & 7) >> 1);
                            const float e0 = c & 1 ? (c < 8 ? s[0][1] : s[1][1]) : (c < 8 ? s[0][0] : s[1][0]);
                            const float e1 = c & 1 ? (c < 8 ? s[0][3] : s[1][3]) : (c < 8 ? s[0][2] : s[1][2]);
                            const float w0 = __shfl_sync(0xffffffffu, e0, from);
                            const float w1 = __shfl_sync(0xffffffffu, e1, from);
                            const bool in = (alive >> c) & 1;
                            const bool in0 = in && visible(key0 + c, p0, a.window, a.sinks);
                            const bool in1 = in && visible(key0 + c, p1, a.window, a.sinks);
#pragma unroll
                            for (int j = 0; j < DP / 8; ++j) {
                                uint32_t raw;
                                asm volatile("ld.shared.b32 %0, [%1];"
                                             : "=r"(raw)
                                             : "r"(vt_s + chunk_at<DP>(c, j) + tq * 4)
                                             : "memory");
                                const float2 v = unpack2<BF16>(raw);
                                if (in0) {
                                    o[j][0] += w0 * v.x;
                                    o[j][1] += w0 * v.y;
                                }
                                if (in1) {
                                    o[j][2] += w1 * v.x;
                                    o[j][3] += w1 * v.y;
                                }
                            }
                        }
                    }
                }
                __syncwarp();  // the stage may be filled again
            }
            cp_async_wait<0>();
            if (!careful) {
                float sum = 0.f;  // not finite if any term is not
#pragma unroll
                for (int j = 0; j < DP / 8; ++j) sum += (o[j][0] + o[j][1]) * 0.f + (o[j][2] + o[j][3]) * 0.f;
                careful = __any_sync(0xffffffffu, !(sum == 0.f));
                if (careful) goto again;
            }
            l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
            l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
            __syncthreads();  // every warp is done with the ring

            // ---- join the four warps' keys
            float* ob = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int j = 0; j < DP / 8; ++j) {
                *reinterpret_cast<float2*>(ob + (warp * kRows + g) * C::kOPad + j * 8 + tq * 2) =
                    make_float2(o[j][0], o[j][1]);
                *reinterpret_cast<float2*>(ob + (warp * kRows + g + 8) * C::kOPad + j * 8 + tq * 2) =
                    make_float2(o[j][2], o[j][3]);
            }
            if (tq == 0) {
                row_m[warp][g] = m0;
                row_m[warp][g + 8] = m1;
                row_l[warp][g] = l0;
                row_l[warp][g + 8] = l1;
            }
            __syncthreads();
            const bool part = n < un.tiles;
            float* ws = part ? a.ws + (static_cast<size_t>(cta) * 2 + (tile0 == 0 ? 1 : 0)) * slot_floats(DP) : nullptr;
            if (part && threadIdx.x == 0 && tile0 > 0) {
                // the range that ends an item's first piece is followed by the one that joins it
                const int64_t first_cta = item_start / share, last_cta = (item_start + un.tiles - 1) / share;
                if (first_cta + 1 == cta) {
                    desc[1] = b;
                    desc[2] = h;
                    desc[3] = rt;
                    desc[4] = static_cast<int>(last_cta);
                    desc[0] = 1;
                }
            }
            {
                const int r = threadIdx.x >> 3, c = threadIdx.x & 7;  // 8 threads a row, DP / 8 columns each
                float m = row_m[0][r];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) m = fmaxf(m, row_m[w][r]);
                const float base = m == -INFINITY ? 0.f : m;
                float f[kWarps], l = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    f[w] = exp2f(row_m[w][r] - base);
                    l += row_l[w][r] * f[w];
                }
                const int row = rt * kRows + r;
                const bool in = row < rows;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint16_t* out = nullptr;
                if (in && !part)
                    out = a.out + (sq.t0 + row / a.group) * a.o_token + (h * a.group + row % a.group) * a.o_head;
                if (part && c == 0) {
                    ws[r] = m;
                    ws[kRows + r] = l;
                }
#pragma unroll
                for (int e = 0; e < DP / 64; ++e) {
                    const int d = (e * 8 + c) * 8;  // neighbouring threads, neighbouring 16-byte chunks
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float* src = ob + (w * kRows + r) * C::kOPad + d;
                        const float4 u = *reinterpret_cast<const float4*>(src);
                        const float4 v = *reinterpret_cast<const float4*>(src + 4);
                        // a warp that saw no key adds nothing
                        if (f[w] != 0.f) {
                            x[0] += f[w] * u.x, x[1] += f[w] * u.y, x[2] += f[w] * u.z, x[3] += f[w] * u.w;
                            x[4] += f[w] * v.x, x[5] += f[w] * v.y, x[6] += f[w] * v.z, x[7] += f[w] * v.w;
                        }
                    }
                    if (part) {
                        float4* dst = reinterpret_cast<float4*>(ws + 2 * kRows + r * DP + d);
                        dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                        dst[1] = make_float4(x[4], x[5], x[6], x[7]);
                    } else if (in && d < a.pages.dim) {
                        *reinterpret_cast<uint4*>(out + d) =
                            make_uint4(pack2<BF16>(x[0] * inv, x[1] * inv), pack2<BF16>(x[2] * inv, x[3] * inv),
                                       pack2<BF16>(x[4] * inv, x[5] * inv), pack2<BF16>(x[6] * inv, x[7] * inv));
                    }
                }
            }
            __syncthreads();  // the ring may be filled again
            at += n;
        }
    }
}

// One CTA per range and four of its 16 rows, a warp a row: adds the pieces of the split
// item that the range is the second to hold, in range order.
template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads) split_join_kernel(const __grid_constant__ AttnArgs a) {
    ptx::grid_dep_wait();
    const int cta = blockIdx.x + 1, ctas = gridDim.x + 1;
    const int* desc = reinterpret_cast<const int*>(a.ws + static_cast<size_t>(ctas) * 2 * slot_floats(DP)) + cta * kDescInts;
    if (desc[0] == 0) return;
    const int b = desc[1], h = desc[2], rt = desc[3], last = desc[4];
    const Seq sq = load_seq(a.seqs, a.pages.page_shift, b);
    const int r = blockIdx.y * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int row = rt * kRows + r;
    if (row >= sq.nq * a.group) return;
    auto piece = [&](int c) {
        return a.ws + (static_cast<size_t>(c) * 2 + (c == cta - 1 ? 1 : 0)) * slot_floats(DP);
    };
    float m = -INFINITY;
    for (int c = cta - 1 + lane; c <= last; c += 32) m = fmaxf(m, piece(c)[r]);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float base = m == -INFINITY ? 0.f : m;
    constexpr int E = DP / 32;
    float x[E] = {}, l = 0.f;
#pragma unroll 4
    for (int c = cta - 1; c <= last; ++c) {
        const float* w = piece(c);
        const float f = exp2f(w[r] - base);
        const float lc = w[kRows + r];
        float v[E];
        if constexpr (E == 4) {
            const float4 u = *reinterpret_cast<const float4*>(w + 2 * kRows + r * DP + lane * 4);
            v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
        } else {
            const float2 u = *reinterpret_cast<const float2*>(w + 2 * kRows + r * DP + lane * 2);
            v[0] = u.x, v[1] = u.y;
        }
        l += lc * f;
        if (f != 0.f) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] += f * v[e];
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* out = a.out + (sq.t0 + row / a.group) * a.o_token + (h * a.group + row % a.group) * a.o_head + lane * E;
    if (lane * E < a.pages.dim) {
#pragma unroll
        for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<BF16>(x[e] * inv, x[e + 1] * inv);
    }
}

template <int DP, bool BF16>
cudaError_t launch_split_t(const AttnArgs& a, const SplitPlan& p, cudaStream_t s) {
    using C = SplitCfg<DP>;
    auto kern = split_kernel<DP, BF16>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), C::kSmem, ready);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, a, p.min_tiles);
    if (e != cudaSuccess || !p.join) return e;
    cfg.gridDim = dim3(p.ctas - 1, kRows / kWarps);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, split_join_kernel<DP, BF16>, a);
}

}  // namespace

SplitPlan plan_split(const AttnArgs& a, int num_sms) {
    SplitPlan p;
    p.min_tiles = 2;
    // what the tables cover bounds the work; the lengths are on the device
    const int64_t covered = static_cast<int64_t>(a.seqs.width) << a.pages.page_shift;
    int64_t tiles = (covered + kTile - 1) / kTile;
    if (a.window)
        tiles = std::min<int64_t>(tiles, (int64_t{a.sinks} + kTile - 1) / kTile +
                                             (int64_t{a.window} + a.seqs.max_q + 2 * kTile - 2) / kTile);
    const int64_t items = static_cast<int64_t>(a.seqs.batch) * a.pages.heads_kv *
                          ((static_cast<int64_t>(a.seqs.max_q) * a.group + kRows - 1) / kRows);
    const int64_t most = std::max<int64_t>(1, (items * tiles + p.min_tiles - 1) / p.min_tiles);
    p.ctas = static_cast<int>(std::min<int64_t>(2 * num_sms, most));
    p.join = p.ctas > 1;
    return p;
}

size_t split_workspace_bytes(const SplitPlan& p, int dim) {
    const int dp = dim <= 64 ? 64 : 128;
    return p.join ? static_cast<size_t>(p.ctas) * (2 * slot_floats(dp) * sizeof(float) + kDescInts * sizeof(int)) : 0;
}

cudaError_t launch_split(const AttnArgs& a, const SplitPlan& p, bool bf16, cudaStream_t s) {
    if (a.pages.dim <= 64) return bf16 ? launch_split_t<64, true>(a, p, s) : launch_split_t<64, false>(a, p, s);
    return bf16 ? launch_split_t<128, true>(a, p, s) : launch_split_t<128, false>(a, p, s);
}

}  // namespace w4a16
