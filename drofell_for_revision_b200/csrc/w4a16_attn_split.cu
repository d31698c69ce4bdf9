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
// Work: every warp is a worker of its own. A unit is a tile of 16 keys of one item (sequence,
// key-value head, 16 rows); all units in item order are cut into equal ranges, one per
// worker, so that uneven lengths balance, loads run on from one item into the next, no warp
// waits for another, and the workspace has a fixed size: at most the first and the last piece
// of a range are parts of an item. Those go to the workspace in fp32 and split_join_kernel
// adds them in range order (the same result for the same lengths, whatever runs when).
#include <algorithm>
#include <atomic>

#include "w4a16_paged.cuh"
#include "w4a16_ptx.cuh"

namespace w4a16 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;  // keys
constexpr int kRows = 16;

template <int DP>
struct SplitCfg {
    static constexpr int kStageBytes = 2 * kTile * DP * 2;  // K and V rows
    static constexpr int kStages = DP == 128 ? 3 : 6;
    static constexpr int kSmem = kWarps * kStages * kStageBytes;  // a ring per warp; two CTAs an SM
};

// Workspace: of each worker two pieces m[16], l[16], o[16][DP] (the one it begins with, the
// one it ends with), then what the item is that it continues: {there is one, sequence, head,
// row tile, its first worker, its last}.
constexpr int piece_floats(int dp) { return 2 * kRows + kRows * dp; }
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

// Units of a sequence: key tiles x row tiles x heads.
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

// A place among the units: a key tile of an item of a sequence.
struct Cursor {
    int b, h, rt, tile;
    Seq sq;
    Units un;
    KeyTiles<kTile> kt;

    __device__ __forceinline__ void load(const AttnArgs& a) {  // of sequence b, or the next with units
        for (;; ++b) {
            sq = load_seq(a.seqs, a.pages.page_shift, b);
            un = units_of(a, sq);
            if (un.units > 0) break;
        }
        kt = KeyTiles<kTile>(sq.p0, sq.p0 + sq.nq - 1, a.window, a.sinks);
    }
    // `off` units into sequence b
    __device__ __forceinline__ Cursor(const AttnArgs& a, int seq, int64_t off) : b(seq), kt(0, -1, 0, 0) {
        load(a);
        const int64_t item = off / un.tiles;
        tile = static_cast<int>(off - item * un.tiles);
        h = static_cast<int>(item / un.row_tiles);
        rt = static_cast<int>(item - static_cast<int64_t>(h) * un.row_tiles);
    }
    // to the first tile of the next item
    __device__ __forceinline__ void next_item(const AttnArgs& a) {
        tile = 0;
        if (++rt < un.row_tiles) return;
        rt = 0;
        if (++h < a.pages.heads_kv) return;
        h = 0;
        ++b;
        load(a);
    }
};

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 2) split_kernel(const __grid_constant__ AttnArgs a, const int min_units) {
    using C = SplitCfg<DP>;
    constexpr int CH = DP / 8;   // 16-byte chunks of a row
    constexpr int KS = DP / 16;  // k steps of the score product
    constexpr int S = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t before[kThreads + 1];  // units before a thread's sequences
    __shared__ uint32_t live[kWarps][S];      // keys of a stage that are seen and lie in valid pages

    ptx::grid_dep_wait();
    ptx::grid_dep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- units before each thread's share of the sequences
    const int per = (a.seqs.batch + kThreads - 1) / kThreads;
    {
        const int b0 = min(a.seqs.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.seqs.batch, b0 + per);
        int64_t sum = 0;
        for (int b = b0; b < b1; ++b) {
            const Seq sq = load_seq(a.seqs, a.pages.page_shift, b);
            const Units un = units_of(a, sq);
            sum += un.units;
            // rows of a sequence without any key are zero
            if (blockIdx.x == b % gridDim.x && sq.nq > 0 && un.tiles == 0) {
                const int chunks = a.pages.dim >> 3;
                for (int i = 0; i < sq.nq * a.heads * chunks; ++i) {
                    const int row = i / chunks, c = i % chunks;
                    *reinterpret_cast<uint4*>(a.out + (sq.t0 + row / a.heads) * a.o_token + (row % a.heads) * a.o_head +
                                              c * 8) = make_uint4(0, 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += o;
        }
        before[threadIdx.x + 1] = sum;
        if (threadIdx.x == 0) before[0] = 0;
    }
    __syncthreads();
    int64_t sums[kWarps + 1] = {0};  // units before each warp's sequences
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sums[w + 1] = sums[w] + before[(w + 1) * 32];
    auto before_of = [&](int i) {  // units before thread i's sequences
        int64_t x = i ? before[i] : 0;
#pragma unroll
        for (int w = 1; w < kWarps; ++w)
            if (i > w * 32) x += before[w * 32];
        return x;
    };

    // ---- this warp's range
    const int worker = blockIdx.x * kWarps + warp, workers = gridDim.x * kWarps;
    const int64_t total = sums[kWarps];
    const int64_t share = max(static_cast<int64_t>(min_units), (total + workers - 1) / workers);
    const int64_t begin = min(total, worker * share), end = min(total, begin + share);
    int* desc = reinterpret_cast<int*>(a.ws + static_cast<size_t>(workers) * 2 * piece_floats(DP)) + worker * kDescInts;
    if (a.ws && lane == 0) desc[0] = 0;
    if (begin >= end) return;
    int seq_lo = 0, seq_hi = kThreads;  // before_of(seq_lo) <= begin < before_of(seq_hi)
    while (seq_hi - seq_lo > 1) {
        const int mid = (seq_lo + seq_hi) >> 1;
        if (before_of(mid) <= begin) {
            seq_lo = mid;
        } else {
            seq_hi = mid;
        }
    }
    int64_t off = begin - before_of(seq_lo);
    int b_first = seq_lo * per;
    for (;; ++b_first) {
        const int64_t n = units_of(a, load_seq(a.seqs, a.pages.page_shift, b_first)).units;
        if (off < n) break;
        off -= n;
    }
    Cursor at(a, b_first, off);
    Cursor ld = at;  // loads run ahead

    const uint32_t ring = ptx::smem_u32(smem) + warp * (S * C::kStageBytes);
    const int g = lane >> 2, tq = lane & 3;
    const int slot_mask = (1 << a.pages.page_shift) - 1;

    // ---- loads: lanes 0..15 find the rows of a tile, all copy chunks
    int64_t ld_left = end - begin;
    int ld_stage = 0;
    // offset of this lane's key of the loading cursor's tile, -1: none; moves the cursor on
    auto find = [&]() -> int64_t {
        if (ld_left <= 0) return -1;
        --ld_left;
        const int key = ld.kt.first(ld.tile) + (lane & 15);
        const int lo = a.window ? max(0, max(ld.sq.p0, 0) + 1 - a.window) : 0;  // first key of the earliest window
        const int32_t* table = a.seqs.tables + ld.b * a.seqs.table_stride;
        const int64_t head = ld.h * a.pages.stride_head;
        const bool seen = key < ld.sq.p0 + ld.sq.nq && (key >= lo || key < a.sinks);  // by any row
        if (++ld.tile == ld.un.tiles && ld_left > 0) ld.next_item(a);
        if (!seen) return -1;
        const int page = table[key >> a.pages.page_shift];
        if (page < 0 || page >= a.pages.num_pages) return -1;
        return page * a.pages.stride_page + (key & slot_mask) * a.pages.stride_token + head;
    };
    auto issue = [&](int64_t row_off) {
        const uint32_t ok = __ballot_sync(0xffffffffu, row_off >= 0) & 0xffffu;
        if (lane == 0) live[warp][ld_stage] = ok;
        const uint32_t dst = ring + ld_stage * C::kStageBytes;
#pragma unroll
        for (int j0 = 0; j0 < kTile * CH; j0 += 32) {
            const int j = j0 + lane, r = j / CH, c = j % CH;
            const int64_t ro = __shfl_sync(0xffffffffu, row_off, r);
            const bool in = ro >= 0 && c * 8 < a.pages.dim;
            const int64_t o = in ? ro + c * 8 : 0;
            const uint32_t n16 = in ? 16u : 0u;
            cp_async16(dst + chunk_at<DP>(r, c), a.pages.k + o, n16);
            cp_async16(dst + kTile * DP * 2 + chunk_at<DP>(r, c), a.pages.v + o, n16);
        }
        ld_stage = ld_stage + 1 == S ? 0 : ld_stage + 1;
        cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < S - 1; ++i) issue(find());  // past the range: a stage of nothing
    int64_t next = find();
    int stage = 0;

    int64_t done = begin;
#pragma unroll 1
    while (done < end) {
        // ---- a piece: tiles [tile0, tile1) of the item at `at`
        const int tile0 = at.tile;
        const int tile1 = static_cast<int>(min(static_cast<int64_t>(at.un.tiles), tile0 + (end - done)));
        const int h = at.h, rows = at.sq.nq * a.group;
        const int r0 = at.rt * kRows + g, r1 = r0 + 8;
        const int i0 = r0 / a.group, i1 = r1 / a.group;
        const int p0 = r0 < rows ? at.sq.p0 + i0 : -1, p1 = r1 < rows ? at.sq.p0 + i1 : -1;
        const int64_t out0 = (at.sq.t0 + i0) * a.o_token + (h * a.group + r0 - i0 * a.group) * a.o_head;
        const int64_t out1 = (at.sq.t0 + i1) * a.o_token + (h * a.group + r1 - i1 * a.group) * a.o_head;
        uint32_t qf[KS][4];  // query rows g and g + 8 of the row tile, as A fragments
        {
            const uint16_t* q0 = a.q + (at.sq.t0 + i0) * a.q_token + (h * a.group + r0 - i0 * a.group) * a.q_head;
            const uint16_t* q1 = a.q + (at.sq.t0 + i1) * a.q_token + (h * a.group + r1 - i1 * a.group) * a.q_head;
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
        // positions of the row tile's first and last row, for the whole-tile test
        const int row_last = min(rows, at.rt * kRows + kRows) - 1;
        const int p_min = at.sq.p0 + (at.rt * kRows) / a.group, p_max = at.sq.p0 + row_last / a.group;

        float o[DP / 8][4];
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll 1
        for (int i = tile0; i < tile1; ++i) {
            issue(next);
            next = find();
            cp_async_wait<S - 1>();
            __syncwarp();
            const uint32_t kt_s = ring + stage * C::kStageBytes, vt_s = kt_s + kTile * DP * 2;
            const int key0 = at.kt.first(i);
            const uint32_t alive = live[warp][stage];
            stage = stage + 1 == S ? 0 : stage + 1;
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
                const bool whole = alive == 0xffffu && key0 + kTile - 1 <= p_min &&
                                   (a.window == 0 || p_max - key0 < a.window || key0 + kTile <= a.sinks);
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int c = j * 8 + tq * 2 + e, key = key0 + c;
                            const bool in = (alive >> c) & 1;
                            if (!in || !visible(key, p0, a.window, a.sinks)) s[j][e] = -INFINITY;
                            if (!in || !visible(key, p1, a.window, a.sinks)) s[j][2 + e] = -INFINITY;
                        }
                }
                float x0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])) * a.scale_log2;
                float x1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])) * a.scale_log2;
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
                if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
                    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
                    const float f0 = x0 > m0 ? exp2_approx(m0 - n0) : 1.f, f1 = x1 > m1 ? exp2_approx(m1 - n1) : 1.f;
                    l0 *= f0;
                    l1 *= f1;
#pragma unroll
                    for (int j = 0; j < DP / 8; ++j) {
                        o[j][0] *= f0;
                        o[j][1] *= f0;
                        o[j][2] *= f1;
                        o[j][3] *= f1;
                    }
                    m0 = n0;
                    m1 = n1;
                }
                const float c0 = m0 == -INFINITY ? 0.f : m0, c1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[j][e] = exp2_approx(s[j][e] * a.scale_log2 - c0);
                        s[j][2 + e] = exp2_approx(s[j][2 + e] * a.scale_log2 - c1);
                        l0 += s[j][e];
                        l1 += s[j][2 + e];
                    }
                // weights as two 16-bit parts, the rounded value and what it leaves: the product
                // then carries 16 (bf16) or 22 (fp16) bits of them, and the second mma costs
                // nothing that HBM does not hide
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
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) {
                    uint32_t vb[4];
                    ldmatrix4_trans(vb, vt_s + chunk_at<DP>(vr, j * 2 + vc));
                    mma16816<BF16>(o[2 * j], hi, vb[0], vb[1]);
                    mma16816<BF16>(o[2 * j + 1], hi, vb[2], vb[3]);
                    mma16816<BF16>(o[2 * j], lo, vb[0], vb[1]);
                    mma16816<BF16>(o[2 * j + 1], lo, vb[2], vb[3]);
                }
            }
            __syncwarp();  // the stage may be filled again
        }
        // ---- the piece's rows: the result, or a part of it
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        const bool part = tile1 - tile0 < at.un.tiles;
        float* ws = part ? a.ws + (static_cast<size_t>(worker) * 2 + (tile0 == 0 ? 1 : 0)) * piece_floats(DP) : nullptr;
        if (part && tile0 > 0 && lane == 0) {
            const int64_t item = done - tile0;
            desc[1] = at.b;
            desc[2] = h;
            desc[3] = at.rt;
            desc[4] = static_cast<int>(item / share);
            desc[5] = static_cast<int>((item + at.un.tiles - 1) / share);
            desc[0] = 1;
        }
        float sum0 = 0.f, sum1 = 0.f;  // 0 if all are finite
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
            sum0 += o[j][0] * 0.f + o[j][1] * 0.f;
            sum1 += o[j][2] * 0.f + o[j][3] * 0.f;
        }
        if (part) {
            if (tq == 0) {
                ws[g] = m0;
                ws[g + 8] = m1;
                ws[kRows + g] = l0;
                ws[kRows + g + 8] = l1;
            }
            float* w0 = ws + 2 * kRows + g * DP + tq * 2;
#pragma unroll
            for (int j = 0; j < DP / 8; ++j) {
                if (r0 < rows) *reinterpret_cast<float2*>(w0 + j * 8) = make_float2(o[j][0], o[j][1]);
                if (r1 < rows) *reinterpret_cast<float2*>(w0 + 8 * DP + j * 8) = make_float2(o[j][2], o[j][3]);
            }
        } else {
            const float inv0 = l0 == 0.f ? 0.f : 1.f / l0, inv1 = l1 == 0.f ? 0.f : 1.f / l1;
#pragma unroll
            for (int j = 0; j < DP / 8; ++j) {
                const int d = j * 8 + tq * 2;
                if (r0 < rows && d < a.pages.dim)
                    *reinterpret_cast<uint32_t*>(a.out + out0 + d) = pack2<BF16>(o[j][0] * inv0, o[j][1] * inv0);
                if (r1 < rows && d < a.pages.dim)
                    *reinterpret_cast<uint32_t*>(a.out + out1 + d) = pack2<BF16>(o[j][2] * inv1, o[j][3] * inv1);
            }
        }
        // A value that a row does not see must not reach it as 0 x inf or 0 x NaN, nor an infinite
        // one as (w - rounded w) x inf. Any such product leaves a sum that is not finite: the row is
        // then taken once more, key by key.
        const uint32_t odd0 = __ballot_sync(0xffffffffu, !(sum0 == 0.f)), odd1 = __ballot_sync(0xffffffffu, !(sum1 == 0.f));
        if (odd0 | odd1) {
            const int rt = at.rt;
#pragma unroll 1
            for (int r = 0; r < kRows; ++r) {
                const int row = rt * kRows + r, token = row / a.group, head = h * a.group + row - token * a.group;
                if (row >= rows || (((r < 8 ? odd0 : odd1) >> ((r & 7) * 4)) & 15u) == 0) continue;
                const RowSum x = careful_row<kTile, BF16>(a, at.b, h, (at.sq.t0 + token) * a.q_token + head * a.q_head,
                                                          at.sq.p0 + token, at.kt, tile0, tile1);
                if (part) {
                    if (lane == 0) {
                        ws[r] = x.m;
                        ws[kRows + r] = x.l;
                    }
                    if (lane * 4 < DP)
                        *reinterpret_cast<float4*>(ws + 2 * kRows + r * DP + lane * 4) = make_float4(x.o[0], x.o[1], x.o[2], x.o[3]);
                } else {
                    x.store<BF16>(a, (at.sq.t0 + token) * a.o_token + head * a.o_head);
                }
            }
        }
        done += tile1 - tile0;
        if (done < end) at.next_item(a);
    }
    cp_async_wait_all();
}

// One CTA per worker that continues an item: the first such of an item, or as many as it has
// rows, take a share of its rows and add the pieces in worker order, a warp a row or several
// when there are many pieces.
constexpr int kJoinWarps = 8;

template <int DP, bool BF16>
__global__ void __launch_bounds__(kJoinWarps * 32) split_join_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int E = DP / 32;
    __shared__ float sums[kJoinWarps][DP + 1];
    ptx::grid_dep_wait();
    const int worker = blockIdx.x + 1, workers = gridDim.x + 1;
    const int* desc =
        reinterpret_cast<const int*>(a.ws + static_cast<size_t>(workers) * 2 * piece_floats(DP)) + worker * kDescInts;
    if (desc[0] == 0) return;
    const int b = desc[1], h = desc[2], rt = desc[3], first = desc[4], last = desc[5];
    const int pieces = last - first + 1, mine = worker - first - 1;
    const Seq sq = load_seq(a.seqs, a.pages.page_shift, b);
    const int rows = min(kRows, sq.nq * a.group - rt * kRows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_row = pieces >= 32 ? 8 : pieces >= 16 ? 4 : pieces >= 8 ? 2 : 1;  // warps
    const int at_once = kJoinWarps / per_row, sub = warp % per_row;
    for (int q = 0; mine + q * (pieces - 1) < rows; q += at_once) {
        const int r = mine + (q + warp / per_row) * (pieces - 1);
        float x[E] = {}, l = 0.f;
        if (r < rows) {
            auto piece = [&](int c) {
                return a.ws + (static_cast<size_t>(c) * 2 + (c == first ? 1 : 0)) * piece_floats(DP);
            };
            float m = -INFINITY;
            for (int c = first + lane; c <= last; c += 32) m = fmaxf(m, piece(c)[r]);
#pragma unroll
            for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
            for (int c = first + sub; c <= last; c += per_row) {
                const float* w = piece(c);
                const float f = exp2_approx(w[r] - base);
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
                // a piece in which the row saw nothing adds nothing
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] += f == 0.f ? 0.f : f * v[e];
            }
        }
        if (per_row > 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = x[e];
            if (lane == 0) sums[warp][DP] = l;
            __syncthreads();
            if (sub == 0 && r < rows) {
                for (int w = warp + 1; w < warp + per_row; ++w) {
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] += sums[w][lane * E + e];
                    l += sums[w][DP];
                }
            }
            __syncthreads();
        }
        if (sub == 0 && r < rows && lane * E < a.pages.dim) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int row = rt * kRows + r, token = row / a.group;
            uint16_t* out = a.out + (sq.t0 + token) * a.o_token + (h * a.group + row - token * a.group) * a.o_head + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<BF16>(x[e] * inv, x[e + 1] * inv);
        }
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
    e = cudaLaunchKernelEx(&cfg, kern, a, p.min_units);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(p.ctas * kWarps - 1);
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, split_join_kernel<DP, BF16>, a);
}

}  // namespace

SplitPlan plan_split(const AttnArgs& a, int num_sms) {
    SplitPlan p;
    p.min_units = 4;
    // what the tables cover bounds the work; the lengths are on the device
    const int64_t covered = static_cast<int64_t>(a.seqs.width) << a.pages.page_shift;
    int64_t tiles = (covered + kTile - 1) / kTile;
    if (a.window)
        tiles = std::min<int64_t>(tiles, (int64_t{a.sinks} + kTile - 1) / kTile +
                                             (int64_t{a.window} + a.seqs.max_q + 2 * kTile - 2) / kTile);
    const int64_t items = static_cast<int64_t>(a.seqs.batch) * a.pages.heads_kv *
                          ((static_cast<int64_t>(a.seqs.max_q) * a.group + kRows - 1) / kRows);
    const int64_t each = int64_t{kWarps} * p.min_units;
    const int64_t most = std::max<int64_t>(1, (items * tiles + each - 1) / each);
    p.ctas = static_cast<int>(std::min<int64_t>(2 * num_sms, most));
    return p;
}

size_t split_workspace_bytes(const SplitPlan& p, int dim) {
    const int dp = dim <= 64 ? 64 : 128;
    return static_cast<size_t>(p.ctas) * kWarps * (2 * piece_floats(dp) * sizeof(float) + kDescInts * sizeof(int));
}

cudaError_t launch_split(const AttnArgs& a, const SplitPlan& p, bool bf16, cudaStream_t s) {
    if (a.pages.dim <= 64) return bf16 ? launch_split_t<64, true>(a, p, s) : launch_split_t<64, false>(a, p, s);
    return bf16 ? launch_split_t<128, true>(a, p, s) : launch_split_t<128, false>(a, p, s);
}

}  // namespace w4a16
