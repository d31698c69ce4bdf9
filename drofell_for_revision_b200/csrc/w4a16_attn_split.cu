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
// worker (an item counts kItemUnits more than its tiles: its query rows and its end), so that
// uneven lengths balance, loads run on from one item into the next, no warp
// waits for another, and the workspace has a fixed size: at most the first and the last piece
// of a range are parts of an item. Those go to the workspace in fp32 and split_join_kernel
// adds them in range order (the same result for the same lengths, whatever runs when).
//
// Measured (keys and values of 128 dimensions): two sequences of 130001 tokens, 64 heads on 8:
// 169 to 190 us by box, 5.6 to 6.3 TB/s; 48 uneven ones of up to 8191: 53 to 54 us, 5.0 TB/s; 24
// under a window of 1024, 40 heads: 47 to 50 us, 5.0 TB/s; one sequence of 777 tokens, 32 heads: 10 us. What
// is left there: some 4 us until the first keys arrive (length, place, page id, key: four
// reads that wait for one another) and 4 us for the join's launch and its two reads.
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
// What an item costs besides its tiles, in tiles: 48 sequences of 1 to 8191 tokens took 104 us
// at 0 (the workers with many short ones came last), 71 at 1, 59 at 2, 57 at 4, 59 at 6.
constexpr int kItemUnits = 4;

// A ring of K and V tiles per warp: as deep as two CTAs an SM allow, or one where there are no
// more CTAs than SMs (DEEP: there latency is what counts, and a worker's few tiles are all in
// flight at once; one sequence of 777 tokens took 14.4 us with the shallow ring).
template <int DP, bool DEEP>
struct SplitCfg {
    static constexpr int kStageBytes = 2 * kTile * DP * 2;  // K and V rows
    static constexpr int kStages = (DP == 128 ? 3 : 6) * (DEEP ? 2 : 1);
    static constexpr int kSmem = kWarps * kStages * kStageBytes;
};

// Workspace: of each worker two pieces m[16], l[16], o[16][DP] (the one it begins with, the
// one it ends with), then what the item is that it continues: {there is one, sequence, head,
// row tile, its first worker, its last, its rows in q: first and number}.
constexpr int piece_floats(int dp) { return 2 * kRows + kRows * dp; }
constexpr int kDescInts = 8;

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
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
// Byte offset of 16-byte chunk c of row r: chunks permuted by the row, so that eight rows
// of one chunk column lie in different banks.
template <int DP>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return static_cast<uint32_t>(r * DP * 2 + ((c ^ (r & 7)) << 4));
}

// Units of a sequence: key tiles (and kItemUnits) x row tiles x heads. The launcher sees to it
// that all of a launch fit 31 bits.
struct Units {
    int tiles, row_tiles, units;
};
__device__ __forceinline__ Units units_of(const AttnArgs& a, const Seq& s) {
    Units u;
    u.tiles = s.nq > 0 ? KeyTiles<kTile>(s.p0, s.p0 + s.nq - 1, a.window, a.sinks).count : 0;
    u.row_tiles = (s.nq * a.group + kRows - 1) / kRows;
    u.units = u.tiles > 0 ? (u.tiles + kItemUnits) * u.row_tiles * a.pages.heads_kv : 0;
    return u;
}

// A place among the units: a key tile of an item of a sequence (or before its first).
struct Cursor {
    int b, h, rt, tile;
    Seq sq;
    Units un;
    KeyTiles<kTile> kt;

    __device__ __forceinline__ void load(const AttnArgs& a) {  // of sequence b, or the next with units
#pragma unroll 1
        for (;; ++b) {
            sq = load_seq(a.seqs, a.pages.page_shift, b);
            un = units_of(a, sq);
            if (un.units > 0) break;
        }
        kt = KeyTiles<kTile>(sq.p0, sq.p0 + sq.nq - 1, a.window, a.sinks);
    }
    // `off` units into sequence b
    __device__ __forceinline__ Cursor(const AttnArgs& a, int seq, int off) : b(seq), kt(0, -1, 0, 0) {
        load(a);
        const int item = off / (un.tiles + kItemUnits);
        tile = off - item * (un.tiles + kItemUnits) - kItemUnits;  // below 0: not begun
        h = item / un.row_tiles;
        rt = item - h * un.row_tiles;
    }
    // to the start of the next item
    __device__ __forceinline__ void next_item(const AttnArgs& a) {
        tile = -kItemUnits;
        if (++rt < un.row_tiles) return;
        rt = 0;
        if (++h < a.pages.heads_kv) return;
        h = 0;
        ++b;
        load(a);
    }
};

template <int DP, bool BF16, bool DEEP>
__global__ void __launch_bounds__(kThreads, DEEP ? 1 : 2) split_kernel(const __grid_constant__ AttnArgs a, const int min_units) {
    using C = SplitCfg<DP, DEEP>;
    constexpr int CH = DP / 8;   // 16-byte chunks of a row
    constexpr int KS = DP / 16;  // k steps of the score product
    constexpr int S = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int before[kThreads];      // units up to a thread's sequences, within its warp
    __shared__ uint32_t live[kWarps][S];      // keys of a stage that are seen and lie in valid pages

    ptx::grid_dep_wait();
    ptx::grid_dep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- units before each thread's share of the sequences
    const int per = (a.seqs.batch + kThreads - 1) / kThreads;
    {
        int sum = 0;
#pragma unroll 1
        for (int i = 0; i < per; ++i) {
            const int b = static_cast<int>(threadIdx.x) * per + i;
            Seq sq = {0, 0, 0};
            bool none = false;
            if (b < a.seqs.batch) {
                sq = load_seq(a.seqs, a.pages.page_shift, b);
                const Units un = units_of(a, sq);
                sum += un.units;
                none = sq.nq > 0 && un.tiles == 0;
            }
            // rows of a sequence without any key are zero: a token a CTA, all lanes over its heads
#pragma unroll 1
            for (uint32_t left = __ballot_sync(0xffffffffu, none); left; left &= left - 1) {
                const int from = __ffs(left) - 1, grid = gridDim.x;
                const int t0 = __shfl_sync(0xffffffffu, sq.t0, from), nq = __shfl_sync(0xffffffffu, sq.nq, from);
                const int first = (static_cast<int>(blockIdx.x) + grid - __shfl_sync(0xffffffffu, b, from) % grid) % grid;
#pragma unroll 1
                for (int t = first; t < nq; t += grid)
#pragma unroll 1
                    for (int h = lane; h < a.heads; h += 32)
#pragma unroll 1
                        for (int d = 0; d < a.pages.dim; d += 8)
                            *reinterpret_cast<uint4*>(a.out + (t0 + t) * a.o_token + h * a.o_head + d) = make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += o;
        }
        before[threadIdx.x] = sum;
    }
    __syncthreads();
    // ---- this warp's range
    const int worker = blockIdx.x * kWarps + warp, workers = gridDim.x * kWarps;
    int warp_end[kWarps];  // units up to each warp's sequences
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) warp_end[w] = total += before[w * 32 + 31];
    const int share = max(min_units, (total + workers - 1) / workers);
    // (a worker behind the last unit may lie behind 31 bits)
    const int begin = static_cast<int>(min(static_cast<int64_t>(total), static_cast<int64_t>(worker) * share));
    const int end = min(total, begin + min(share, total - begin));
    int* desc = reinterpret_cast<int*>(a.ws + static_cast<size_t>(workers) * 2 * piece_floats(DP)) + worker * kDescInts;
    if (a.ws && lane == 0) desc[0] = 0;
    if (begin >= end) return;
    // the thread whose sequences hold `begin`: how many end at or before it
    int holder = 0, off = begin, warp_start = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const bool past = warp_start + before[w * 32 + lane] <= begin;
        holder += __popc(__ballot_sync(0xffffffffu, past));
        warp_start = warp_end[w];
    }
    if (holder > 0) off -= before[holder - 1] + (holder > 32 ? warp_end[(holder - 1) / 32 - 1] : 0);
    int b_first = holder * per;
    if (per > 1) {
#pragma unroll 1
        for (;; ++b_first) {
            const int n = units_of(a, load_seq(a.seqs, a.pages.page_shift, b_first)).units;
            if (off < n) break;
            off -= n;
        }
    }
    Cursor at(a, b_first, off);
    Cursor ld = at;  // loads run ahead

    const uint32_t ring = ptx::smem_u32(smem) + warp * (S * C::kStageBytes);
    const int g = lane >> 2, tq = lane & 3;
    const int slot_mask = (1 << a.pages.page_shift) - 1;

    // ---- loads: lanes 0..15 find the rows of a tile, all copy chunks
    int ld_left = end - begin;
    int ld_stage = 0;
    // page ids of the loading cursor's sequence, a lane each from `page0` on: one read of the table
    // for 32 pages
    int pages = -1, page0 = 0, page_b = -1;
    // offset of this lane's key of the loading cursor's tile, -1: none; moves the cursor on
    auto find = [&]() -> int64_t {
        if (ld.tile < 0) {  // an item begins
            ld_left += ld.tile;
            ld.tile = 0;
            if (ld_left > 0) {  // its query rows on their way to L2
                const int row = ld.rt * kRows + (lane & 15), token = row / a.group;
                if (row < ld.sq.nq * a.group && (lane >> 4) * 64 < a.pages.dim)
                    prefetch_l2(a.q + (ld.sq.t0 + token) * a.q_token + (ld.h * a.group + row - token * a.group) * a.q_head +
                                (lane >> 4) * 64);
            }
        }
        if (ld_left <= 0) return -1;
        --ld_left;
        const int key0 = ld.kt.first(ld.tile), key = key0 + (lane & 15), keys = ld.sq.p0 + ld.sq.nq;
        const int lo = a.window ? max(0, max(ld.sq.p0, 0) + 1 - a.window) : 0;  // first key of the earliest window
        const bool seen = key < keys && (key >= lo || key < a.sinks);           // by any row
        const int64_t head = ld.h * a.pages.stride_head;
        const int want = key0 >> a.pages.page_shift, want2 = (min(key0 + kTile, keys) - 1) >> a.pages.page_shift;
        if (ld.b != page_b || want < page0 || want2 >= page0 + 32) {
            page_b = ld.b;
            page0 = want;
            const int i = page0 + lane;
            pages = i <= (keys - 1) >> a.pages.page_shift ? a.seqs.tables[ld.b * a.seqs.table_stride + i] : -1;
        }
        const int page = __shfl_sync(0xffffffffu, pages, (key >> a.pages.page_shift) - page0);
        if (++ld.tile == ld.un.tiles && ld_left > 0) ld.next_item(a);
        if (!seen || page < 0 || page >= a.pages.num_pages) return -1;
        return page * a.pages.stride_page + (key & slot_mask) * a.pages.stride_token + head;
    };
    auto issue = [&](int64_t row_off) {
        const uint32_t ok = __ballot_sync(0xffffffffu, row_off >= 0) & 0xffffu;
        if (lane == 0) live[warp][ld_stage] = ok;
        if (ok) {  // a tile of no key is not read either
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
        }
        ld_stage = ld_stage + 1 == S ? 0 : ld_stage + 1;
        cp_async_commit();
    };

    // ---- one loop over the tiles: what an item begins and ends with inside it, so that its code
    // is there once (fetching instructions is a good part of a small call)
    int done = begin;
    int64_t next = -1;
    int stage = 1 % S;  // the first stage holds nothing
    int tile0 = 0, tile1 = 0;  // of the piece at hand
    int rows = 0, r0 = 0, r1 = 0, p0 = 0, p1 = 0, p_min = 0, p_max = 0;
    uint32_t qf[KS][4];  // query rows g and g + 8 of the row tile, as A fragments
    float o[DP / 8][4], m0 = 0.f, m1 = 0.f, l0 = 0.f, l1 = 0.f;
    bool begins = true;
#pragma unroll 1
    for (int step = 0;; ++step) {
        issue(next);
        next = find();
        if (step < S) continue;
        if (begins) {
            // ---- a piece: tiles [tile0, tile1) of the item at `at`
            if (at.tile < 0) {
                done -= at.tile;
                at.tile = 0;
            }
            if (done >= end) break;
            begins = false;
            tile0 = at.tile;
            tile1 = min(at.un.tiles, tile0 + (end - done));
            rows = at.sq.nq * a.group;
            r0 = at.rt * kRows + g;
            r1 = r0 + 8;
            const int i0 = r0 / a.group, i1 = r1 / a.group;
            p0 = r0 < rows ? at.sq.p0 + i0 : -1;
            p1 = r1 < rows ? at.sq.p0 + i1 : -1;
            const uint16_t* q0 = a.q + (at.sq.t0 + i0) * a.q_token + (at.h * a.group + r0 - i0 * a.group) * a.q_head;
            const uint16_t* q1 = a.q + (at.sq.t0 + i1) * a.q_token + (at.h * a.group + r1 - i1 * a.group) * a.q_head;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = ks * 16 + e * 8 + tq * 2;
                    const bool in = d < a.pages.dim;
                    qf[ks][2 * e] = r0 < rows && in ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
                    qf[ks][2 * e + 1] = r1 < rows && in ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
                }
            // positions of the row tile's first and last row, for the whole-tile test
            p_min = at.sq.p0 + (at.rt * kRows) / a.group;
            p_max = at.sq.p0 + (min(rows, at.rt * kRows + kRows) - 1) / a.group;
#pragma unroll
            for (int j = 0; j < DP / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            m0 = m1 = -INFINITY;
            l0 = l1 = 0.f;
        }
        {
            cp_async_wait<S - 1>();
            __syncwarp();
            const uint32_t kt_s = ring + stage * C::kStageBytes, vt_s = kt_s + kTile * DP * 2;
            const int key0 = at.kt.first(at.tile);
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
                float x0 = __fmul_rn(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), a.scale_log2);
                float x1 = __fmul_rn(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])), a.scale_log2);
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
                        s[j][e] = weight_of(s[j][e], a.scale_log2, c0, kWeightBias<BF16, kTile>);
                        s[j][2 + e] = weight_of(s[j][2 + e], a.scale_log2, c1, kWeightBias<BF16, kTile>);
                        l0 += s[j][e];
                        l1 += s[j][2 + e];
                    }
                // weights as two 16-bit parts, the rounded value and what it leaves: the product
                // then carries 16 (bf16) or 22 (fp16) bits of them, and the second mma costs
                // nothing that HBM does not hide. fp16 parts end at 2^-24, 2^-39 of the largest
                // weight: below 2^-18 of it bits are lost one by one, and n keys lose less
                // than n 2^-40 of the whole.
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
        if (++at.tile < tile1) continue;

        // ---- the piece's rows: the result, or a part of it
        const int h = at.h;
        const int i0 = r0 / a.group, i1 = r1 / a.group;
        const int64_t out0 = (at.sq.t0 + i0) * a.o_token + (h * a.group + r0 - i0 * a.group) * a.o_head;
        const int64_t out1 = (at.sq.t0 + i1) * a.o_token + (h * a.group + r1 - i1 * a.group) * a.o_head;
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        const bool part = tile1 - tile0 < at.un.tiles;
        float* ws = part ? a.ws + (static_cast<size_t>(worker) * 2 + (tile0 == 0 ? 1 : 0)) * piece_floats(DP) : nullptr;
        if (part && tile0 > 0 && lane == 0) {
            const int item = done - tile0;  // of its first tile
            reinterpret_cast<int4*>(desc)[0] = make_int4(1, at.b, at.h, at.rt);
            reinterpret_cast<int4*>(desc)[1] = make_int4(item / share, (item + at.un.tiles - 1) / share, at.sq.t0, rows);
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
        // bits: rows of the row tile whose sums are not finite while their sums of weights are
        const uint32_t odd0 = __ballot_sync(0xffffffffu, !(sum0 == 0.f) && r0 < rows && l0 == l0);
        const uint32_t odd1 = __ballot_sync(0xffffffffu, !(sum1 == 0.f) && r1 < rows && l1 == l1);
        if (odd0 | odd1) {
            uint32_t bad = 0;
#pragma unroll 1
            for (int r = 0; r < kRows; ++r)
                if (((r < 8 ? odd0 : odd1) >> ((r & 7) * 4)) & 15u) bad |= 1u << r;
            settle_rows<kTile, DP, BF16>(a, at.b, h, at.sq.t0, at.sq.p0, at.rt * kRows, bad, at.kt, tile0, tile1, ws, kRows, 0);
        }
        done += tile1 - tile0;
        if (done >= end) break;
        at.next_item(a);
        begins = true;
    }
    cp_async_wait_all();
}

// One CTA per worker that continues an item: the first such of an item, or as many as it has
// rows, take a share of its rows and add the pieces in worker order, a warp a row or several
// when there are many pieces. A warp has eight pieces in flight at once: latency is all there
// is to it.
constexpr int kJoinWarps = 4, kJoinPieces = 8;

template <int DP, bool BF16>
__global__ void __launch_bounds__(kJoinWarps * 32) split_join_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int E = DP / 32;
    __shared__ float sums[kJoinWarps][DP + 2];
    ptx::grid_dep_wait();
    const int worker = blockIdx.x + 1, workers = gridDim.x + 1;
    const int4* desc =
        reinterpret_cast<const int4*>(a.ws + static_cast<size_t>(workers) * 2 * piece_floats(DP)) + worker * (kDescInts / 4);
    const int4 d0 = desc[0], d1 = desc[1];
    if (d0.x == 0) return;
    const int h = d0.z, rt = d0.w, first = d1.x, last = d1.y, t0 = d1.z;
    const int pieces = last - first + 1, mine = worker - first - 1;
    const int rows = min(kRows, d1.w - rt * kRows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_row = pieces > 2 * kJoinPieces ? 4 : pieces > kJoinPieces ? 2 : 1;  // warps
    const int at_once = kJoinWarps / per_row, sub = warp % per_row;
#pragma unroll 1
    for (int q = 0; mine + q * (pieces - 1) < rows; q += at_once) {
        const int r = mine + (q + warp / per_row) * (pieces - 1);
        float x[E] = {}, m = -INFINITY, l = 0.f;
        if (r < rows) {
#pragma unroll 1
            for (int c0 = first + sub * kJoinPieces; c0 <= last; c0 += per_row * kJoinPieces) {
                float v[kJoinPieces][E];
#pragma unroll
                for (int i = 0; i < kJoinPieces; ++i) {
                    const int c = min(c0 + i, last);
                    const float* w = a.ws + (static_cast<size_t>(c) * 2 + (c == first ? 1 : 0)) * piece_floats(DP) + 2 * kRows +
                                     r * DP + lane * E;
                    if constexpr (E == 4) {
                        const float4 u = *reinterpret_cast<const float4*>(w);
                        v[i][0] = u.x, v[i][1] = u.y, v[i][2] = u.z, v[i][3] = u.w;
                    } else {
                        const float2 u = *reinterpret_cast<const float2*>(w);
                        v[i][0] = u.x, v[i][1] = u.y;
                    }
                }
                // maximum and sum of piece c0 + (lane & 7)
                const int c = c0 + (lane & (kJoinPieces - 1));
                const float* w = a.ws + (static_cast<size_t>(min(c, last)) * 2 + (c == first ? 1 : 0)) * piece_floats(DP) + r;
                const float mc = c <= last ? w[0] : -INFINITY, lc = c <= last ? w[kRows] : 0.f;
                float m2 = fmaxf(m, mc);
#pragma unroll
                for (int d = kJoinPieces / 2; d; d >>= 1) m2 = fmaxf(m2, __shfl_xor_sync(0xffffffffu, m2, d));
                const float base = m2 == -INFINITY ? 0.f : m2;
                const float old = m == -INFINITY ? 0.f : exp2_approx(m - base), f = exp2_approx(mc - base + kJoinBias);
                m = m2;
                float sum = lc * f;
#pragma unroll
                for (int d = kJoinPieces / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                l = l * old + sum;
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = share_of(old, x[e]);
#pragma unroll
                for (int i = 0; i < kJoinPieces; ++i) {
                    const float fi = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] += share_of(fi, v[i][e]);
                }
            }
        }
        if (per_row > 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = x[e];
            if (lane == 0) {
                sums[warp][DP] = m;
                sums[warp][DP + 1] = l;
            }
            __syncthreads();
            if (sub == 0 && r < rows) {
                float top = m;
                for (int w = warp + 1; w < warp + per_row; ++w) top = fmaxf(top, sums[w][DP]);
                const float base = top == -INFINITY ? 0.f : top;
                const float f = exp2_approx(m - base);
                l *= f;
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = share_of(f, x[e]);
#pragma unroll 1
                for (int w = warp + 1; w < warp + per_row; ++w) {
                    const float fw = exp2_approx(sums[w][DP] - base);
                    l += sums[w][DP + 1] * fw;
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] += share_of(fw, sums[w][lane * E + e]);
                }
            }
            __syncthreads();
        }
        if (sub == 0 && r < rows && lane * E < a.pages.dim) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int row = rt * kRows + r, token = row / a.group;
            uint16_t* out = a.out + (t0 + token) * a.o_token + (h * a.group + row - token * a.group) * a.o_head + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<BF16>(x[e] * inv, x[e + 1] * inv);
        }
    }
}

template <int DP, bool BF16, bool DEEP>
cudaError_t launch_split_t(const AttnArgs& a, const SplitPlan& p, cudaStream_t s) {
    using C = SplitCfg<DP, DEEP>;
    auto kern = split_kernel<DP, BF16, DEEP>;
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

// The most units that one sequence can have: what the tables cover bounds its length, which is
// on the device.
int64_t most_units(const AttnArgs& a) {
    const int64_t covered = static_cast<int64_t>(a.seqs.width) << a.pages.page_shift;
    int64_t tiles = (covered + kTile - 1) / kTile;
    if (a.window)
        tiles = std::min<int64_t>(tiles, (int64_t{a.sinks} + kTile - 1) / kTile +
                                             (int64_t{a.window} + a.seqs.max_q + 2 * kTile - 2) / kTile);
    return (tiles + kItemUnits) * a.pages.heads_kv * ((static_cast<int64_t>(a.seqs.max_q) * a.group + kRows - 1) / kRows);
}
constexpr int64_t kMostUnits = (int64_t{1} << 31) - (int64_t{1} << 20);

}  // namespace

bool split_fits(const AttnArgs& a) { return most_units(a) <= kMostUnits; }

SplitPlan plan_split(const AttnArgs& a, int num_sms) {
    SplitPlan p;
    p.min_units = 2;  // one sequence of 777 tokens: 10.8 us at 1, 10.1 at 2, 10.3 at 3, 11.2 at 4
    const int64_t each = int64_t{kWarps} * p.min_units;
    const int64_t most = std::max<int64_t>(1, (a.seqs.batch * most_units(a) + each - 1) / each);
    p.ctas = static_cast<int>(std::min<int64_t>(2 * num_sms, most));
    p.deep = p.ctas <= num_sms;
    return p;
}

size_t split_workspace_bytes(const SplitPlan& p, int dim) {
    const int dp = dim <= 64 ? 64 : 128;
    return static_cast<size_t>(p.ctas) * kWarps * (2 * piece_floats(dp) * sizeof(float) + kDescInts * sizeof(int));
}

cudaError_t launch_split(const AttnArgs& all, const SplitPlan& p, bool bf16, cudaStream_t s) {
    // as many sequences a launch as have units that fit 31 bits: all of them but for tables of
    // many millions of tokens
    const int most = static_cast<int>(std::min<int64_t>(all.seqs.batch, kMostUnits / most_units(all)));
    for (int b = 0; b < all.seqs.batch; b += most) {
        AttnArgs a = all;
        a.seqs.batch = std::min(most, all.seqs.batch - b);
        a.seqs.tables += b * a.seqs.table_stride;
        a.seqs.lens += b;
        if (a.seqs.cu_q) {
            a.seqs.cu_q += b;
        } else {
            a.q += b * a.q_token;
            a.out += b * a.o_token;
            a.seqs.tokens = a.seqs.batch;
        }
        cudaError_t e;
        if (a.pages.dim <= 64) {
            e = p.deep ? (bf16 ? launch_split_t<64, true, true>(a, p, s) : launch_split_t<64, false, true>(a, p, s))
                       : (bf16 ? launch_split_t<64, true, false>(a, p, s) : launch_split_t<64, false, false>(a, p, s));
        } else {
            e = p.deep ? (bf16 ? launch_split_t<128, true, true>(a, p, s) : launch_split_t<128, false, true>(a, p, s))
                       : (bf16 ? launch_split_t<128, true, false>(a, p, s) : launch_split_t<128, false, false>(a, p, s));
        }
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace w4a16
