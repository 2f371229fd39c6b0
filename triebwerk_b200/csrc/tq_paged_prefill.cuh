// Causal attention of several new tokens per request over paged packed caches (tcgen05 + tensor memory), sm_100a.
//
// Query i of request g, of its n new tokens, stands at position p = L - n + i of its L tokens and attends to tokens 0 .. p:
//   out = R (softmax_t(R q . norm_K[t] centroids_K[t] / sqrt(128)) . norm_V[t] centroids_V[t])
// with q rotated once and one R product at the end (tq_prefill_fa.cuh has the mathematics; the slots, the softmax and the order of
// products are that kernel's).  What differs: the batch is ragged, requests have earlier tokens, rows come by way of block tables, and the
// codes become fp16 centroids INSIDE the kernel, so that a call needs no scratch for the contexts, whose lengths the host does not know
// (16384 tokens and 8 KV heads as fp16 are 64 MB a request), and reads the packed bytes alone.
//   * A block = 128 score rows = 128 / GRP query tokens x the GRP query heads of a KV head.  MT = 2: a CTA has two blocks, which share
//     every K and V tile; MT = 1: one block, whose two slots take the even and the odd tiles and are combined at the end.
//   * The 16 softmax warps are the producers too: a thread fetches 16 (2-bit: 8) bytes of one row of the next K and V tile into registers
//     as soon as it has made the present one, and turns them into centroids through a shared-memory table with a column
//     per lane.  So the table look-ups and operand stores fill the time in which the tensor core works on the slot's own products.
//   * All 16 warps make a share of every tile.  MT = 2: K of tile j + 1 before the softmax of tile j, V behind it.  MT = 1: after tile j, which is
//     one slot's, K of tile j + 2 and V of tile j + 1, so that the other slot's warps need not wait for tile j's products.
//   * Three warps fetch the tiles' rows (one page number for each 32 tokens) and norms ahead, into a ring in shared memory.
//   * SPLIT (MT = 1): few query rows, long contexts: the tiles of every block are cut into as many parts as the SMs have room for, whose
//     sums meet in paged_merge_kernel.  How many blocks there are is known here, not on the host, which knows no request's share of the
//     batch's tokens: single tokens beside a chunk have no block of this kernel (4-bit 32/8 heads, 63 beside 64 tokens behind 30000: 560 us uncut, 186 cut).
// Blocks are found without a table: every CTA takes the running sum of the requests' blocks (BT query tokens each) and looks where its number
// falls; the launch has room for as many as there can be, and those behind the last end at once.  Requests of few rows (small_rows) have none: those
// are tq_paged_rows.cuh's.
// Every wait on a barrier is bounded, as there.
//
// 4-bit: 8 prompts of 512, 16/8 heads, 45 us; 4 x 1024 behind 5100 to 8192, 32/8 heads, 605 to 639 us (0.70 to 0.74 PFLOP/s; GPUs differ).  What bounds it is the number of
// instructions, 6500 a warp-wide pair of tiles (issue slots 57 %, products 40 % of the cycles; stamps: 5000 cycles a pair), and at the ends of short prompts a
// CTA's start (5800 cycles: table, queries times R, first rows) and end.
#pragma once

#include <climits>

#include "tq_paged.cuh"

namespace tq {

struct PagedPrefillParams {
    const uint8_t* ck;
    const uint8_t* cv;
    const __half* kn;
    const __half* vn;
    const int* block_table;
    const int* lens;          // [G]; 0 and less: no token
    const int* start;         // [G + 1]
    __half* out;
    float* partials;          // SPLIT: [parts][T][H][PART_STRIDE]
    int* status;
    int table_stride, page_shift, num_pages, most_tokens;
    int T, G, H, Hkv, grp, out_stride;
    int small_rows;           // requests of up to so many score rows (new tokens x heads of a KV head) are not served here
    int room, most_parts;     // SPLIT: see prefill_parts
};
// Parts that every block's tiles are cut into: as many as give `room` CTAs a part each.
__device__ __forceinline__ int prefill_parts(int blocks, int Hkv, int room, int most) {  // blocks: of 128 rows, of all requests and one KV head
    return (int)max(1ll, min((long long)most, room / ((long long)max(blocks, 1) * Hkv)));
}

constexpr int PPF_THREADS = 32 * PFT_SOFT_WARPS + 128;  // softmax and operands; one warp for the products, three for rows and norms
constexpr int PPF_MEET = 32 * PFT_SOFT_WARPS + 32;      // all but those
// (No register split: 96 each are enough, and the thread that issues the products spilled with fewer -- 64 for it, 104 for the rest, 4 x 1024 tokens
// behind 8192 took 618 us, with 32 and 112 1072.)
constexpr int PPF_STAGES = 4;                          // of a tile's norms and rows: fetched ahead, and the slots may be far apart
struct PpfSmem {
    static constexpr uint32_t Q = 0;                       // 2 tiles; at the end: the results
    static constexpr uint32_t K = 2 * PFT_TILE;            // 2 stages; at the start R in the second
    static constexpr uint32_t V = K + 2 * PFT_TILE;        // 2 stages; at the end R in the free one
    static constexpr uint32_t LUT = V + 2 * PFT_TILE;      // byte (4-bit) or nibble -> two centroids, a column per lane; at the end (MT = 1) the slots' maxima and sums
    static constexpr uint32_t LUT_BYTES = 32768u;
    static constexpr uint32_t INFO = LUT + LUT_BYTES;      // [stage]: K norms, V norms as halves, first row of each 32 tokens, a V norm that is not finite
    static constexpr uint32_t INFO_ROWS = 4u * PFT_KT, INFO_ODD = INFO_ROWS + 16u, INFO_BYTES = INFO_ODD + 16u;
    static constexpr uint32_t CTRL = INFO + PPF_STAGES * INFO_BYTES;
    static constexpr uint32_t BYTES = CTRL + 256u;
};
static_assert(PpfSmem::BYTES <= 227 * 1024, "one CTA's shared memory");
constexpr uint32_t PPF_XCH = PpfSmem::LUT;  // (the table is no longer needed then)

template <int BITS, int MT, bool SPLIT>
__global__ void __launch_bounds__(PPF_THREADS, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmR, const PagedPrefillParams p) {
    static_assert(!SPLIT || MT == 1, "few rows");
    extern __shared__ __align__(1024) uint8_t ppf_smem[];
    const uint32_t sb = smem_u32(ppf_smem);
    uint8_t* const gb = ppf_smem;
    if ((sb & 1023u) != 0u) {
        if (threadIdx.x == 0) atomicMax(p.status, ST_SMEM_LAYOUT);
        return;
    }
    constexpr int MMA_WARP = PFT_SOFT_WARPS;
    constexpr int BPH = HEAD_DIM * BITS / 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int GRP = p.grp, QT = PFT_ROWS / GRP, BT = MT * QT;

    // ---- once: tensor memory, barriers, table ----
    const uint32_t ctrl = sb + PpfSmem::CTRL;
    const uint32_t bar_kfull = ctrl, bar_vfull = ctrl + 16u, bar_kfree = ctrl + 32u, bar_vfree = ctrl + 48u;  // [2] each
    const uint32_t bar_sfull = ctrl + 64u, bar_pfull = ctrl + 80u;                                            // [2 slots] each
    const uint32_t bar_rot = ctrl + 96u, bar_done = ctrl + 104u, bar_q = ctrl + 112u, bar_r = ctrl + 120u, bar_done1 = ctrl + 248u;
    const uint32_t bar_rows = ctrl + 128u, bar_norms = ctrl + 160u, bar_used = ctrl + 192u;                   // [PPF_STAGES] each
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(gb + PpfSmem::CTRL + 224);
    if (warp == 0) {
        tmem_alloc(ctrl + 224u, 512u);
        tmem_relinquish();
    }
    if (tid == 32 * MMA_WARP) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_kfull + 8u * i, PFT_SOFT_WARPS);
            mbar_init(bar_vfull + 8u * i, PFT_SOFT_WARPS);
            mbar_init(bar_kfree + 8u * i, 1);
            mbar_init(bar_vfree + 8u * i, 1);
            mbar_init(bar_sfull + 8u * i, 1);
            mbar_init(bar_pfull + 8u * i, PFT_SOFT_WARPS / 2);
        }
        for (int i = 0; i < PPF_STAGES; ++i) {
            mbar_init(bar_rows + 8u * i, 1);
            mbar_init(bar_norms + 8u * i, 1);
            mbar_init(bar_used + 8u * i, PFT_SOFT_WARPS);
        }
        mbar_init(bar_rot, 1);
        mbar_init(bar_done, 1);
        mbar_init(bar_done1, 1);
        mbar_init(bar_q, 1);
        mbar_init(bar_r, 1);
        fence_mbar_init();
    }
    {
        // (entry (tid >> 3) + 64 i, four lanes' columns: a thread's entries share their first code)
        constexpr float c = PPF_CENT<BITS>;
        const int e = tid >> 3;
        const float first = c * (BITS == 4 ? kCent4[e & 15] : kCent2[e & 3]);
#pragma unroll
        for (int i = 0; i < (BITS == 4 ? 4 : 1); ++i) {
            const uint32_t u = pack_half2(first, c * (BITS == 4 ? kCent4[((tid >> 7) & 3) + 4 * i] : kCent2[(e >> 2) & 3]));
            if (BITS == 4 ? tid < 512 : tid < 128) *reinterpret_cast<uint4*>(gb + PpfSmem::LUT + 16u * (uint32_t)(tid + 512 * i)) = make_uint4(u, u, u, u);
        }
    }
    pdl_wait();  // (lengths, tables, caches, queries: all of earlier launches)
    pdl_launch_dependents();  // (behind the wait: what starts now knows that those have finished)
    // ---- the request and the block of this CTA ----
    const int kvh = (int)blockIdx.x % p.Hkv;
    int y = (int)blockIdx.x / p.Hkv;  // SPLIT: all blocks' first parts, then their second ones
    // First query, queries of the request, the block's first one, request; SPLIT: part and parts.  (They wait in shared memory for the end, which is what else needs them: in
    // registers they cost spills, and those come back from L2, see below.)  The warps' block counts lie where K comes later.
    volatile int* const kept = reinterpret_cast<volatile int*>(gb + PpfSmem::CTRL + 228);
    int* const scratch = reinterpret_cast<int*>(gb + PpfSmem::K);
    constexpr int WARPS = PPF_THREADS / 32;
    if (tid == 0) kept[3] = -1;
    tc_fence_before();
    int before = 0, part = 0, parts = 1;
    auto blocks_of = [&](int i, int& a, int& m) {
        a = m = 0;
        if (i < p.G) {
            a = max(p.start[i], 0);
            m = max(min(p.start[i + 1], p.T) - a, 0);
        }
        return m * GRP > p.small_rows ? (m + BT - 1) / BT : 0;
    };
    auto cut = [&](int blocks) {  // of all requests
        parts = prefill_parts(blocks, p.Hkv, p.room, p.most_parts);
        part = y / max(blocks, 1);
        y = part < parts ? y - part * blocks : INT_MAX;
        if (tid == 0) kept[4] = part | parts << 8;
    };
    if (SPLIT && p.G > PPF_THREADS) {  // (otherwise the sum is at hand below)
        int sum = 0, a, m;
        for (int i = tid; i < p.G; i += PPF_THREADS) sum += blocks_of(i, a, m);
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) scratch[warp] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < WARPS; ++w) sum += scratch[w];
        cut(sum);
        __syncthreads();
    }
    for (int first = 0; first < p.G; first += PPF_THREADS) {
        const int i = first + tid;
        int a, m;
        const int blocks = blocks_of(i, a, m);
        int incl = blocks;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scratch[warp] = incl;
        __syncthreads();
        int mine = before, all = 0;
        for (int w = 0; w < WARPS; ++w) {
            const int v = scratch[w];
            mine += w < warp ? v : 0;
            all += v;
        }
        if (SPLIT && p.G <= PPF_THREADS) cut(all);
        const int at = y - (mine + incl - blocks);
        if (at >= 0 && at < blocks) {  // (the last blocks of a request, whose causal prefixes are the longest, first)
            kept[0] = a;
            kept[1] = m;
            kept[2] = (blocks - 1 - at) * BT;
            kept[3] = i;
        }
        before += all;
        __syncthreads();  // (what was made above is in place too)
        if (before > y) break;
    }
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int s0 = kept[0], n = kept[1], q0 = kept[2], g = kept[3];
    if (g < 0) {  // no such block
        if (warp == 0) tmem_dealloc(tmem, 512u);
        return;
    }
    if (tid == 32 * MMA_WARP) {
        mbar_arrive_expect_tx(bar_q, (uint32_t)(MT * QT * GRP) * 256u + PFT_TILE);
        for (int m = 0; m < MT; ++m) {  // (rows of other requests or past the end: a row's garbage stays in that row and is never stored)
            tma_load_4d(sb + PpfSmem::Q + m * PFT_TILE, &tmQ, bar_q, 0, kvh * GRP, s0 + q0 + m * QT, 0);
            tma_load_4d(sb + PpfSmem::Q + m * PFT_TILE + PFT_TILE / 2, &tmQ, bar_q, 0, kvh * GRP, s0 + q0 + m * QT, 1);
        }
        tma_load_3d(sb + PpfSmem::K + PFT_TILE, &tmR, bar_q, 0, 0, 0);
    }
    const int L = min(max(p.lens[g], 0), p.most_tokens), pos0 = L - n;  // position of the request's first new token
    // tiles that the block whose first query is `first` reads
    auto tiles_to = [&](int first) { return first < n ? (int)(((unsigned)max(pos0 + min(first + QT, n), 0) + (PFT_KT - 1u)) / PFT_KT) : 0; };
    const int t_lo = SPLIT ? (int)((long long)tiles_to(q0) * part / parts) : 0;
    const int n_all = (SPLIT ? (int)((long long)tiles_to(q0) * (part + 1) / parts) : tiles_to(q0)) - t_lo;
    const int n0 = MT == 2 ? n_all : (n_all + 1) / 2, n1 = MT == 2 ? tiles_to(q0 + QT) : n_all / 2;
    const int n_tiles = MT == 2 ? max(n0, n1) : n_all;
    auto tile_of = [&](int s, int i) { return MT == 2 ? i : 2 * i + s; };  // (behind t_lo)

    auto joined = [&]() { return SPLIT && kept[4] >> 8 > 1; };  // (uniform) the results are paged_merge_kernel's

    bool dead = false;
    auto wait_bar = [&](uint32_t bar, uint32_t parity) {
        if (!dead && !mbar_try_wait(bar, parity) && !mbar_wait_bounded_hint(bar, parity, 1u << 17, 2000u)) {
            dead = true;
            atomicMax(p.status, ST_TMA_WAIT_TIMEOUT);
        }
    };
    const int slot = (warp >> 2) & 1, row0 = 32 * (warp & 3) + 16 * (warp >> 3), gl = lane >> 2, t4 = lane & 3;
    const int my_first = q0 + (MT == 2 ? slot * QT : 0);
    auto make_by_grp = [&]() {  // row / GRP by a multiplication, exact below 128
        uint32_t d = (uint32_t)GRP;
        asm volatile("" : "+r"(d));
        return (65536u + d - 1u) / d;
    };
    auto token_in = [&](int row, uint32_t by_grp) { return (int)(((uint32_t)row * by_grp) >> 16); };
    auto token_of = [&](int row, uint32_t by_grp) { return token_in(row, by_grp) < QT ? my_first + token_in(row, by_grp) : n; };  // (n: a row of no query)
    const uint32_t my_lanes = tmem + ((uint32_t)row0 << 16);
    auto put_frag = [&](uint32_t tile, int c0, const float (&v)[32]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                auto two = [&](int b) { return pack_half2(v[4 * b + 2 * h], v[4 * b + 2 * h + 1]); };
                stmatrix_x4(sb + tile + pft_chunk(row0 + 8 * h + (lane & 7), (c0 >> 3) + j + (lane >> 3)), two(j), two(j + 1), two(j + 2), two(j + 3));
            }
    };
    constexpr int PCOLS = MT == 2 ? 128 : 64;
    const int pcol0 = MT == 2 ? 0 : 64 * slot;
    const uint32_t pslot = MT == 2 ? (uint32_t)slot : 0u;

    if (warp >= MMA_WARP) {
      if (warp == MMA_WARP) {
        // ================= one thread issues every product =================
        if (lane == 0) {
            wait_bar(bar_q, 0u);
            tc_fence_after();
            if (!dead) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        umma_lo(tmem + 128u * m, pft_lo_k(sb + PpfSmem::Q + m * PFT_TILE) + pft_kstep(ks), pft_lo_k(sb + PpfSmem::K + PFT_TILE) + pft_kstep(ks), PFT_IDESC_K, ks != 0);
            }
            umma_commit(bar_rot);
        }
        __syncwarp();
        named_barrier(1, PPF_MEET);  // the rotated queries are in place
        tc_fence_after();
        if (lane == 0) {
            auto issue_scores = [&](int s, int i) {
                const int j = tile_of(s, i), st = j & 1;
                wait_bar(bar_kfull + 8u * st, (uint32_t)((j >> 1) & 1));
                tc_fence_after();
                if (dead) return;
                const uint32_t a = pft_lo_k(sb + PpfSmem::Q + (MT == 2 ? s * PFT_TILE : 0u)), b = pft_lo_k(sb + PpfSmem::K + st * PFT_TILE);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) umma_lo(tmem + 128u * s, a + pft_kstep(ks), b + pft_kstep(ks), PFT_IDESC_K, ks != 0);
                umma_commit(bar_sfull + 8u * s);
                if (MT == 1 || s == (j < n1 ? 1 : 0)) umma_commit(bar_kfree + 8u * st);  // its last reader
            };
            auto issue_values = [&](int s, int i) {
                const int j = tile_of(s, i), st = j & 1;
                wait_bar(bar_vfull + 8u * st, (uint32_t)((j >> 1) & 1));
                wait_bar(bar_pfull + 8u * s, (uint32_t)(i & 1));
                tc_fence_after();
                if (dead) return;
                const uint32_t b = pft_lo_mn(sb + PpfSmem::V + st * PFT_TILE);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    umma_lo_ta(tmem + 256u + 128u * s, tmem + 128u * s + 8u * ks, b + 128u * ks, PFT_IDESC_MN, ks == 0 ? (uint32_t)(i != 0) : 1u);
                if (MT == 1 || s == (j < n1 ? 1 : 0)) umma_commit(bar_vfree + 8u * st);
            };
            if (n0 > 0) issue_scores(0, 0);
            if (n1 > 0) issue_scores(1, 0);
            // R again, for the results, where V of the tile in front of the last was: as soon as its products are done
            auto fetch_rotation = [&]() {
                if (joined()) return;
                if (n_tiles >= 2) wait_bar(bar_vfree + 8u * (n_tiles & 1), (uint32_t)(((n_tiles - 2) >> 1) & 1));
                if (dead) return;
                mbar_arrive_expect_tx(bar_r, PFT_TILE);
                tma_load_3d(sb + PpfSmem::V + (uint32_t)(n_tiles & 1) * PFT_TILE, &tmR, bar_r, 0, 0, 0);
            };
            // MT = 2: the slots end apart, each with a barrier of its own; MT = 1: together
            if (MT == 2 && n0 == 0) umma_commit(bar_done);
            if (MT == 2 && n1 == 0) umma_commit(bar_done1);
            for (int i = 0; i < max(n0, n1); ++i) {
                if (i < n0) {
                    issue_values(0, i);
                    if (i + 1 < n0) issue_scores(0, i + 1);
                    else if (MT == 2) umma_commit(bar_done);
                }
                if (MT == 2 && i + 1 == n_tiles) fetch_rotation();  // (the products of the tile in front are all on their way)
                if (i < n1) {
                    issue_values(1, i);
                    if (i + 1 < n1) issue_scores(1, i + 1);
                    else if (MT == 2) umma_commit(bar_done1);
                }
            }
            if (MT == 1) umma_commit(bar_done);
            if (MT == 1 || n_tiles == 0) fetch_rotation();
        }
        __syncwarp();
        if (!joined()) {
            // out[d] = sum_k R[k][d] * acc[k]
            auto rotate_back = [&](int m, uint32_t bar) {
                if (lane == 0) {
                    wait_bar(bar_r, 0u);
                    tc_fence_after();
                    if (!dead) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            umma_lo(tmem + 128u * m, pft_lo_k(sb + PpfSmem::Q + m * PFT_TILE) + pft_kstep(ks), pft_lo_mn(sb + PpfSmem::V + (uint32_t)(n_tiles & 1) * PFT_TILE) + 128u * ks,
                                    PFT_IDESC_MN, ks != 0);
                    }
                    umma_commit(bar);
                }
                __syncwarp();
            };
            if (MT == 1) {
                named_barrier(1, PPF_MEET);
                rotate_back(0, bar_rot);
            } else {
                named_barrier(3, PPF_MEET / 2 + 16);
                rotate_back(0, bar_rot);
                named_barrier(4, PPF_MEET / 2 + 16);
                rotate_back(1, bar_q);
            }
        }
      } else {
        // ================= rows and norms of the tiles, three warps in turn =================
        const int* const my_pages = p.block_table + (size_t)g * p.table_stride;
        for (int j = warp - MMA_WARP - 1; j < n_tiles; j += 3) {
            const int st = j & (PPF_STAGES - 1), t0 = (t_lo + j) * PFT_KT;
            if (j >= PPF_STAGES) wait_bar(bar_used + 8u * st, (uint32_t)((j / PPF_STAGES - 1) & 1));
            uint8_t* const info = gb + PpfSmem::INFO + (uint32_t)st * PpfSmem::INFO_BYTES;
            // pages hold 32 tokens at least.  (Behind the request's last token: some row of the cache; its norm counts as zero.)
            uint32_t row = 0u;
            if (lane < 4 && t0 + 32 * lane < L)
                row = (min((uint32_t)__ldg(my_pages + ((t0 + 32 * lane) >> p.page_shift)), (uint32_t)p.num_pages - 1u) << p.page_shift) + (uint32_t)((t0 + 32 * lane) & ((1 << p.page_shift) - 1));
            if (lane < 4) reinterpret_cast<uint32_t*>(info + PpfSmem::INFO_ROWS)[lane] = row;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_rows + 8u * st);
            unsigned short kn[4], vn[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const size_t at = (size_t)(__shfl_sync(0xffffffffu, row, k) + (uint32_t)lane) * p.Hkv + kvh;
                kn[k] = vn[k] = 0;
                if (t0 + 32 * k + lane < L) {
                    kn[k] = __ldg(reinterpret_cast<const unsigned short*>(p.kn) + at);
                    vn[k] = __ldg(reinterpret_cast<const unsigned short*>(p.vn) + at);
                }
            }
            bool odd = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                reinterpret_cast<unsigned short*>(info)[32 * k + lane] = kn[k];
                reinterpret_cast<unsigned short*>(info)[PFT_KT + 32 * k + lane] = vn[k];
                odd = odd || (vn[k] & 0x7fffu) >= 0x7c00u;
            }
            odd = __any_sync(0xffffffffu, odd);
            __syncwarp();
            if (lane == 0) {
                *reinterpret_cast<uint32_t*>(info + PpfSmem::INFO_ODD) = odd ? 1u : 0u;
                mbar_arrive(bar_norms + 8u * st);
            }
        }
      }
    } else {
        // ================= operands and softmax =================
        // ---- a thread's share of every tile: piece tid & 3 of row tid >> 2 ----
        const int mrow = tid >> 2, piece = tid & 3;
        uint4 kc, vc;                   // codes of the next tile (2-bit: x, y)
        auto info_of = [&](int j) { return gb + PpfSmem::INFO + (uint32_t)(j & (PPF_STAGES - 1)) * PpfSmem::INFO_BYTES; };
        // (four words in the order in which put_codes takes them)
        auto fetch = [&](int j, const uint8_t* codes, uint4& c) {
            const uint32_t row = reinterpret_cast<const uint32_t*>(info_of(j) + PpfSmem::INFO_ROWS)[mrow >> 5] + (uint32_t)(mrow & 31);
            const uint8_t* const src = codes + ((size_t)row * (uint32_t)p.Hkv + (uint32_t)kvh) * BPH;
            if (BITS == 4) {
                const uint2 a = __ldg(reinterpret_cast<const uint2*>(src + 16 * piece + 4 * (piece & 2))), b = __ldg(reinterpret_cast<const uint2*>(src + 16 * piece + 8 - 4 * (piece & 2)));
                c = make_uint4(a.x, a.y, b.x, b.y);
            } else {
                const uint2 a = __ldg(reinterpret_cast<const uint2*>(src) + piece);
                c.x = a.x; c.y = a.y;
            }
        };
        auto fetch_k = [&](int j) {  // (the norms' barrier: rows come before them)
            if (j >= n_tiles) return;
            wait_bar(bar_norms + 8u * (j & (PPF_STAGES - 1)), (uint32_t)((j / PPF_STAGES) & 1));
            fetch(j, p.ck, kc);
        };
        auto fetch_v = [&](int j) {  // (K's fetch of that tile came before)
            if (j < n_tiles) fetch(j, p.cv, vc);
        };
        uint32_t lut;  // (made here, behind the barrier that the table waits for: the look-ups take it into their address)
        asm volatile("mov.u32 %0, %1;" : "=r"(lut) : "r"(sb + PpfSmem::LUT + 4u * (uint32_t)lane) : "memory");
        // 32 codes as centroids times a norm into the row's 16-byte pieces 4 piece .. + 3, in an order in which a quarter-warp's stores meet no
        // bank twice: the f-th is piece f ^ (piece & 2) of the four.  The norm is in the operands, rounded to fp16 once more: for each score and
        // weight, 64 a thread and tile, it cost a fifth of all instructions.
        const uint32_t my_at = sb + (uint32_t)(piece >> 1) * (PFT_TILE / 2) + (uint32_t)mrow * 128u + (uint32_t)(((4 * (piece & 1)) ^ (piece & 2) ^ (mrow & 7)) << 4);
        auto put_codes = [&](uint32_t tile, const uint4 c, uint32_t norm) {
            const __half2 n2 = __half2half2(__ushort_as_half((unsigned short)norm));
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const uint32_t first = (piece & 2) ? c.y : c.x, second = (piece & 2) ? c.x : c.y;  // (2-bit: 16 bits a piece)
                const uint32_t w = BITS == 4 ? (f == 0 ? c.x : f == 1 ? c.y : f == 2 ? c.z : c.w) : (f & 2 ? second : first) >> ((f & 1) * 16);
                uint32_t u[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const uint32_t at = BITS == 4 ? (b == 0 ? (w << 7) & 0x7f80u : (w >> (8 * b - 7)) & 0x7f80u)
                                                  : (b < 2 ? (w << (7 - 4 * b)) & 0x780u : (w >> (4 * b - 7)) & 0x780u);
                    u[b] = ldsp32(lut + at);
                    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&u[b]), n2);
                    u[b] = *reinterpret_cast<const uint32_t*>(&v);
                }
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"((my_at ^ (uint32_t)(f << 4)) + tile), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
            }
        };
        auto handed = [&](uint32_t bar) {  // this warp's stores are in place
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // The share's K codes of tile j; then the next tile's are requested.
        auto make_k = [&](int j) {
            if (j >= n_tiles) return;
            const int st = j & 1;
            if (j >= 2) wait_bar(bar_kfree + 8u * st, (uint32_t)(((j >> 1) - 1) & 1));
            put_codes(PpfSmem::K + st * PFT_TILE, kc, reinterpret_cast<const unsigned short*>(info_of(j))[mrow]);
            handed(bar_kfull + 8u * st);
            fetch_k(j + 1);
        };
        // ... its V codes.  V's norm goes into V too, unless it is not finite: it would reach queries that the token is hidden from (0 x inf).
        // Then the weights take it, those that count (below).
        auto make_v = [&](int j) {
            if (j >= n_tiles) return;
            const int st = j & 1;
            if (j >= 2) wait_bar(bar_vfree + 8u * st, (uint32_t)(((j >> 1) - 1) & 1));
            const uint32_t norm = reinterpret_cast<const unsigned short*>(info_of(j))[PFT_KT + mrow];
            put_codes(PpfSmem::V + st * PFT_TILE, vc, (norm & 0x7fffu) >= 0x7c00u ? 0x3c00u : norm);
            handed(bar_vfull + 8u * st);
            fetch_v(j + 1);
        };
        kc = vc = make_uint4(0u, 0u, 0u, 0u);
        if (n_tiles > 0) {  // (the first tile's norms are on their way while its codes are)
            wait_bar(bar_rows, 0u);
            fetch(0, p.ck, kc);
            fetch(0, p.cv, vc);
            wait_bar(bar_norms, 0u);
        }
        make_k(0);
        // ---- q_rot = Q . R^T, scaled by log2(e) / sqrt(128), back into the Q tiles ----
        wait_bar(bar_rot, 0u);
        tc_fence_after();
#pragma unroll 1
        for (int c0 = pcol0; c0 < pcol0 + PCOLS; c0 += 64) {
            uint32_t r[32];
            tmem_ld_frag64(my_lanes + 128u * pslot + (uint32_t)c0, r);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]) * (PFT_SCALE / PPF_CENT<BITS>);
            put_frag(PpfSmem::Q + pslot * PFT_TILE, c0, v);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        named_barrier(1, PPF_MEET);
        tc_fence_after();
        make_v(0);
        if (MT == 1) make_k(1);  // (goes where R was)

        // ---- softmax of slot `slot`, rows row0 + gl and row0 + gl + 8 ----
        const uint32_t s_col = my_lanes + 128u * slot, o_col = s_col + 256u;
        const int nt = slot ? n1 : n0;
        const bool some_row = token_of(row0, make_by_grp()) < n;  // (uniform for the warp)
        const int first_pos = pos0 + my_first;                    // position of the slot's first query
        // last tokens that the thread's rows attend to (none: a row of no query)
        const int tok0 = token_of(row0 + gl, make_by_grp()), tok1 = token_of(row0 + gl + 8, make_by_grp());
        const int last0 = tok0 < n ? pos0 + tok0 : -1, last1 = tok1 < n ? pos0 + tok1 : -1;
        float m_run[2] = {-1e30f, -1e30f}, l_run[2] = {0.0f, 0.0f};  // (sums: of this thread's columns)
        for (int j = 0; j < n_tiles; ++j) {
            if (MT == 2) make_k(j + 1);
            if (MT == 2 ? j < nt : (j & 1) == slot) {
                const int i = MT == 2 ? j : j >> 1, col0 = (t_lo + j) * PFT_KT;
                wait_bar(bar_sfull + 8u * slot, (uint32_t)(i & 1));
                tc_fence_after();
                if (some_row) {
                    const bool diagonal = col0 + PFT_KT - 1 > first_pos;  // (uniform for the slot)
                    const uint8_t* const info = info_of(j);
                    const bool select = *reinterpret_cast<const uint32_t*>(info + PpfSmem::INFO_ODD) != 0u;  // a norm of V that is not finite
                    // Scores of 64 columns at a time, masked: [row][column block].  The second half is read once for the
                    // row maxima and once more for its weights: with all 128 in registers the compiler spilled, and what is spilled comes back
                    // from L2 (shared memory leaves no L1): 4 x 1024 tokens behind 8192 took 990 us, 60 % of them waits for such loads.
                    auto scores = [&](int c, float2 (&x)[2][8]) {
                        uint32_t r[32];
                        tmem_ld_frag64(s_col + 64u * c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int b = 0; b < 8; ++b)
#pragma unroll
                            for (int h = 0; h < 2; ++h) x[h][b] = make_float2(__uint_as_float(r[4 * b + 2 * h]), __uint_as_float(r[4 * b + 2 * h + 1]));
                        if (diagonal) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int lim = (h ? last1 : last0) - col0 - 64 * c - 2 * t4;  // columns up to here count
#pragma unroll
                                for (int b = 0; b < 8; ++b) {
                                    if (8 * b > lim) x[h][b].x = -1e30f;
                                    if (8 * b + 1 > lim) x[h][b].y = -1e30f;
                                }
                            }
                        }
                    };
                    float mx[2] = {-1e30f, -1e30f};
                    auto largest = [&](const float2 (&x)[2][8]) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float m2 = -1e30f;
#pragma unroll
                            for (int b = 0; b < 8; b += 2) {
                                mx[h] = fmaxf(mx[h], fmaxf(x[h][b].x, x[h][b].y));
                                m2 = fmaxf(m2, fmaxf(x[h][b + 1].x, x[h][b + 1].y));
                            }
                            mx[h] = fmaxf(mx[h], m2);
                        }
                    };
                    float2 x[2][8];
#pragma unroll
                    for (int c = 1; c >= 0; --c) {
                        scores(c, x);
                        largest(x);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                    }
                    const bool grew0 = mx[0] > m_run[0] + PFT_SLACK, grew1 = mx[1] > m_run[1] + PFT_SLACK;
                    if (__any_sync(0xffffffffu, grew0 || grew1)) {
                        const float mn0 = grew0 ? mx[0] : m_run[0], mn1 = grew1 ? mx[1] : m_run[1];
                        const float corr0 = ex2_approx(m_run[0] - mn0), corr1 = ex2_approx(m_run[1] - mn1);
                        m_run[0] = mn0; m_run[1] = mn1;
                        l_run[0] *= corr0; l_run[1] *= corr1;
                        if (i > 0) {  // S(i) is there, so P(i - 1) V has finished: O is at rest
#pragma unroll 1
                            for (int c = 0; c < 4; ++c) {
                                uint32_t r[16];
                                tmem_ld_frag32(o_col + 32u * c, r);
                                tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * ((e & 2) ? corr1 : corr0));
                                tmem_st_frag32(o_col + 32u * c, r);
                            }
                        }
                    }
                    // ---- P as fp16 over S ----
                    float2 lsum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                    float2 minus[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)  // (no column counts yet: all weights 0)
                        minus[h] = m_run[h] <= -1e29f ? make_float2(0.0f, 0.0f) : make_float2(-m_run[h], -m_run[h]);
                    auto weights = [&](int c, auto masked_is_zero) {
                        uint32_t pr[16];
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            float2 v2;
                            if constexpr (decltype(masked_is_zero)::value) {
                                v2 = __half22float2(reinterpret_cast<const __half2*>(info + 2 * PFT_KT)[32 * c + 4 * b + t4]);
                                if (fabsf(v2.x) < INFINITY) v2.x = 1.0f;
                                if (fabsf(v2.y) < INFINITY) v2.y = 1.0f;
                            }
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float2 a = add2(x[h][b], minus[h]);
                                a = make_float2(ex2_approx(a.x), ex2_approx(a.y));
                                lsum[h] = add2(lsum[h], a);
                                if constexpr (decltype(masked_is_zero)::value)
                                    a = make_float2(x[h][b].x <= -1e30f ? 0.0f : a.x * v2.x, x[h][b].y <= -1e30f ? 0.0f : a.y * v2.y);
                                pr[2 * b + h] = pack_half2(a.x, a.y);
                            }
                        }
                        tmem_st_pack32(s_col + 32u * c, pr);
                    };
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c) scores(1, x);
                        if (select) weights(c, std::true_type{});
                        else weights(c, std::false_type{});
                    }
                    l_run[0] += lsum[0].x + lsum[0].y;
                    l_run[1] += lsum[1].x + lsum[1].y;
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_pfull + 8u * slot);
            }
            if (lane == 0) mbar_arrive(bar_used + 8u * (j & (PPF_STAGES - 1)));
            if (MT == 1) make_k(j + 2);
            make_v(j + 1);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
        }
        wait_bar(MT == 2 && slot ? bar_done1 : bar_done, 0u);  // every product (of the slot) has completed
        tc_fence_after();
        const int s0_e = kept[0], n_e = kept[1], first_e = kept[2] + (MT == 2 ? slot * QT : 0);
        const uint32_t lanes_e = *tmem_slot + ((uint32_t)row0 << 16);
        auto token_e = [&](int row, uint32_t by_grp) { return token_in(row, by_grp) < QT ? first_e + token_in(row, by_grp) : n_e; };

        // ================= results =================
        float w0[2], w1[2] = {0.0f, 0.0f};  // by row: weights of the slots' sums, normalised (MT = 2: of its own; joined: not normalised)
        float M_all[2], Z_all[2];
        if constexpr (MT == 1) {
            named_barrier(2, 32 * PFT_SOFT_WARPS);  // (every warp has made its last tile)
            float2* const xch = reinterpret_cast<float2*>(gb + PPF_XCH);
            if (t4 == 0) {
                xch[slot * 128 + row0 + gl] = make_float2(m_run[0], l_run[0]);
                xch[slot * 128 + row0 + gl + 8] = make_float2(m_run[1], l_run[1]);
            }
            named_barrier(2, 32 * PFT_SOFT_WARPS);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 a = xch[row0 + gl + 8 * h], b = xch[128 + row0 + gl + 8 * h];
                const float M = fmaxf(a.x, b.x), e0 = n0 > 0 ? ex2_approx(a.x - M) : 0.0f, e1 = n1 > 0 ? ex2_approx(b.x - M) : 0.0f;
                M_all[h] = M;
                Z_all[h] = a.y * e0 + b.y * e1;
                const float inv = (1.0f / PPF_CENT<BITS>) * (joined() ? 1.0f : 1.0f / (Z_all[h] + 1e-8f));
                w0[h] = e0 * inv;
                w1[h] = e1 * inv;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) w0[h] = (1.0f / PPF_CENT<BITS>) / (l_run[h] + 1e-8f);
        }
        // rows that attend to nothing (no tile at all, or none up to their position) give zeros whatever tensor memory holds
        auto sees = [&](int r) {
            const int tok = token_e(row0 + r, make_by_grp());
            return tok < n_e && first_pos + tok - first_e >= 0 && (MT == 1 || nt > 0);
        };
        const bool on[2] = {sees(gl), sees(gl + 8)};
        auto result = [&](int c0, float (&v)[32]) {  // columns c0 .. c0 + 63 in fragment order
            uint32_t r[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.0f;
            if (MT == 2 ? nt > 0 : n0 > 0) {
                tmem_ld_frag64((MT == 2 ? o_col : lanes_e + 256u) + (uint32_t)c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = on[(e >> 1) & 1] ? __uint_as_float(r[e]) * w0[(e >> 1) & 1] : 0.0f;
            }
            if (MT == 1 && n1 > 0) {
                tmem_ld_frag64(lanes_e + 384u + (uint32_t)c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = on[(e >> 1) & 1] ? fmaf(__uint_as_float(r[e]), w1[(e >> 1) & 1], v[e]) : 0.0f;
            }
        };
        if constexpr (SPLIT) {
            if (joined()) {
                // the sums as they are, with maximum and sum of weights behind them
                const uint32_t by_grp = make_by_grp();
                const int c0 = pcol0;
                float v[32];
                result(c0, v);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = row0 + gl + 8 * h, tok = token_e(row, by_grp);
                    if (tok >= n_e) continue;
                    float* const dst = p.partials + (((size_t)(kept[4] & 255) * p.T + s0_e + tok) * p.H + (size_t)(kvh * GRP + row - token_in(row, by_grp) * GRP)) * PART_STRIDE;
#pragma unroll
                    for (int b = 0; b < 8; ++b) *reinterpret_cast<float2*>(dst + c0 + 8 * b + 2 * t4) = make_float2(v[4 * b + 2 * h], v[4 * b + 2 * h + 1]);
                    if (slot == 0 && t4 == 0) *reinterpret_cast<float2*>(dst + HEAD_DIM) = on[h] ? make_float2(M_all[h], Z_all[h]) : make_float2(-1e30f, 0.0f);
                }
            }
        }
        if (!joined()) {
            // The normalised rows as fp16 over the Q tile, times R.  (One rounding more, relative to a row 2^-11 at most, as R changes no length; with
            // a low part beside it the way from the last tile to the end, a third of a short prompt's time, was twice as many products and stores.)
            const uint32_t qtile = PpfSmem::Q + pslot * PFT_TILE;
#pragma unroll 1
            for (int c0 = pcol0; c0 < pcol0 + PCOLS; c0 += 64) {
                float v[32];
                result(c0, v);
                put_frag(qtile, c0, v);
            }
            fence_proxy_async_smem();
            tc_fence_before();
            named_barrier(MT == 1 ? 1 : 3 + slot, MT == 1 ? PPF_MEET : PPF_MEET / 2 + 16);
            wait_bar(MT == 2 && slot ? bar_q : bar_rot, 1u);
            tc_fence_after();
            // the finished values as fp16 through the (consumed) query tile, so that 16 lanes store 256 contiguous bytes of a row
#pragma unroll 1
            for (int c0 = pcol0; c0 < pcol0 + PCOLS; c0 += 64) {
                float v[32];
                uint32_t r[32];
                tmem_ld_frag64(lanes_e + 128u * pslot + (uint32_t)c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]);
                put_frag(qtile, c0, v);
            }
            __syncwarp();
            constexpr int CH = PCOLS / 8;  // 16-byte pieces per row
            const uint32_t by_grp = make_by_grp();
            __half* const out_seq = p.out + (size_t)s0_e * p.out_stride;
#pragma unroll
            for (int k = 0; k < CH / 2; ++k) {
                const int at = 32 * k + lane, row = row0 + at / CH, ch = (pcol0 >> 3) + at % CH, tok = token_e(row, by_grp);
                if (tok < n_e) {
                    const uint4 u = *reinterpret_cast<const uint4*>(gb + qtile + pft_chunk(row, ch));
                    *(reinterpret_cast<uint4*>(out_seq + (size_t)tok * p.out_stride + (size_t)(kvh * GRP + row - token_in(row, by_grp) * GRP) * HEAD_DIM) + ch) = u;
                }
            }
        }
        tc_fence_before();
    }
    if (dead) {  // copies and products may still be in flight: a bounded chance to land before shared and tensor memory go away
        mbar_wait_bounded_hint(bar_q, 0u, 1u << 10, 2000u);
        mbar_wait_bounded_hint(bar_r, 0u, 1u << 10, 2000u);
        mbar_wait_bounded_hint(bar_done, 0u, 1u << 10, 2000u);
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, 512u);
}

// The parts of a request whose tokens were cut: out[tok][h] = R (sum_z 2^(m_z - M) acc_z / sum_z 2^(m_z - M) l_z).  16 (token, head) rows per CTA, two a
// warp; fp16 high and low parts of the sums times R on mma.sync, a warp 16 output coordinates.
struct PagedMergeParams {
    const float* partials;        // PagedPrefillParams::partials
    const float* small_partials;  // PagedRowsParams::partials
    int part_tokens, by_request;
    const __half* rotation;       // R row-major
    const int* start;        // [G + 1]
    __half* out;
    int room, most_parts;  // PagedPrefillParams' (most_parts 0: no request of more than small_rows rows is cut)
    int small_splits;      // parts of the others (0: there are none)
    int small_rows;
    int T, G, H, Hkv, grp, out_stride;
};
static __global__ void __launch_bounds__(256) paged_merge_kernel(const PagedMergeParams p) {
    __shared__ __align__(16) __half r_s[HEAD_DIM / 2][HEAD_DIM + 8];
    __shared__ __align__(16) __half a_s[2][16][HEAD_DIM + 8];
    __shared__ int blocks_s[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t4 = lane & 3;
    pdl_launch_dependents();
    // (the kernels before let this one start when what came before the call has finished: R and the batch may be read; the sums not yet)
    const int s0 = max(p.start[blockIdx.y], 0), n = max(min(p.start[blockIdx.y + 1], p.T) - s0, 0);
    const bool large = n * p.grp > p.small_rows;
    const long long rows = (long long)n * p.H;
    int splits = p.small_splits;
    if (large) {
        splits = 0;
        if (p.most_parts > 0 && 16ll * blockIdx.x < rows) {  // as the kernel that made them
            const int qt = PFT_ROWS / p.grp;
            int blocks = 0;
            for (int i = tid; i < p.G; i += 256) {
                const int m = max(min(p.start[i + 1], p.T) - max(p.start[i], 0), 0);
                if (m * p.grp > p.small_rows) blocks += (m + qt - 1) / qt;
            }
            blocks = __reduce_add_sync(0xffffffffu, blocks);
            if (lane == 0) blocks_s[warp] = blocks;
            __syncthreads();
            blocks = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) blocks += blocks_s[w];
            splits = prefill_parts(blocks, p.Hkv, p.room, p.most_parts);
            if (splits == 1) splits = 0;  // (the results are in place)
        }
    }
    if (splits == 0 || 16ll * blockIdx.x >= rows) {
        if (blockIdx.x + blockIdx.y == 0) pdl_wait();  // (this launch ends behind the ones before; whoever has work waits below)
        return;
    }
    uint32_t bf[2][8][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = tid + 256 * i;
            *reinterpret_cast<uint4*>(&r_s[at >> 4][8 * (at & 15)]) = reinterpret_cast<const uint4*>(p.rotation)[1024 * half + at];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t r[4];
            ldmatrix_x4_trans(r, smem_u32(&r_s[16 * j + (lane & 15)][16 * warp + 8 * (lane >> 4)]));
            bf[0][4 * half + j][0] = r[0]; bf[0][4 * half + j][1] = r[1];
            bf[1][4 * half + j][0] = r[2]; bf[1][4 * half + j][1] = r[3];
        }
    }
    pdl_wait();
    const size_t part = (size_t)(large ? p.T : p.part_tokens) * p.H * PART_STRIDE;
    const float* const sums = (large ? p.partials : p.small_partials) + (size_t)(!large && p.by_request ? (int)blockIdx.y * p.by_request : s0) * p.H * PART_STRIDE;
    for (long long row0 = 16ll * blockIdx.x; row0 < rows; row0 += 16ll * gridDim.x) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int rr = 2 * warp + k;
            const float* const src = sums + (size_t)(row0 + rr) * PART_STRIDE;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row0 + rr < rows) {
                float2 ml = make_float2(-1e30f, 0.0f);
                if (lane < splits) ml = __ldcg(reinterpret_cast<const float2*>(src + lane * part + HEAD_DIM));
                float M = ml.x;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
                const float e = lane < splits ? ex2_approx(ml.x - M) : 0.0f;
                float Z = ml.y * e;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) Z += __shfl_xor_sync(0xffffffffu, Z, o);
                const float sc = e / (Z + 1e-8f);
#pragma unroll 4
                for (int z = 0; z < splits; ++z) {
                    const float4 v = __ldcg(reinterpret_cast<const float4*>(src + z * part) + lane);
                    const float w = __shfl_sync(0xffffffffu, sc, z);
                    a.x = fmaf(w, v.x, a.x); a.y = fmaf(w, v.y, a.y); a.z = fmaf(w, v.z, a.z); a.w = fmaf(w, v.w, a.w);
                }
            }
            *reinterpret_cast<uint2*>(&a_s[0][rr][4 * lane]) = make_uint2(pack_half2(a.x, a.y), pack_half2(a.z, a.w));
            *reinterpret_cast<uint2*>(&a_s[1][rr][4 * lane]) = make_uint2(pack_low_half2(a.x, a.y), pack_low_half2(a.z, a.w));
        }
        __syncthreads();
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int part2 = 0; part2 < 2; ++part2)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t a[4];
                ldmatrix_x4(a, smem_u32(&a_s[part2][lane & 15][16 * j + 8 * (lane >> 4)]));
#pragma unroll
                for (int i = 0; i < 2; ++i) mma16816(c[i], a[0], a[1], a[2], a[3], bf[i][j][0], bf[i][j][1]);
            }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const long long row = row0 + gl + 8 * r, tok = row / p.H;
            if (row >= rows) continue;
            __half* const dst = p.out + (s0 + tok) * p.out_stride + (row - tok * p.H) * HEAD_DIM + 16 * warp + 2 * t4;
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<__half2*>(dst + 8 * i) = __floats2half2_rn(c[i][2 * r], c[i][2 * r + 1]);
        }
        __syncthreads();  // (the next rows)
    }
}

}  // namespace tq
