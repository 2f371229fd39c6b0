// Attention of requests with few new tokens over paged packed caches, on mma.sync, sm_100a: the part of tq_paged_prefill_attention for
// requests with at most ROWS_MOST score rows (new tokens x query heads) per KV head; tq_paged_prefill.cuh, whose tcgen05 products take 128
// rows whatever there is, has the others.
//
//   * A CTA has up to 8 NCB rows of one request and KV head, and a share of its tokens (one of `parts`).  Its warps take 16 tokens at a
//     time, in turn, each on its own: codes go from global memory into registers in fragment order, a tile ahead, and become fp16
//     centroids through a shared-memory table (the cluster kernel's layout, tq_decode_cluster.cuh), with no barrier in the loop.
//   * S^T = K Q^T (tokens in the M dimension, rows of queries in N, 8 to a block) and O^T += V^T P^T.  What is made of the codes is used
//     for all row blocks: 190 instructions a warp and 16 tokens, and 78 for each block.  (tcgen05: 6500 warp instructions per 128 tokens.)
//     So a CTA takes all blocks that its registers hold: two with two CTAs per SM, three with one.
//   * The queries are rotated at the start (R from L2, in fragments) and lie in shared memory in fragment order.
//   * The warps' sums meet in shared memory, halves in turn; the CTA's go to the workspace, paged_merge_kernel adds the parts up.
//
// What bounds it is instruction issue (54 % of the slots used under a profiler) and a CTA's start and end, 5 to 11 us in all: 32 requests of 5 tokens behind
// 4000, 2-bit, 32/8 heads (71 MB of codes and norms, 11 us at the copy rate) take 118 us with the merge, 4-bit 146; of 1 to 5 tokens behind 2000 to 4000 88 us,
// 131 us on the tcgen05 kernel.
#pragma once

#include "tq_decode_cluster.cuh"
#include "tq_paged_prefill.cuh"

namespace tq {

constexpr int ROWS_MOST = 32;
constexpr int ROWS_SORTED = 128;
template <int NCB>
constexpr int ROWS_WARPS = NCB <= 2 ? 8 : 12;  // (two CTAs per SM, or one whose sums take the room)
template <int NCB>
constexpr int ROWS_THREADS = 32 * ROWS_WARPS<NCB>;
constexpr uint32_t ROWS_LUT_ABS = 0x8000u;  // one entry (a column per lane) every 256 bytes: one PRMT makes a look-up's address
constexpr uint32_t ROWS_MAX_BASE = 0x480u;  // dynamic shared memory starts at or below this address

struct PagedRowsParams {
    const uint8_t* ck;
    const uint8_t* cv;
    const __half* kn;
    const __half* vn;
    const __half* q;
    const __half* rotation;
    const int* block_table;
    const int* lens;
    const int* start;
    float* partials;  // [parts][part_tokens][H][PART_STRIDE], token: of the batch, or by_request times the request plus its own
    int part_tokens, by_request;
    int* status;
    int table_stride, page_shift, num_pages, most_tokens;
    int T, G, H, Hkv, grp, q_stride, parts;
    int behind;       // see the kernel
    int row_blocks;   // CTAs per request, KV head and part: ROWS_MOST / (8 NCB), rounded up
};

template <int NCB>
struct RowsSmem {
    static constexpr uint32_t Q = 0;                                     // rotated queries [8 NCB][136] halves
    static constexpr uint32_t FRAG = 8u * NCB * MERGE_ROW * 2u;          // ... in fragment order [NCB][4][32 lanes][16 B]
    static constexpr uint32_t END = FRAG + NCB * 2048u;
    static constexpr uint32_t WARP = 9u * 32u * 16u;                     // a warp's sums of one row block, at the end: [9][32 lanes][4 floats]
};
template <int BITS>
constexpr size_t rows_smem_bytes() {  // counted from address 0
    return ROWS_LUT_ABS + (BITS == 4 ? 0x10000u : 0x1000u);
}

template <int BITS, int NCB>
__global__ void __launch_bounds__(ROWS_THREADS<NCB>, NCB <= 2 ? 2 : 1) paged_rows_kernel(const PagedRowsParams p) {
    extern __shared__ __align__(1024) uint8_t rows_smem[];
    constexpr int WARPS = ROWS_WARPS<NCB>, THREADS = ROWS_THREADS<NCB>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t4 = lane & 3;
    const uint32_t base = (smem_u32(rows_smem) + 127u) & ~127u;
    uint8_t* const gb = rows_smem + (base - smem_u32(rows_smem));
    static_assert(ROWS_MAX_BASE + RowsSmem<NCB>::END <= ROWS_LUT_ABS && ROWS_MAX_BASE + (WARPS / 2) * RowsSmem<NCB>::WARP <= ROWS_LUT_ABS, "below the table");
    if (base > ROWS_MAX_BASE) {
        if (tid == 0) atomicMax(p.status, ST_SMEM_LAYOUT);
        pdl_wait();
        return;
    }
    constexpr int BPH = HEAD_DIM * BITS / 8;
    // behind: paged_prefill_kernel comes before, which lets this launch start when all before it has finished and has nothing to do with these
    // requests.  So its end is waited for at this one's end only (which stands for both to whatever follows).
    if (!p.behind) pdl_wait();
    pdl_launch_dependents();
    auto leave = [&]() { if (p.behind) pdl_wait(); };
    int rest = (int)blockIdx.x / p.Hkv;
    const int kvh = (int)blockIdx.x - rest * p.Hkv, by_blocks = rest / p.row_blocks, r0 = 8 * NCB * (rest - by_blocks * p.row_blocks);
    int g = by_blocks / p.parts;
    const int part = by_blocks - g * p.parts;
    // The longest contexts first, so that the last CTAs to run are short ones: the request whose length is the g-th.  (2-bit 32/8 heads 32 x 5 behind 100 to 4000
    // 91 -> 70 us, 4-bit behind 1000 to 8000 185 -> 145, 16/8 48 x 1 behind 100 to 4000 74 -> 59; equal contexts cost 1 to 4 % more.  More requests than this have enough turns of CTAs to even out.)
    auto request = [&](int i) {  // first query, queries, tokens
        const int s = max(p.start[i], 0);
        return make_int4(s, min(p.start[i + 1], p.T) - s, min(max(p.lens[i], 0), p.most_tokens), 0);
    };
    int4 mine = make_int4(0, 0, 0, 0);
    if (p.G > 1 && p.G <= ROWS_SORTED) {
        // (where the queries' fragments lie later, behind another barrier)
        int* const lens_s = reinterpret_cast<int*>(gb + RowsSmem<NCB>::FRAG);
        volatile int4* const pick = reinterpret_cast<volatile int4*>(gb + RowsSmem<NCB>::FRAG) + ROWS_SORTED / 4;
        if (tid < p.G) mine = request(tid);
        const int key = tid >= p.G ? -2 : mine.y > 0 && mine.y * p.grp <= ROWS_MOST ? mine.z : -1;
        if (tid < ROWS_SORTED) lens_s[tid] = key;
        if (tid == 0) pick->y = 0;
        if (__syncthreads_or(key >= 0 && mine.y * p.grp > r0) && tid < p.G) {  // (some request has that many rows)
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < p.G; j += 4) {
                const int4 l = *reinterpret_cast<const int4*>(lens_s + j);
                rank += (l.x > key || (l.x == key && j < tid)) + (l.y > key || (l.y == key && j + 1 < tid)) + (l.z > key || (l.z == key && j + 2 < tid)) +
                        (l.w > key || (l.w == key && j + 3 < tid));
            }
            if (rank == g) {
                pick->x = mine.x;
                pick->y = mine.y;
                pick->z = mine.z;
                pick->w = tid;
            }
        }
        __syncthreads();
        mine.x = pick->x;
        mine.y = pick->y;
        mine.z = pick->z;
        g = pick->w;
    } else {
        mine = request(g);
    }
    const int s0 = mine.x, n = mine.y, all_rows = n * p.grp;
    const int L = mine.z, pos0 = L - n;
    const int rows = min(8 * NCB, all_rows - r0);                     // this CTA's: r0 .., row = token * grp + head
    if (n <= 0 || all_rows > ROWS_MOST || rows <= 0) {
        leave();
        return;
    }
    {
        // (entry (tid >> 3) + 32 i, four lanes' columns: a thread's entries share their first code)
        constexpr float c = PPF_CENT<BITS>;
        const int e = tid >> 3;
        const float first = c * (BITS == 4 ? kCent4[e & 15] : kCent2[e & 3]);
#pragma unroll
        for (int i = 0; i < (BITS == 4 ? 8 : 1); ++i) {
            const uint32_t u = pack_half2(first, c * (BITS == 4 ? kCent4[(tid >> 7) + 2 * i] : kCent2[(e >> 2) & 3]));
            if (BITS == 4 ? tid < 256 : e < 16)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ROWS_LUT_ABS + (uint32_t)(e + 32 * i) * 256u + (uint32_t)(tid & 7) * 16u), "r"(u) : "memory");
        }
    }
    const int used = (rows + 7) >> 3;                                 // row blocks
    const int first_last = pos0 + r0 / p.grp;                         // last token that the first row attends to
    const int end = max(pos0 + (r0 + rows - 1) / p.grp + 1, 0);       // tokens that count for any
    const int blocks = (end + 15) / 16;                               // of 16 tokens
    const int b_lo = (int)((long long)blocks * part / p.parts), b_hi = (int)((long long)blocks * (part + 1) / p.parts);
    auto row_token = [&](int r) { return (r0 + r) / p.grp; };

    // ---- a warp's tokens: 16 at a time, in turn; the first ones are requested before all else ----
    const int* const my_pages = p.block_table + (size_t)g * p.table_stride;
    uint32_t page = 0u;
    size_t row0 = 0;
    uint4 kw[2];                 // K rows gl, gl + 8: the lane's 32 coordinates 32 t4 .. (2-bit: x, y)
    uint2 vw[4];                 // V rows 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9: its 16 coordinates 16 gl .. (2-bit: x)
    unsigned short kn_h[2], vn_h[2];  // norms of rows gl, gl + 8
    auto fetch_page = [&](int b) { if (b < b_hi) page = (uint32_t)__ldg(my_pages + ((16 * b) >> p.page_shift)); };
    auto use_page = [&](int b) {  // (16 tokens lie within one page; its number is requested a turn ahead)
        row0 = ((size_t)min(page, (uint32_t)p.num_pages - 1u) << p.page_shift) + (size_t)((16 * b) & ((1 << p.page_shift) - 1));
        fetch_page(b + WARPS);
    };
    // (rows behind the last token: zero codes with zero norms)
    auto load_k = [&](int b) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int t = 8 * r + gl;
            kw[r] = make_uint4(0u, 0u, 0u, 0u);
            kn_h[r] = 0;
            if (16 * b + t < L) {
                const size_t at = (row0 + t) * p.Hkv + kvh;
                if (BITS == 4) {
                    kw[r] = __ldg(reinterpret_cast<const uint4*>(p.ck + at * BPH) + t4);
                } else {
                    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p.ck + at * BPH) + t4);
                    kw[r].x = u.x; kw[r].y = u.y;
                }
                kn_h[r] = __ldg(reinterpret_cast<const unsigned short*>(p.kn) + at);
            }
        }
    };
    auto load_v = [&](int b) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = 2 * t4 + (r & 1) + 8 * (r >> 1);
            vw[r] = make_uint2(0u, 0u);
            if (16 * b + t < L) {
                const uint8_t* const src = p.cv + ((row0 + t) * p.Hkv + kvh) * BPH;
                if (BITS == 4) vw[r] = __ldg(reinterpret_cast<const uint2*>(src) + gl);
                else vw[r].x = __ldg(reinterpret_cast<const uint32_t*>(src) + gl);
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int t = 8 * r + gl;
            vn_h[r] = 16 * b + t < L ? __ldg(reinterpret_cast<const unsigned short*>(p.vn) + (row0 + t) * p.Hkv + kvh) : (unsigned short)0;
        }
    };
    int b = b_lo + warp;
    if (b < b_hi) {
        fetch_page(b);
        use_page(b);
        load_k(b);
        load_v(b);
    }

    // R's fragments: rows 16 warp .. + 15; step (m, e) of lane t4 covers k = 32 m + 8 t4 + 4 e .. + 3, on both sides
    uint4 bf[2][4];
    if (warp < 8)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < 4; ++m) bf[i][m] = ldg128_now(reinterpret_cast<const uint4*>(p.rotation + (size_t)(8 * (2 * warp + i) + gl) * HEAD_DIM) + t4 + 4 * m);
    // ---- queries: rot[r][c] = sum_k q[r][k] R[c][k], scaled by log2(e) / sqrt(128); a warp has the coordinates 16 warp .. + 15 ----
    {
        if (warp < 8)
#pragma unroll
        for (int mt = 0; mt < (NCB + 1) / 2; ++mt) {
            uint4 a[2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 16 * mt + 8 * r + gl;
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    a[r][m] = make_uint4(0u, 0u, 0u, 0u);
                    if (row < rows) {
                        const int tok = row_token(row);
                        a[r][m] = __ldg(reinterpret_cast<const uint4*>(p.q + (size_t)(s0 + tok) * p.q_stride + (size_t)(kvh * p.grp + r0 + row - tok * p.grp) * HEAD_DIM) + t4 + 4 * m);
                    }
                }
            }
            float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mma16816(c[i], a[0][m].x, a[1][m].x, a[0][m].y, a[1][m].y, bf[i][m].x, bf[i][m].y);
                    mma16816(c[i], a[0][m].z, a[1][m].z, a[0][m].w, a[1][m].w, bf[i][m].z, bf[i][m].w);
                }
            constexpr float sc = PFT_SCALE / PPF_CENT<BITS>;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (16 * mt + 8 * r < 8 * NCB)
                        *reinterpret_cast<uint32_t*>(gb + RowsSmem<NCB>::Q + (uint32_t)((16 * mt + 8 * r + gl) * MERGE_ROW + 8 * (2 * warp + i) + 2 * t4) * 2u) =
                            pack_half2(c[i][2 * r] * sc, c[i][2 * r + 1] * sc);
        }
        __syncthreads();
        for (int i = tid; i < NCB * 128; i += THREADS) {  // lane l of row block nb: row l / 4, coordinates 32 (l & 3) + 8 m ..
            const int nb = i >> 7, m = (i >> 5) & 3, l = i & 31;
            *reinterpret_cast<uint4*>(gb + RowsSmem<NCB>::FRAG + 16u * (uint32_t)i) =
                *reinterpret_cast<const uint4*>(gb + RowsSmem<NCB>::Q + (uint32_t)((8 * nb + (l >> 2)) * MERGE_ROW + 32 * (l & 3) + 8 * m) * 2u);
        }
        __syncthreads();
    }
    uint32_t lutlane;  // (made behind the barrier that the table waits for: the look-ups take it into their address)
    asm volatile("mov.u32 %0, %1;" : "=r"(lutlane) : "r"((uint32_t)lane << 2) : "memory");
    auto lut = [&](uint32_t w, int byte) -> uint32_t {
        uint32_t r;
        asm("ld.shared.u32 %0, [%1 + %2];" : "=r"(r) : "r"(prmt(w, lutlane, 0x7604u | ((uint32_t)byte << 4))), "n"(ROWS_LUT_ABS));
        return r;
    };
    const uint32_t frag = base + RowsSmem<NCB>::FRAG + 16u * (uint32_t)lane;  // (read by volatile loads: else all of it would be kept in registers)

    int last[NCB][2];  // last token of the rows of this lane's columns 2 t4, 2 t4 + 1
    float m_run[NCB][2], l_run[NCB][2], acc[NCB][8][4];
#pragma unroll
    for (int nb = 0; nb < NCB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * nb + 2 * t4 + e;
            last[nb][e] = r < rows ? pos0 + row_token(r) : -1;
            m_run[nb][e] = -1e30f;
            l_run[nb][e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[nb][i][0] = acc[nb][i][1] = acc[nb][i][2] = acc[nb][i][3] = 0.0f;
    }
    // (one copy of the loop for each number of row blocks in use: a branch around every product cost a third of the time)
    auto walk = [&](auto used_) {
    constexpr int USED = decltype(used_)::value;
    for (; b < b_hi; b += WARPS) {
        const int t0 = 16 * b, next = b + WARPS;
        // ---- scores: tokens gl and gl + 8, rows 2 t4 and 2 t4 + 1 of each block ----
        float c[USED][4];
#pragma unroll
        for (int nb = 0; nb < USED; ++nb) c[nb][0] = c[nb][1] = c[nb][2] = c[nb][3] = 0.0f;
#pragma unroll
        for (int j2 = 0; j2 < 4; ++j2) {  // two steps of 16 coordinates
            uint32_t a[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = 2 * j2 + h;
                if constexpr (BITS == 4) {
                    const uint32_t lo = j2 == 0 ? kw[0].x : j2 == 1 ? kw[0].y : j2 == 2 ? kw[0].z : kw[0].w, hi = j2 == 0 ? kw[1].x : j2 == 1 ? kw[1].y : j2 == 2 ? kw[1].z : kw[1].w;
                    a[h][0] = lut(lo, 2 * h); a[h][1] = lut(hi, 2 * h);
                    a[h][2] = lut(lo, 2 * h + 1); a[h][3] = lut(hi, 2 * h + 1);
                } else {
                    const uint32_t lo = j < 4 ? kw[0].x : kw[0].y, hi = j < 4 ? kw[1].x : kw[1].y;
                    a[h][0] = lut(lo & 0x0f0f0f0fu, j & 3); a[h][1] = lut(hi & 0x0f0f0f0fu, j & 3);
                    a[h][2] = lut((lo >> 4) & 0x0f0f0f0fu, j & 3); a[h][3] = lut((hi >> 4) & 0x0f0f0f0fu, j & 3);
                }
            }
#pragma unroll
            for (int nb = 0; nb < USED; ++nb) {
                const uint4 qf = ldsv128(frag + (uint32_t)(nb * 2048 + j2 * 512));
                mma16816(c[nb], a[0][0], a[0][1], a[0][2], a[0][3], qf.x, qf.y);
                mma16816(c[nb], a[1][0], a[1][1], a[1][2], a[1][3], qf.z, qf.w);
            }
        }
        const float kn0 = __half2float(__ushort_as_half(kn_h[0])), kn1 = __half2float(__ushort_as_half(kn_h[1]));
        const float vn0 = __half2float(__ushort_as_half(vn_h[0])), vn1 = __half2float(__ushort_as_half(vn_h[1]));
        if (next < b_hi) {
            use_page(next);
            load_k(next);
        }
        const float slack = fmaxf(vn0, vn1) <= 65504.0f / (float)(1 << (int)PFT_SLACK) ? PFT_SLACK : 0.0f;
        const bool masked = t0 + 15 > first_last;  // (uniform) some row does not count all of them
        uint32_t pb[USED][2];  // weights times V norms: B operand of the value product
#pragma unroll
        for (int nb = 0; nb < USED; ++nb) {
            float s[2][2] = {{c[nb][0] * kn0, c[nb][1] * kn0}, {c[nb][2] * kn1, c[nb][3] * kn1}};  // [token][row]
            if (masked) {
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (t0 + 8 * r + gl > last[nb][e]) s[r][e] = -1e30f;
            }
            float mx[2] = {fmaxf(s[0][0], s[1][0]), fmaxf(s[0][1], s[1][1])};
            // The reference point follows the maximum only when that has grown by more than PFT_SLACK (weights stay below 2^PFT_SLACK; times a norm of
            // 4094 they still fit fp16, tokens with a larger one are given no slack): one of 16 rows has a new maximum nearly always.
            if (__any_sync(0xffffffffu, fmaxf(mx[0] - m_run[nb][0], mx[1] - m_run[nb][1]) > slack)) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], o));
                    const float mn = fmaxf(m_run[nb][e], mx[e]), f = ex2_approx(m_run[nb][e] - mn);
                    l_run[nb][e] *= f;
                    m_run[nb][e] = mn;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        acc[nb][i][e] *= f;
                        acc[nb][i][2 + e] *= f;
                    }
                }
            }
            float w[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    w[r][e] = ex2_approx(s[r][e] - m_run[nb][e]);
                    if (masked && s[r][e] <= -1e30f) w[r][e] = 0.0f;
                    l_run[nb][e] += w[r][e];
                    w[r][e] *= r ? vn1 : vn0;
                    if (masked && s[r][e] <= -1e30f) w[r][e] = 0.0f;  // (0 x a norm that is not finite is not 0)
                }
            pb[nb][0] = movmatrix_trans(pack_half2(w[0][0], w[0][1]));
            pb[nb][1] = movmatrix_trans(pack_half2(w[1][0], w[1][1]));
        }
        // ---- values ----
        auto product = [&](int i, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, int byte) {
            const uint32_t a0 = lut(w0, byte), a1 = lut(w1, byte), a2 = lut(w2, byte), a3 = lut(w3, byte);
#pragma unroll
            for (int nb = 0; nb < USED; ++nb) mma16816(acc[nb][i], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
        };
        if constexpr (BITS == 4) {
#pragma unroll
            for (int w2 = 0; w2 < 2; ++w2) {  // (code of token A, code of token B) per byte, even and odd coordinates
                const uint32_t wa = w2 ? vw[0].y : vw[0].x, wb = w2 ? vw[1].y : vw[1].x, wc = w2 ? vw[2].y : vw[2].x, wd = w2 ? vw[3].y : vw[3].x;
                const uint32_t ev_ab = (wa & 0x0f0f0f0fu) | ((wb << 4) & 0xf0f0f0f0u), od_ab = ((wa >> 4) & 0x0f0f0f0fu) | (wb & 0xf0f0f0f0u);
                const uint32_t ev_cd = (wc & 0x0f0f0f0fu) | ((wd << 4) & 0xf0f0f0f0u), od_cd = ((wc >> 4) & 0x0f0f0f0fu) | (wd & 0xf0f0f0f0u);
#pragma unroll
                for (int i = 0; i < 4; ++i) product(4 * w2 + i, ev_ab, od_ab, ev_cd, od_cd, i);
            }
        } else {
            const uint32_t wa = vw[0].x, wb = vw[1].x, wc = vw[2].x, wd = vw[3].x;
            const uint32_t ev_ab = (wa & 0x33333333u) | ((wb << 2) & 0xccccccccu), od_ab = ((wa >> 2) & 0x33333333u) | (wb & 0xccccccccu);
            const uint32_t ev_cd = (wc & 0x33333333u) | ((wd << 2) & 0xccccccccu), od_cd = ((wc >> 2) & 0x33333333u) | (wd & 0xccccccccu);
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // coordinates 2 i, 2 i + 1 of the lane's 16: nibble i of `ev`, `od`
                auto nib = [&](uint32_t w) { return ((i & 1) ? w >> 4 : w) & 0x0f0f0f0fu; };
                product(i, nib(ev_ab), nib(od_ab), nib(ev_cd), nib(od_cd), i >> 1);
            }
        }
        if (next < b_hi) load_v(next);
    }
    };
    if (NCB == 1 || used == 1) walk(std::integral_constant<int, 1>());
    else if (NCB > 2 && used == 2) walk(std::integral_constant<int, NCB < 2 ? 1 : 2>());
    else walk(std::integral_constant<int, NCB>());

    // ---- the warps' sums meet: the upper half of those left hand theirs to the lower half, lane by lane ----
#pragma unroll
    for (int nb = 0; nb < NCB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l_run[nb][e] += __shfl_xor_sync(0xffffffffu, l_run[nb][e], o);
#pragma unroll 1
    for (int left = WARPS; left > 1;) {
        const int half = (left + 1) / 2;  // (an odd number: the one in the middle keeps its own)
        float4* const mine = reinterpret_cast<float4*>(gb + (uint32_t)(warp >= half ? warp - half : warp) * RowsSmem<NCB>::WARP) + lane;
#pragma unroll
        for (int nb = 0; nb < NCB; ++nb) {
            if (nb >= used) continue;  // (uniform)
            __syncthreads();  // (queries are no longer read; the sums before have been)
            if (warp >= half && warp < left) {
#pragma unroll
                for (int i = 0; i < 8; ++i) mine[i * 32] = make_float4(acc[nb][i][0], acc[nb][i][1], acc[nb][i][2], acc[nb][i][3]);
                mine[8 * 32] = make_float4(m_run[nb][0], m_run[nb][1], l_run[nb][0], l_run[nb][1]);
            }
            __syncthreads();
            if (warp < left - half) {
                const float4 s = mine[8 * 32];
                const float m2[2] = {s.x, s.y}, l2[2] = {s.z, s.w};
                float f[2], f2[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m_run[nb][e], m2[e]);
                    f[e] = ex2_approx(m_run[nb][e] - mn);
                    f2[e] = ex2_approx(m2[e] - mn);
                    m_run[nb][e] = mn;
                    l_run[nb][e] = l_run[nb][e] * f[e] + l2[e] * f2[e];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 a = mine[i * 32];
                    acc[nb][i][0] = acc[nb][i][0] * f[0] + a.x * f2[0];
                    acc[nb][i][1] = acc[nb][i][1] * f[1] + a.y * f2[1];
                    acc[nb][i][2] = acc[nb][i][2] * f[0] + a.z * f2[0];
                    acc[nb][i][3] = acc[nb][i][3] * f[1] + a.w * f2[1];
                }
            }
        }
        left = half;
    }
    leave();
    if (warp > 0) return;
    // ---- the CTA's: acc[i]: coordinates 16 gl + 2 i (and + 1) of the rows 2 t4, 2 t4 + 1 ----
#pragma unroll
    for (int nb = 0; nb < NCB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * nb + 2 * t4 + e;
            if (r >= rows) continue;
            const int tok = row_token(r);
            float* const dst = p.partials + (((size_t)part * p.part_tokens + (p.by_request ? g * p.by_request : s0) + tok) * p.H + (size_t)(kvh * p.grp + r0 + r - tok * p.grp)) * PART_STRIDE;
            constexpr float k = 1.0f / PPF_CENT<BITS>;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(dst + 16 * gl + 4 * i) = make_float4(k * acc[nb][2 * i][e], k * acc[nb][2 * i][2 + e], k * acc[nb][2 * i + 1][e], k * acc[nb][2 * i + 1][2 + e]);
            if (gl == 0) *reinterpret_cast<float2*>(dst + HEAD_DIM) = make_float2(m_run[nb][e], l_run[nb][e]);
        }
}

}  // namespace tq
