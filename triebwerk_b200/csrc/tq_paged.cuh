// Paged packed caches, sm_100a: block tables and slot maps from request lengths, and rows of a slot map back as vectors.
//
// A cache array is the packed one of the other kernels ([rows][kv_dim / codes per byte], norms [rows][KV heads]) cut into pages of
// 1 << page_shift consecutive rows; request g's token t is row table[g][t >> page_shift] << page_shift plus t's place in the page.
// The writes into such a cache are the append kernels' (tq_layer_prep.cuh, tq_prefill_tc.cuh, SLOTS), the attention of single tokens is
// the decode kernels' (tq_attention.cuh, tq_decode_cluster.cuh, PAGED).
#pragma once

#include "tq_prefill_fa.cuh"

namespace tq {

// The centroids times these have fp16 neighbours 3.4 times (2-bit: over 1000 times) as close as the centroids themselves (2^-11 x 0.22 and 0.0004
// against 0.73 and 0.54, relative): the tables hold them scaled, queries and results carry the inverse.
template <int BITS>
constexpr float PPF_CENT = BITS == 4 ? 1.211955f : 1.591824f;

// ---- block tables and slot maps -----------------------------------------------------------------------------------------------------
// With c the tokens that request g holds (0 where it has ended), n its new ones, P the page size:
//   pages back      ceil(old / P) of every ended request, in order, on top of the stack of free pages;
//   pages taken     need = ceil((c + n) / P) - ceil(c / P); the k-th page of the call, in the order of requests, is the k-th from the top;
//   admitted        c + n fits the table, and nothing is wanted, or the slot map holds it and (no page is wanted, or the pages wanted
//                   up to and including it are there).  A request that does not fit the table counts for no page;
//   token t         of the slot map belongs to the request whose range of running sums of n holds t.
// Three running sums over the requests, then scattered writes of a few bytes each: bound by latency (a trip for the lengths, one for the
// table entries and free pages, one for the stores), so one CTA does the bookkeeping, and the slot map too where it is short.  A long map
// is filled by a second launch over all SMs, which takes lengths and starts from the first.
struct PagePlanParams {
    int* table;                      // [G][width], rows table_stride apart
    int* free_pages;                 // the stack: [num_pages]
    const int* free_count;
    int* free_count_out;
    const int* context;              // [G] tokens held; ~tokens of a request that was not admitted
    const int* new_tokens;           // [G]
    const unsigned char* finished;   // [G] or null
    int* lens;                       // [G]
    int* start;                      // [G + 1]
    long long* slots;                // [T]
    int* positions;                  // [T] or null
    int G, T, num_pages, table_stride, width, page_shift;
};

constexpr int PLAN_THREADS = 1024;
// Slots that the first launch writes itself.  (us, one / two launches: 64 x 16 new tokens 4.7 / 6.1, 256 x 4 5.2 / 6.8, 64 x 32 5.5 / 6.2, 64 x 64 7.0 / 6.3,
// 256 x 16 7.7 / 7.1, 64 x 128 9.7 / 6.3, 64 x 1024 51 / 6.6.)
constexpr int PLAN_ONE_LAUNCH = 2048;

// Token t of the slot map is request a's, start[a] <= t < start[a + 1].
constexpr int SLOTS_THREADS = 256, SLOTS_SHARED = 8192;  // starts that are searched in shared memory
static __global__ void __launch_bounds__(SLOTS_THREADS) page_slots_kernel(const PagePlanParams p) {
    __shared__ int start_s[SLOTS_SHARED];
    pdl_launch_dependents();
    pdl_wait();
    const int* start = p.start;
    if (p.G < SLOTS_SHARED) {
        for (int i = threadIdx.x; i <= p.G; i += SLOTS_THREADS) start_s[i] = p.start[i];
        __syncthreads();
        start = start_s;
    }
    const int used = start[p.G];
    for (int t = blockIdx.x * SLOTS_THREADS + threadIdx.x; t < p.T; t += gridDim.x * SLOTS_THREADS) {
        long long slot = -1;
        int pos = -1;
        if (t < used) {
            int a = 0, b = p.G;
            while (b - a > 1) {
                const int mid = (a + b) >> 1;
                if (start[mid] <= t) a = mid;
                else b = mid;
            }
            const int len = p.lens[a];
            if (len > 0) {  // (a request that was not admitted: negative)
                pos = len - (start[a + 1] - t);
                slot = ((long long)p.table[(size_t)a * p.table_stride + (pos >> p.page_shift)] << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
            }
        }
        p.slots[t] = slot;
        if (p.positions) p.positions[t] = pos;
    }
}

// The request of a chunk (requests base .. base + PLAN_THREADS - 1) whose range of running sums holds q: the last one with sums[r] <= q.
__device__ __forceinline__ int plan_row(const int* sums, int rows, int q) {
    int a = 0, b = rows;
    while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (sums[mid] <= q) a = mid;
        else b = mid;
    }
    return a;
}

// Pages and slots are dealt out to the threads one by one, whichever request they belong to (its number by a search in the running sums): with
// a warp for 32 requests, in turn, 64 prompts of 28 pages on average waited for as many trips to memory one behind the other, 26 us of 30 with
// the slot map (12.8 now, alone and from cold caches; 18.4 -> 8.6 us in a stream of calls).  256 requests with a token each: 5.9 us, three trips.
static __global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const PagePlanParams p) {
    __shared__ long long sums[2][2][PLAN_THREADS / 32];
    __shared__ int page_sum[PLAN_THREADS], token_sum[PLAN_THREADS], first_s[PLAN_THREADS], held_s[PLAN_THREADS];
    __shared__ unsigned long long taken_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) taken_s = 0;
    pdl_launch_dependents();
    pdl_wait();
    const int P1 = (1 << p.page_shift) - 1;
    auto pages_of = [&](long long tokens) { return (int)((tokens + P1) >> p.page_shift); };
    // running sums over the threads: of a and b before this thread's own, and of all
    auto scan = [&](long long (&a)[2], int buf, long long (&all)[2]) {
        long long incl[2] = {a[0], a[1]};
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v0 = __shfl_up_sync(0xffffffffu, incl[0], o), v1 = __shfl_up_sync(0xffffffffu, incl[1], o);
            if (lane >= o) {
                incl[0] += v0;
                incl[1] += v1;
            }
        }
        if (lane == 31) {
            sums[buf][0][warp] = incl[0];
            sums[buf][1][warp] = incl[1];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            long long s = sums[buf][i][lane], before = lane < warp ? s : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                before += __shfl_xor_sync(0xffffffffu, before, o);
            }
            all[i] = s;
            a[i] = before + incl[i] - a[i];
        }
    };
    struct Request {
        int held, n;
        bool ended;
    };
    auto load = [&](int g) {
        Request r{0, 0, false};
        if (g < p.G) {
            const int c = p.context[g];
            r.n = max(p.new_tokens[g], 0);
            r.ended = p.finished && p.finished[g] != 0;
            r.held = c < 0 ? ~c : c;
        }
        return r;
    };
    const Request first_chunk = load(tid);
    long long have = min(max(*p.free_count, 0), p.num_pages);
    // ---- pages of ended requests ----
    if (p.finished) {
        for (int base = 0; base < p.G; base += PLAN_THREADS) {
            const Request r = base == 0 ? first_chunk : load(base + tid);
            if (!__syncthreads_or(r.ended)) continue;
            long long sum[2] = {r.ended ? min(pages_of(r.held), p.width) : 0, 0}, all[2];
            scan(sum, 0, all);
            page_sum[tid] = (int)min(sum[0], (long long)p.num_pages);
            __syncthreads();
            const int back = (int)min(all[0], (long long)p.num_pages - have), rows = min(PLAN_THREADS, p.G - base);  // (a stack that is full takes no more)
            for (int q = tid; q < back; q += PLAN_THREADS) {
                const int row = plan_row(page_sum, rows, q);
                p.free_pages[have + q] = p.table[(size_t)(base + row) * p.table_stride + q - page_sum[row]];
            }
            have += back;
            // (the stack's new entries, the rows that new tokens may now replace, the sums)
            __syncthreads();
        }
    }
    // ---- new tokens ----
    long long wanted = 0, tokens = 0;
    for (int base = 0; base < p.G; base += PLAN_THREADS) {
        const Request r = base == 0 ? first_chunk : load(base + tid);
        const int g = base + tid, rows = min(PLAN_THREADS, p.G - base);
        const long long c = r.ended ? 0 : r.held, n = r.n;
        const bool fits = c + n <= (long long)p.width << p.page_shift;
        const int first = pages_of(c), need = fits ? pages_of(c + n) - first : 0;
        long long sum[2] = {need, n}, all[2];
        scan(sum, 1, all);
        const long long k = wanted + sum[0], t = tokens + sum[1];
        const bool ok = fits && (n == 0 || (t + n <= p.T && (need == 0 || k + need <= have)));
        if (g < p.G) {
            p.lens[g] = ok ? (int)(c + n) : ~(int)c;
            p.start[g] = (int)min(t, (long long)p.T);
            if (g == p.G - 1) p.start[p.G] = (int)min(t + n, (long long)p.T);
        }
        // (sums behind what is there count as that; a request that was not admitted: -1)
        page_sum[tid] = (int)min(k, have);
        first_s[tid] = ok ? first : -1;
        const bool dealt = p.T <= PLAN_ONE_LAUNCH;
        if (dealt) {
            token_sum[tid] = (int)min(t, (long long)p.T);
            held_s[tid] = (int)c;
        }
        long long mine = ok ? need : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0 && mine > 0) atomicAdd(&taken_s, (unsigned long long)mine);
        const bool several = __syncthreads_or(dealt && n > 1);
        const int page_end = (int)min(wanted + all[0], have);
        for (int q = (int)min(wanted, have) + tid; q < page_end; q += PLAN_THREADS) {
            const int row = plan_row(page_sum, rows, q), f = first_s[row];
            if (f >= 0) p.table[(size_t)(base + row) * p.table_stride + f + q - page_sum[row]] = p.free_pages[have - 1 - q];
        }
        if (dealt) {
            // token i of a request: its page is in the table already, or on the stack
            auto put = [&](int row, int t, int c, int i, int first, int sum) {
                const int pos = c + i, j = pos >> p.page_shift;
                long long slot = -1;
                if (first >= 0) slot = ((long long)(j < first ? p.table[(size_t)(base + row) * p.table_stride + j] : p.free_pages[have - 1 - (sum + j - first)]) << p.page_shift) + (pos & P1);
                p.slots[t + i] = slot;
                if (p.positions) p.positions[t + i] = first >= 0 ? pos : -1;
            };
            if (!several && n == 1 && t < p.T) put(tid, (int)t, (int)c, 0, ok ? first : -1, (int)min(k, have));
            const int token_end = several ? (int)min(tokens + all[1], (long long)p.T) : 0;
            for (int q = (int)min(tokens, (long long)p.T) + tid; q < token_end; q += PLAN_THREADS) {
                const int row = plan_row(token_sum, rows, q), i = q - token_sum[row];
                put(row, token_sum[row], held_s[row], i, first_s[row], page_sum[row]);
            }
        }
        wanted += all[0];
        tokens += all[1];
        if (base + PLAN_THREADS < p.G) __syncthreads();  // (the sums may be written again)
    }
    __syncthreads();
    if (tid == 0) *p.free_count_out = (int)(have - (long long)taken_s);
    if (p.T > PLAN_ONE_LAUNCH) return;
    for (long long t = tokens + tid; t < p.T; t += PLAN_THREADS) {
        p.slots[t] = -1;
        if (p.positions) p.positions[t] = -1;
    }
}

// ---- rows of a slot map as vectors ------------------------------------------------------------------------------------------------------
// out[t][h] = norm * R^T c, c the centroids of row slots[t], head h (zeros where the slot is no row).  Vectors are the M dimension of mma.sync,
// 64 at a time; a warp owns 32 of them and 32 output coordinates, whose part of R stays in its registers; the centroids, and then the results,
// go through shared memory, so that whole rows leave.  Two dependent trips to memory (slot, codes) stand before a vector's arithmetic: both
// are made a tile ahead.  8192 tokens, 8 KV heads, 4-bit (42 MB, 6.5 us at the copy rate): 19.8 us; 34.4 with neither, results stored as the
// products leave them and every warp on all 64 vectors for 16 coordinates (the operand is then read eight times, not four: 22 us by itself).
// What bounds it now is the table look-ups and operand traffic of shared memory.  64 tokens: the launch and the two trips.
struct PagedReadParams {
    const uint8_t* ck;
    const __half* kn;
    const uint8_t* cv;
    const __half* vn;
    const __half* rotation;      // R row-major
    const long long* slots;      // [T]
    __half* k_out;               // [T][stride]
    __half* v_out;
    long long total_rows, stride;
    int T, Hkv;
};
constexpr int READ_THREADS = 256, READ_VECTORS = 64;

template <int BITS>
__global__ void __launch_bounds__(READ_THREADS, 2) paged_read_kernel(const PagedReadParams p) {
    constexpr int BPH = HEAD_DIM * BITS / 8, ENTRIES = BITS == 4 ? 256 : 16;
    constexpr int COPIES = 16;  // of the table: two lanes share a bank
    __shared__ uint32_t lut[ENTRIES * COPIES];
    __shared__ __align__(16) __half a_s[READ_VECTORS][HEAD_DIM + 8];
    __shared__ float norm_s[READ_VECTORS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t4 = lane & 3;
    const int v_part = 32 * (warp >> 2), c_part = 32 * (warp & 3);  // first vector, first output coordinate of the warp
    for (int i = tid; i < ENTRIES * COPIES; i += READ_THREADS) {
        constexpr float c = PPF_CENT<BITS>;  // (the table's centroids times this are closer to fp16 numbers)
        const int e = i / COPIES;
        lut[i] = BITS == 4 ? pack_half2(c * kCent4[e & 15], c * kCent4[(e >> 4) & 15]) : pack_half2(c * kCent2[e & 3], c * kCent2[(e >> 2) & 3]);
    }
    pdl_launch_dependents();
    pdl_wait();
    // four threads a vector, 32 coordinates each.  A tile's vectors: their slots (requested two tiles ahead), then codes and norm (one).
    const uint32_t per_kind = (uint32_t)p.T * p.Hkv, tiles = (per_kind + READ_VECTORS - 1) / READ_VECTORS;
    const uint2 by_heads = fastdiv_make((uint32_t)p.Hkv);
    auto token_of = [&](uint32_t v) { return (uint32_t)fastdiv((int)v, by_heads); };
    auto slot_of = [&](uint32_t tile) -> long long {
        if (tile >= 2 * tiles) return -1;
        const uint32_t v = (tile >= tiles ? tile - tiles : tile) * READ_VECTORS + (uint32_t)(tid >> 2);
        return v < per_kind ? __ldg(p.slots + token_of(v)) : -1;
    };
    uint4 codes;
    unsigned short norm;
    auto fetch = [&](uint32_t tile, long long row) {
        codes = make_uint4(0u, 0u, 0u, 0u);
        norm = 0;
        if (row < 0 || row >= p.total_rows) return;
        const bool is_v = tile >= tiles;
        const uint32_t v = (is_v ? tile - tiles : tile) * READ_VECTORS + (uint32_t)(tid >> 2);
        const size_t at = (size_t)row * p.Hkv + (v - token_of(v) * (uint32_t)p.Hkv);
        const uint8_t* const src = (is_v ? p.cv : p.ck) + at * BPH + (BPH / 4) * (tid & 3);
        if (BITS == 4) {
            codes = __ldg(reinterpret_cast<const uint4*>(src));
        } else {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(src));
            codes = make_uint4(u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16);
        }
        if ((tid & 3) == 0) norm = __ldg(reinterpret_cast<const unsigned short*>(is_v ? p.vn : p.kn) + at);
    };
    const uint32_t step = gridDim.x;
    long long next_row = slot_of(blockIdx.x);
    // B fragments: coordinates n = c_part + 8 i + gl, k = 16 j + 2 t4, + 1 (+ 8); R passes through the operand's place, 64 rows at a time
    uint32_t bf[4][8][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = tid + READ_THREADS * i;
            *reinterpret_cast<uint4*>(&a_s[at >> 4][8 * (at & 15)]) = reinterpret_cast<const uint4*>(p.rotation)[1024 * half + at];
        }
        if (half == 0) {
            fetch(blockIdx.x, next_row);
            next_row = slot_of(blockIdx.x + step);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                uint32_t r[4];
                ldmatrix_x4_trans(r, smem_u32(&a_s[16 * j + (lane & 15)][c_part + 8 * i + 8 * (lane >> 4)]));
                bf[i][4 * half + j][0] = r[0]; bf[i][4 * half + j][1] = r[1];
                bf[i + 1][4 * half + j][0] = r[2]; bf[i + 1][4 * half + j][1] = r[3];
            }
    }
    for (uint32_t tile = blockIdx.x; tile < 2 * tiles; tile += step) {
        const bool is_v = tile >= tiles;
        const uint32_t v0 = (is_v ? tile - tiles : tile) * READ_VECTORS;
        __syncthreads();  // (the last tile's results have left)
        {
            const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
            const int copy = tid & (COPIES - 1);
            if ((tid & 3) == 0) norm_s[tid >> 2] = (1.0f / PPF_CENT<BITS>) * __half2float(__ushort_as_half(norm));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4 u;
                constexpr uint32_t M = ENTRIES - 1, W = BITS == 4 ? 8 : 4;
                u.x = lut[(w[i] & M) * COPIES + copy]; u.y = lut[((w[i] >> W) & M) * COPIES + copy];
                u.z = lut[((w[i] >> (2 * W)) & M) * COPIES + copy]; u.w = lut[((w[i] >> (3 * W)) & M) * COPIES + copy];
                *reinterpret_cast<uint4*>(&a_s[tid >> 2][32 * (tid & 3) + 8 * i]) = u;
            }
        }
        fetch(tile + step, next_row);
        next_row = slot_of(tile + 2 * step);
        __syncthreads();
        float c[2][4][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[m][i][0] = c[m][i][1] = c[m][i][2] = c[m][i][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t a[4];
                ldmatrix_x4(a, smem_u32(&a_s[v_part + 16 * m + (lane & 15)][16 * j + 8 * (lane >> 4)]));
#pragma unroll
                for (int i = 0; i < 4; ++i) mma16816(c[m][i], a[0], a[1], a[2], a[3], bf[i][j][0], bf[i][j][1]);
            }
        }
        __syncthreads();  // the operand has been read: the results take its place
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int at = v_part + 16 * m + gl + 8 * r;
                const float n = norm_s[at];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<__half2*>(&a_s[at][c_part + 8 * i + 2 * t4]) = __floats2half2_rn(c[m][i][2 * r] * n, c[m][i][2 * r + 1] * n);
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < READ_VECTORS * 16 / READ_THREADS; ++i) {  // 16 lanes a row
            const int at = (tid >> 4) + (READ_THREADS / 16) * i;
            const uint32_t v = v0 + (uint32_t)at, t = token_of(v);
            if (v < per_kind)
                *(reinterpret_cast<uint4*>((is_v ? p.v_out : p.k_out) + (size_t)t * p.stride + (size_t)(v - t * (uint32_t)p.Hkv) * HEAD_DIM) + (tid & 15)) =
                    *reinterpret_cast<const uint4*>(&a_s[at][8 * (tid & 15)]);
        }
    }
}

}  // namespace tq
